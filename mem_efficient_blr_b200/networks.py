"""Network-level glue around the structured linears: a Llama-7B-shaped decoder, a ViT-B/16-shaped encoder and a
DiT-XL/2-shaped denoiser.

The reference times whole HuggingFace models whose nn.Linear layers were swapped for its structured modules
(models/llama7b.py:24-92, models/vit_b_patch16_224.py:69-131, utils.py:46-116).  No checkpoint or tokenizer can be
fetched here, so the networks are built from the shapes alone with random weights: the same layer list, the same
linears swapped (Llama: q/k/v/o and gate/up/down of every layer, lm_head stays dense; ViT: fused qkv, intermediate
and output of every layer, the attention output projection stays dense), and around them plain PyTorch - RMSNorm /
LayerNorm, rotary embedding, `scaled_dot_product_attention`, SwiGLU / GELU.  Those surrounding pieces are
placeholders for what a serving stack would fuse; the structured linears are what this package is about.

Decode runs against a static key/value cache (one write position per step, attention over the whole cache), so a
step has fixed shapes and can be captured in a CUDA graph (`GraphedCall`).
"""
from __future__ import annotations

import contextlib
import math
from dataclasses import dataclass, field
from typing import Optional

import torch
import torch.nn as nn
import torch.nn.functional as F
from torch.nn.modules.module import _has_any_global_hook

from . import _lib as L
from . import blast_kernels as bk
from . import blast_sym_quant_kernels as bq


# ------------------------------------------------------------------------------------------------ structured linears
_EMPTY_INIT = False


@contextlib.contextmanager
def empty_init():
    """Inside this context the networks and layers of this module are built with uninitialised weights (no random
    numbers, and quantised layers without their 16-bit factors ever existing): the skeleton for
    packed.load_packed_into."""
    global _EMPTY_INIT
    keep, _EMPTY_INIT = _EMPTY_INIT, True
    try:
        yield
    finally:
        _EMPTY_INIT = keep


# A fused operator may stand for a module only where a call of that module would run exactly the code that the operator was written for.
_CALL = nn.Module.__call__
_FORWARD = {nn.Linear: nn.Linear.forward}   # the classes of which that is known, with their own forward


def _known(cls):
    _FORWARD[cls] = cls.forward
    return cls


def _stock(m) -> bool:
    """Whether m(...) is the forward of one of these classes and nothing else: no subclass, no forward put on the object or patched onto the
    class, no hook on the module or on all modules, not compiled in place."""
    t, d = type(m), m.__dict__   # (the dictionary: half the time of nn.Module's attributes, and an encoder pass asks fifty times)
    return (_FORWARD.get(t) is t.forward and t.__call__ is _CALL and "forward" not in d and d.get("_compiled_call_impl") is None
            and not (d["_forward_hooks"] or d["_forward_pre_hooks"] or d["_backward_hooks"] or d["_backward_pre_hooks"] or _has_any_global_hook()))


def _stock_blast(m) -> bool:
    return type(m) in (BlastTorchLinear, BlastQuantLinear) and _stock(m) and m.U_device_ok()


@_known
class BlastTorchLinear(nn.Module):
    """BLAST linear on the torch layouts U (b,Q,R), Vt (b,R,P), S (b,b,R) (torch_funcs/blast_funcs.py:3-47), with a
    variance-preserving random init: x ~ N(0,1) gives out ~ N(0,1) (Vt ~ N(0,1/P), S ~ U(0.5,1.5), U ~ N(0,1/(R b E[S^2])))."""

    def __init__(self, in_features, out_features, b, rank, bias=False, device="cuda", dtype=torch.float16, generator=None):
        super().__init__()
        assert in_features % b == 0 and out_features % b == 0
        self.in_features, self.out_features, self.b, self.rank = in_features, out_features, b, rank
        P, Q = in_features // b, out_features // b
        g = generator
        gd = g.device if g is not None else "cpu"   # a CUDA generator fills the factors on the device (large models)
        if _EMPTY_INIT:
            for name, shp in (("U", (b, Q, rank)), ("Vt", (b, rank, P)), ("S", (b, b, rank))):
                setattr(self, name, nn.Parameter(torch.empty(shp, device=device, dtype=dtype), requires_grad=False))
            self.bias = nn.Parameter(torch.zeros(out_features, device=device, dtype=dtype), requires_grad=False) if bias else None
            return
        rn = lambda *s: torch.randn(*s, generator=g, device=gd)
        self.U = nn.Parameter((rn(b, Q, rank) / math.sqrt(rank * b * 13.0 / 12.0)).to(device=device, dtype=dtype), requires_grad=False)
        self.Vt = nn.Parameter((rn(b, rank, P) / math.sqrt(P)).to(device=device, dtype=dtype), requires_grad=False)
        self.S = nn.Parameter((torch.rand(b, b, rank, generator=g, device=gd) + 0.5).to(device=device, dtype=dtype), requires_grad=False)
        self.bias = nn.Parameter(torch.zeros(out_features, device=device, dtype=dtype), requires_grad=False) if bias else None

    def forward(self, x, out_act=None):
        """out_act ("gelu" | "gelu_tanh"): the activation that follows the layer, applied in the kernels' epilogue where
        the fused call applies."""
        if self.bias is not None or out_act is not None:   # (bias and activation in the kernels' epilogue where the fused call applies)
            return bk.blast_multi_torch_layout(x, [(self.U, self.Vt, self.S)], biases=[self.bias], out_act=out_act)[0]
        return bk.blast_torch_layout(x, self.U, self.Vt, self.S)

    def U_device_ok(self) -> bool:
        return self.U.is_cuda

    def quantized(self, bits: int, group: int = 0) -> "BlastQuantLinear":
        return BlastQuantLinear(self, bits, group)


def _factors16(m):
    """(U, Vt, S, bias) of a stock BLAST layer on 16-bit factors, for the extension's functions over several layers; None: not one."""
    if type(m) is not BlastTorchLinear or not _stock(m):
        return None
    p = m.__dict__["_parameters"]
    return (p["U"], p["Vt"], p["S"], p["bias"]) if p.keys() >= {"U", "Vt", "S", "bias"} else None


@_known
class BlastQuantLinear(nn.Module):
    """The same layer with int8 / packed-int4 factors and fp16 scales (the format of blr_blast_wq)."""

    def __init__(self, src: Optional[BlastTorchLinear], bits: int, group: int = 0):
        super().__init__()
        self.bits, self.group = bits, group
        if src is None:
            return   # BlastQuantLinear.empty fills the rest
        self.in_features, self.out_features, self.b, self.rank = src.in_features, src.out_features, src.b, src.rank
        Uq, us, Vq, vs = bq.quantize_blast_factors(src.U.data, src.Vt.data, bits, group)
        for name, t in (("Uq", Uq), ("u_scale", us), ("Vq", Vq), ("v_scale", vs), ("S", src.S.data)):
            self.register_buffer(name, t)
        self.bias = src.bias

    @classmethod
    def empty(cls, in_features, out_features, b, rank, bits, group=0, bias=False, device="cuda", dtype=torch.float16):
        """The layer with uninitialised buffers of the right shapes (to be filled from a packed-weight file)."""
        m = cls(None, bits, group)
        m.in_features, m.out_features, m.b, m.rank = in_features, out_features, b, rank
        P, Q, per = in_features // b, out_features // b, (1 if bits == 8 else 2)
        e = lambda shp, dt: torch.empty(shp, device=device, dtype=dt)
        m.register_buffer("Uq", e((b, Q, rank // per), torch.int8 if bits == 8 else torch.uint8))
        m.register_buffer("u_scale", e((b, Q) if group == 0 else (b, Q, rank // group), torch.float16))
        m.register_buffer("Vq", e((b, rank, P // per), torch.int8 if bits == 8 else torch.uint8))
        m.register_buffer("v_scale", e((b, rank) if group == 0 else (b, rank, P // group), torch.float16))
        m.register_buffer("S", e((b, b, rank), dtype))
        m.bias = nn.Parameter(torch.zeros(out_features, device=device, dtype=dtype), requires_grad=False) if bias else None
        return m

    def U_device_ok(self) -> bool:
        return self.Uq.is_cuda

    def forward(self, x, out_act=None):
        if self.bias is not None or out_act is not None:
            return bq.blast_wq_multi(x, [(self.Uq, self.u_scale, self.Vq, self.v_scale, self.S)], self.bits, self.group,
                                     biases=[self.bias], out_act=out_act)[0]
        return bq.blast_wq(x, self.Uq, self.u_scale, self.Vq, self.v_scale, self.S, self.bits, self.group)


def make_linear(method: str, in_features: int, out_features: int, b: int, rank: int, bias: bool, device, dtype, generator):
    """method: 'blast' (16-bit factors), 'blast_int8', 'blast_int4', or 'dense' (nn.Linear, the unstructured bar)."""
    if method == "dense":
        lin = nn.Linear(in_features, out_features, bias=bias, device=device, dtype=dtype)
        gd = generator.device if generator is not None else "cpu"
        if _EMPTY_INIT:
            return lin.requires_grad_(False)
        with torch.no_grad():
            lin.weight.copy_((torch.randn(out_features, in_features, generator=generator, device=gd) / math.sqrt(in_features)).to(dtype))
            if bias:
                lin.bias.zero_()
        return lin.requires_grad_(False)
    if _EMPTY_INIT and method in ("blast_int8", "blast_int4"):
        return BlastQuantLinear.empty(in_features, out_features, b, rank, 8 if method == "blast_int8" else 4, 0, bias, device, dtype)
    base = BlastTorchLinear(in_features, out_features, b, rank, bias, device, dtype, generator)
    if method == "blast":
        return base
    if method in ("blast_int8", "blast_int4"):
        return base.quantized(8 if method == "blast_int8" else 4)
    raise ValueError(f"unknown method {method!r}")


def linear_act(m, x, act: str):
    """act(m(x)) for act = "gelu" | "gelu_tanh": inside the layer's kernels where it is a stock BLAST layer of this module, else
    torch's activation on the layer's result."""
    if _stock_blast(m):
        return m(x, out_act=act)
    return F.gelu(m(x), approximate="tanh" if act == "gelu_tanh" else "none")


def structured_multi(mods, x, x_mul=None, residual=None):
    """[m(x') (+ residual) for m in mods] with x' = x, or silu(x) * x_mul: the layers of `mods` share their input.
    BLAST layers of equal shape go through the fused operators (one pair of launches at decode sizes, with the SwiGLU
    product, the bias and the residual folded in); anything else runs layer by layer."""
    res = None if residual is None else [residual] * len(mods)
    if not all(_stock_blast(m) for m in mods):
        pass   # a replaced or hooked layer (tests put the oracle there), a dense one or CPU tensors: layer by layer below
    elif all(isinstance(m, BlastTorchLinear) for m in mods):
        return bk.blast_multi_torch_layout(x, [(m.U, m.Vt, m.S) for m in mods], x_mul, [m.bias for m in mods], res)
    elif all(isinstance(m, BlastQuantLinear) for m in mods) and len({(m.bits, m.group) for m in mods}) == 1:
        return bq.blast_wq_multi(x, [(m.Uq, m.u_scale, m.Vq, m.v_scale, m.S) for m in mods], mods[0].bits, mods[0].group,
                                 x_mul, [m.bias for m in mods], res)
    xe = x if x_mul is None else F.silu(x) * x_mul
    return [m(xe) if residual is None else residual + m(xe) for m in mods]


class MonarchSwiGLU(nn.Module):
    """SwiGLU MLP on Monarch linears, torch layouts (w1_t (b, rank, P), w2_t (b, Qs, rank)): down(silu(gate(x)) * up(x)).
    chain = "ideal": gate and up leave their outputs in the block-major order of the reference's right_ideal variant
    (no interleave; contiguous stores) and down takes block l of that order as its input block l - the chaining of
    configs/networks/llama7b.yaml:164,180; "interleaved": every layer emits the interleaved order (the reference's
    `right`).  The two are different networks on the same factors (monarch_kernels.ideal_order_index)."""

    def __init__(self, d, ffn, b, rank, chain="ideal", device="cuda", dtype=torch.float16, generator=None):
        super().__init__()
        assert chain in ("ideal", "interleaved") and d % b == 0 and ffn % b == 0 and rank % b == 0
        self.d, self.ffn, self.b, self.rank, self.chain = d, ffn, b, rank, chain
        gd = generator.device if generator is not None else "cpu"
        rn = lambda *s: torch.randn(*s, generator=generator, device=gd)
        mk_ = lambda t: nn.Parameter(t.to(device=device, dtype=dtype), requires_grad=False)
        for name, (i_f, o_f) in (("gate", (d, ffn)), ("up", (d, ffn)), ("down", (ffn, d))):
            setattr(self, name + "_w1", mk_(rn(b, rank, i_f // b) / math.sqrt(i_f // b)))
            setattr(self, name + "_w2", mk_(rn(b, o_f // b, rank) / math.sqrt(rank)))

    def forward(self, x):
        from . import monarch_kernels as mk
        ideal = self.chain == "ideal"
        g = mk.monarch_torch_layout(x, self.gate_w1, self.gate_w2, ideal)
        u = mk.monarch_torch_layout(x, self.up_w1, self.up_w2, ideal)
        return mk.monarch_torch_layout(F.silu(g) * u, self.down_w1, self.down_w2)


# ------------------------------------------------------------------------------------------------ Llama-shaped decoder
@dataclass
class LlamaShape:
    """Llama-7B: 32 layers, d = 4096, 32 heads, FFN 11008 (SwiGLU), vocabulary 32000; BLAST b = 16 with the ranks of
    the reference's configs/networks/llama7b.yaml (q/k/v/o 1024, gate/up/down 1488: 50 % of the dense parameters)."""
    layers: int = 32
    d: int = 4096
    heads: int = 32
    ffn: int = 11008
    vocab: int = 32000
    b: int = 16
    rank_attn: int = 1024
    rank_mlp: int = 1488
    rope_theta: float = 10000.0
    eps: float = 1e-6


class RMSNorm(nn.Module):
    def __init__(self, d, eps, device, dtype):
        super().__init__()
        self.weight = nn.Parameter(torch.ones(d, device=device, dtype=dtype), requires_grad=False)
        self.eps = eps

    def forward(self, x):
        if x.is_cuda and x.dtype in (torch.float16, torch.bfloat16) and x.shape[-1] % 8 == 0:
            from . import ops
            out = ops.rmsnorm(x, self.weight, self.eps, or_none=True)   # one kernel instead of five element-wise ones
            if out is not None:
                return out
        v = x.float()
        v = v * torch.rsqrt(v.pow(2).mean(-1, keepdim=True) + self.eps)
        return (v * self.weight.float()).to(x.dtype)


@_known
class LayerNorm(nn.LayerNorm):
    """nn.LayerNorm whose 16-bit CUDA forward is the package's kernel (a warp per row: 12.6 k rows of 768 values took
    torch's kernel 33 us, a sixth of the memory rate); anything else runs torch's."""

    def forward(self, x):
        d = x.shape[-1]
        if x.is_cuda and x.dtype in (torch.float16, torch.bfloat16) and d % 8 == 0 and d <= 2048 and self.normalized_shape == (d,) \
                and not torch.compiler.is_compiling():
            from . import ops
            out = ops.layernorm(x, self.weight, self.bias, self.eps, or_none=True)
            if out is not None:
                return out
        return super().forward(x)


_HALF = (torch.float16, torch.bfloat16)


def _one_kernel(x):
    """Whether the package's norm kernels may stand for what happens to x here: 16-bit rows on the GPU that a warp holds, nothing that
    records or compiles the call."""
    return (x.is_cuda and x.dtype in _HALF and x.size(-1) % 8 == 0 and x.size(-1) <= 2048
            and not torch.compiler.is_compiling() and not torch.jit.is_tracing() and not (x.requires_grad and torch.is_grad_enabled()))


def _plain_norm(norm, d) -> bool:
    """A LayerNorm of this module over rows of d values, of which a fused operator that takes no affine parameters needs eps alone."""
    return type(norm) is LayerNorm and norm.normalized_shape == (d,) and norm.weight is None and norm.bias is None and _stock(norm)


def add_norm(x, y, norm):
    """(t, norm(t)) for t = x + y: a block's residual and the norm behind it, in one kernel where x, y and the norm allow it."""
    if type(norm) is LayerNorm and norm.normalized_shape == (x.size(-1),) and _one_kernel(x) \
            and not (y.requires_grad and torch.is_grad_enabled()) and _stock(norm):
        from . import ops
        out = ops.add_layernorm(x, y, norm.weight, norm.bias, norm.eps, or_none=True)
        if out is not None:
            return out
    t = x + y
    return t, norm(t)


def _rope(q, k, cos, sin):
    """q, k (B, H, T, hd); cos, sin (T, hd/2): rotate pairs (first half, second half) like HF's Llama."""
    def rot(t):
        t1, t2 = t.float().chunk(2, dim=-1)
        return torch.cat((t1 * cos - t2 * sin, t2 * cos + t1 * sin), dim=-1).to(t.dtype)
    return rot(q), rot(k)


class LlamaLayer(nn.Module):
    def __init__(self, shape: LlamaShape, method: str, device, dtype, generator):
        super().__init__()
        s, mk = shape, lambda i, o, r: make_linear(method, i, o, shape.b, r, False, device, dtype, generator)
        self.heads, self.hd = s.heads, s.d // s.heads
        # Batches up to this size use the package's attention kernel (ops.attention_decode), larger ones torch's
        # scaled_dot_product_attention.  Measured through the whole decode step at 2048 keys (ms, torch | package):
        # batch 1 3.08 | 3.23, 4: 3.94 | 4.28, 16: 7.34 | 8.56, 64: 15.5 | 18.0 - torch's flash-decoding kernel streams the
        # cache at 6.3 - 7.3 TB/s, the package's at 4.4 - 5.7: the library kernel serves every batch size.
        self.fused_attention_max_batch = 0
        self.q_proj, self.k_proj, self.v_proj, self.o_proj = (mk(s.d, s.d, s.rank_attn) for _ in range(4))
        self.gate_proj, self.up_proj = mk(s.d, s.ffn, s.rank_mlp), mk(s.d, s.ffn, s.rank_mlp)
        self.down_proj = mk(s.ffn, s.d, s.rank_mlp)
        self.input_layernorm = RMSNorm(s.d, s.eps, device, dtype)
        self.post_attention_layernorm = RMSNorm(s.d, s.eps, device, dtype)

    def structured(self):
        return [self.q_proj, self.k_proj, self.v_proj, self.o_proj, self.gate_proj, self.up_proj, self.down_proj]

    def _decode_fused(self, x, cos_table, sin_table, kc, vc, pos):
        """One new token per sequence on the GPU: four structured-linear calls and four small kernels (two norms,
        rotary embedding + cache append, attention over the cache) instead of some thirty element-wise launches."""
        from . import ops
        B, _, d = x.shape
        h = self.input_layernorm(x)
        q, k, v = (t.view(B, d) for t in structured_multi([self.q_proj, self.k_proj, self.v_proj], h))
        ops.rope_append(q, k, v, cos_table, sin_table, pos, kc, vc, 1)
        if B <= self.fused_attention_max_batch:
            a = ops.attention_decode(q, kc, vc)
        else:
            a = F.scaled_dot_product_attention(q.view(B, self.heads, 1, self.hd), kc, vc).view(B, d)
        (x,) = structured_multi([self.o_proj], a.view(B, 1, d), residual=x)
        h = self.post_attention_layernorm(x)
        g, u = structured_multi([self.gate_proj, self.up_proj], h)
        (x,) = structured_multi([self.down_proj], g, x_mul=u, residual=x)
        return x

    def forward_q8(self, x, tables, cache, start, n_new=None, kernels: bool = True):
        """The layer on an 8-bit cache (ops.Q8Cache) or one in pages (ops.PagedCache): x (B, T, d), the next T tokens of each sequence from slot start[b] on, of which the
        first n_new[b] (None: all) are tokens.  kernels = False reads the cache back and leaves the attention to torch."""
        from . import ops
        B, T, d = x.shape
        paged = isinstance(cache, ops.PagedCache)
        h = self.input_layernorm(x)
        q, k, v = (t.view(B * T, d) for t in structured_multi([self.q_proj, self.k_proj, self.v_proj], h))
        q = (ops.rope_append_paged if paged else ops.rope_append_q8)(q, k, v, tables[0], tables[1], start, cache, n_new)
        if kernels:
            a = (ops.attention_paged if paged else ops.attention_q8)(q, cache, start, n_new)
        else:
            last = start[:, None] + torch.arange(T, device=x.device)   # (slots behind a row's own are masked, and zeros where nobody wrote)
            if paged:
                there = cache.table >= 0
                kc, vc = (t[cache.table.clamp(min=0).long()].transpose(1, 2).reshape(B, self.heads, -1, self.hd) for t in cache[:2])
                written = torch.arange(kc.shape[2], device=x.device) < (start + (T if n_new is None else n_new))[:, None]
                written &= there.repeat_interleave(cache.k.shape[2], 1)
                kc, vc = (t.masked_fill(~written[:, None, :, None], 0) for t in (kc, vc))
            else:
                kc, vc = ops.cache_read_q8(cache, x.dtype, start + (T if n_new is None else n_new))
            seen = torch.arange(kc.shape[2], device=x.device) <= last[..., None]
            if paged:
                seen = seen & written[:, None]
            a = F.scaled_dot_product_attention(q.view(B, T, self.heads, self.hd).transpose(1, 2), kc, vc, attn_mask=seen[:, None]).transpose(1, 2)
        (x,) = structured_multi([self.o_proj], a.reshape(B, T, d), residual=x)
        h = self.post_attention_layernorm(x)
        g, u = structured_multi([self.gate_proj, self.up_proj], h)
        (x,) = structured_multi([self.down_proj], g, x_mul=u, residual=x)
        return x

    def forward(self, x, cos, sin, kc, vc, pos, causal: bool, tables=None):
        """x (B, T, d); kc, vc (B, H, S, hd) static cache; pos (T,) int64 cache slots of these tokens; cos, sin (T, hd/2)
        the angles of those slots.  causal: the T tokens are the whole sequence so far (prefill); else they attend to
        the whole cache.  tables: the full (S, hd/2) cos / sin tables, which selects the fused decode path."""
        B, T, d = x.shape
        if tables is not None and not causal:
            return self._decode_fused(x, tables[0], tables[1], kc, vc, pos)
        h = self.input_layernorm(x)
        if tables is not None:
            # prefill on the GPU (slots 0 .. T-1): one kernel rotates q in place and writes the rotated k and v into the
            # cache, whose first T slots then serve as the keys and values (torch's rotate / cat / index_copy chain was
            # about 390 us per layer at 2048 tokens, 30 % of the prefill)
            from . import ops
            q, k, v = structured_multi([self.q_proj, self.k_proj, self.v_proj], h)
            ops.rope_append(q.view(B * T, d), k.view(B * T, d), v.view(B * T, d), tables[0], tables[1], pos, kc, vc, T)
            a = F.scaled_dot_product_attention(q.view(B, T, self.heads, self.hd).transpose(1, 2), kc[:, :, :T], vc[:, :, :T], is_causal=True)
        else:
            q, k, v = (t.view(B, T, self.heads, self.hd).transpose(1, 2) for t in
                       structured_multi([self.q_proj, self.k_proj, self.v_proj], h))
            q, k = _rope(q, k, cos, sin)
            kc.index_copy_(2, pos, k)
            vc.index_copy_(2, pos, v)
            a = F.scaled_dot_product_attention(q, k, v, is_causal=True) if causal else F.scaled_dot_product_attention(q, kc, vc)
        (x,) = structured_multi([self.o_proj], a.transpose(1, 2).reshape(B, T, -1), residual=x)
        h = self.post_attention_layernorm(x)
        g, u = structured_multi([self.gate_proj, self.up_proj], h)
        (x,) = structured_multi([self.down_proj], g, x_mul=u, residual=x)   # down(silu(gate) * up) + x
        return x


class LlamaDecoder(nn.Module):
    """Decoder of the shape above with a static cache for `cache_len` positions and `batch` sequences.  kv_cache "int8" or "e4m3": the cache in 8 bits with
    a scale for each kv_block slots and head (ops.Q8Cache; CUDA, heads of 64 or 128), which a token attends to up to its own slot; sequences may then be
    at different positions (`extend`, `generate`).  "paged": the same in the activations' 16-bit type, in pages of kv_block slots out of kv_pages for all sequences
    (ops.PagedCache), which `reserve` gives to sequences and `release` takes back; kv_pages None: every sequence has its pages from the beginning.  None: a static cache in the
    activations' 16-bit type."""

    def __init__(self, shape: LlamaShape, method: str, batch: int, cache_len: int, device="cuda", dtype=torch.float16, seed=0,
                 init_on_device: bool = False, kv_cache: Optional[str] = None, kv_block: int = 16, kv_pages: Optional[int] = None):
        super().__init__()
        g = torch.Generator(device=device if init_on_device else "cpu").manual_seed(seed)
        self.shape, self.method, self.batch, self.cache_len = shape, method, batch, cache_len
        self.fused_decode = True   # False: prefill and decode step run torch modules around the linears (no rotary / cache / norm-fusing kernels)
        self.embed_tokens = nn.Embedding(shape.vocab, shape.d, device=device, dtype=dtype)
        with torch.no_grad():
            if not _EMPTY_INIT:
                self.embed_tokens.weight.copy_(torch.randn(shape.vocab, shape.d, generator=g, device=g.device).to(dtype))
        self.embed_tokens.requires_grad_(False)
        self.layers = nn.ModuleList(LlamaLayer(shape, method, device, dtype, g) for _ in range(shape.layers))
        self.norm = RMSNorm(shape.d, shape.eps, device, dtype)
        self.lm_head = make_linear("dense", shape.d, shape.vocab, 0, 0, False, device, dtype, g)
        hd = shape.d // shape.heads
        inv = 1.0 / (shape.rope_theta ** (torch.arange(0, hd, 2, dtype=torch.float32) / hd))
        ang = torch.outer(torch.arange(cache_len, dtype=torch.float32), inv)
        self.register_buffer("cos", ang.cos().to(device), persistent=False)
        self.register_buffer("sin", ang.sin().to(device), persistent=False)
        self.q8cache = None
        self.paged = None
        if kv_pages is not None and kv_cache != "paged":
            raise ValueError("kv_pages is for a cache in pages (kv_cache='paged')")
        if kv_cache == "paged":
            from . import ops
            each = -(-cache_len // kv_block)
            self.kv_pages, self.kv_page = batch * each if kv_pages is None else kv_pages, kv_block
            self.page_table = torch.full((batch, each), -1, dtype=torch.int32, device=device)   # (the layers' caches share it)
            self.paged = [ops.paged_cache(batch, shape.heads, self.kv_pages, each, hd, kv_block, dtype, device)._replace(table=self.page_table) for _ in range(shape.layers)]
            self._pages, self._free = [[] for _ in range(batch)], list(range(self.kv_pages))[::-1]
            if kv_pages is None:
                self.reserve([cache_len] * batch)
        elif kv_cache is not None:
            from . import ops
            codes = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn}.get(kv_cache)
            if codes is None:
                raise ValueError(f"unknown kv_cache {kv_cache!r}")
            self.q8cache = [ops.q8_cache(batch, shape.heads, cache_len, hd, kv_block, codes, device) for _ in range(shape.layers)]
        n16 = shape.layers if kv_cache is None else 0
        self.kcache = [torch.zeros(batch, shape.heads, cache_len, hd, device=device, dtype=dtype) for _ in range(n16)]
        self.vcache = [torch.zeros(batch, shape.heads, cache_len, hd, device=device, dtype=dtype) for _ in range(n16)]

    def structured_linears(self):
        return [m for layer in self.layers for m in layer.structured()]

    def reserve(self, lengths) -> None:
        """Pages for the first lengths[b] slots of sequence b (one number for each of the first sequences), out of those that are free; what a sequence has stays.  Raises
        where there are too few, or where the table cannot be written (inside a stream capture), and then nothing has changed.  The table is written behind what the current stream has been given so far."""
        if self.paged is None:
            raise RuntimeError("reserve needs a decoder with a cache in pages (kv_cache='paged')")
        lengths = [int(n) for n in lengths]
        if len(lengths) > self.batch or any(n < 0 or n > self.cache_len for n in lengths):
            raise ValueError(f"lengths of at most {self.batch} sequences, up to {self.cache_len} slots each")
        more = [max(0, -(-n // self.kv_page) - len(have)) for n, have in zip(lengths, self._pages)]
        if sum(more) > len(self._free):
            raise RuntimeError(f"{sum(more)} more pages are needed, {len(self._free)} are free")
        if sum(more) == 0:
            return
        new = self._free[::-1][:sum(more)]
        dev = torch.tensor(new, dtype=torch.int32).to(self.page_table.device)   # (what a stream capture refuses comes first)
        del self._free[-len(new):]
        for have, row, n in zip(self._pages, self.page_table, more):
            row[len(have):len(have) + n] = dev[:n]
            have.extend(new[:n])
            new, dev = new[n:], dev[n:]

    def release(self, sequences) -> None:
        """Takes back the pages of these sequences (their numbers in the batch); of none where one of them does not exist."""
        if self.paged is None:
            raise RuntimeError("release needs a decoder with a cache in pages (kv_cache='paged')")
        sequences = list(sequences)
        for b in sequences:
            if not 0 <= b < self.batch:
                raise ValueError(f"there is no sequence {b}")
        for b in sequences:
            self._free.extend(reversed(self._pages[b]))
            self._pages[b] = []
            self.page_table[b].fill_(-1)

    def _caches(self):
        """The caches of sequences at positions of their own, one for each layer; None: the static cache."""
        return self.paged if self.paged is not None else self.q8cache

    def _hidden_q8(self, ids, start, n_new=None):
        self._fit(ids)
        x, B = self.embed_tokens(ids), ids.shape[0]
        for layer, cache in zip(self.layers, self._caches()):
            x = layer.forward_q8(x, (self.cos, self.sin), cache.first(B), start, n_new, self.fused_decode)
        return x

    def _run(self, ids, pos, causal):
        logits = self.lm_head(self.norm(self._hidden(ids, pos, causal)[:, -1]))
        return logits if self._caches() is None or causal else self._nan_outside(logits, pos, ids.shape[1])

    def _nan_outside(self, logits, start, n):
        """NaN for sequences whose n tokens from `start` on do not all have a place in the cache: those outside are written nowhere, and the host, which does not
        see the positions, cannot refuse them."""
        outside = start.clamp(min=0).clamp(max=self.cache_len - n) != start
        if self.paged is not None:
            table = self.page_table[:logits.shape[0]]
            at = torch.arange(table.shape[1], device=start.device) * self.kv_page
            first, end = start.clamp(0, self.cache_len), (start.clamp(0, self.cache_len) + n).clamp(max=self.cache_len)
            outside = outside | ((table < 0) & (at + self.kv_page > first[:, None]) & (at < end[:, None])).any(1)
        return logits.masked_fill_(outside[:, None], float("nan"))

    def _fit(self, ids):
        if ids.shape[1] > self.cache_len:
            raise ValueError(f"{ids.shape[1]} tokens do not fit a cache of {self.cache_len} slots")

    def _hidden(self, ids, pos, causal):
        self._fit(ids)
        if self._caches() is not None:
            B = ids.shape[0]
            if self.paged is not None and causal:
                self.reserve([ids.shape[1]] * B)
            return self._hidden_q8(ids, pos.new_zeros(B) if causal else pos if pos.numel() == B else pos.expand(B).contiguous())
        x = self.embed_tokens(ids)
        B = ids.shape[0]   # a smaller batch than the cache was built for uses the first B sequences' slots
        # one new token per sequence on the GPU with 16-bit activations takes the fused decode path
        hd = self.shape.d // self.shape.heads
        kernels = x.is_cuda and x.dtype in (torch.float16, torch.bfloat16) and hd in (8, 16, 32, 64, 128, 256) and self.fused_decode
        # one new token per sequence: the fused decode step; a prefill (the whole sequence so far, slots 0 .. T-1): the rotary
        # / cache kernel in front of torch's causal attention
        fused = kernels and ((not causal and ids.shape[1] == 1) or causal)
        tables = (self.cos, self.sin) if fused else None
        cos, sin = (None, None) if fused else (self.cos.index_select(0, pos), self.sin.index_select(0, pos))
        for i, layer in enumerate(self.layers):
            x = layer(x, cos, sin, self.kcache[i][:B], self.vcache[i][:B], pos, causal, tables)
        return x

    @torch.no_grad()
    def prefill(self, ids: torch.Tensor) -> torch.Tensor:
        """ids (B, T), T <= cache_len: fills cache slots 0..T-1, returns the logits of the last position (B, vocab)."""
        pos = torch.arange(ids.shape[1], device=ids.device)
        return self._run(ids, pos, True)

    @torch.no_grad()
    def decode_step(self, ids: torch.Tensor, pos: torch.Tensor) -> torch.Tensor:
        """ids (B, 1): one new token per sequence, written to cache slot pos (1,) and attending to the whole cache
        (slots beyond the sequence's length must hold real keys: the benchmark decodes at a full cache).  On an 8-bit cache it attends to the slots up to
        its own, and pos may be (B,), one for each sequence; a position outside the cache gives NaN."""
        return self._run(ids, pos, False)

    @torch.no_grad()
    def extend(self, ids: torch.Tensor, start: torch.Tensor, n_new: Optional[torch.Tensor] = None) -> torch.Tensor:
        """The next tokens of sequences at different positions, on an 8-bit cache or one in pages: ids (B, T) go to slots start[b] .. (start (B,) int64), of each row the
        first n_new[b] ((B,) int64; None: all).  Returns the logits behind each sequence's last new token (B, vocab); those of a sequence without a new
        token mean nothing, and those of one with a token outside the cache are NaN."""
        if self._caches() is None:
            raise RuntimeError("extend needs a decoder with an 8-bit cache or one in pages (kv_cache='int8', 'e4m3' or 'paged')")
        x = self._hidden_q8(ids, start, n_new)
        last = x[:, -1] if n_new is None else x[torch.arange(ids.shape[0], device=ids.device), (n_new - 1).clamp(0, ids.shape[1] - 1)]
        T = ids.shape[1]
        return self._nan_outside(self.lm_head(self.norm(last)), start, T if n_new is None else n_new.clamp(0, T))

    @torch.no_grad()
    def generate(self, ids: torch.Tensor, new_tokens: int, uniform: Optional[torch.Tensor] = None, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0,
                 n_new: Optional[torch.Tensor] = None):
        """Goes on from prompts ids (B, T), of each row the first n_new[b] ((B,) int64; None: all), by new_tokens tokens, each chosen as ops.sample does from its
        uniform number (B, new_tokens) fp32 (None: torch.rand) with these settings.  On an 8-bit cache or one in pages, whose first B sequences it begins anew; in pages it reserves
        each sequence's prompt and what it appends, n_new[b] + new_tokens - 1 slots (the last token is the caller's to append, and to reserve for).  Returns (ids, log probabilities), (B, new_tokens) each; a
        sequence without a token has ids -1 and NaN, and so has one that does not fit the cache from there on."""
        from . import ops
        if self._caches() is None:
            raise RuntimeError("generate needs a decoder with an 8-bit cache or one in pages (kv_cache='int8', 'e4m3' or 'paged')")
        B, T = ids.shape
        if uniform is None:
            uniform = torch.rand(B, new_tokens, device=ids.device)
        if uniform.shape != (B, new_tokens):
            raise ValueError(f"uniform: a number for each of {new_tokens} tokens of {B} sequences")
        if self.paged is not None:
            # the last token that is chosen is not appended.  n_new is read back only where not everybody has the pages of a whole row already
            slots = lambda n: min(n + max(new_tokens - 1, 0), self.cache_len) if n > 0 else 0   # noqa: E731
            lengths = [slots(T)] * B
            if n_new is not None and B <= self.batch and any(len(have) * self.kv_page < lengths[0] for have in self._pages[:B]):
                lengths = [slots(n) for n in n_new.clamp(0, T).tolist()]
            self.reserve(lengths)
        pos = ids.new_zeros(B) if n_new is None else n_new
        pos = pos + T if n_new is None else pos.clamp(0, T)
        chosen, logprobs, each = [], [], uniform.t().contiguous()
        logits = self.extend(ids, torch.zeros_like(pos), n_new)
        if n_new is not None:
            logits = logits.masked_fill_((pos == 0)[:, None], float("nan"))
        for i in range(new_tokens):
            token, lp = ops.sample(logits, each[i], temperature, top_k, top_p, min_p)
            chosen.append(token)
            logprobs.append(lp)
            if i + 1 < new_tokens:
                # (a sequence without a token has NaN for its logits from here on: the position that its next one would have is outside the cache)
                pos = torch.where(token < 0, -1, pos)
                logits = self.decode_step(token.clamp(min=0)[:, None], pos)
                pos = torch.where(pos < 0, pos, pos + 1)
        if not chosen:
            return ids.new_zeros(B, 0), uniform
        return torch.stack(chosen, 1), torch.stack(logprobs, 1)

    @torch.no_grad()
    def score(self, ids: torch.Tensor, top: int = 0):
        """How likely a text is: ids (B, T), a prefill of all of it; of each position but the last (log probability of the token that follows, entropy, log
        probabilities of the `top` likeliest tokens, their ids), (B, T - 1) and (B, T - 1, top), as ops.token_logprobs gives them."""
        from . import ops
        x = self._hidden(ids, torch.arange(ids.shape[1], device=ids.device), True)
        return ops.token_logprobs(self.lm_head(self.norm(x[:, :-1])), ids[:, 1:], top)


# ------------------------------------------------------------------------------------------------ ViT-shaped encoder
@dataclass
class ViTShape:
    """ViT-B/16 at 224 x 224: 12 layers, d = 768, 12 heads, MLP 3072, 196 patches + class token = 197 tokens.
    BLAST b = 16 with ranks for 50 % of the dense parameters: R (I + O + b^2) = I O / 2."""
    layers: int = 12
    d: int = 768
    heads: int = 12
    mlp: int = 3072
    image: int = 224
    patch: int = 16
    b: int = 16
    eps: float = 1e-12
    ranks: dict = field(default_factory=lambda: {"qkv": 256, "intermediate": 288, "output": 288})


@_known
class ViTLayer(nn.Module):
    def __init__(self, shape: ViTShape, method: str, device, dtype, generator):
        super().__init__()
        s = shape
        mk = lambda i, o, r: make_linear(method, i, o, s.b, r, True, device, dtype, generator)
        self.heads = s.heads
        self.qkv = mk(s.d, 3 * s.d, s.ranks["qkv"])                 # fused like fuse_qkv_in_vit (vit_b_patch16_224.py:14-66)
        self.attn_out = make_linear("dense", s.d, s.d, 0, 0, True, device, dtype, generator)  # skipped by the reference's swap
        self.intermediate = mk(s.d, s.mlp, s.ranks["intermediate"])
        self.output = mk(s.mlp, s.d, s.ranks["output"])
        self.ln1 = LayerNorm(s.d, eps=s.eps, device=device, dtype=dtype).requires_grad_(False)
        self.ln2 = LayerNorm(s.d, eps=s.eps, device=device, dtype=dtype).requires_grad_(False)

    def structured(self):
        return [self.qkv, self.intermediate, self.output]

    def forward(self, x):
        x, y = self.parts(x, self.ln1(x))
        return x + y

    def parts(self, x, h):
        """The two terms of the layer's result for an input x whose norm is h = ln1(x)."""
        x, h = add_norm(x, self.attention(h), self.ln2)
        return x, self.mlp(h)

    def attention(self, h):
        dr = L.direct()   # (the same calls from one native function: an eager pass on a batch of images is bound by its host time)
        if dr is not None and _stock(self.attn_out) and type(self.attn_out) is nn.Linear:
            layer, lin = _factors16(self.qkv), self.attn_out.__dict__["_parameters"]   # (a weight may also be a plain attribute)
            out = dr.attention(h, layer, self.heads, lin["weight"], lin["bias"]) if layer is not None and lin.keys() >= {"weight", "bias"} else None
            if out is not None:
                return out
        B, T, d = h.shape
        q, k, v = self.qkv(h).view(B, T, 3, self.heads, d // self.heads).permute(2, 0, 3, 1, 4)
        a = F.scaled_dot_product_attention(q, k, v)
        return self.attn_out(a.transpose(1, 2).reshape(B, T, d))

    def mlp(self, h):
        dr = L.direct()
        if dr is not None:
            first, second = _factors16(self.intermediate), _factors16(self.output)
            out = None if first is None or second is None else dr.mlp(h, first, second, L.ACT_OUT["gelu"])
            if out is not None:
                return out
        return self.output(linear_act(self.intermediate, h, "gelu"))


class ViTEncoder(nn.Module):
    def __init__(self, shape: ViTShape, method: str, device="cuda", dtype=torch.float16, seed=0, init_on_device: bool = False):
        super().__init__()
        g = torch.Generator(device=device if init_on_device else "cpu").manual_seed(seed)
        s = shape
        self.shape, self.method = shape, method
        self.patch = nn.Conv2d(3, s.d, s.patch, s.patch, device=device, dtype=dtype).requires_grad_(False)
        ntok = (s.image // s.patch) ** 2 + 1
        self.cls = nn.Parameter((torch.randn(1, 1, s.d, generator=g, device=g.device) * 0.02).to(device=device, dtype=dtype), requires_grad=False)
        self.posemb = nn.Parameter((torch.randn(1, ntok, s.d, generator=g, device=g.device) * 0.02).to(device=device, dtype=dtype), requires_grad=False)
        self.layers = nn.ModuleList(ViTLayer(s, method, device, dtype, g) for _ in range(s.layers))
        self.ln = LayerNorm(s.d, eps=s.eps, device=device, dtype=dtype).requires_grad_(False)

    def structured_linears(self):
        return [m for layer in self.layers for m in layer.structured()]

    @torch.no_grad()
    def forward(self, images: torch.Tensor) -> torch.Tensor:
        """images (B, 3, 224, 224) -> features (B, 197, d)."""
        # the patch embedding as one GEMM over unfolded patches (the convolution's weights, viewed (d, 3 p p)): the strided
        # convolution took 0.48 ms at batch 64 with its layout changes, a twentieth of the whole forward
        B, C, H, W = images.shape
        p = self.shape.patch
        x = images.view(B, C, H // p, p, W // p, p).permute(0, 2, 4, 1, 3, 5).reshape(B, (H // p) * (W // p), C * p * p)
        x = F.linear(x, self.patch.weight.view(self.patch.weight.shape[0], -1), self.patch.bias)
        # class token and position embedding written straight into the token stream: one add over the patch rows instead
        # of a concatenation (62 us at batch 64) followed by an add
        tok = torch.empty(B, x.shape[1] + 1, x.shape[2], device=x.device, dtype=x.dtype)
        tok[:, :1] = self.cls + self.posemb[:, :1]
        torch.add(x, self.posemb[:, 1:], out=tok[:, 1:])
        x = tok
        if len(self.layers) == 0 or not (_one_kernel(x) and all(type(layer) is ViTLayer and _stock(layer) for layer in self.layers)):
            for layer in self.layers:
                x = layer(x)
            return self.ln(x)
        # a layer's last addition together with the norm that follows: the next layer's first, or the encoder's
        h = self.layers[0].ln1(x)
        for layer, norm in zip(self.layers, [layer.ln1 for layer in self.layers[1:]] + [self.ln]):
            x, h = add_norm(*layer.parts(x, h), norm)
        return h


# ------------------------------------------------------------------------------------------------ DiT-shaped denoiser
@dataclass
class DiTShape:
    """DiT-XL/2 on 32 x 32 x 4 latents (256 x 256 images): 28 blocks, d = 1152, 16 heads, MLP 4608, patch 2 -> 256
    tokens, 1000 classes, adaLN-Zero conditioning on timestep + class.  Structured linears and their BLAST settings as
    in the reference's configs/networks/dit_xl.yaml: attn.qkv (rank 384), mlp.fc1 (256), adaLN_modulation.1 (256),
    all with b = 9; attn.proj and mlp.fc2 stay dense."""
    layers: int = 28
    d: int = 1152
    heads: int = 16
    mlp: int = 4608
    latent: int = 32
    patch: int = 2
    channels: int = 4
    classes: int = 1000
    b: int = 9
    freq: int = 256
    eps: float = 1e-6
    ranks: dict = field(default_factory=lambda: {"qkv": 384, "fc1": 256, "adaln": 256})


def _modulate(x, shift, scale):
    """x * (1 + scale) + shift with shift, scale (B, d) broadcast over the tokens: one small add and one fused multiply-add."""
    return torch.addcmul(shift.unsqueeze(1), x, (scale + 1).unsqueeze(1))


@_known
class DiTBlock(nn.Module):
    """x <- x + gate_a * attn(mod(norm(x))), x <- x + gate_m * mlp(mod(norm(x))); the six modulation vectors come
    from one linear on silu(c), c (B, d) the conditioning of the image (one token per image: a decode-size call)."""

    def __init__(self, shape: DiTShape, method: str, device, dtype, generator):
        super().__init__()
        s = shape
        mk = lambda i, o, r: make_linear(method, i, o, s.b, r, True, device, dtype, generator)
        dense = lambda i, o: make_linear("dense", i, o, 0, 0, True, device, dtype, generator)
        self.heads = s.heads
        self.qkv = mk(s.d, 3 * s.d, s.ranks["qkv"])
        self.proj = dense(s.d, s.d)
        self.fc1 = mk(s.d, s.mlp, s.ranks["fc1"])
        self.fc2 = dense(s.mlp, s.d)
        self.adaln = mk(s.d, 6 * s.d, s.ranks["adaln"])
        self.norm1 = LayerNorm(s.d, eps=s.eps, elementwise_affine=False, device=device, dtype=dtype)
        self.norm2 = LayerNorm(s.d, eps=s.eps, elementwise_affine=False, device=device, dtype=dtype)

    def structured(self):
        return [self.qkv, self.fc1, self.adaln]

    def fused(self, x, h, mods, after):
        """x with h, the modulated norm of it -> the block's result and that one's modulated norm, after = (shift, scale, eps): every
        gated residual in one kernel with the norm behind it."""
        from . import ops
        B, T, d = x.shape
        _, _, ga, sm, cm, gm = mods
        q, k, v = self.qkv(h).view(B, T, 3, self.heads, d // self.heads).permute(2, 0, 3, 1, 4)
        a = F.scaled_dot_product_attention(q, k, v)
        x, h = ops.gated_add_modulate(x, ga, self.proj(a.transpose(1, 2).reshape(B, T, d)), sm, cm, self.norm2.eps)
        return ops.gated_add_modulate(x, gm, self.fc2(linear_act(self.fc1, h, "gelu_tanh")), *after)

    def forward(self, x, c):
        B, T, d = x.shape
        sa, ca, ga, sm, cm, gm = self.adaln(F.silu(c)).chunk(6, dim=1)
        # 16-bit tensors on the GPU: norm + modulation in one kernel and the gated residuals in another (torch's broadcast
        # element-wise kernels ran at 1 TB/s: a quarter of the denoiser's time at batch 64)
        fast = x.is_cuda and x.dtype in (torch.float16, torch.bfloat16) and d % 8 == 0 and d <= 2048 and not torch.compiler.is_compiling()
        if fast:
            from . import ops
            mod = lambda norm, t, shift, scale: (ops.layernorm_modulate(t, shift, scale, norm.eps) if _plain_norm(norm, d)
                                                 else _modulate(norm(t), shift, scale))
            gated = ops.gated_add
        else:
            mod = lambda norm, t, shift, scale: _modulate(norm(t), shift, scale)
            gated = lambda t, gate, y: torch.addcmul(t, gate.unsqueeze(1), y)
        q, k, v = self.qkv(mod(self.norm1, x, sa, ca)).view(B, T, 3, self.heads, d // self.heads).permute(2, 0, 3, 1, 4)
        a = F.scaled_dot_product_attention(q, k, v)
        x = gated(x, ga, self.proj(a.transpose(1, 2).reshape(B, T, d)))
        return gated(x, gm, self.fc2(linear_act(self.fc1, mod(self.norm2, x, sm, cm), "gelu_tanh")))


class DiTDenoiser(nn.Module):
    """Latents (B, C, H, W), timesteps (B,), class labels (B,) -> (B, 2C, H, W) (noise and variance channels).  Patch
    embedding, positional embedding, timestep MLP on sinusoidal features, class embedding, the blocks, and an
    adaLN-modulated linear back to patches.  Random weights of the shape (no checkpoint can be fetched here)."""

    def __init__(self, shape: DiTShape, method: str, device="cuda", dtype=torch.float16, seed=0, init_on_device: bool = False):
        super().__init__()
        g = torch.Generator(device=device if init_on_device else "cpu").manual_seed(seed)
        s = shape
        self.shape, self.method = shape, method
        self.x_embed = nn.Conv2d(s.channels, s.d, s.patch, s.patch, device=device, dtype=dtype).requires_grad_(False)
        ntok = (s.latent // s.patch) ** 2
        self.posemb = nn.Parameter((torch.randn(1, ntok, s.d, generator=g, device=g.device) * 0.02).to(device=device, dtype=dtype), requires_grad=False)
        dense = lambda i, o: make_linear("dense", i, o, 0, 0, True, device, dtype, g)
        self.t_fc1, self.t_fc2 = dense(s.freq, s.d), dense(s.d, s.d)
        self.y_embed = nn.Embedding(s.classes + 1, s.d, device=device, dtype=dtype).requires_grad_(False)
        self.blocks = nn.ModuleList(DiTBlock(s, method, device, dtype, g) for _ in range(s.layers))
        self.final_norm = LayerNorm(s.d, eps=s.eps, elementwise_affine=False, device=device, dtype=dtype)
        self.final_adaln = dense(s.d, 2 * s.d)
        self.final = dense(s.d, s.patch * s.patch * 2 * s.channels)
        half = s.freq // 2
        self.register_buffer("freqs", torch.exp(-math.log(10000.0) * torch.arange(half, dtype=torch.float32) / half).to(device), persistent=False)

    def structured_linears(self):
        return [m for blk in self.blocks for m in blk.structured()]

    @torch.no_grad()
    def forward(self, latents: torch.Tensor, t: torch.Tensor, y: torch.Tensor) -> torch.Tensor:
        s = self.shape
        B = latents.shape[0]
        # patch embedding as a GEMM over unfolded patches, which also leaves x token-major and contiguous (the transposed
        # view of a convolution's output made every element-wise kernel after it a strided one and every norm a copy)
        C, p = s.channels, s.patch
        hh = s.latent // p
        x = latents.view(B, C, hh, p, hh, p).permute(0, 2, 4, 1, 3, 5).reshape(B, hh * hh, C * p * p)
        x = F.linear(x, self.x_embed.weight.view(self.x_embed.weight.shape[0], -1), self.x_embed.bias) + self.posemb
        ang = t.float()[:, None] * self.freqs[None]
        temb = torch.cat((ang.cos(), ang.sin()), dim=-1).to(x.dtype)
        c = self.t_fc2(F.silu(self.t_fc1(temb))) + self.y_embed(y)
        a = F.silu(c)
        shift, scale = self.final_adaln(a).chunk(2, dim=1)
        blocks = list(self.blocks)
        if blocks and _one_kernel(x) and _plain_norm(self.final_norm, s.d) and all(
                type(blk) is DiTBlock and _stock(blk) and _stock(blk.adaln) and _plain_norm(blk.norm1, s.d) and _plain_norm(blk.norm2, s.d)
                for blk in blocks):
            # the modulations of all blocks depend on c alone: three blocks' linears at a time share one call
            mods = [m.chunk(6, dim=1) for i in range(0, len(blocks), 3) for m in structured_multi([blk.adaln for blk in blocks[i:i + 3]], a)]
            from . import ops
            h = ops.layernorm_modulate(x, *mods[0][:2], blocks[0].norm1.eps)
            ends = [(*m[:2], blk.norm1.eps) for m, blk in zip(mods[1:], blocks[1:])] + [(shift, scale, self.final_norm.eps)]
            for blk, m, after in zip(blocks, mods, ends):
                x, h = blk.fused(x, h, m, after)
            x = self.final(h)
        else:
            for blk in blocks:
                x = blk(x, c)
            x = self.final(_modulate(self.final_norm(x), shift, scale))
        # patches back to the image grid: (B, h, w, p, p, C) -> (B, C, h p, w p)
        h = s.latent // s.patch
        x = x.view(B, h, h, s.patch, s.patch, 2 * s.channels).permute(0, 5, 1, 3, 2, 4)
        return x.reshape(B, 2 * s.channels, h * s.patch, h * s.patch)


# ------------------------------------------------------------------------------------------------ CUDA-graph replay
class GraphedCall:
    """Captures `fn(*static_inputs)` once in a CUDA graph and replays it; inputs are updated by copying into the
    static tensors.  The structured operators launch on the current stream from caller-provided tensors and their
    per-stream workspace exists after the warm-up calls, so a capture contains no allocation of theirs."""

    def __init__(self, fn, *static_inputs, warmup: int = 2):
        self.fn, self.inputs = fn, static_inputs
        self.stream = torch.cuda.Stream()
        self.stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(self.stream):
            for _ in range(warmup):
                self.out = fn(*static_inputs)
            self.stream.synchronize()
            self.graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(self.graph, stream=self.stream):
                self.out = fn(*static_inputs)
        torch.cuda.current_stream().wait_stream(self.stream)

    def __call__(self, *new_inputs):
        for dst, src in zip(self.inputs, new_inputs):
            dst.copy_(src)
        self.graph.replay()
        return self.out
