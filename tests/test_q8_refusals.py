"""What the operators around the 8-bit cache and the log probabilities refuse, checked without a GPU: every check comes before the device is touched."""
import ctypes as C

import pytest
import torch

ARG, SHAPE, UNSUPPORTED, WORKSPACE = -1, -2, -6, -4


@pytest.fixture(scope="module")
def L():
    from mem_efficient_blr_b200 import build as b
    b.build()
    from mem_efficient_blr_b200 import _lib
    _lib.load()
    return _lib


def _desc(L, **kw):
    d = dict(k=256, v=256, k_scale=256, v_scale=256, n_seq=2, kv_heads=2, slots=40, head_dim=64, block=16, code=0) | kw
    return L.Q8CacheDesc(*d.values())


P = 4096   # an aligned address that nothing reads


def _append(L, desc, q=P, ldq=256, n_tok=1, heads=4, dtype=0, ldo=256, start=P):
    return L.load().blr_rope_append_q8(q, ldq, P, 128, P, 128, P, P, start, None, n_tok, heads, dtype, desc, P, ldo, None)


def _attend(L, desc, q=P, ldq=256, n_tok=1, heads=4, dtype=0, out=P, scratch=P, nbytes=1 << 30, start=P, scale=1.0):
    return L.load().blr_attention_q8(q, ldq, desc, start, None, n_tok, heads, scale, dtype, out, 256, scratch, nbytes, None, None)


@pytest.mark.parametrize("bad", [dict(head_dim=96), dict(head_dim=256), dict(block=8), dict(block=48), dict(block=256), dict(code=2), dict(kv_heads=0), dict(slots=0),
                                 dict(n_seq=-1), dict(k=None), dict(v_scale=None), dict(v=264), dict(k_scale=258)])
def test_caches_that_are_none(L, bad):
    d, lib = _desc(L, **bad), L.load()
    assert _append(L, d) < 0 and _attend(L, d) < 0
    assert lib.blr_cache_read_q8(d, None, 0, P, P, None) < 0
    assert lib.blr_last_error()


def test_arguments_of_the_cache_operators(L):
    d, lib = _desc(L), L.load()
    assert _append(L, d, dtype=2) == ARG and _attend(L, d, dtype=2) == ARG and lib.blr_cache_read_q8(d, None, 3, P, P, None) == ARG
    assert _append(L, d, q=None) == ARG and _attend(L, d, q=None) == ARG and _attend(L, d, start=None) == ARG and _append(L, d, start=None) == ARG
    assert _append(L, d, q=P + 8) == ARG and _attend(L, d, out=P + 8) == ARG and lib.blr_cache_read_q8(d, None, 0, P + 2, P, None) == ARG
    assert _append(L, d, ldq=252) == ARG and _append(L, d, ldo=252) == ARG and _attend(L, d, ldq=252) == ARG
    assert _append(L, d, n_tok=-1) == ARG and _append(L, d, heads=0) == ARG
    assert _attend(L, d, heads=3) == ARG and _attend(L, d, heads=0) == ARG and _attend(L, d, n_tok=-1) == SHAPE
    assert all(_attend(L, d, scale=s) == ARG for s in (0.0, -1.0, float("inf"), float("nan")))
    wide = _desc(L, n_seq=1, kv_heads=1, slots=100000, head_dim=128)
    need = lib.blr_attention_q8_scratch_bytes(wide, 1, 1)
    assert need > 0 and _attend(L, wide, heads=1, nbytes=need - 1) == WORKSPACE and _attend(L, wide, heads=1, scratch=None) == WORKSPACE
    # nothing to do: no launch, no pointer looked at
    none = _desc(L, n_seq=0, k=None, v=None, k_scale=None, v_scale=None)
    assert _append(L, none, q=None) == 0 and _attend(L, none, q=None) == 0 and lib.blr_cache_read_q8(none, None, 0, None, None, None) == 0
    assert _append(L, d, n_tok=0, q=None) == 0 and _attend(L, d, n_tok=0, q=None) == 0


def test_arguments_of_the_log_probabilities(L):
    f = L.load().blr_token_logprobs
    call = lambda logits=P, ld=100, rows=2, vocab=100, kind=0, ids=P, top=3, tl=P: f(logits, ld, rows, vocab, kind, ids, top, P, P, tl, P, None)   # noqa: E731
    assert call(kind=3) == ARG and call(ld=99) == ARG and call(vocab=0) == ARG and call(rows=-1) == ARG
    assert call(top=65) == ARG and call(top=-1) == ARG and call(vocab=2, top=3) == ARG
    assert call(vocab=900000, ld=900000) == UNSUPPORTED and call(vocab=450000, ld=450000, kind=2) == UNSUPPORTED and call(logits=P + 1) == ARG
    assert call(logits=None) == ARG and call(ids=None) == ARG and call(tl=None) == ARG
    assert call(rows=0, logits=None) == 0


def test_the_python_layer_refuses_before_any_launch(L):
    from mem_efficient_blr_b200 import ops
    cache = ops.q8_cache(1, 2, 32, 64, device="cpu")
    x, i = torch.zeros(1, 128, dtype=torch.float16), torch.zeros(1, dtype=torch.int64)
    tab = torch.zeros(32, 32)
    for call in (lambda: ops.rope_append_q8(x, x, x, tab, tab, i, cache), lambda: ops.attention_q8(x, cache, i),
                 lambda: ops.cache_read_q8(cache, torch.float16), lambda: ops.token_logprobs(x, i)):
        with pytest.raises(RuntimeError, match="no CPU implementation"):
            call()
    g = x.clone().requires_grad_(True)
    for call in (lambda: ops.rope_append_q8(x, g, x, tab, tab, i, cache), lambda: ops.attention_q8(g, cache, i), lambda: ops.token_logprobs(g, i)):
        with pytest.raises(RuntimeError, match="no derivative"):
            call()
    for bad in (dict(head_dim=96), dict(block=24), dict(dtype=torch.uint8)):
        with pytest.raises(AssertionError):
            ops.q8_cache(**(dict(n_seq=1, kv_heads=1, slots=16, head_dim=64, device="cpu") | bad))


def test_decoders_of_another_kind_refuse():
    from mem_efficient_blr_b200 import networks as nw
    shape = nw.LlamaShape(layers=1, d=128, heads=2, ffn=128, vocab=32, b=4, rank_attn=16, rank_mlp=16)
    with pytest.raises(ValueError, match="kv_cache"):
        nw.LlamaDecoder(shape, "dense", batch=1, cache_len=8, device="cpu", dtype=torch.float32, kv_cache="int4")
    plain = nw.LlamaDecoder(shape, "dense", batch=1, cache_len=8, device="cpu", dtype=torch.float32)
    with pytest.raises(RuntimeError, match="8-bit cache"):
        plain.extend(torch.zeros(1, 2, dtype=torch.int64), torch.zeros(1, dtype=torch.int64))
    q8 = nw.LlamaDecoder(shape, "dense", batch=1, cache_len=8, device="cpu", dtype=torch.float16, kv_cache="int8")
    assert not q8.kcache and q8.q8cache[0].k.dtype == torch.int8
    with pytest.raises(ValueError, match="9 tokens"):
        q8.prefill(torch.zeros(1, 9, dtype=torch.int64))
