"""The operators around an 8-bit key/value cache and a decoder's answers, as measured: what is called, on which inputs, and what comes out.

* ``append``: rotary embedding of new tokens and the write of their keys and values into a cache of 8-bit codes with one fp32 scale for each block
  of slots and head (``ops.rope_append_q8``);
* ``read``: that cache read back in 16 bits (``ops.cache_read_q8``);
* ``attend``: causal attention of the newest tokens of each sequence over that cache (``ops.attention_q8``), from one token to whole prompts;
* ``logprobs``: log probability of given tokens, entropy and top alternatives of rows of logits (``ops.token_logprobs``).

With ``own`` false ``run`` computes them from elementary torch operations in fp32."""
import math

import torch

own = False
_own_ops = None

DEV = "cuda"
HALF = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
CODE = {"int8": torch.int8, "e4m3": torch.float8_e4m3fn}
TOP = {"int8": 127.0, "e4m3": 448.0}          # the largest code of each kind
LEAST = torch.finfo(torch.float32).tiny       # a block whose scale would be smaller is held as zeros


def _ops():
    global _own_ops
    if _own_ops is None:
        from mem_efficient_blr_b200 import ops
        _own_ops = ops
    return _own_ops


# ------------------------------------------------------------------------------------------------ cases
def listed():
    return [
        # one decode step of 16 sequences of a 32-head decoder: each writes one token somewhere into its cache (latency; some blocks' scales grow)
        dict(name="append_decode_16", op="append", seqs=16, tokens=1, heads=32, kv_heads=32, hd=128, slots=2048, keys=2011, ragged=True, idle=0,
             block=16, code="int8", dtype="fp16"),
        # a whole prompt of 2048 tokens written by one layer
        dict(name="append_prompt_2048", op="append", seqs=1, tokens=2048, heads=32, kv_heads=32, hd=128, slots=2048, keys=2048, ragged=False, idle=0,
             block=16, code="int8", dtype="fp16"),
        # one sequence's cache of one layer handed to something that reads 16 bits
        dict(name="read_1x2048", op="read", seqs=1, kv_heads=32, hd=128, slots=2048, keys=2048, ragged=False, block=16, code="int8", dtype="fp16"),
        # a padded batch of caches of shared heads, an odd number of slots, blocks of 32
        dict(name="read_ragged_16x4099", op="read", seqs=16, kv_heads=8, hd=64, slots=4099, keys=4090, ragged=True, block=32, code="e4m3", dtype="bf16"),
        # decode of one sequence at 2048 keys (latency: 17 MB of codes)
        dict(name="attend_decode_1x2048", op="attend", seqs=1, tokens=1, heads=32, kv_heads=32, hd=128, slots=2048, keys=2048, ragged=False, idle=0,
             block=16, code="int8", dtype="fp16"),
        # decode of a full batch, 64 sequences at 2048 keys
        dict(name="attend_decode_64x2048", op="attend", seqs=64, tokens=1, heads=32, kv_heads=32, hd=128, slots=2048, keys=2048, ragged=False, idle=0,
             block=16, code="int8", dtype="fp16"),
        # decode at long, uneven lengths with shared heads, one place of the batch idle
        dict(name="attend_decode_7x32768", op="attend", seqs=7, tokens=1, heads=32, kv_heads=8, hd=128, slots=32768, keys=32763, ragged=True, idle=1,
             block=64, code="e4m3", dtype="bf16"),
        # five drafted tokens a sequence looked over in one call
        dict(name="attend_drafted_8x5", op="attend", seqs=8, tokens=5, heads=32, kv_heads=8, hd=128, slots=4096, keys=4001, ragged=True, idle=0,
             block=32, code="int8", dtype="bf16"),
        # the next 257 tokens of three prompts of different lengths, heads of 64
        dict(name="attend_chunk_3x257", op="attend", seqs=3, tokens=257, heads=16, kv_heads=4, hd=64, slots=6001, keys=6001, ragged=True, idle=0,
             block=16, code="e4m3", dtype="bf16"),
        # a long prompt at once
        dict(name="attend_prompt_8192", op="attend", seqs=1, tokens=8192, heads=32, kv_heads=8, hd=128, slots=8192, keys=8192, ragged=False, idle=0,
             block=16, code="int8", dtype="fp16"),
        # the answer of a decode step: log probabilities of the chosen tokens with five alternatives
        dict(name="logprobs_step_4", op="logprobs", rows=4, vocab=32000, top=5, dtype="fp16", masked=False),
        # scoring a text of 2047 predicted tokens
        dict(name="logprobs_text_2047", op="logprobs", rows=2047, vocab=32000, top=8, dtype="bf16", masked=False),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _heads(rng):
    kv = rng.choice([1, 2, 4, 8, 16, 32])
    return kv * rng.choice([g for g in (1, 2, 4, 7, 8) if kv * g <= 40]), kv


def _draw(rng):
    op = rng.choice(["append", "read", "attend", "attend", "logprobs"])
    if op == "logprobs":
        return dict(op=op, rows=_log(rng, 1, 4096), vocab=_log(rng, 300, 160000), top=rng.choice([0, 1, 5, 8, 20]),
                    dtype=rng.choice(["fp16", "bf16", "fp32"]), masked=rng.random() < 0.3)
    heads, kv = _heads(rng)
    c = dict(op=op, seqs=_log(rng, 1, 64), kv_heads=kv, hd=rng.choice([64, 128]), block=rng.choice([16, 32, 64, 128]),
             code=rng.choice(["int8", "e4m3"]), dtype=rng.choice(["fp16", "bf16"]), ragged=rng.random() < 0.6)
    keys = _log(rng, 1, 32768)
    if op != "read":
        tokens = 1 if rng.random() < 0.4 else _log(rng, 1, 4096)
        keys = max(keys, tokens)
        c |= dict(tokens=tokens, heads=heads, idle=rng.choice([0, 0, 1]) if c["seqs"] > 1 else 0)
    return c | dict(keys=keys, slots=keys + rng.choice([0, 0, 1, 37, 500]))


def draw(rng):
    most = {}
    for c in listed():
        w = work(c)
        most[c["op"]] = max(most.get(c["op"], (0, 0)), (w["bytes"], w["flops"]), key=lambda p: p[0] / 6.5e12 + p[1] / 1.6e15)
    while True:
        c = _draw(rng)
        w = work(c)
        b, f = most[c["op"]]
        scores = c.get("seqs", 1) * c.get("tokens", 1) * c.get("heads", 1) * c.get("slots", 1) if c["op"] == "attend" else 0
        if w["bytes"] / 6.5e12 + w["flops"] / 1.6e15 <= b / 6.5e12 + f / 1.6e15 and scores <= 32 * 8192 * 8192:
            return c


def _lengths(c):
    """Slots in use of each sequence behind the call: all of `keys`, or down to about half of it."""
    n, t = c["seqs"], c.get("tokens", 1)
    return [max(min(t, c["keys"]), c["keys"] - (b * c["keys"] // (2 * n) if c["ragged"] else 0)) for b in range(n)]


def _new(c):
    """New tokens of each sequence: the last `idle` sequences have none, and in a ragged batch every third has about half."""
    n, t = c["seqs"], c["tokens"]
    return [0 if b >= n - c["idle"] else max(1, t // 2) if c["ragged"] and t > 1 and b % 3 == 2 else t for b in range(n)]


def work(case):
    c = case
    if c["op"] == "logprobs":
        e = HALF[c["dtype"]].itemsize
        return {"bytes": c["rows"] * (c["vocab"] * e + 16 + 12 * c["top"]), "flops": 6 * c["rows"] * c["vocab"]}
    kv, hd, blk = c["kv_heads"], c["hd"], c["block"]
    if c["op"] == "read":
        n = sum(_lengths(c))
        return {"bytes": 2 * kv * (n * hd + 4 * (n // blk + 1)) + 2 * 2 * c["seqs"] * kv * c["slots"] * hd, "flops": 2 * kv * n * hd}
    lens, new = _lengths(c), _new(c)
    rows = sum(new)
    if c["op"] == "append":
        by = rows * hd * (2 * 2 * c["heads"] + 2 * kv * (2 + 1)) + rows * 4 * hd + 2 * 4 * kv * (rows // blk + c["seqs"])
        return {"bytes": by, "flops": rows * hd * (3 * c["heads"] + 6 * kv)}
    seen, pairs = 0, 0
    for ln, t in zip(lens, new):
        first = ln - t if t else 0
        seen += ln if t else 0
        pairs += t * first + t * (t + 1) // 2
    by = 2 * kv * (seen * hd + 4 * (seen // blk + 1)) + 2 * 2 * rows * c["heads"] * hd
    return {"bytes": by, "flops": 4 * hd * c["heads"] * pairs}


# ------------------------------------------------------------------------------------------------ inputs
def _generator(seed):
    return torch.Generator(device=DEV).manual_seed(int(seed) * 7919 + 11)


def _codes(shape, code, g):
    """Codes as a quantised normal variable leaves them: a block's largest value near the largest code, most of the others well below."""
    v = torch.randn(shape, generator=g, device=DEV).mul_(TOP[code] / 4)
    return (v.round_() if code == "int8" else v).clamp_(-TOP[code], TOP[code]).to(CODE[code])


def _cache(c, g):
    shape = (c["seqs"], c["kv_heads"], c["slots"], c["hd"])
    nb = -(-c["slots"] // c["block"])
    scale = lambda: (torch.rand(*shape[:2], nb, generator=g, device=DEV) + 0.6) * (4 / TOP[c["code"]])  # noqa: E731
    return dict(k=_codes(shape, c["code"], g), v=_codes(shape, c["code"], g), k_scale=scale(), v_scale=scale(), block=c["block"])


def prepare(case, seed):
    c, g = dict(case), _generator(seed)
    dt = HALF[c["dtype"]]
    if c["op"] == "logprobs":
        # peaked rows, as a trained model gives: one token in a hundred well above the rest
        x = torch.randn(c["rows"], c["vocab"], generator=g, device=DEV) * 2
        x += 4 * (torch.rand(c["rows"], c["vocab"], generator=g, device=DEV) < 0.01)
        if c["masked"]:   # tokens that a grammar rules out
            x.masked_fill_(torch.rand(c["rows"], c["vocab"], generator=g, device=DEV) < 0.5, -math.inf)
            x[:, 0] = 0.0
        ids = torch.randint(0, c["vocab"], (c["rows"],), generator=g, device=DEV)
        return dict(c=c, logits=x.to(dt), ids=ids)
    s = dict(c=c, cache=_cache(c, g))
    lens = _lengths(c)
    if c["op"] == "read":
        s["lengths"] = torch.tensor(lens, device=DEV)
        return s
    new = _new(c)
    s["start"] = torch.tensor([ln - t for ln, t in zip(lens, new)], device=DEV)
    s["n_new"] = torch.tensor(new, device=DEV)
    rows = c["seqs"] * c["tokens"]
    rn = lambda h: (torch.randn(rows, h * c["hd"], generator=g, device=DEV) * (2.0 if c["op"] == "attend" else 1.0)).to(dt)  # noqa: E731
    s["q"] = rn(c["heads"])
    if c["op"] == "append":
        s["kn"], s["vn"] = rn(c["kv_heads"]), rn(c["kv_heads"])
        inv = 10000.0 ** (-torch.arange(0, c["hd"], 2, device=DEV, dtype=torch.float64) / c["hd"])
        ang = torch.outer(torch.arange(c["slots"], device=DEV, dtype=torch.float64), inv)
        s["cos"], s["sin"] = ang.cos().float(), ang.sin().float()
    return s


# ------------------------------------------------------------------------------------------------ one pass
def run(state):
    s, c = state, state["c"]
    if own:
        o = _ops()
        if c["op"] == "logprobs":
            return o.token_logprobs(s["logits"], s["ids"], c["top"])
        cache = o.Q8Cache(**s["cache"])
        if c["op"] == "read":
            return o.cache_read_q8(cache, HALF[c["dtype"]], s["lengths"])
        if c["op"] == "attend":
            return o.attention_q8(s["q"], cache, s["start"], s["n_new"])
        q = o.rope_append_q8(s["q"], s["kn"], s["vn"], s["cos"], s["sin"], s["start"], cache, s["n_new"])
        return q, cache.k, cache.v, cache.k_scale, cache.v_scale
    return {"append": _append, "read": _read, "attend": _attend, "logprobs": _logprobs}[c["op"]](s, c)


def _per_slot(scale, block, slots):
    """(.., blocks) -> (.., slots, 1): each slot's scale."""
    return scale.repeat_interleave(block, dim=-1)[..., :slots].unsqueeze(-1)


def _rotate(x, cos, sin):
    a, b = x.chunk(2, dim=-1)
    return torch.cat((a * cos - b * sin, b * cos + a * sin), dim=-1)


def _quantised(v, code):
    return (v.round() if code == "int8" else v).clamp(-TOP[code], TOP[code]).to(CODE[code])


def _write(codes, scale, new, slot, start, n_new, c):
    """new (B, T, KV, hd) fp32 into the slots (B, T) of codes (B, KV, S, hd), scale (B, KV, blocks), in place: a block's scale is the largest that its
    tokens asked for since the block was begun, and codes that were there before are brought to a scale that has grown."""
    B, T, KV, hd = new.shape
    blk, S, top = c["block"], c["slots"], TOP[c["code"]]
    t = torch.arange(T, device=new.device)
    have = t[None] < n_new[:, None]
    which = (slot // blk).clamp(0, scale.shape[2] - 1)
    need = torch.where(have[..., None], new.abs().amax(-1), 0.0).transpose(1, 2)                       # (B, KV, T)
    most = torch.zeros_like(scale).scatter_reduce_(2, which[:, None].expand(B, KV, T), need, "amax")
    begun = torch.arange(scale.shape[2], device=new.device) * blk >= start[:, None]                     # a block that begins with this call
    touched = torch.zeros_like(begun, dtype=torch.int32).scatter_reduce_(1, which, have.int(), "amax")[:, None].bool()
    asked = most / top
    asked = torch.where(asked < LEAST, 0.0, asked)
    before = torch.where(begun[:, None], 0.0, scale)
    after = torch.where(touched, torch.maximum(before, asked), scale)
    inverse = torch.where(after > 0, 1.0 / after, 0.0)
    # the one block that may hold older tokens: the block of the first new slot
    b0 = (start // blk).clamp(0, scale.shape[2] - 1)
    at = (b0[:, None] * blk + torch.arange(blk, device=new.device)).clamp(max=S - 1)                    # (B, blk)
    at4 = at[:, None, :, None].expand(B, KV, blk, hd)
    old = codes.view(torch.uint8).gather(2, at4).view(codes.dtype)
    one = b0[:, None, None].expand(B, KV, 1)
    ratio = before.gather(2, one) * inverse.gather(2, one)
    grown = (after.gather(2, one) > before.gather(2, one)) & (at < start[:, None])[:, None]             # (B, KV, blk)
    kept = torch.where(grown[..., None], _quantised(old.float() * ratio[..., None], c["code"]).view(torch.uint8), old.view(torch.uint8))
    codes.view(torch.uint8).scatter_(2, at4, kept)
    # the new tokens; places behind a sequence's last one repeat that one, and a sequence without any rewrites what is there
    tt = torch.minimum(t[None].expand(B, T), (n_new - 1).clamp(min=0)[:, None])
    to = slot.gather(1, tt).clamp(0, S - 1)
    val = new.gather(1, tt[..., None, None].expand(B, T, KV, hd)).transpose(1, 2)
    inv = inverse.gather(2, (to // blk)[:, None].expand(B, KV, T))
    to4 = to[:, None, :, None].expand(B, KV, T, hd)
    put = torch.where((n_new > 0)[:, None, None, None], _quantised(val * inv[..., None], c["code"]).view(torch.uint8),
                      codes.view(torch.uint8).gather(2, to4))
    codes.view(torch.uint8).scatter_(2, to4, put)
    scale.copy_(after)


def _append(s, c):
    B, T, H, KV, hd = c["seqs"], c["tokens"], c["heads"], c["kv_heads"], c["hd"]
    t = torch.arange(T, device=s["q"].device)
    slot = s["start"][:, None] + t
    at = slot.clamp(0, c["slots"] - 1)
    cos, sin = s["cos"][at][:, :, None], s["sin"][at][:, :, None]
    q = _rotate(s["q"].view(B, T, H, hd).float(), cos, sin)
    q = torch.where((t[None] < s["n_new"][:, None])[..., None, None], q, 0.0).to(s["q"].dtype).view(B * T, H * hd)
    k = _rotate(s["kn"].view(B, T, KV, hd).float(), cos, sin)
    m = s["cache"]
    _write(m["k"], m["k_scale"], k, slot, s["start"], s["n_new"], c)
    _write(m["v"], m["v_scale"], s["vn"].view(B, T, KV, hd).float(), slot, s["start"], s["n_new"], c)
    return q, m["k"], m["v"], m["k_scale"], m["v_scale"]


def _read(s, c):
    m, S = s["cache"], c["slots"]
    live = (torch.arange(S, device=DEV) < s["lengths"][:, None])[:, None, :, None]
    one = lambda x, sc: torch.where(live, x.float() * _per_slot(sc, c["block"], S), 0.0).to(HALF[c["dtype"]])  # noqa: E731
    return one(m["k"], m["k_scale"]), one(m["v"], m["v_scale"])


def _attend(s, c):
    B, T, H, KV, hd, S = c["seqs"], c["tokens"], c["heads"], c["kv_heads"], c["hd"], c["slots"]
    m, G = s["cache"], c["heads"] // c["kv_heads"]
    k = m["k"].float() * _per_slot(m["k_scale"], c["block"], S)
    v = m["v"].float() * _per_slot(m["v_scale"], c["block"], S)
    q = s["q"].view(B, T, KV, G, hd).permute(0, 2, 1, 3, 4).reshape(B, KV, T * G, hd).float() * hd ** -0.5
    x = (q @ k.transpose(2, 3)).view(B, KV, T, G, S)
    t = torch.arange(T, device=DEV)
    seen = torch.where(t[None] < s["n_new"][:, None], s["start"][:, None] + t + 1, 0)                   # (B, T) slots that a row sees
    x.masked_fill_((torch.arange(S, device=DEV) >= seen[..., None])[:, None, :, None], -math.inf)
    top = x.amax(-1, keepdim=True)
    p = x.sub_(torch.where(top == -math.inf, 0.0, top)).exp_()
    total = p.sum(-1, keepdim=True)
    out = (p.view(B, KV, T * G, S) @ v).view(B, KV, T, G, hd) / torch.where(total == 0, 1.0, total)
    return out.permute(0, 2, 1, 3, 4).reshape(B * T, H * hd).to(HALF[c["dtype"]])


def _logprobs(s, c):
    x = s["logits"].float()
    top = x.amax(-1, keepdim=True)
    e = (x - top).exp()
    total = e.sum(-1, keepdim=True)
    lse = top + total.log()
    entropy = (lse - (torch.where(e > 0, x, 0.0) * e).sum(-1, keepdim=True) / total)[:, 0]
    given = (x.gather(1, s["ids"][:, None]) - lse)[:, 0]
    best, at = x.sort(dim=-1, descending=True, stable=True)   # ties to the lowest index
    return given, entropy, (best[:, :c["top"]] - lse).contiguous(), at[:, :c["top"]].contiguous()


# ------------------------------------------------------------------------------------------------ the definition in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    c = s["c"]
    if c["op"] == "logprobs":
        parts = [_exact_logprobs(x.double(), i, c["top"]) for x, i in zip(s["logits"].split(64), s["ids"].split(64))]
        return tuple(torch.cat(p) for p in zip(*parts))
    m, blk = s["cache"], c["block"]
    of_slot = torch.arange(c["slots"], device=DEV) // blk
    if c["op"] == "read":
        outs = []
        for x, sc in ((m["k"], m["k_scale"]), (m["v"], m["v_scale"])):
            o = torch.zeros(x.shape, dtype=torch.float64, device=DEV)
            for b, n in enumerate(_lengths(c)):
                o[b, :, :n] = x[b, :, :n].to(torch.float64) * sc[b].double()[:, of_slot[:n], None]
            outs.append(o)
        return tuple(outs)
    B, T, H, KV, hd = c["seqs"], c["tokens"], c["heads"], c["kv_heads"], c["hd"]
    new, first = s["n_new"].tolist(), s["start"].tolist()
    if c["op"] == "append":
        q = torch.zeros(B, T, H, hd // 2, dtype=torch.complex128, device=DEV)
        scales = [m["k_scale"].double(), m["v_scale"].double()]
        for b in range(B):
            if not new[b]:
                continue
            at = torch.arange(first[b], first[b] + new[b], device=DEV)
            turn = torch.complex(s["cos"][at].double(), s["sin"][at].double())[:, None]                 # a pair as one complex number
            pairs = lambda x, h: torch.complex(*x.view(B, T, h, 2, hd // 2)[b, :new[b]].double().unbind(2))  # noqa: E731
            q[b, :new[b]] = pairs(s["q"], H) * turn
            k = pairs(s["kn"], KV) * turn
            size = [torch.maximum(k.real.abs(), k.imag.abs()).amax(-1), s["vn"].view(B, T, KV, hd)[b, :new[b]].double().abs().amax(-1)]
            for j in range(first[b] // blk, (first[b] + new[b] - 1) // blk + 1):
                here = (at // blk) == j
                for sc, z in zip(scales, size):
                    asked = z[here].amax(0) / TOP[c["code"]]
                    sc[b, :, j] = asked if j * blk >= first[b] else torch.maximum(sc[b, :, j], asked)
        q = torch.cat((q.real, q.imag), -1).reshape(B * T, H * hd)
        return q, None, None, scales[0], scales[1]
    out = torch.zeros(B, T, H, hd, dtype=torch.float64, device=DEV)
    for b in range(B):
        n, f = new[b], first[b]
        if not n:
            continue
        sees = torch.arange(f, f + n, device=DEV)
        for h in range(KV):
            dq = lambda x, sc: x[b, h, :f + n].to(torch.float64) * sc[b, h].double()[of_slot[:f + n], None]  # noqa: E731
            k, v = dq(m["k"], m["k_scale"]), dq(m["v"], m["v_scale"])
            for g in range(H // KV):
                head = h * (H // KV) + g
                x = s["q"].view(B, T, H, hd)[b, :n, head].double() @ k.T / math.sqrt(hd)
                x = x.masked_fill(torch.arange(f + n, device=DEV) > sees[:, None], -math.inf)
                out[b, :n, head] = torch.softmax(x, -1) @ v
    return out.view(B * T, H * hd)


def _exact_logprobs(x, ids, top):
    lp = torch.log_softmax(x, -1)
    entropy = torch.special.entr(lp.exp()).sum(-1)
    order = x.argsort(dim=-1, descending=True, stable=True)[:, :top]
    return lp.gather(1, ids[:, None])[:, 0], entropy, lp.gather(1, order), order
