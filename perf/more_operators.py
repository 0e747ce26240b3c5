"""The operators around a key/value cache in pages and the choice of the next token, as measured: what is called, on which inputs, and what comes out.

* ``append``: rotary embedding of new tokens and the write of their keys and values into a cache whose slots lie in pages of a common pool
  (``ops.rope_append_paged``);
* ``attend``: causal attention of the newest tokens of each sequence over that cache (``ops.attention_paged``), from one token to whole prompts;
* ``sample``: the next token of rows of logits from given uniform numbers, with temperature, top-k, top-p and min-p (``ops.sample``).

With ``own`` false ``run`` computes them from elementary torch operations, in fp32, and the choice of a token in 64 bits."""
import math

import torch

own = False
_own_ops = None

DEV = "cuda"
TYPE = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}


def _ops():
    global _own_ops
    if _own_ops is None:
        from mem_efficient_blr_b200 import ops
        _own_ops = ops
    return _own_ops


# ------------------------------------------------------------------------------------------------ cases
def listed():
    return [
        # one decode step of 16 sequences of a 32-head decoder: each writes one token into its last page (latency)
        dict(name="append_step_16", op="append", seqs=16, tokens=1, heads=32, kv_heads=32, hd=128, keys=2011, ragged=True, idle=0, page=16, dtype="fp16"),
        # a whole prompt of 2048 tokens written by one layer
        dict(name="append_prompt_2048", op="append", seqs=1, tokens=2048, heads=32, kv_heads=32, hd=128, keys=2048, ragged=False, idle=0, page=64, dtype="fp16"),
        # the next pieces of five prompts of different lengths, shared heads, one place of the batch idle
        dict(name="append_pieces_5x777", op="append", seqs=5, tokens=777, heads=28, kv_heads=4, hd=64, keys=3001, ragged=True, idle=1, page=32, dtype="bf16"),
        # decode of one sequence at 2048 keys (latency: 34 MB of keys and values)
        dict(name="attend_step_1x2048", op="attend", seqs=1, tokens=1, heads=32, kv_heads=32, hd=128, keys=2048, ragged=False, idle=0, page=16, dtype="fp16"),
        # decode of a full batch, 64 sequences at 2048 keys
        dict(name="attend_step_64x2048", op="attend", seqs=64, tokens=1, heads=32, kv_heads=32, hd=128, keys=2048, ragged=False, idle=0, page=16, dtype="fp16"),
        # decode at long, uneven lengths with shared heads, one place of the batch idle
        dict(name="attend_step_7x32763", op="attend", seqs=7, tokens=1, heads=32, kv_heads=8, hd=128, keys=32763, ragged=True, idle=1, page=64, dtype="bf16"),
        # five drafted tokens a sequence looked over in one call
        dict(name="attend_drafted_8x5", op="attend", seqs=8, tokens=5, heads=32, kv_heads=8, hd=128, keys=4001, ragged=True, idle=0, page=32, dtype="bf16"),
        # the next 257 tokens of three prompts of different lengths, heads of 64
        dict(name="attend_pieces_3x257", op="attend", seqs=3, tokens=257, heads=16, kv_heads=4, hd=64, keys=6001, ragged=True, idle=0, page=16, dtype="bf16"),
        # a long prompt at once
        dict(name="attend_prompt_8192", op="attend", seqs=1, tokens=8192, heads=32, kv_heads=8, hd=128, keys=8192, ragged=False, idle=0, page=128, dtype="fp16"),
        # the next token of a few sequences, as a chat is answered
        dict(name="sample_step_4", op="sample", rows=4, vocab=32000, dtype="fp16", top_k=50, top_p=0.95, min_p=0.0, masked=False),
        # a large batch by nucleus alone, each row with its own settings
        dict(name="sample_nucleus_256", op="sample", rows=256, vocab=32000, dtype="bf16", top_k=0, top_p=0.9, min_p=0.02, masked=False),
        # many rows from the whole distribution, logits in fp32, some tokens ruled out
        dict(name="sample_whole_1024", op="sample", rows=1024, vocab=50001, dtype="fp32", top_k=0, top_p=1.0, min_p=0.0, masked=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _heads(rng):
    kv = rng.choice([1, 2, 4, 8, 16, 32])
    return kv * rng.choice([g for g in (1, 2, 4, 7, 8) if kv * g <= 40]), kv


def _draw(rng):
    op = rng.choice(["append", "attend", "attend", "sample", "sample"])
    if op == "sample":
        return dict(op=op, rows=_log(rng, 1, 1024), vocab=_log(rng, 300, 160000), dtype=rng.choice(["fp16", "bf16", "fp32"]),
                    top_k=rng.choice([0, 0, 1, 20, 50, 200, 1000]), top_p=rng.choice([1.0, 1.0, 0.5, 0.9, 0.95, 0.99]), min_p=rng.choice([0.0, 0.0, 0.02, 0.1]),
                    masked=rng.random() < 0.3)
    heads, kv = _heads(rng)
    seqs = _log(rng, 1, 64)
    tokens = 1 if rng.random() < 0.4 else _log(rng, 1, 4096)
    return dict(op=op, seqs=seqs, tokens=tokens, heads=heads, kv_heads=kv, hd=rng.choice([64, 128]), keys=max(tokens, _log(rng, 1, 32768)),
                ragged=rng.random() < 0.6, idle=rng.choice([0, 0, 1]) if seqs > 1 else 0, page=rng.choice([16, 32, 64, 128]), dtype=rng.choice(["fp16", "bf16"]))


def _cost(c):
    w = work(c)
    return w["bytes"] / 6.5e12 + w["flops"] / 1.6e15


def _held(c):
    """Bytes of the pool that a case needs."""
    return 0 if c["op"] == "sample" else 4 * c["seqs"] * c["kv_heads"] * c["keys"] * c["hd"]


def draw(rng):
    most, held = {}, {}
    for c in listed():
        most[c["op"]] = max(most.get(c["op"], 0), _cost(c))
        held[c["op"]] = max(held.get(c["op"], 0), _held(c))
    while True:
        c = _draw(rng)
        if c.get("top_k", 0) > c.get("vocab", 0):
            continue
        scores = c["seqs"] * c["tokens"] * c["heads"] * c["keys"] if c["op"] == "attend" else 0   # (the plain form holds them all)
        if _cost(c) <= most[c["op"]] and _held(c) <= held[c["op"]] and scores <= 32 * 8192 * 8192:
            return c


def _lengths(c):
    """Slots in use of each sequence behind the call: all of `keys`, or down to about half of it."""
    n, t = c["seqs"], c["tokens"]
    return [max(min(t, c["keys"]), c["keys"] - (b * c["keys"] // (2 * n) if c["ragged"] else 0)) for b in range(n)]


def _new(c):
    """New tokens of each sequence: the last `idle` sequences have none, and in a ragged batch every third has about half."""
    n, t = c["seqs"], c["tokens"]
    return [0 if b >= n - c["idle"] else max(1, t // 2) if c["ragged"] and t > 1 and b % 3 == 2 else t for b in range(n)]


def work(case):
    c = case
    if c["op"] == "sample":   # each logit once, the row's number and settings in, its token and log probability out
        return {"bytes": c["rows"] * (c["vocab"] * TYPE[c["dtype"]].itemsize + 24 + 12), "flops": 6 * c["rows"] * c["vocab"]}
    kv, hd = c["kv_heads"], c["hd"]
    lens, new = _lengths(c), _new(c)
    rows = sum(new)
    if c["op"] == "append":
        return {"bytes": rows * hd * (2 * 2 * c["heads"] + 2 * 2 * 2 * kv) + rows * 4 * hd, "flops": rows * hd * 3 * (c["heads"] + kv)}
    seen, pairs = 0, 0
    for ln, t in zip(lens, new):
        first = ln - t if t else 0
        seen += ln if t else 0
        pairs += t * first + t * (t + 1) // 2
    return {"bytes": 2 * 2 * kv * seen * hd + 2 * 2 * rows * c["heads"] * hd, "flops": 4 * hd * c["heads"] * pairs}


# ------------------------------------------------------------------------------------------------ inputs
def _generator(seed):
    return torch.Generator(device=DEV).manual_seed(int(seed) * 7919 + 11)


def prepare(case, seed):
    c, g = dict(case), _generator(seed)
    dt = TYPE[c["dtype"]]
    if c["op"] == "sample":
        return _prepare_sample(c, g, dt)
    # pages in no order, some of them spare; no page behind a sequence's last
    lens, new, P = _lengths(c), _new(c), c["page"]
    each = -(-c["keys"] // P)
    need = [-(-n // P) for n in lens]
    pages = sum(need) + 3
    order = torch.randperm(pages, generator=g, device=DEV).to(torch.int32).split([*need, 3])
    table = torch.full((c["seqs"], each), -1, dtype=torch.int32, device=DEV)
    for b, mine in enumerate(order[:-1]):
        table[b, :need[b]] = mine
    pool = lambda: torch.randn(pages, c["kv_heads"], P, c["hd"], generator=g, device=DEV, dtype=dt)  # noqa: E731
    s = dict(c=c, k=pool(), v=pool(), table=table)
    s["start"] = torch.tensor([n - t for n, t in zip(lens, new)], device=DEV)
    s["n_new"] = torch.tensor(new, device=DEV)
    rows = c["seqs"] * c["tokens"]
    rn = lambda h: (torch.randn(rows, h * c["hd"], generator=g, device=DEV) * (2.0 if c["op"] == "attend" else 1.0)).to(dt)  # noqa: E731
    s["q"] = rn(c["heads"])
    if c["op"] == "append":
        s["kn"], s["vn"] = rn(c["kv_heads"]), rn(c["kv_heads"])
        inv = 10000.0 ** (-torch.arange(0, c["hd"], 2, device=DEV, dtype=torch.float64) / c["hd"])
        ang = torch.outer(torch.arange(each * P, device=DEV, dtype=torch.float64), inv)
        s["cos"], s["sin"] = ang.cos().float(), ang.sin().float()
    return s


def _prepare_sample(c, g, dt):
    """Rows as a trained model gives them: the r-th likeliest token has a probability like r^-a, with an a of the row's own from hardly to very sure."""
    R, V = c["rows"], c["vocab"]
    uni = lambda lo, hi: torch.rand(R, generator=g, device=DEV) * (hi - lo) + lo  # noqa: E731
    x = torch.empty(R, V, device=DEV).exponential_(generator=g).mul_(uni(0.9, 2.2)[:, None]).add_(uni(-12.0, -4.0)[:, None])
    if c["masked"]:   # tokens that a grammar rules out
        x.masked_fill_(torch.rand(R, V, generator=g, device=DEV) < 0.4, -math.inf)
        x[:, 0] = 0.0
    row = torch.arange(R, device=DEV)
    k, p, mp = c["top_k"], c["top_p"], c["min_p"]
    t = uni(0.6, 1.2)
    t[row % 16 == 15] = 0.0   # a request in sixteen wants the likeliest token
    return dict(c=c, logits=x.to(dt), uniform=uni(0.0, 1.0), temperature=t,
                top_k=torch.where(row % 7 == 6, k + k // 2, k), top_p=p if p >= 1.0 else uni(p - 0.05, p), min_p=mp if mp <= 0.0 else uni(0.0, mp))


# ------------------------------------------------------------------------------------------------ one pass
def run(state):
    s, c = state, state["c"]
    if own:
        o = _ops()
        if c["op"] == "sample":
            return o.sample(s["logits"], s["uniform"], s["temperature"], s["top_k"], s["top_p"], s["min_p"])
        cache = o.PagedCache(s["k"], s["v"], s["table"])
        if c["op"] == "attend":
            return o.attention_paged(s["q"], cache, s["start"], s["n_new"])
        return o.rope_append_paged(s["q"], s["kn"], s["vn"], s["cos"], s["sin"], s["start"], cache, s["n_new"]), cache.k, cache.v
    return {"append": _append, "attend": _attend, "sample": _sample}[c["op"]](s, c)


def _rotate(x, cos, sin):
    a, b = x.chunk(2, dim=-1)
    return torch.cat((a * cos - b * sin, b * cos + a * sin), dim=-1)


def _append(s, c):
    B, T, H, KV, hd, P = c["seqs"], c["tokens"], c["heads"], c["kv_heads"], c["hd"], c["page"]
    t = torch.arange(T, device=s["q"].device)
    have = t[None] < s["n_new"][:, None]
    slot = (s["start"][:, None] + t).clamp(max=s["table"].shape[1] * P - 1)
    cos, sin = s["cos"][slot][:, :, None], s["sin"][slot][:, :, None]
    q = _rotate(s["q"].view(B, T, H, hd).float(), cos, sin)
    q = torch.where(have[..., None, None], q, 0.0).to(s["q"].dtype).view(B * T, H * hd)
    k = _rotate(s["kn"].view(B, T, KV, hd).float(), cos, sin).to(s["k"].dtype)
    page = s["table"].long().gather(1, slot // P)
    at = (page[have], slice(None), (slot % P)[have])
    s["k"][at] = k[have]
    s["v"][at] = s["vn"].view(B, T, KV, hd)[have]
    return q, s["k"], s["v"]


def _attend(s, c):
    B, T, H, KV, hd, P = c["seqs"], c["tokens"], c["heads"], c["kv_heads"], c["hd"], c["page"]
    G, S = H // KV, s["table"].shape[1] * P
    flat = lambda pool: pool[s["table"].clamp(min=0).long()].transpose(1, 2).reshape(B, KV, S, hd).float()  # noqa: E731
    q = s["q"].view(B, T, KV, G, hd).permute(0, 2, 1, 3, 4).reshape(B, KV, T * G, hd).float() * hd ** -0.5
    x = (q @ flat(s["k"]).transpose(2, 3)).view(B, KV, T, G, S)
    t = torch.arange(T, device=DEV)
    seen = torch.where(t[None] < s["n_new"][:, None], s["start"][:, None] + t + 1, 0)                   # (B, T) slots that a row sees
    x.masked_fill_((torch.arange(S, device=DEV) >= seen[..., None])[:, None, :, None], -math.inf)
    top = x.amax(-1, keepdim=True)
    p = x.sub_(torch.where(top == -math.inf, 0.0, top)).exp_()
    total = p.sum(-1, keepdim=True)
    out = (p.view(B, KV, T * G, S) @ flat(s["v"])).view(B, KV, T, G, hd) / torch.where(total == 0, 1.0, total)
    return out.permute(0, 2, 1, 3, 4).reshape(B * T, H * hd).to(s["q"].dtype)


def _column(v, like):
    """A setting as a column in 64 bits: one for all rows, which the operator holds in 32, or one for each."""
    return v.double()[:, None] if torch.is_tensor(v) else torch.full((like.shape[0], 1), v, dtype=torch.float32, device=like.device).double()


def _sample(s, c):
    """Tokens in the order of falling logits decide what is kept, in their own order which one is drawn; 64 bits, since a sum may end next to a border."""
    x = s["logits"].double()
    R, V = x.shape
    T, tp, mp, u = (_column(s[n], x) for n in ("temperature", "top_p", "min_p", "uniform"))
    top_k = s["top_k"][:, None]
    best, order = x.sort(dim=-1, descending=True, stable=True)
    place = torch.arange(V, device=x.device)[None]
    gap = best - best[:, :1]
    w = torch.where(T > 0, torch.exp(gap / torch.where(T > 0, T, 1.0)), (place == 0).double())
    w = torch.where((top_k <= 0) | (place < top_k), w, 0.0)
    before = w.cumsum(-1) - w
    w = torch.where((tp >= 1) | (place == 0) | (before < tp * w.sum(-1, keepdim=True)), w, 0.0)
    w = torch.where(w >= mp.clamp(max=1.0), w, 0.0)
    byid = torch.zeros_like(w).scatter_(1, order, w)
    upto = byid.cumsum(-1)
    total = upto[:, -1:]
    ids = (upto > u * total).int().argmax(-1)
    return ids, (byid.gather(1, ids[:, None]) / total).log()[:, 0].float()


# ------------------------------------------------------------------------------------------------ the definition in 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    c = s["c"]
    if c["op"] == "sample":
        rows = [_exact_row(s, r) for r in range(c["rows"])]
        return torch.stack([i for i, _ in rows]), torch.stack([p for _, p in rows])
    B, T, H, KV, hd, P = c["seqs"], c["tokens"], c["heads"], c["kv_heads"], c["hd"], c["page"]
    new, first = s["n_new"].tolist(), s["start"].tolist()
    if c["op"] == "append":
        q = torch.zeros(B, T, H, hd // 2, dtype=torch.complex128, device=DEV)
        kp, vp = s["k"].double(), s["v"].double()
        for b in range(B):
            if not new[b]:
                continue
            at = torch.arange(first[b], first[b] + new[b], device=DEV)
            turn = torch.complex(s["cos"][at].double(), s["sin"][at].double())[:, None]                 # a pair as one complex number
            pairs = lambda x, h: torch.complex(*x.view(B, T, h, 2, hd // 2)[b, :new[b]].double().unbind(2))  # noqa: E731
            q[b, :new[b]] = pairs(s["q"], H) * turn
            k = pairs(s["kn"], KV) * turn
            page, inside = s["table"][b].long()[at // P], at % P
            kp[page, :, inside] = torch.cat((k.real, k.imag), -1)
            vp[page, :, inside] = s["vn"].view(B, T, KV, hd)[b, :new[b]].double()
        return torch.cat((q.real, q.imag), -1).reshape(B * T, H * hd), kp, vp
    out = torch.zeros(B, T, H, hd, dtype=torch.float64, device=DEV)
    for b in range(B):
        n, f = new[b], first[b]
        if not n:
            continue
        sees, live = torch.arange(f, f + n, device=DEV), -(-(f + n) // P)
        pages = s["table"][b, :live].long()
        for h in range(KV):
            k, v = (s[name][pages, h].reshape(live * P, hd)[:f + n].double() for name in ("k", "v"))
            for g in range(H // KV):
                head = h * (H // KV) + g
                x = s["q"].view(B, T, H, hd)[b, :n, head].double() @ k.T / math.sqrt(hd)
                x = x.masked_fill(torch.arange(f + n, device=DEV) > sees[:, None], -math.inf)
                out[b, :n, head] = torch.softmax(x, -1) @ v
    return out.view(B * T, H * hd)


def _exact_row(s, r):
    """One row, by taking tokens away from it."""
    setting = lambda n: (s[n][r] if torch.is_tensor(s[n]) else torch.tensor(s[n], device=DEV)).float().double()  # noqa: E731
    x, u, T = s["logits"][r].double(), setting("uniform"), setting("temperature")
    if T == 0:
        return (x == x.max()).nonzero()[0, 0], torch.zeros((), dtype=torch.float64, device=DEV)
    ids = x.argsort(descending=True, stable=True)
    k = int(s["top_k"][r])
    ids = ids[:k] if k > 0 else ids
    p = torch.softmax(x[ids] / T, 0)
    if setting("top_p") < 1:
        n = int(torch.searchsorted(p.cumsum(0), setting("top_p"))) + 1
        ids, p = ids[:n], p[:n]
    likely = p >= setting("min_p").clamp(max=1.0) * p[0]
    ids, back = ids[likely].sort()
    p = p[likely][back] / p[likely].sum()
    at = torch.searchsorted(p.cumsum(0), u, right=True).clamp(max=ids.numel() - 1)
    return ids[at], p[at].log()
