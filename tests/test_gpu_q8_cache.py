"""The 8-bit key / value cache (append with rotary embedding, read back, attention) and the log probabilities of given tokens against plain
implementations: codes and scales bit for bit against the formula in fp32 (each product and sum rounded by itself), the rest against 64 bits with tolerances
that count roundings (half a step, eps / 2, each)."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
TOP = {torch.int8: 127.0, torch.float8_e4m3fn: 448.0}
I8, E4 = torch.int8, torch.float8_e4m3fn


@pytest.fixture(scope="module")
def ops():
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")
    from mem_efficient_blr_b200 import ops as o
    return o


def _half(dtype):
    return torch.finfo(dtype).eps / 2


def _subnormal(dtype):
    return torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps


def _values(codes):
    return codes.float() if codes.dtype == I8 else codes.to(torch.float32)


def _coded(v, code):
    v = torch.nan_to_num(v, nan=0.0)
    return (v.round() if code == I8 else v).clamp(-TOP[code], TOP[code]).to(code)


def _tables(slots, hd):
    ang = torch.outer(torch.arange(slots, dtype=torch.float64), 10000.0 ** (-torch.arange(0, hd, 2, dtype=torch.float64) / hd))
    return ang.cos().float(), ang.sin().float()


def _rot(x, c, s):
    a, b = x.chunk(2, dim=-1)
    return torch.cat((a * c - b * s, b * c + a * s), dim=-1)


def _write(codes, scale, x, s, start, block):
    """x (n, hd) fp32 to slots start .. of one head's codes (slots, hd) and scale (blocks,), in place: the formula, block by block."""
    slots, code = codes.shape[0], codes.dtype
    first, end = max(start, 0), min(start + x.shape[0], slots)
    if first >= end:
        return
    for j in range(first // block, (end - 1) // block + 1):
        lo, hi = max(first, j * block), min(end, (j + 1) * block)
        new = x[lo - start:hi - start]
        big = new.abs().max()   # (a NaN stays one)
        asked = big * torch.tensor(1.0 / TOP[code])
        if asked < torch.finfo(torch.float32).tiny:
            asked = torch.zeros(())
        before = torch.zeros(()) if j * block >= first else scale[j].clone()
        after = before if before.isnan() else torch.maximum(before, asked)
        inv = 1.0 / after if after > 0 and not after.isinf() else torch.zeros(())
        if not bool(after == before) and j * block < first:
            old = slice(j * block, first)
            codes[old] = _coded(_values(codes[old]) * (before * inv), code)
        codes[lo:hi] = _coded(torch.where(inv == 0, torch.zeros(()), new * inv), code)
        scale[j] = after


def _cache(ops, B, KV, slots, hd, block, code, g, spread=1.0):
    nb = -(-slots // block)
    codes = lambda: _coded(torch.randn(B, KV, slots, hd, generator=g) * TOP[code] / 4, code)   # noqa: E731
    scale = lambda: (torch.rand(B, KV, nb, generator=g) * spread + 0.3) * 4 / TOP[code]        # noqa: E731
    return [codes(), codes(), scale(), scale()]


def _on(ops, parts, block):
    return ops.Q8Cache(*(t.to(DEV) for t in parts), block)


APPENDS = [  # B, T, H, KV, hd, slots, block, starts, new
    (1, 1, 1, 1, 64, 1, 16, [0], None),
    (3, 1, 8, 2, 128, 33, 16, [0, 17, 32], None),
    (2, 1, 4, 4, 64, 130, 128, [127, 128], None),
    (1, 16, 2, 2, 128, 64, 16, [16], None),
    (2, 19, 6, 3, 64, 45, 32, [26, 0], [19, 7]),
    (4, 5, 4, 1, 128, 40, 64, [0, 33, 38, -2], [0, 5, 5, 5]),     # none; ordinary; past the end; before the beginning
    (1, 300, 32, 8, 128, 301, 128, [1], None),
    (2, 257, 5, 5, 64, 400, 16, [3, 100], [257, 256]),
]


@pytest.mark.parametrize("code", [I8, E4], ids=["int8", "e4m3"])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("case", APPENDS, ids=[str(i) for i in range(len(APPENDS))])
def test_append(ops, case, dtype, code):
    B, T, H, KV, hd, slots, block, starts, new = case
    g = torch.Generator().manual_seed(T + slots)
    parts = _cache(ops, B, KV, slots, hd, block, code, g)
    rn = lambda h: torch.randn(B * T, h * hd, generator=g).to(dtype)   # noqa: E731
    q, k, v = rn(H), rn(KV), rn(KV)
    cos, sin = _tables(slots, hd)
    dev = _on(ops, parts, block)
    out = ops.rope_append_q8(q.to(DEV), k.to(DEV), v.to(DEV), cos.to(DEV), sin.to(DEV), torch.tensor(starts, device=DEV), dev,
                             None if new is None else torch.tensor(new, device=DEV))
    torch.cuda.synchronize()
    want = [t.clone() for t in parts]
    want_q, room = torch.zeros(B, T, H, hd, dtype=torch.float64), torch.zeros(B, T, H, hd, dtype=torch.float64)
    for b in range(B):
        n = T if new is None else new[b]
        for t in range(n):
            at = starts[b] + t
            if 0 <= at < slots:
                x = q.view(B, T, H, hd)[b, t].double()
                want_q[b, t] = _rot(x, cos[at].double(), sin[at].double())
                room[b, t] = _rot(x.abs(), cos[at].abs().double(), -sin[at].abs().double()).abs()   # |a c| + |b s| of the first half, at least
                room[b, t, :, hd // 2:] = (x[:, hd // 2:] * cos[at].double()).abs() + (x[:, :hd // 2] * sin[at].double()).abs()
        slot = (torch.arange(n) + starts[b]).clamp(0, slots - 1)
        for h in range(KV):
            kh = _rot(k.view(B, T, KV, hd)[b, :n, h].float(), cos[slot], sin[slot])
            _write(want[0][b, h], want[2][b, h], kh, sin, starts[b], block)
            _write(want[1][b, h], want[3][b, h], v.view(B, T, KV, hd)[b, :n, h].float(), sin, starts[b], block)
    got_q = out.cpu().double().view(B, T, H, hd)
    # one rounding to 16 bits, three of fp32 ahead of it
    tiny = _subnormal(dtype)
    assert ((got_q - want_q).abs() <= _half(dtype) * want_q.abs() * 1.001 + 4 * 2.0 ** -24 * room + tiny).all()
    for a, w in zip(dev[:4], want):
        assert torch.equal(a.cpu().view(torch.uint8), w.view(torch.uint8))


def test_a_block_filled_token_by_token(ops):
    """Growing values: the scale grows at every token and older codes follow it; what comes out is off by half a step for each time, no more."""
    B, H, hd, slots, block = 2, 3, 64, 48, 16
    g = torch.Generator().manual_seed(5)
    cos, sin = _tables(slots, hd)
    cache = ops.q8_cache(B, H, slots, hd, block, I8, DEV)
    want = [t.cpu().clone() for t in cache[:4]]
    true = torch.zeros(B, H, slots, hd, dtype=torch.float64)
    for t in range(slots):
        q, k, v = ((torch.randn(B, H * hd, generator=g) * (1 + t % 16)).half() for _ in range(3))
        ops.rope_append_q8(q.to(DEV), k.to(DEV), v.to(DEV), cos.to(DEV), sin.to(DEV), torch.full((B,), t, device=DEV), cache)
        true[:, :, t] = v.view(B, H, hd).double()
        for b in range(B):
            for h in range(H):
                _write(want[0][b, h], want[2][b, h], _rot(k.view(B, H, hd)[b, h:h + 1].float(), cos[t], sin[t]), None, t, block)
                _write(want[1][b, h], want[3][b, h], v.view(B, H, hd)[b, h:h + 1].float(), None, t, block)
    for a, w in zip(cache[:4], want):
        assert torch.equal(a.cpu(), w)
    _, vr = ops.cache_read_q8(cache, torch.float16)
    step = cache.v_scale.cpu().double().repeat_interleave(block, -1)[..., None]
    assert ((vr.cpu().double() - true).abs() <= (8.01 * step + _half(torch.float16) * true.abs())).all()   # 16 growths, each at most half a step of a smaller scale


@pytest.mark.parametrize("code", [I8, E4], ids=["int8", "e4m3"])
def test_append_of_values_that_are_no_numbers(ops, code):
    """A NaN or an infinity makes its own block of its own head NaN, and nothing else; a block of values too small for a scale is zeros; a block begun
    again is sound again."""
    hd, slots, block = 64, 48, 16
    cos, sin = _tables(slots, hd)
    cache = ops.q8_cache(1, 2, slots, hd, block, code, DEV)
    x = torch.ones(48, 2 * hd, dtype=torch.bfloat16)
    x[3, 5], x[20, hd + 1] = math.nan, math.inf
    x[32:] = 1e-38
    put = lambda x, n, at: ops.rope_append_q8(x[:n].to(DEV), x[:n].to(DEV), x[:n].to(DEV), cos.to(DEV), sin.to(DEV), torch.tensor([at], device=DEV), cache)   # noqa: E731
    put(x, 48, 0)
    for t in ops.cache_read_q8(cache, torch.bfloat16):
        t = t.cpu().float()
        assert t[0, 0, :16].isnan().all() and t[0, 1, 16:32].isnan().all()
        assert not t[0, 1, :16].isnan().any() and not t[0, 0, 16:32].isnan().any() and (t[0, :, 32:] == 0).all()
    put(x[40:], 4, 4)     # into the middle of the bad block: still bad
    assert ops.cache_read_q8(cache, torch.bfloat16)[1][0, 0, :16].isnan().all()
    put(torch.ones_like(x), 16, 0)
    assert (ops.cache_read_q8(cache, torch.bfloat16)[1][0, 0, :16] - 1).abs().max() <= (0.5 / 127 if code == I8 else 0) + _half(torch.bfloat16)


@pytest.mark.parametrize("code", [I8, E4], ids=["int8", "e4m3"])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("B,KV,hd,slots,block,lengths", [(1, 1, 64, 1, 16, None), (3, 2, 128, 77, 32, [0, 77, 50]), (2, 5, 64, 301, 128, [1000, -3])])
def test_read(ops, B, KV, hd, slots, block, lengths, dtype, code):
    g = torch.Generator().manual_seed(slots)
    parts = _cache(ops, B, KV, slots, hd, block, code, g)
    got = ops.cache_read_q8(_on(ops, parts, block), dtype, None if lengths is None else torch.tensor(lengths, device=DEV))
    for codes, scale, o in zip(parts[:2], parts[2:], got):
        want = _values(codes).double() * scale.double().repeat_interleave(block, -1)[..., :slots, None]
        for b in range(B):
            want[b, :, max(0, slots if lengths is None else lengths[b]):] = 0
        tiny = _subnormal(dtype)
        assert o.dtype == dtype and ((o.cpu().double() - want).abs() <= _half(dtype) * want.abs() * 1.001 + tiny).all()


def _attention(q, parts, block, starts, new, scale):
    """(out, allowance without the output's rounding) in 64 bits; q (B, T, H, hd).  Allowed: p is rounded to fp16 (half a step, at most 2^-11 of it, to either side;
    what its exponent's argument and the sums of fp32 add is below 2^-16) and below 2^-14 to multiples of 2^-24 of the largest value's scale, sixteen times that
    where a larger scale came first; l is at least the sum taken against the true maximum."""
    B, T, H, hd = q.shape
    KV, slots = parts[0].shape[1:3]
    k, v = (_values(c).double() * s.double().repeat_interleave(block, -1)[..., :slots, None] for c, s in ((parts[0], parts[2]), (parts[1], parts[3])))
    out, room = torch.zeros(B, T, H, hd, dtype=torch.float64), torch.zeros(B, T, H, hd, dtype=torch.float64)
    for b in range(B):
        rows = T if new is None else max(0, min(T, new[b]))
        seen = (torch.arange(rows) + starts[b] + 1).clamp(0, slots)
        n = int(seen.max()) if rows else 0
        if n == 0:
            continue
        out_of_sight = torch.arange(n) >= seen[:, None]
        for h in range(H):
            kh, vh = k[b, h // (H // KV), :n], v[b, h // (H // KV), :n]
            x = (q[b, :rows, h].double() @ kh.T * scale).masked_fill(out_of_sight, -math.inf)
            p = torch.exp(x - x.amax(1, keepdim=True).clamp(min=-1e300))
            l = p.sum(1, keepdim=True).clamp(min=1e-300)
            most = vh.abs().amax(1).cummax(0).values[seen.clamp(min=1) - 1]   # the largest value that the row sees
            out[b, :rows, h] = p @ vh / l
            room[b, :rows, h] = 2.0 ** -11 * (p @ vh.abs()) / l + torch.where(seen > 0, seen * 2.0 ** -21 * most, torch.zeros(()).double())[:, None] / l.clamp(min=1e-3)
    return out, room


ATTENDS = [  # B, T, H, KV, hd, slots, block, starts, new
    (1, 1, 1, 1, 64, 1, 16, [0], None),
    (2, 1, 4, 2, 128, 17, 16, [16, 3], None),
    (3, 1, 8, 8, 128, 600, 32, [599, 0, 255], None),
    (2, 1, 8, 1, 64, 1100, 128, [1099, 64], None),
    (4, 1, 4, 2, 64, 50, 16, [10, -1, 200, 49], [1, 1, 1, 0]),    # ordinary; sees nothing; past the end: all slots; no token
    (1, 3, 14, 2, 128, 90, 64, [87], None),
    (2, 5, 8, 2, 64, 700, 16, [300, 650], [5, 2]),
    (1, 40, 4, 4, 128, 333, 16, [293], None),
    (2, 70, 6, 2, 64, 300, 32, [0, 211], [70, 33]),
    (1, 130, 2, 1, 128, 130, 16, [0], None),
    (2, 150, 3, 3, 128, 420, 128, [1, 270], [0, 150]),
    (1, 260, 4, 1, 64, 517, 64, [257], None),
    (2, 410, 4, 2, 128, 900, 32, [490, 100], [410, 77]),
    (2, 1520, 8, 1, 64, 1560, 32, [25, -7], [1520, 800]),         # (codes widened ahead)
    (1, 1540, 8, 1, 128, 1600, 16, [60], None),
]


@pytest.mark.parametrize("code", [I8, E4], ids=["int8", "e4m3"])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("case", ATTENDS, ids=[str(i) for i in range(len(ATTENDS))])
def test_attention(ops, case, dtype, code):
    B, T, H, KV, hd, slots, block, starts, new = case
    g = torch.Generator().manual_seed(slots + T)
    parts = _cache(ops, B, KV, slots, hd, block, code, g)
    q = (torch.randn(B, T, H, hd, generator=g) * 2).to(dtype)
    args = (torch.tensor(starts, device=DEV), None if new is None else torch.tensor(new, device=DEV))
    dirty = [t.clone() for t in parts]
    for b in range(B):   # what nobody has written yet may be anything: the largest scales and NaN codes
        end = max(0, min(slots, starts[b] + (T if new is None else new[b])))
        for c, s in ((dirty[0], dirty[2]), (dirty[1], dirty[3])):
            c.view(torch.uint8)[b, :, end:] = 0x7f
            s[b, :, -(-end // block):] = math.nan
    got = ops.attention_q8(q.view(B * T, H * hd).to(DEV), _on(ops, dirty, block), *args)
    want, room = _attention(q, parts, block, starts, new, hd ** -0.5)
    got = got.cpu().double().view(B, T, H, hd)
    assert ((got - want).abs() <= _half(dtype) * want.abs() * 1.001 + room + _subnormal(dtype)).all()
    again = ops.attention_q8(q.view(B * T, H * hd).to(DEV), _on(ops, parts, block), *args, scale=hd ** -0.5)
    assert torch.equal(again.cpu().double().view(B, T, H, hd), got)   # the same sums in the same order


@pytest.mark.parametrize("T", [1, 7, 160])
def test_attention_of_uneven_values(ops, T):
    """Scores that climb along the keys (the running maximum moves all the time), value scales from 1e-6 to 1e3 block by block, rows of q of very different
    size, one of zeros: the same bounds hold."""
    B, H, KV, hd, slots, block = 1, 4, 2, 128, 700, 16
    g = torch.Generator().manual_seed(T)
    parts = _cache(ops, B, KV, slots, hd, block, I8, g)
    parts[2] *= torch.linspace(0.1, 3, parts[2].shape[2])
    parts[3] = 10.0 ** (torch.rand(parts[3].shape, generator=g) * 9 - 6)
    parts[3][:, :, 3] = 0
    q = (torch.randn(B, T, H, hd, generator=g) * 10.0 ** (torch.arange(H) * 0.5 - 1.5)[:, None]).bfloat16()
    q[:, :, 1] = 0
    start = torch.tensor([slots - T], device=DEV)
    got = ops.attention_q8(q.view(T, H * hd).to(DEV), _on(ops, parts, block), start).cpu().double().view(B, T, H, hd)
    want, room = _attention(q, parts, block, [slots - T], None, hd ** -0.5)
    assert ((got - want).abs() <= _half(torch.bfloat16) * want.abs() * 1.001 + room).all()


@pytest.mark.parametrize("T,H,KV", [(3, 2, 2), (150, 2, 1)])
def test_a_bad_block_reaches_only_the_rows_that_see_it(ops, T, H, KV):
    hd, slots, block = 64, 300, 16
    g = torch.Generator().manual_seed(1)
    parts = _cache(ops, 1, KV, slots, hd, block, I8, g)
    q = torch.randn(T, H * hd, generator=g).half()
    start = 160 - T + 2   # slots 160 and 161, the block's first two, belong to the last two rows
    for bad in (math.nan, math.inf):
        for which in (2, 3):
            spoilt = [t.clone() for t in parts]
            spoilt[which][:, :, 10] = bad
            out = ops.attention_q8(q.to(DEV), _on(ops, spoilt, block), torch.tensor([start], device=DEV)).cpu()
            sound = ops.attention_q8(q.to(DEV), _on(ops, parts, block), torch.tensor([start], device=DEV)).cpu()
            assert out[-2:].isnan().all() if bad != math.inf else not out[-2:].isfinite().all()
            assert torch.equal(out[:-2], sound[:-2])


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("T,H", [(2, 4), (90, 2)])
def test_a_row_of_q_that_is_no_number_stays_alone(ops, T, H, dtype):
    g = torch.Generator().manual_seed(6)
    parts = _cache(ops, 1, H, 200, 128, 32, I8, g)
    q = torch.randn(T, H, 128, generator=g).to(dtype)
    call = lambda q: ops.attention_q8(q.view(T, -1).to(DEV), _on(ops, parts, 32), torch.tensor([200 - T], device=DEV)).cpu().view(T, H, 128)   # noqa: E731
    sound = call(q)
    q[1, 1, 7], q[0, 0, 3] = math.nan, math.inf
    got = call(q)
    assert got[1, 1].isnan().all() and not got[0, 0].isfinite().all()
    got[1, 1], got[0, 0] = sound[1, 1], sound[0, 0]
    assert torch.equal(got, sound)


@pytest.mark.parametrize("T", [1, 70])
def test_a_cache_beyond_32_bit_offsets(ops, T):
    """5 GB of codes for the keys and as many for the values: the last 16 slots are written, everything before them has scale 0, so that its keys score 0 and
    its values are 0: out = sum p v / (n + sum p) over the last slots."""
    hd, slots, block = 128, 40_000_016, 16
    cache = ops.q8_cache(1, 1, slots, hd, block, I8, DEV)
    cos, sin = torch.ones(1, hd // 2, device=DEV), torch.zeros(1, hd // 2, device=DEV)   # (angles of 0: nothing turns)
    g = torch.Generator().manual_seed(8)
    new = slots - 16 - (T - 16 if T > 16 else 0)
    k, v, q = (torch.randn(T, hd, generator=g).bfloat16() for _ in range(3))
    tables = (cos.expand(slots, -1).contiguous(), sin.expand(slots, -1).contiguous())
    start = torch.tensor([new], device=DEV)
    r = ops.rope_append_q8(q.to(DEV), k.to(DEV), v.to(DEV), *tables, start, cache)
    assert torch.equal(r.cpu(), q)
    got = ops.attention_q8(r, cache, start).cpu().double()
    del tables
    kq, vq = (c[0, 0, new:new + T].cpu().double() * sc[0, 0, new // block:].cpu().double().repeat_interleave(block)[new % block:][:T, None]
              for c, sc in ((cache.k, cache.k_scale), (cache.v, cache.v_scale)))
    x = (q.double() @ kq.T * hd ** -0.5 + math.log(1e6)).exp().tril()   # (weights times 10^6, for the sake of the sums here)
    total = 1e6 * new + x.sum(1, keepdim=True)
    # the output's rounding, p's (2^-11), and 2^-19 for sums of up to 2^25 fp32 terms, most of them equal to 1, over some hundred threads
    assert ((got - x @ vq / total).abs() <= (2.0 ** -8 + 2.0 ** -19) * (x @ vq / total).abs() * 1.001 + 2.0 ** -11 * (x @ vq.abs() / total)).all()


def test_strides_and_streams(ops):
    """q, k, v as columns of a fused projection's rows, and as views that the kernels do not take; a stream of its own."""
    B, T, H, KV, hd, slots = 2, 6, 4, 2, 64, 40
    g = torch.Generator().manual_seed(2)
    wide = torch.randn(B * T, (H + 2 * KV) * hd, generator=g).half().to(DEV)
    q, k, v = wide.split([H * hd, KV * hd, KV * hd], dim=1)
    cos, sin = (t.to(DEV) for t in _tables(slots, hd))
    start = torch.tensor([0, 30], device=DEV)

    def both(q, k, v):
        c = ops.q8_cache(B, KV, slots, hd, 16, I8, DEV)
        r = ops.rope_append_q8(q, k, v, cos, sin, start, c)
        return [r, ops.attention_q8(r, c, start), *c[:4]]

    want = both(q.contiguous(), k.contiguous(), v.contiguous())
    odd = torch.zeros(B * T, KV * hd + 3, dtype=torch.float16, device=DEV)[:, 3:]
    odd.copy_(k)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = both(q, odd, v)
    s.synchronize()
    for a, b in zip(want, got):
        assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))


def test_captured_and_replayed(ops):
    """A graph of append and attention whose positions move by an in-place addition in the graph itself, against eager calls; two graphs of the same calls
    replayed in turn on two streams share nothing."""
    B, H, KV, hd, slots = 2, 4, 2, 128, 2048
    cos, sin = (t.to(DEV) for t in _tables(slots, hd))
    g = torch.Generator().manual_seed(3)
    xs = [torch.randn(3, B, h * hd, generator=g).half().to(DEV) for h in (H, KV, KV)]

    def make():
        c = ops.q8_cache(B, KV, slots, hd, 16, I8, DEV)
        start = torch.tensor([5, 1029], device=DEV)
        return c, start, [x[0].clone() for x in xs]

    def step(c, start, x):
        r = ops.rope_append_q8(*x, cos, sin, start, c)
        o = ops.attention_q8(r, c, start)
        start.add_(1)
        return o

    eager = make()
    want = []
    for i in range(3):
        for d, s in zip(eager[2], xs):
            d.copy_(s[i])
        want.append(step(*eager).clone())
    graphs = []
    for _ in range(2):
        state = make()
        st = torch.cuda.Stream()
        st.wait_stream(torch.cuda.current_stream())
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.stream(st):
            with torch.cuda.graph(graph, stream=st):
                out = step(*state)
        graphs.append((graph, st, state, out))
    torch.cuda.synchronize()
    for i in range(3):
        for graph, st, state, out in graphs:
            with torch.cuda.stream(st):
                for d, s in zip(state[2], xs):
                    d.copy_(s[i])
                graph.replay()
        torch.cuda.synchronize()
        for graph, st, state, out in graphs:
            assert torch.equal(out, want[i])


def test_refusals_on_the_device(ops):
    c = ops.q8_cache(1, 2, 32, 64, device=DEV)
    cos, sin = (t.to(DEV) for t in _tables(32, 64))
    x, start = torch.zeros(2, 128, dtype=torch.float16, device=DEV), torch.zeros(1, dtype=torch.int64, device=DEV)
    bad = [lambda: ops.rope_append_q8(x, x[:1], x, cos, sin, start, c), lambda: ops.rope_append_q8(x, x, x.bfloat16(), cos, sin, start, c),
           lambda: ops.rope_append_q8(x, x, x, cos[:31], sin[:31], start, c), lambda: ops.rope_append_q8(x, x, x, cos, sin.double(), start, c),
           lambda: ops.rope_append_q8(x, x, x, cos, sin, start.int(), c), lambda: ops.rope_append_q8(x, x, x, cos, sin, start.expand(2), c),
           lambda: ops.rope_append_q8(x, x, x, cos, sin, start.cpu(), c), lambda: ops.attention_q8(x[:, :64], c, start), lambda: ops.attention_q8(x.float(), c, start),
           lambda: ops.attention_q8(x, c._replace(block=32), start), lambda: ops.attention_q8(x, c._replace(k=c.k.float()), start),
           lambda: ops.attention_q8(x, c._replace(k=c.k.transpose(1, 2)), start), lambda: ops.attention_q8(x, c._replace(v_scale=c.v_scale.half()), start),
           lambda: ops.cache_read_q8(c, torch.float32), lambda: ops.cache_read_q8(c, torch.float16, start.int()),
           lambda: ops.token_logprobs(x, start), lambda: ops.token_logprobs(x.double(), start.expand(2)), lambda: ops.token_logprobs(x, start.expand(2).int())]
    for call in bad:
        with pytest.raises(AssertionError):
            call()
    with pytest.raises(RuntimeError, match="0 to 64"):
        ops.token_logprobs(x, start.expand(2), 65)
    with pytest.raises((AssertionError, RuntimeError)):
        ops.attention_q8(x, ops.Q8Cache(*(t[..., :48].contiguous() for t in c[:2]), *c[2:4], 16), start)


# ------------------------------------------------------------------------------------------------ log probabilities
def _rows(rows, vocab, dtype, g, kind):
    x = torch.randn(rows, vocab, generator=g) * 3
    if kind == "masked":
        x[torch.rand(rows, vocab, generator=g) < 0.7] = -math.inf
        x[:, vocab // 2] = 1.0
    elif kind == "equal":
        x[:] = 0.25
    elif kind == "lowest":   # places masked with the type's lowest number
        x[:, 1:] = torch.finfo(dtype).min
    elif kind == "all lowest":   # a row that is masked as a whole in that way is an even distribution
        x[:] = torch.finfo(dtype).min
        x[1:, ::3] = 0
    elif kind == "ends":
        x[:, 1], x[:, vocab // 2], x[1:, 3] = torch.finfo(dtype).min, -math.inf, torch.finfo(dtype).max
    elif kind == "large":
        x = x * 1e4
    elif kind == "steps":    # many ties
        x = x.round()
    return x.to(dtype)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows,vocab,top,kind", [(1, 1, 1, ""), (1, 5, 5, ""), (3, 257, 64, ""), (4, 32000, 5, ""), (5, 1001, 8, "masked"), (2, 4096, 64, "equal"),
                                                 (2, 333, 3, "lowest"), (3, 2048, 4, "large"), (37, 50257, 0, ""), (7, 20011, 20, "steps"), (300, 515, 2, ""),
                                                 (2, 131072, 7, "steps"), (1, 151936, 33, "masked"), (160, 40000, 64, "equal"),
                                                 # (many rows of 16 to 64 KB)
                                                 (311, 9001, 8, ""), (300, 20000, 64, "masked"), (602, 15011, 33, "steps"), (296, 16000, 40, "equal"), (299, 8300, 0, "lowest"), (2, 1030, 4, "all lowest"), (3, 40003, 9, "ends")])
def test_logprobs(ops, rows, vocab, top, kind, dtype):
    g = torch.Generator().manual_seed(rows + vocab)
    x = _rows(rows, vocab, dtype, g, kind)
    ids = torch.randint(0, vocab, (rows,), generator=g)
    lp, ent, tl, ti = (t.cpu() for t in ops.token_logprobs(x.to(DEV), ids.to(DEV), top))
    d = x.double()
    want = torch.log_softmax(d, -1)
    far = d - d.amax(-1, keepdim=True)
    log_s = far.exp().sum(-1, keepdim=True).log()
    # S: e to 2^-21 and 2^-23 of its exponent's argument, sums over at most vocab / 256 + 64 terms in a row; then a difference of two fp32 numbers
    rel_s = 2.0 ** -21 + (vocab / 256 + 64) * 2.0 ** -24
    allow = rel_s + 2.0 ** -23 * (far.abs().nan_to_num(posinf=0) + log_s)
    # (fp16 rows of "large" hold infinities: NaN in both)
    ok = lambda got, ref, room: bool((((got.double() - ref).abs() <= room) | (got.double() == ref) | (got.isnan() & ref.isnan())).all())   # noqa: E731
    assert ok(lp, want.gather(1, ids[:, None])[:, 0], allow.gather(1, ids[:, None])[:, 0])
    e = torch.special.entr(want.exp()).sum(-1)
    spread = (want.exp() * far.nan_to_num(neginf=0).abs()).sum(-1)   # sum p |x - M|: each term to rel_s and 2^-23 of its argument
    assert ok(ent, e, rel_s * (1 + 2 * spread) + 2.0 ** -22 * (want.exp() * far.nan_to_num(neginf=0) ** 2).sum(-1) + 2.0 ** -23 * (log_s[:, 0] + spread))
    order = x.float().sort(dim=-1, descending=True, stable=True).indices[:, :top]
    assert tl.shape == ti.shape == (rows, top) and ti.dtype == torch.int64 and torch.equal(ti, order)
    assert ok(tl, want.gather(1, order), allow.gather(1, order))


# Rows short enough for one or four warps (up to 96 and 2048 vectors of 16 bytes), around both limits, and more alternatives than a warp has threads.  At most 2048 x 8 values
# for 128 threads with two sums each, 64 terms in a row, or 96 x 8 for 32, 12 (and 8 more for the joining): fewer than the vocab / 256 + 64 that test_logprobs allows.
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows,vocab,top,kind", [(700, 300, 20, ""), (33, 20, 20, "steps"), (301, 97, 32, "masked"), (40, 300, 33, ""), (40, 300, 64, "masked"), (50, 768, 9, "equal"),
                                                 (50, 776, 32, ""), (50, 384, 32, "steps"), (50, 388, 5, "lowest"), (2, 300, 4, "all lowest"), (5, 500, 7, "ends"),
                                                 (310, 4111, 20, "masked"), (300, 8191, 64, ""), (300, 8192, 64, "equal"), (298, 8200, 64, "steps"), (297, 16384, 20, "large"),
                                                 (297, 16399, 20, "")])
def test_logprobs_of_short_rows(ops, rows, vocab, top, kind, dtype):
    test_logprobs(ops, rows, vocab, top, kind, dtype)


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows,vocab,left,top,ruled_out", [(3, 32001, 3, 8, "inf"), (300, 32000, 3, 64, "inf"), (2, 32003, 70, 64, "lowest"), (300, 9001, 5, 20, "lowest"), (9, 2000, 0, 7, "lowest"),
                                                           (300, 4099, 1, 33, "inf"), (5, 700, 2, 20, "inf"), (301, 9000, 2, 40, "below"), (2, 700, 2, 20, "below")])
def test_logprobs_with_few_tokens_left(ops, rows, vocab, left, top, ruled_out, dtype):
    g = torch.Generator().manual_seed(vocab)
    low = torch.finfo(dtype).min
    x = torch.full((rows, vocab), -math.inf if ruled_out == "inf" else low)
    if ruled_out == "below":   # (numbers below the one that most have, at the front and among them)
        x[:, :] = -2.0
        x[:, :top] = -math.inf
        x[:, 100::3] = low
    at = torch.rand(rows, vocab, generator=g).argsort(-1)[:, :left]
    x.scatter_(1, at, torch.randn(rows, left, generator=g))
    x = x.to(dtype)
    ids = at[:, 0].contiguous() if left else torch.zeros(rows, dtype=torch.int64)
    lp, ent, tl, ti = (t.cpu() for t in ops.token_logprobs(x.to(DEV), ids.to(DEV), top))
    order = x.float().sort(dim=-1, descending=True, stable=True).indices[:, :top]
    assert torch.equal(ti, order)
    d = x.double()
    want = torch.log_softmax(d, -1)
    far = (d - d.amax(-1, keepdim=True)).abs()
    allow = 2.0 ** -21 + (vocab / 256 + 64) * 2.0 ** -24 + 2.0 ** -23 * (far + math.log(vocab))   # (as test_logprobs has it; log S is at most log vocab)
    for got, ref, room in ((tl, want.gather(1, order), allow.gather(1, order)), (lp, want.gather(1, ids[:, None])[:, 0], allow.gather(1, ids[:, None])[:, 0])):
        assert bool((((got.double() - ref).abs() <= room) | (got.double() == ref) | ((got == -math.inf) & (ref < -3.4e38))).all())   # (fp32: the lowest less M may pass the range)
    assert ent.isfinite().all()


@pytest.mark.parametrize("vocab,top", [(12, 12), (300, 8), (300, 40)])
def test_logprobs_of_short_rows_with_a_nan_or_infinity(ops, vocab, top):
    x = torch.randn(4, vocab, generator=torch.Generator().manual_seed(vocab))
    x[0, 7], x[1, 11], x[2, :] = math.nan, math.inf, -math.inf
    lp, ent, tl, ti = (t.cpu() for t in ops.token_logprobs(x.half().to(DEV), torch.tensor([1, 2, 3, 4], device=DEV), top))
    assert lp[:2].isnan().all() and ent[:2].isnan().all() and ti[0, 0] == 7 and ti[1, 0] == 11
    assert lp[2] == -math.inf and ent[2] == 0 and ti[2].tolist() == list(range(top))
    assert torch.equal(ti[3], x[3].half().float().sort(descending=True, stable=True).indices[:top]) and lp[3].isfinite()
    assert torch.equal(ti[0, 1:], x[0].half().float().nan_to_num(-math.inf).sort(descending=True, stable=True).indices[:top - 1])


@pytest.mark.parametrize("many", [1, 60])   # (60 times six rows of 9000: the kernel for many rows)
def test_logprobs_of_rows_without_a_distribution(ops, many):
    x = torch.zeros(6, 700 if many == 1 else 9000)
    if many > 1:
        x[:, 700:] = -math.inf
    x[0] = -math.inf
    x[1, 3], x[1, 600] = math.nan, 5.0
    x[2, 9], x[2, 8] = math.inf, 1.0
    x[3, :] = -math.inf
    x[3, 699] = -2.0
    x[4, 100::2] = -0.0
    for dtype in (torch.float16, torch.float32):
        ids = torch.tensor([1, 2, 9, 699, x.shape[1], -1], device=DEV)
        every = [t.cpu() for t in ops.token_logprobs(x.to(dtype).to(DEV).repeat(many, 1), ids.repeat(many), 3)]
        lp, ent, tl, ti = (t[-6:] for t in every)
        assert all(torch.equal(t[:6].nan_to_num(7.0), t[-6:].nan_to_num(7.0)) for t in every)
        assert lp[0] == -math.inf and ent[0] == 0 and (tl[0] == -math.inf).all() and ti[0].tolist() == [0, 1, 2]
        assert lp[1].isnan() and ent[1].isnan() and ti[1].tolist() == [3, 600, 0]
        assert lp[2].isnan() and ent[2].isnan() and ti[2].tolist() == [9, 8, 0]
        assert lp[3] == 0 and ent[3] == 0 and tl[3].tolist() == [0, -math.inf, -math.inf] and ti[3].tolist() == [699, 0, 1]
        assert lp[4].isnan() and ti[4].tolist() == [0, 1, 2]     # an id beyond the vocabulary; -0 ties with 0
        assert lp[5] == 0


def test_logprobs_shapes_and_strides(ops):
    g = torch.Generator().manual_seed(9)
    x = torch.randn(3, 4, 1003, generator=g).half().to(DEV)
    ids = torch.randint(0, 1000, (3, 4), generator=g).to(DEV)
    want = ops.token_logprobs(x[..., :1000].contiguous(), ids, 4)
    for got in (ops.token_logprobs(x[..., :1000], ids, 4), ops.token_logprobs(x[..., :1000].transpose(0, 1), ids.t(), 4)):
        for a, b in zip(want, got):
            b = b if b.shape[0] == 3 else b.transpose(0, 1)
            # (the order of a row's sums goes by its alignment: each result is within rel_s + 2^-23 (|x - M| + log S) of the exact one, see test_logprobs, with
            # |x - M| < 9 and log S < 8 here, so two are within twice that of each other)
            assert a.shape[:2] == (3, 4) and a.shape == b.shape and (a - b).abs().max() <= (0 if a.dtype == torch.int64 else 2 * (2.0 ** -21 + 68 * 2.0 ** -24 + 17 * 2.0 ** -23))
    one = ops.token_logprobs(x[0, 0, 1:1001], ids[0, 0])
    assert one[0].shape == () and one[2].shape == (0,) and one[0].isfinite()
    none = ops.token_logprobs(x[:0], ids[:0], 2)
    assert none[0].shape == (0, 4) and none[3].shape == (0, 4, 2)


# ------------------------------------------------------------------------------------------------ together, as a decoder uses them
@pytest.mark.parametrize("code", ["int8", "e4m3"])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_decoder_on_an_8_bit_cache(ops, code, dtype):
    from mem_efficient_blr_b200 import networks as nw
    shape = nw.LlamaShape(layers=2, d=512, heads=8, ffn=1024, vocab=384, b=16, rank_attn=64, rank_mlp=96)
    B, T, S = 3, 41, 64
    ids = torch.randint(0, shape.vocab, (B, T), generator=torch.Generator().manual_seed(1)).to(DEV)
    make = lambda **kw: nw.LlamaDecoder(shape, "blast", batch=B, cache_len=S, device=DEV, dtype=dtype, seed=3, **kw)   # noqa: E731
    rel = lambda a, b: float((a.double() - b.double()).norm() / b.double().norm())   # noqa: E731
    m, slow, plain = make(kv_cache=code), make(kv_cache=code, kv_block=32), make()
    slow.fused_decode = False
    a, c = m.prefill(ids[:, :T - 1]), plain.prefill(ids[:, :T - 1])
    # quantising: a value is off by at most half a step, 1/254 of its block's largest (2^-4 of itself in e4m3), in both operands of both products of two layers
    assert rel(a, c) < (0.1 if code == "e4m3" else 0.03)
    step = m.decode_step(ids[:, T - 1:], torch.tensor([T - 1], device=DEV))
    # the same tokens in pieces, sequences at different positions and a padded batch
    n = torch.tensor([30, 17, 1], device=DEV)
    p = make(kv_cache=code)
    p.extend(ids[:, :30], torch.zeros(B, dtype=torch.int64, device=DEV), n)
    idx = (n[:, None] + torch.arange(T - 1, device=DEV)).clamp(max=T - 1)
    p.extend(ids.gather(1, idx), n, T - 1 - n)
    piece = p.decode_step(ids[:, T - 1:], torch.full((B,), T - 1, device=DEV))
    tol = 0.1 if code == "e4m3" else 0.03    # (a block's codes depend on how the block was filled)
    assert rel(piece, step) < tol
    # reading back and torch's attention, on blocks of 32
    slow.prefill(ids[:, :T - 1])
    assert rel(slow.decode_step(ids[:, T - 1:], torch.tensor([T - 1], device=DEV)), step) < tol
    # scoring: the last position's distribution is the prefill's
    lp, ent, tl, ti = m.score(ids, 3)
    assert lp.shape == (B, T - 1) and tl.shape == (B, T - 1, 3)
    want = torch.log_softmax(a.double(), -1)
    assert (lp[:, -1].double() - want.gather(1, ids[:, -1:])[:, 0]).abs().max() < 0.05 and (lp <= 0).all() and (ent >= 0).all()
    assert (plain.score(ids)[0] - lp).abs().mean() < (0.3 if code == "e4m3" else 0.1)


def test_graphed_decode_on_an_8_bit_cache(ops):
    from mem_efficient_blr_b200 import networks as nw
    shape = nw.LlamaShape(layers=2, d=512, heads=8, ffn=1024, vocab=384, b=16, rank_attn=64, rank_mlp=96)
    ids = torch.randint(0, shape.vocab, (2, 40), generator=torch.Generator().manual_seed(4)).to(DEV)
    m = [nw.LlamaDecoder(shape, "blast_int8", batch=2, cache_len=48, device=DEV, seed=3, kv_cache="int8") for _ in range(2)]
    for x in m:
        x.prefill(ids[:, :36])
    pos = torch.tensor([36], device=DEV)
    step = nw.GraphedCall(m[0].decode_step, ids[:, 36:37].clone(), pos.clone())
    for i in range(36, 40):
        at = torch.tensor([i], device=DEV)
        assert torch.equal(step(ids[:, i:i + 1], at), m[1].decode_step(ids[:, i:i + 1], at))
