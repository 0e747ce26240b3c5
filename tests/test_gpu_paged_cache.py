"""The key / value cache in pages (append with rotary embedding, attention) against plain implementations in 64 bits, with tolerances that count roundings (half a step,
eps / 2, each)."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F16, BF16 = torch.float16, torch.bfloat16


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


def _tables(slots, hd):
    ang = torch.outer(torch.arange(slots, dtype=torch.float64), 10000.0 ** (-torch.arange(0, hd, 2, dtype=torch.float64) / hd))
    return ang.cos().float(), ang.sin().float()


def _rot(x, c, s):
    a, b = x.chunk(2, dim=-1)
    return torch.cat((a * c - b * s, b * c + a * s), dim=-1)


def _pool(B, KV, hd, page, per, dtype, g, gaps=()):
    """(k, v, table): pages of a shuffled pool with two to spare; `gaps`: places of the table without a page, by numbers that are none."""
    pages = B * per + 2
    k, v = (torch.randn(pages, KV, page, hd, generator=g).to(dtype) for _ in range(2))
    table = torch.randperm(pages, generator=g)[:B * per].to(torch.int32).view(B, per)
    for i, (b, j) in enumerate(gaps):
        table[b, j] = (-1, pages, 2 ** 31 - 1, -2 ** 31)[i % 4]
    return k, v, table


def _on(ops, k, v, table):
    return ops.PagedCache(k.to(DEV), v.to(DEV), table.to(DEV))


def _dev(x):
    return None if x is None else torch.tensor(x, device=DEV)


APPENDS = [  # B, T, H, KV, hd, page, pages of a sequence, starts, new, gaps
    (1, 1, 1, 1, 64, 16, 1, [0], None, []),
    (3, 1, 8, 2, 128, 16, 3, [0, 17, 47], None, []),
    (2, 1, 4, 4, 64, 128, 2, [127, 128], None, []),
    (1, 16, 2, 2, 128, 16, 4, [16], None, []),
    (2, 19, 6, 3, 64, 32, 2, [26, 0], [19, 7], []),
    (4, 5, 4, 1, 128, 64, 1, [0, 33, 62, -2], [0, 5, 5, 5], []),      # none; ordinary; past the end; ahead of the beginning
    (3, 40, 4, 2, 64, 16, 4, [0, 5, 2 ** 62], [40, 40, 3], [(0, 1), (1, 0)]),   # tokens without a page; far outside
    (1, 300, 32, 8, 128, 128, 3, [1], None, []),
    (2, 257, 5, 5, 64, 16, 25, [3, 100], [257, 256], []),
    (2, 700, 28, 4, 64, 32, 30, [0, 250], [700, 9], [(1, 8)]),
]


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("case", APPENDS, ids=[str(i) for i in range(len(APPENDS))])
def test_append(ops, case, dtype):
    B, T, H, KV, hd, page, per, starts, new, gaps = case
    g = torch.Generator().manual_seed(T + per)
    pk, pv, table = _pool(B, KV, hd, page, per, dtype, g, gaps)
    rn = lambda h: torch.randn(B * T, h * hd, generator=g).to(dtype)   # noqa: E731
    q, k, v = rn(H), rn(KV), rn(KV)
    cos, sin = _tables(page * per, hd)
    c = _on(ops, pk, pv, table)
    out = ops.rope_append_paged(q.to(DEV), k.to(DEV), v.to(DEV), cos.to(DEV), sin.to(DEV), _dev(starts), c, _dev(new)).cpu().double().view(B, T, H, hd)

    def turned(x, h):   # with the sum of what its terms may be off
        x = x.view(B, T, h, hd).double()
        want, room, there = torch.zeros_like(x), torch.zeros_like(x), torch.zeros(B, T, dtype=torch.long)
        for b in range(B):
            for t in range(T if new is None else new[b]):
                at = starts[b] + t
                if 0 <= at < page * per and 0 <= table[b, at // page] < len(pk):
                    cc, ss = cos[at].double(), sin[at].double()
                    want[b, t], there[b, t] = _rot(x[b, t], cc, ss), 1
                    lo, hi = x[b, t].abs().chunk(2, -1)
                    room[b, t] = torch.cat((lo * cc.abs() + hi * ss.abs(), hi * cc.abs() + lo * ss.abs()), -1)
        return want, room, there

    def near(got, want, room):   # one rounding to 16 bits, three of fp32 ahead of it
        return bool(((got - want).abs() <= _half(dtype) * want.abs() * 1.001 + 4 * 2.0 ** -24 * room + _subnormal(dtype)).all())

    want, room, there = turned(q, H)
    assert near(out, want, room) and not out[there == 0].any()
    want, room, _ = turned(k, KV)
    gk, gv = c.k.cpu(), c.v.cpu()
    for b in range(B):
        for t in range(T):
            if there[b, t]:
                at = starts[b] + t
                here = (int(table[b, at // page]), slice(None), at % page)
                assert near(gk[here].double(), want[b, t], room[b, t])
                assert torch.equal(gv[here], v.view(B, T, KV, hd)[b, t])
                gk[here], gv[here] = pk[here], pv[here]
    assert torch.equal(gk, pk) and torch.equal(gv, pv)   # nothing else is touched
    assert torch.equal(c.table.cpu(), table)


def test_positions_without_an_angle(ops):
    """Tables that end ahead of the cache's last page."""
    c = ops.paged_cache(1, 1, 2, 2, 64, 16, F16, DEV)
    c.table.copy_(torch.tensor([[1, 0]]))
    cos, sin = (t.to(DEV) for t in _tables(20, 64))
    x = torch.ones(8, 64, dtype=F16, device=DEV)
    out = ops.rope_append_paged(x, x, x, cos, sin, _dev([16]), c)
    assert out[:4].any(1).all() and not out[4:].any()
    assert c.v[0, 0, :4].all() and not c.v[0, 0, 4:].any() and not c.v[1].any()


# ------------------------------------------------------------------------------------------------ attention
def _attention(q, k, v, table, starts, new, scale):
    """(result, room for the error, row by row and value by value) in 64 bits.  The kernels round q, k, v nowhere; the exponent's argument is off by the sum of hd products in fp32
    (hd / 8 roundings of 2^-23 of the sum of their sizes at most: the tensor cores add 8 or more at a time) and two roundings; ex2 by 2^-22; p is rounded to fp16 (2^-11 of itself,
    or 2^-25 of the heaviest), for bf16 to the sum of two bf16 numbers (the first one cut, which leaves less than 2^-7, that rounded: 2^-15; up to 32 rows of a kv head) or to one (2^-8); sums of n terms, by threads and in parts: 2^-18 in all."""
    B, T, H, hd = q.shape
    pages, KV, page, _ = k.shape
    slots = table.shape[1] * page
    there = ((table >= 0) & (table < pages)).repeat_interleave(page, 1)
    at = table.clamp(0, pages - 1).long()
    flat = lambda x: x[at].transpose(1, 2).reshape(B, KV, slots, hd).double()   # noqa: E731
    k, v = flat(k), flat(v)
    out, room = torch.zeros(B, T, H, hd, dtype=torch.float64), torch.zeros(B, T, H, hd, dtype=torch.float64)
    p_step = 2.0 ** -11 if q.dtype == F16 else 2.0 ** -15 if T * (H // KV) <= 32 else 2.0 ** -8
    for b in range(B):
        rows = T if new is None else max(0, min(T, new[b]))
        seen = (torch.arange(rows) + min(starts[b], slots) + 1).clamp(0, slots)
        n = int(seen.max()) if rows else 0
        if n == 0:
            continue
        sight = (torch.arange(n) < seen[:, None]) & there[b, :n]
        kz, vz = (torch.where(sight.any(0)[:, None], x[b, :, :n], 0.0) for x in (k, v))
        for h in range(H):
            kh, vh, qh = kz[h // (H // KV)], vz[h // (H // KV)], q[b, :rows, h].double()
            x = (qh @ kh.T * scale).masked_fill(~sight, -math.inf)
            p = torch.exp(x - x.amax(1, keepdim=True).clamp(min=-1e300))
            l = p.sum(1, keepdim=True).clamp(min=1e-300)
            off = (hd / 8 * 2.0 ** -23 * (qh.abs() @ kh.abs().T * scale) + 2.0 ** -22 * x.abs()).masked_fill(~sight, 0.0).amax(1, keepdim=True)
            most = torch.where(sight[:, :, None], vh.abs()[None], 0.0).amax(1)
            out[b, :rows, h] = p @ vh / l
            room[b, :rows, h] = (p_step + 2 * (off + 2.0 ** -22) + 2.0 ** -18) * (p @ vh.abs()) / l + n * 2.0 ** -25 * most / l * (l > 1e-200)
    return out, room


ATTENDS = [  # B, T, H, KV, hd, page, pages of a sequence, starts, new, gaps
    (1, 1, 1, 1, 64, 16, 1, [0], None, []),
    (2, 1, 4, 2, 128, 16, 2, [16, 3], None, []),
    (3, 1, 8, 8, 128, 32, 19, [599, 0, 255], None, []),
    (2, 1, 8, 1, 64, 128, 9, [1099, 64], None, []),
    (4, 1, 4, 2, 64, 16, 4, [10, -1, 200, 49], [1, 1, 1, 0], []),     # ordinary; sees nothing; past the end: all slots; no token
    (3, 1, 4, 2, 128, 16, 50, [799, 400, 20], None, [(0, 3), (0, 17), (0, 49), (1, 0), (1, 25), (2, 0), (2, 1)]),   # pages that are none, the last one sees nothing
    (2, 1, 8, 8, 64, 64, 40, [2559, 7], [1, -3], []),
    (1, 3, 14, 2, 128, 64, 2, [87], None, []),
    (2, 5, 8, 2, 64, 16, 44, [300, 650], [5, 2], [(0, 19)]),
    (1, 40, 4, 4, 128, 16, 21, [293], None, []),
    (2, 70, 6, 2, 64, 32, 10, [0, 211], [70, 33], []),
    (1, 130, 2, 1, 128, 16, 9, [0], None, [(0, 0)]),
    (2, 150, 3, 3, 128, 128, 4, [1, 270], [0, 150], []),
    (1, 260, 4, 1, 64, 64, 9, [257], None, []),
    (2, 410, 4, 2, 128, 32, 29, [490, 100], [410, 77], [(0, 2), (0, 20)]),
    (2, 1520, 8, 1, 64, 32, 49, [25, -7], [1520, 800], []),
    (1, 1540, 8, 1, 128, 16, 100, [60], None, [(0, 7)]),
    (1, 200, 2, 2, 64, 16, 200, [2990], None, []),
]


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("case", ATTENDS, ids=[str(i) for i in range(len(ATTENDS))])
def test_attention(ops, case, dtype):
    B, T, H, KV, hd, page, per, starts, new, gaps = case
    g = torch.Generator().manual_seed(per + T)
    pk, pv, table = _pool(B, KV, hd, page, per, dtype, g, gaps)
    q = (torch.randn(B, T, H, hd, generator=g) * 2).to(dtype)
    want, room = _attention(q, pk, pv, table, starts, new, hd ** -0.5)
    dirty = [torch.full_like(pk, math.nan), torch.full_like(pv, math.nan)]   # what no row sees may be anything
    for b in range(B):
        end = max(0, min(page * per, starts[b] + (T if new is None else new[b])))
        for j in range(-(-end // page)):
            i = int(table[b, j])
            if 0 <= i < len(pk):
                for d, x in zip(dirty, (pk, pv)):
                    d[i, :, :min(page, end - j * page)] = x[i, :, :min(page, end - j * page)]
    args = (_dev(starts), _dev(new))
    got = ops.attention_paged(q.view(B * T, H * hd).to(DEV), _on(ops, *dirty, table), *args).cpu().double().view(B, T, H, hd)
    assert ((got - want).abs() <= _half(dtype) * want.abs() * 1.001 + room + _subnormal(dtype)).all()
    again = ops.attention_paged(q.view(B * T, H * hd).to(DEV), _on(ops, pk, pv, table), *args, scale=hd ** -0.5)
    assert torch.equal(again.cpu().double().view(B, T, H, hd), got)   # the same sums in the same order


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("T", [1, 7, 160])
def test_attention_of_uneven_values(ops, T, dtype):
    """Scores that climb along the keys (the running maximum moves all the time), rows of q of very different size, one of zeros."""
    B, H, KV, hd, page, per = 1, 4, 2, 128, 16, 44
    g = torch.Generator().manual_seed(T)
    k, v, table = _pool(B, KV, hd, page, per, dtype, g)
    order = torch.linspace(0.1, 3, per)
    for j in range(per):
        k[table[0, j].long()] *= order[j].to(dtype)
    q = (torch.randn(B, T, H, hd, generator=g) * 10.0 ** (torch.arange(H) * 0.5 - 1.5)[:, None]).to(dtype)
    q[:, :, 1] = 0
    start = [page * per - T]
    got = ops.attention_paged(q.view(T, H * hd).to(DEV), _on(ops, k, v, table), _dev(start)).cpu().double().view(B, T, H, hd)
    want, room = _attention(q, k, v, table, start, None, hd ** -0.5)
    assert ((got - want).abs() <= _half(dtype) * want.abs() * 1.001 + room + _subnormal(dtype)).all()


@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("T,H,KV,hd,back", [(3, 2, 2, 64, 2), (5, 8, 2, 128, 3), (150, 2, 1, 64, 2), (300, 2, 1, 128, 131), (300, 4, 4, 128, 290)])
def test_a_bad_value_reaches_only_the_rows_that_see_it(ops, T, H, KV, hd, back, dtype, bad):
    page, per = 16, 25
    g = torch.Generator().manual_seed(1)
    k, v, table = _pool(1, KV, hd, page, per, dtype, g)
    q = torch.randn(T, H * hd, generator=g).to(dtype)
    slot = 320 - back                      # seen by the last `back` rows
    start = _dev([320 - T])
    sound = ops.attention_paged(q.to(DEV), _on(ops, k, v, table), start).cpu()
    for which in (0, 1):
        spoilt = [k.clone(), v.clone()]
        spoilt[which][table[0, slot // page].long(), :, slot % page, 5] = bad
        out = ops.attention_paged(q.to(DEV), _on(ops, *spoilt, table), start).cpu()
        assert torch.equal(out[:-back], sound[:-back])
        rows = out[-back:].view(back, H, hd)
        if which == 1:   # one value of each head, and only that
            assert (rows[..., 5].isnan() if bad != bad else rows[..., 5] == bad).all()
            assert (rows[..., :5].double() - sound[-back:].view(back, H, hd)[..., :5].double()).abs().max() <= 2 * _half(dtype) * 4   # (summed another way: two roundings of values below 4)
        elif bad != bad:
            assert rows.isnan().all()


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("T,H", [(2, 4), (90, 2), (300, 2)])
def test_a_row_of_q_that_is_no_number_stays_alone(ops, T, H, dtype):
    g = torch.Generator().manual_seed(6)
    pool = _pool(1, H, 128, 32, 11, dtype, g)
    q = torch.randn(T, H, 128, generator=g).to(dtype)
    call = lambda q: ops.attention_paged(q.view(T, -1).to(DEV), _on(ops, *pool), _dev([352 - T])).cpu().view(T, H, 128)   # noqa: E731
    sound = call(q)
    q[1, 1, 7], q[0, 0, 3] = math.nan, math.inf
    got = call(q)
    assert got[1, 1].isnan().all() and not got[0, 0].isfinite().all()
    got[1, 1], got[0, 0] = sound[1, 1], sound[0, 0]
    assert torch.equal(got, sound)


@pytest.mark.parametrize("T", [1, 70])
def test_a_pool_beyond_32_bit_offsets(ops, T):
    """Pools of 2.4 G values each, of which the last pages are used."""
    hd, page, pages = 128, 128, 147_000
    g = torch.Generator().manual_seed(8)
    small = _pool(1, 1, hd, page, 3, BF16, g)
    k, v = (torch.empty(pages, 1, page, hd, dtype=BF16, device=DEV) for _ in range(2))
    base = pages - small[0].shape[0]
    k[base:], v[base:] = small[0].to(DEV), small[1].to(DEV)
    big = ops.PagedCache(k, v, (small[2] + base).to(DEV))
    ref = _on(ops, *small)
    cos, sin = (t.to(DEV) for t in _tables(3 * page, hd))
    x = [torch.randn(T, h * hd, generator=g).bfloat16().to(DEV) for h in (4, 1, 1)]
    start = _dev([300])
    qs = [ops.rope_append_paged(*x, cos, sin, start, c) for c in (big, ref)]
    assert torch.equal(*qs) and torch.equal(k[base:], ref.k) and torch.equal(v[base:], ref.v)
    assert torch.equal(*(ops.attention_paged(qs[0], c, start) for c in (big, ref)))


def test_strides_and_streams(ops):
    """q, k, v as columns of a fused projection's rows, and as views that the kernels do not take; keys and values as parts of one tensor, heads within slots; a table with
    room behind its rows; a stream of its own."""
    B, T, H, KV, hd, page, per = 2, 6, 4, 2, 64, 16, 3
    g = torch.Generator().manual_seed(2)
    wide = torch.randn(B * T, (H + 2 * KV) * hd, generator=g).half().to(DEV)
    q, k, v = wide.split([H * hd, KV * hd, KV * hd], dim=1)
    cos, sin = (t.to(DEV) for t in _tables(page * per, hd))
    start = _dev([0, 30])
    pk, pv, table = (t.to(DEV) for t in _pool(B, KV, hd, page, per, F16, g))

    def both(q, k, v, cache):
        r = ops.rope_append_paged(q, k, v, cos, sin, start, cache)
        return [r, ops.attention_paged(r, cache, start), ops.attention_paged(r[:B], cache, start), cache.k.contiguous(), cache.v.contiguous()]

    want = both(q.contiguous(), k.contiguous(), v.contiguous(), ops.PagedCache(pk.clone(), pv.clone(), table))
    odd = torch.zeros(B * T, KV * hd + 3, dtype=torch.float16, device=DEV)[:, 3:]
    odd.copy_(k)
    one = torch.empty(len(pk), page, 2, KV, hd, dtype=F16, device=DEV)        # slot by slot
    two = torch.empty(len(pk), KV, page, 2, hd + 8, dtype=F16, device=DEV)    # keys and values by turns, with a gap
    loose = torch.full((B, per + 5), -1, dtype=torch.int32, device=DEV)
    loose[:, :per] = table
    s = torch.cuda.Stream()
    for ck, cv in ((one[:, :, 0].transpose(1, 2), one[:, :, 1].transpose(1, 2)), (two[..., 0, :hd], two[..., 1, :hd])):
        ck.copy_(pk), cv.copy_(pv)
        s.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(s):
            got = both(q, odd, v, ops.PagedCache(ck, cv, loose[:, :per]))
        s.synchronize()
        for a, b in zip(want, got):
            assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("T,hd", [(90, 128), (300, 64)])
@pytest.mark.parametrize("layout", ["slots", "turns", "heads", "odd"])
def test_many_rows_on_other_layouts(ops, T, hd, dtype, layout):
    """Prompts over pools whose strides rise in other orders, and over one (odd) that the copy engine cannot describe, where a head's stride is no multiple of a slot's."""
    B, H, KV, page, per = 2, 4, 2, 32, 12
    g = torch.Generator().manual_seed(T)
    pk, pv, table = _pool(B, KV, hd, page, per, dtype, g, [(1, 3)])
    n = len(pk)

    def pools():
        if layout == "slots":
            one = torch.zeros(n, page, 2, KV, hd, dtype=dtype, device=DEV)
            return one[:, :, 0].transpose(1, 2), one[:, :, 1].transpose(1, 2)
        if layout == "turns":
            one = torch.zeros(n, KV, page, 2, hd + 8, dtype=dtype, device=DEV)
            return one[..., 0, :hd], one[..., 1, :hd]
        if layout == "heads":
            return tuple(torch.zeros(KV, n, page, hd, dtype=dtype, device=DEV).transpose(0, 1) for _ in range(2))
        sizes = (KV * (page * (hd + 8) + 8) + 16, page * (hd + 8) + 8, hd + 8, 1)
        return tuple(torch.zeros(n * sizes[0], dtype=dtype, device=DEV).as_strided((n, KV, page, hd), sizes) for _ in range(2))

    k, v = pools()
    k.copy_(pk), v.copy_(pv)
    q = (torch.randn(B, T, H, hd, generator=g) * 2).to(dtype)
    starts = [page * per - T, 11]
    got = ops.attention_paged(q.view(B * T, -1).to(DEV), ops.PagedCache(k, v, table.to(DEV)), _dev(starts)).cpu().double().view(B, T, H, hd)
    want, room = _attention(q, pk, pv, table, starts, None, hd ** -0.5)
    assert ((got - want).abs() <= _half(dtype) * want.abs() * 1.001 + room + _subnormal(dtype)).all()
    if layout != "odd":   # (there the rows go through the kernel for few, which sums in another order)
        assert torch.equal(ops.attention_paged(q.view(B * T, -1).to(DEV), _on(ops, pk, pv, table), _dev(starts)).cpu().double().view(B, T, H, hd), got)


@pytest.mark.parametrize("T", [1, 70])
def test_lazily_negated_rows_and_odd_columns(ops, T):
    """Views that the kernels do not take as they are give what their copies give."""
    H, KV, hd, page, per = 4, 2, 64, 16, 8
    g = torch.Generator().manual_seed(9)
    pk, pv, table = _pool(1, KV, hd, page, per, F16, g)
    cos, sin = (t.to(DEV) for t in _tables(page * per, hd))
    q, k, v = (torch.randn(T, h * hd, generator=g).half().to(DEV) for h in (H, KV, KV))
    start = _dev([50])
    a, b = _on(ops, pk, pv, table), _on(ops, pk, pv, table)
    x = ops.rope_append_paged(-q, -k, -v, cos, sin, start, a)
    y = ops.rope_append_paged(*(torch._neg_view(t) for t in (q, k, v)), cos, sin, start, b)
    assert torch.equal(x, y) and torch.equal(a.k, b.k) and torch.equal(a.v, b.v)
    odd = torch.empty(T, H * hd + 1, dtype=F16, device=DEV)[:, 1:]
    odd.copy_(-x)
    assert torch.equal(ops.attention_paged(x, a, start), ops.attention_paged(torch._neg_view(odd), a, start))


def test_two_streams_at_once(ops):
    """Calls on two streams that share a pool and q, but neither scratch nor results."""
    B, H, KV, hd, page, per = 2, 8, 2, 128, 16, 64
    g = torch.Generator().manual_seed(12)
    c = _on(ops, *_pool(B, KV, hd, page, per, BF16, g))
    calls = [(torch.randn(B * T, H * hd, generator=g).bfloat16().to(DEV), _dev([1024 - T, 700])) for T in (1, 3, 200)]
    want = [ops.attention_paged(q, c, start) for q, start in calls]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [[], []]
    for _ in range(10):
        for st, to in zip(streams, got):
            with torch.cuda.stream(st):
                to.extend(ops.attention_paged(q, c, start) for q, start in calls)
    torch.cuda.synchronize()
    for to in got:
        for i, o in enumerate(to):
            assert torch.equal(o, want[i % 3])


def test_sequences_that_share_pages(ops):
    """Two sequences on the pages of one prompt, each with a last page of its own."""
    KV, H, hd, page = 2, 4, 128, 16
    g = torch.Generator().manual_seed(4)
    k, v, table = _pool(2, KV, hd, page, 5, F16, g)
    table[1, :4] = table[0, :4]
    q = torch.randn(2, 1, H, hd, generator=g).half()
    got = ops.attention_paged(q.view(2, -1).to(DEV), _on(ops, k, v, table), _dev([70, 66])).cpu().double().view(2, 1, H, hd)
    want, room = _attention(q, k, v, table, [70, 66], None, hd ** -0.5)
    assert ((got - want).abs() <= _half(F16) * want.abs() * 1.001 + room).all()


@pytest.mark.parametrize("T", [1, 40])
def test_captured_and_replayed(ops, T):
    """A graph of append and attention whose positions move by an in-place addition in the graph itself, and whose table changes between replays, against eager calls;
    two graphs of the same calls replayed in turn on two streams share nothing."""
    B, H, KV, hd, page, per = 2, 4, 2, 128, 16, 128
    cos, sin = (t.to(DEV) for t in _tables(page * per, hd))
    g = torch.Generator().manual_seed(3)
    xs = [torch.randn(3, B * T, h * hd, generator=g).half().to(DEV) for h in (H, KV, KV)]
    pool = _pool(B, KV, hd, page, per, F16, g)

    def make():
        return _on(ops, *pool), _dev([5, 1029]), [x[0].clone() for x in xs]

    def step(c, start, x):
        r = ops.rope_append_paged(*x, cos, sin, start, c)
        o = ops.attention_paged(r, c, start)
        start.add_(T)
        return o

    def change(state, i):
        for d, s in zip(state[2], xs):
            d.copy_(s[i])
        state[0].table[:, 2 * i].fill_(-1)

    eager = make()
    want = []
    for i in range(3):
        change(eager, i)
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
                change(state, i)
                graph.replay()
        torch.cuda.synchronize()
        for graph, st, state, out in graphs:
            assert torch.equal(out, want[i])


@pytest.mark.parametrize("direct", [True, False])
def test_both_routes_give_the_same(ops, monkeypatch, direct):
    """The extension's direct calls and the general route, against each other on odd strides of dimensions of one."""
    from mem_efficient_blr_b200 import _lib as L
    if not direct:
        monkeypatch.setattr(L, "direct", lambda: None)
    g = torch.Generator().manual_seed(5)
    k, v, table = _pool(1, 1, 64, 16, 4, F16, g)
    c = ops.PagedCache(k.to(DEV).as_strided(k.shape, (1024, 3, 64, 1)), v.to(DEV), table.to(DEV))
    x = torch.randn(6, 64, generator=g).half().to(DEV)
    cos, sin = (t.to(DEV) for t in _tables(64, 64))
    r = ops.rope_append_paged(x, x, x, cos, sin, _dev([9]), c)
    o = ops.attention_paged(r, c, _dev([9])).cpu()
    want, room = _attention(r.cpu().view(1, 6, 1, 64), c.k.cpu(), c.v.cpu(), table, [9], None, 0.125)
    assert ((o.view(1, 6, 1, 64).double() - want).abs() <= _half(F16) * want.abs() * 1.001 + room).all()


def test_refusals_on_the_device(ops):
    c = ops.paged_cache(1, 2, 3, 2, 64, 16, F16, DEV)
    cos, sin = (t.to(DEV) for t in _tables(32, 64))
    x, start = torch.zeros(2, 128, dtype=torch.float16, device=DEV), torch.zeros(1, dtype=torch.int64, device=DEV)
    bad = [lambda: ops.rope_append_paged(x, x[:1], x, cos, sin, start, c), lambda: ops.rope_append_paged(x, x, x.bfloat16(), cos, sin, start, c),
           lambda: ops.rope_append_paged(x, x, x, cos[:31], sin, start, c), lambda: ops.rope_append_paged(x, x, x, cos, sin.double(), start, c),
           lambda: ops.rope_append_paged(x, x, x, cos, sin, start.int(), c), lambda: ops.rope_append_paged(x, x, x, cos, sin, start.expand(2), c),
           lambda: ops.rope_append_paged(x, x, x, cos, sin, start.cpu(), c), lambda: ops.attention_paged(x[:, :64], c, start), lambda: ops.attention_paged(x.float(), c, start),
           lambda: ops.attention_paged(x.bfloat16(), c, start), lambda: ops.attention_paged(x, c._replace(k=c.k.float()), start),
           lambda: ops.attention_paged(x, c._replace(v=c.v[:2]), start), lambda: ops.attention_paged(x, c._replace(table=c.table.long()), start),
           lambda: ops.attention_paged(x, c._replace(table=c.table[0]), start), lambda: ops.attention_paged(x, c._replace(table=c.table.new_zeros(1, 4)[:, ::2]), start),
           lambda: ops.attention_paged(x, c._replace(v=torch._neg_view(c.v)), start), lambda: ops.attention_paged(x, c._replace(table=c.table[:0]), start),
           lambda: ops.attention_paged(x, c._replace(k=c.k.transpose(2, 3)), start)]
    for call in bad:
        with pytest.raises(AssertionError):
            call()
    for k in (c.k[:1].expand(3, 2, 16, 64), torch.zeros(3, 2, 16, 68, dtype=F16, device=DEV)[..., :64], torch.zeros(8 + c.k.numel(), dtype=F16, device=DEV)[4:-4].view(c.k.shape)):
        with pytest.raises(RuntimeError, match="paged cache"):
            ops.attention_paged(x, c._replace(k=k), start)
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.attention_paged(x, c._replace(table=c.table.cpu()), start)
    for scale in (-1.0, math.inf, math.nan):
        with pytest.raises(RuntimeError, match="positive"):
            ops.attention_paged(x, c, start, None, scale)


def test_nothing_to_read(ops):
    """A pool without a page; sequences without a token; no rows."""
    empty = ops.paged_cache(2, 2, 0, 4, 64, 16, F16, DEV)
    x, start = torch.ones(2, 128, dtype=F16, device=DEV), torch.zeros(2, dtype=torch.int64, device=DEV)
    cos, sin = (t.to(DEV) for t in _tables(64, 64))
    assert not ops.rope_append_paged(x, x, x, cos, sin, start, empty).any() and not ops.attention_paged(x, empty, start).any()
    c = ops.paged_cache(2, 2, 8, 4, 64, 16, F16, DEV)
    assert not ops.attention_paged(x, c, start).any() and not ops.attention_paged(x, c, start, start).any()
    assert ops.attention_paged(x[:0], c, start).shape == (0, 128) and ops.rope_append_paged(x[:0], x[:0], x[:0], cos, sin, start, c).shape == (0, 128)
