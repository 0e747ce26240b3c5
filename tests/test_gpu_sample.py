"""The choice of the next token against the definition in 64 bits, row by row.  Ids have to be equal: the kernel's weights and sums are 64-bit too, and a draw that lies within
2^-45 of a border has a chance of some 1e-9 here.  Log probabilities are off by their rounding to fp32 (2^-24 of themselves) and what the sums of at most 2^19 terms leave."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F16, BF16, F32 = torch.float16, torch.bfloat16, torch.float32


@pytest.fixture(scope="module")
def ops():
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")
    from mem_efficient_blr_b200 import ops as o
    return o


def _row(x, u, T, k, p, mp):
    """(id, log probability) of one row of logits; settings as they are held, in fp32."""
    x = x.double()
    if bool(x.isnan().any()) or x.max() == -math.inf or not T >= 0 or p != p or mp != mp or u != u:
        return -1, math.nan
    order = (x + 0.0).sort(descending=True, stable=True).indices
    M = x[order[0]]
    if T == 0:
        return int(order[0]), 0.0
    w = torch.where(x == M, 1.0, torch.exp((x - M) / T)).nan_to_num(0.0)
    w[x == -math.inf] = 0
    if M == math.inf:
        w = (x == M).double()
    kept = order[:k] if 0 < k < len(x) else order
    if p < 1:
        upto = w[kept].cumsum(0)
        kept = kept[:int((upto - w[kept] < p * upto[-1]).sum())] if p > 0 else kept[:1]
    kept = kept[w[kept] >= min(mp, 1.0)]
    ids = kept.sort().values
    ids = ids[w[ids] > 0]
    upto = w[ids].cumsum(0)
    n = len(ids) - 1 if u >= 1 else min(int((upto <= max(u, 0.0) * upto[-1]).sum()), len(ids) - 1)
    return int(ids[n]), float(torch.log(w[ids[n]] / upto[-1]))


def _want(x, u, T, k, p, mp):
    R = len(x)
    col = lambda v, t: [float(torch.tensor(v, dtype=torch.float32))] * R if not torch.is_tensor(v) else v.expand(R).tolist()   # noqa: E731
    k = [k] * R if not torch.is_tensor(k) else k.expand(R).tolist()
    rows = [_row(*a) for a in zip(x, u.tolist(), col(T, x), k, col(p, x), col(mp, x))]
    return torch.tensor([r[0] for r in rows]), torch.tensor([r[1] for r in rows], dtype=torch.float64)


def _check(got, want):
    ids, lp = (t.cpu() for t in got)
    assert ids.dtype == torch.int64 and lp.dtype == torch.float32
    assert torch.equal(ids, want[0])
    assert ((lp.isnan() & want[1].isnan()) | ((lp.double() - want[1]).abs() <= 2.0 ** -23 * want[1].abs() + 2.0 ** -32)).all()


def _rows(rows, vocab, dtype, g, kind):
    x = torch.empty(rows, vocab).exponential_(generator=g) * (torch.rand(rows, 1, generator=g) * 1.5 + 0.5) - 7   # the r-th likeliest token has a weight like r^-a
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
    elif kind == "normal":
        x = torch.randn(rows, vocab, generator=g) * 3
    elif kind == "steps":    # many ties
        x = (x * 2).round() / 2
    elif kind == "zeros":
        x = torch.where(torch.rand(rows, vocab, generator=g) < 0.5, 0.0, -0.0)
    return x.to(dtype)


SETTINGS = [  # temperature, top_k, top_p, min_p
    (1.0, 0, 1.0, 0.0), (0.0, 5, 0.5, 0.1), (0.7, 1, 1.0, 0.0), (0.8, 50, 0.95, 0.0), (1.3, 0, 0.9, 0.0), (1.0, 0, 0.3, 0.05), (2.0, 40, 1.0, 0.2), (0.5, 0, 1.0, 0.1),
    (1.0, 700, 0.99, 0.0), (1.0, 0, 0.0, 0.0), (1.0, 0, 1.0, 1.5), (1e-3, 0, 0.999, 0.0), (50.0, 0, 0.97, 0.0), (1.0, 3000, 0.8, 0.0),
]
SHAPES = [(1, 1, ""), (3, 5, ""), (4, 257, ""), (4, 257, "equal"), (3, 1001, "masked"), (3, 1001, "steps"), (2, 333, "lowest"), (2, 1030, "all lowest"), (3, 4003, "ends"),
          (2, 4096, "zeros"), (4, 32000, ""), (3, 32000, "steps"), (2, 32000, "normal"), (150, 5000, ""), (300, 777, "steps"), (2, 50001, ""), (1, 151936, ""), (2, 131072, "normal"), (2, 600, ""), (3, 4111, "steps"), (150, 24600, ""), (2, 49000, "steps"), (150, 52000, "masked")]


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("rows,vocab,kind", SHAPES)
def test_sample(ops, rows, vocab, kind, dtype):
    g = torch.Generator().manual_seed(rows + vocab)
    x = _rows(rows, vocab, dtype, g, kind)
    xd = x.to(DEV)
    for s in SETTINGS if rows < 100 else SETTINGS[3:6]:
        u = torch.rand(rows, generator=g)
        _check(ops.sample(xd, u.to(DEV), *s), _want(x, u, *s))


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
def test_settings_of_each_row(ops, dtype):
    g = torch.Generator().manual_seed(7)
    n = len(SETTINGS)
    x = _rows(n, 9001, dtype, g, "")
    T, k, p, mp = (torch.tensor(c, dtype=torch.int64 if i == 1 else F32) for i, c in enumerate(zip(*SETTINGS)))
    for _ in range(3):
        u = torch.rand(n, generator=g)
        _check(ops.sample(x.to(DEV), u.to(DEV), T.to(DEV), k.to(DEV), p.to(DEV), mp.to(DEV)), _want(x, u, T, k, p, mp))
        _check(ops.sample(x.to(DEV), u.to(DEV), T.to(DEV), 20, p.to(DEV), 0.01), _want(x, u, T, 20, p, 0.01))


def test_ties_and_borders(ops):
    """Whole weights, so that sums are exact and draws can lie on borders: 1000 equal tokens, of which top-k and top-p keep the first by id."""
    x = torch.zeros(12, 1000)
    u = torch.tensor([0.0, 0.25, 0.5, 0.75, 0.999, 1 - 2.0 ** -24, 1.0, 7.0, -1.0, 2.0 ** -30, 0.125, 0.3])
    for s, kept in (((1.0, 0, 1.0, 0.0), 1000), ((1.0, 8, 1.0, 0.0), 8), ((3.0, 0, 0.5, 0.0), 500), ((1.0, 64, 0.125, 1.0), 8), ((0.3, 0, 0.0005, 0.0), 1), ((1.0, 0, 0.501, 0.0), 501)):
        ids, lp = (t.cpu() for t in ops.sample(x.to(DEV), u.to(DEV), *s))
        want = (u.double().clamp(0, 1) * kept).floor().clamp(max=kept - 1).long()
        assert torch.equal(ids, want) and (lp.double() + math.log(kept)).abs().max() <= 2.0 ** -23 * math.log(kept)
    # the border lies between values: the third largest three times, of which two are kept
    y = torch.full((1, 3000), -5.0)
    y[0, [7, 100, 2000, 2999, 50]] = torch.tensor([2.0, 1.0, 1.0, 1.0, 3.0])
    got = {int(ops.sample(y.to(DEV), torch.tensor([v], device=DEV), 1e6, 4)[0]) for v in (0.1, 0.3, 0.6, 0.9)}
    assert got == {7, 50, 100, 2000}


@pytest.mark.parametrize("dtype", [F16, F32])
@pytest.mark.parametrize("vocab,many", [(700, 1), (9000, 1), (9000, 50)])
def test_rows_without_a_distribution(ops, vocab, many, dtype):
    x = torch.randn(9, vocab, generator=torch.Generator().manual_seed(1))
    x[0] = -math.inf
    x[1, 3] = math.nan
    x[2, 9] = x[2, 600] = math.inf
    x[3] = -math.inf
    x[3, 699] = -2.0
    x[4, vocab - 1] = math.nan
    x = x.to(dtype).repeat(many, 1)
    u = torch.full((9 * many,), 0.7)
    T = torch.tensor([1.0, 1.0, 1.0, 1.0, 0.0, -1.0, math.nan, math.inf, 1.0]).repeat(many)
    p = torch.tensor([1.0] * 8 + [math.nan]).repeat(many)
    for k in (0, 30):
        got = ops.sample(x.to(DEV), u.to(DEV), T.to(DEV), k, p.to(DEV))
        ids, lp = (t.cpu().view(many, 9) for t in got)
        assert (ids == ids[0]).all()
        assert ids[0, [0, 1, 4, 5, 6, 8]].eq(-1).all() and lp[:, [0, 1, 4, 5, 6, 8]].isnan().all()
        assert ids[0, 2] == 600 and abs(lp[0, 2] + math.log(2)) < 1e-6 and ids[0, 3] == 699 and lp[0, 3] == 0
        if k == 0:   # no temperature at all: an even choice
            assert ids[0, 7] == int(float(u[0]) * vocab)   # (0.7 is a little less in fp32)
    bad = ops.sample(x[5:6].to(DEV), torch.tensor([math.nan], device=DEV))
    assert bad[0] == -1 and bad[1].isnan()
    bad = ops.sample(x[5:6].to(DEV), torch.tensor([0.5], device=DEV), 1.0, 0, 1.0, torch.tensor([math.nan], device=DEV))
    assert bad[0] == -1


def test_frequencies(ops):
    """20000 draws of one row: how often each token comes up is within six standard deviations of its weight's share."""
    x = torch.tensor([1.0, 3.0, 2.0, 0.0, 2.5, -1.0, 2.0])
    n = 20000
    u = torch.rand(n, generator=torch.Generator().manual_seed(3))
    ids, lp = ops.sample(x.expand(n, 7).contiguous().to(DEV), u.to(DEV), 0.9, 5, 0.93)
    w = torch.exp(x.double() / 0.9)
    w[[3, 5, 0]] = 0   # (0.93 of the five is reached by four)
    share = w / w.sum()
    seen = torch.bincount(ids.cpu(), minlength=7).double() / n
    assert ((seen - share).abs() <= 6 * (share * (1 - share) / n).sqrt()).all()
    assert ((lp.cpu().double() - share.log()[ids.cpu()]).abs() <= 2.0 ** -22).all()


def test_shapes_strides_and_streams(ops):
    g = torch.Generator().manual_seed(9)
    x = torch.randn(3, 4, 1003, generator=g).half().to(DEV)
    u = torch.rand(3, 4, generator=g).to(DEV)
    want = ops.sample(x[..., :1000].contiguous(), u, 0.9, 40, 0.9)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = [ops.sample(x[..., :1000], u, 0.9, 40, 0.9), [t.t() for t in ops.sample(x[..., :1000].transpose(0, 1), u.t(), 0.9, 40, 0.9)],
               ops.sample(x[..., :1000], u, torch.tensor(0.9, device=DEV), torch.full((3, 4), 40, device=DEV), torch.full((4, 3), 0.9, device=DEV).t()),
               ops.sample(torch._neg_view(-x[..., :1000]), torch._neg_view(-u), 0.9, 40, 0.9)]
    s.synchronize()
    for ids, lp in got:
        # (the order of a row's sums goes by its alignment; 64 bits)
        assert ids.shape == lp.shape == (3, 4) and torch.equal(ids, want[0]) and (lp - want[1]).abs().max() <= 2.0 ** -22
    one = ops.sample(x[0, 0, 1:1001], u[0, 0])
    assert one[0].shape == one[1].shape == () and 0 <= one[0] < 1000
    none = ops.sample(x[:0], u[:0])
    assert none[0].shape == none[1].shape == (0, 4)


def test_captured_and_replayed(ops):
    g = torch.Generator().manual_seed(11)
    x, u = torch.randn(4, 5, 20000, generator=g).to(DEV) * 3, torch.rand(4, 5, generator=g).to(DEV)
    T = torch.tensor([1.0, 0.5, 0.0, 2.0, 0.8], device=DEV)
    want = [[t.clone() for t in ops.sample(x[i], u[i], T, 100, 0.9)] for i in range(4)]
    graphs = []
    for _ in range(2):
        xs, us = x[0].clone(), u[0].clone()
        st = torch.cuda.Stream()
        st.wait_stream(torch.cuda.current_stream())
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.stream(st):
            with torch.cuda.graph(graph, stream=st):
                out = ops.sample(xs, us, T, 100, 0.9)
        graphs.append((graph, st, xs, us, out))
    torch.cuda.synchronize()
    for i in range(4):
        for graph, st, xs, us, out in graphs:
            with torch.cuda.stream(st):
                xs.copy_(x[i]), us.copy_(u[i])
                graph.replay()
        torch.cuda.synchronize()
        for *_, out in graphs:
            assert torch.equal(out[0], want[i][0]) and torch.equal(out[1], want[i][1])


@pytest.mark.parametrize("dtype,vocab", [(BF16, 786000), (F32, 393000), (F16, 2097151), (F32, 1048576)])
def test_the_longest_rows(ops, dtype, vocab):
    g = torch.Generator().manual_seed(vocab)
    x = _rows(2, vocab, dtype, g, "")
    for s in SETTINGS[:6]:
        u = torch.rand(2, generator=g)
        _check(ops.sample(x.to(DEV), u.to(DEV), *s), _want(x, u, *s))


def test_refusals_on_the_device(ops):
    x, u = torch.zeros(2, 10, device=DEV), torch.zeros(2, device=DEV)
    each = torch.ones(2, device=DEV)
    bad = [lambda: ops.sample(x, u[:1]), lambda: ops.sample(x, u.double()), lambda: ops.sample(x, u.cpu()), lambda: ops.sample(x.double(), u), lambda: ops.sample(x.int(), u),
           lambda: ops.sample(x, u, -0.1), lambda: ops.sample(x, u, math.nan), lambda: ops.sample(x, u, each.double()), lambda: ops.sample(x, u, each.cpu()),
           lambda: ops.sample(x, u, 1.0, each), lambda: ops.sample(x, u, 1.0, each.int()), lambda: ops.sample(x, u, 1.0, 0, each[:1]), lambda: ops.sample(x, u, 1.0, 0, 1.0, each.half())]
    for call in bad:
        with pytest.raises(AssertionError):
            call()
    for call in (lambda: ops.sample(x, u, 1.0, 0, math.nan), lambda: ops.sample(x, u, 1.0, 0, 1.0, math.nan)):
        with pytest.raises(RuntimeError, match="numbers"):
            call()
    with pytest.raises(RuntimeError, match="rows of at most"):
        ops.sample(torch.zeros(1, 1048577, device=DEV), u[:1])
