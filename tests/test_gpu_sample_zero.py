"""The choice of the next token on rows whose search for the edge goes on below, or begins at, a logit of exactly 0, against the definition in 64 bits.  Ids have to be equal;
log probabilities are off by their rounding to fp32 (2^-24 of themselves) and what sums of at most 2^19 terms leave."""
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


def _want(x, u, T, k, p, mp):
    """(ids, log probabilities) of one row of logits for each number of u; settings as they are held, in fp32."""
    T, p, mp = (float(torch.tensor(v, dtype=F32)) for v in (T, p, mp))
    x = x.double() + 0.0
    order = x.sort(descending=True, stable=True).indices
    w = torch.exp((x - x.max()) / T)
    kept = order[:k] if k > 0 else order
    if p < 1:
        upto = w[kept].cumsum(0)
        kept = kept[:int((upto - w[kept] < p * upto[-1]).sum())]
    kept = kept[w[kept] >= min(mp, 1.0)]
    ids = kept.sort().values
    ids = ids[w[ids] > 0]
    upto = w[ids].cumsum(0)
    at = torch.searchsorted(upto, u.double() * upto[-1], right=True).clamp(max=len(ids) - 1)
    return ids[at], torch.log(w[ids[at]] / upto[-1])


def _check(ops, x, T, k, p, mp=0.0):
    u = (torch.arange(24) + 0.37) / 24
    ids, lp = (t.cpu() for t in ops.sample(x.to(DEV).expand(24, -1), u.to(DEV), T, k, p, mp))
    want, want_lp = _want(x, u, T, k, p, mp)
    assert torch.equal(ids, want)
    assert ((lp.double() - want_lp).abs() <= 2.0 ** -23 * want_lp.abs() + 2.0 ** -32).all()


# (the row by 128 threads and 512 that keep it, and by 1024 that read it again)
SIZES = [3000, 32000, 150000]


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("vocab", SIZES)
@pytest.mark.parametrize("every", [107, 53])
def test_the_likeliest_are_zeros(ops, vocab, every, dtype):
    """Some hundred logits of 0, of either sign, are the largest, and the nucleus reaches into what lies below."""
    x = torch.full((vocab,), -3.0)
    x[::every] = 0.0
    x[::5 * every] = -0.0
    for p in (0.05, 0.5, 0.9, 0.999):
        _check(ops, x.to(dtype), 1.0, 0, p)
    y = x.clone()
    y[1::7] = -1.0
    y[2::9] = -3.25
    y[5] = 0.5
    for p in (0.3, 0.6, 0.9, 0.97):
        _check(ops, y.to(dtype), 1.0, 0, p)
        _check(ops, y.to(dtype), 0.7, 2000, p)
        _check(ops, y.to(dtype), 1.1, 0, p, 0.01)


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("vocab", SIZES)
def test_a_search_down_to_zero(ops, vocab, dtype):
    """The search for the edge of a nucleus covers weights from 1 to e^-24, that is down to a logit of exactly 0 here, and the edge lies there or below."""
    g = torch.Generator().manual_seed(vocab)
    x = -torch.rand(vocab, generator=g) * 2
    x[torch.rand(vocab, generator=g) < 0.5] = 0.0
    x[vocab // 3] = 24.0
    for p in (1 - 2.0 ** -20, 1 - 2.0 ** -22, 1 - 2.0 ** -23, 1 - 2.0 ** -24):
        _check(ops, x.to(dtype), 1.0, 0, p)
        _check(ops, (x / 4).to(dtype), 0.25, 0, p)
    # the same with a greater share: of many large logits, and of what T makes of it
    y = torch.where(torch.rand(vocab, generator=g) < 0.01, 3.0, x.clamp(max=0.0))
    for p in (0.3, 0.6, 0.8, 0.9, 0.95, 0.99):
        _check(ops, y.to(dtype), 0.125, 0, p)
        _check(ops, y.to(dtype), 2.0, 0, p)


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
@pytest.mark.parametrize("vocab", SIZES)
def test_an_edge_by_count_around_zero(ops, vocab, dtype):
    """More than can be listed are to be counted, and the last one is a zero, the next one above or the next one below."""
    g = torch.Generator().manual_seed(vocab + 1)
    x = torch.randn(vocab, generator=g)
    x = torch.where(x.abs() < 0.4, 0.0, x)
    tiny = float(torch.finfo(dtype).smallest_normal)
    x[7::50] = tiny
    x[9::50] = -tiny
    above, zeros = int((x > 0).sum()), int((x == 0).sum())
    for k in (above, above + 1, above + zeros // 2, above + zeros, above + zeros + 1):
        _check(ops, x.to(dtype), 1.0, k, 1.0)
        _check(ops, x.to(dtype), 1.0, k, 0.97)


@pytest.mark.parametrize("dtype", [F16, BF16, F32])
def test_many_rows(ops, dtype):
    """More rows than there are SMs, each with zeros of its own."""
    for vocab in (900, 32000, 60000):
        g = torch.Generator().manual_seed(vocab)
        rows = 160
        x = torch.full((rows, vocab), -3.0)
        x[torch.rand(rows, vocab, generator=g) < torch.rand(rows, 1, generator=g) * 0.05] = 0.0
        x[:, 11] = 0.0
        x = x.to(dtype)
        u = torch.rand(rows, generator=g)
        ids, lp = (t.cpu() for t in ops.sample(x.to(DEV), u.to(DEV), 1.0, 0, 0.9))
        for r in range(rows):
            want, want_lp = _want(x[r], u[r:r + 1], 1.0, 0, 0.9, 0.0)
            assert ids[r] == want[0] and abs(float(lp[r]) - float(want_lp[0])) <= 2.0 ** -23 * abs(float(want_lp[0])) + 2.0 ** -32
