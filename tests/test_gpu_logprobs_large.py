"""Log probabilities of rows whose largest value is large: a row that is masked as a whole with a number like -1e10 is an even distribution, and what
is compared within a row are differences, however far from 0 it lies."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.fixture(scope="module")
def ops():
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")
    from mem_efficient_blr_b200 import ops as o
    return o


def _check(ops, x, top):
    rows, vocab = x.shape
    ids = torch.randint(0, vocab, (rows,), generator=torch.Generator().manual_seed(rows))
    lp, ent, tl, ti = (t.cpu() for t in ops.token_logprobs(x.to(DEV), ids.to(DEV), top))
    d = x.double()
    want = torch.log_softmax(d, -1)
    far = d - d.amax(-1, keepdim=True)
    log_s = far.exp().sum(-1, keepdim=True).log()
    # S: e to 2^-21 and 2^-22 of its exponent's argument, whose mean size is at most log S; sums of at most vocab / 256 + 64 terms in a row; then a difference of
    # two fp32 numbers
    rel_s = 2.0 ** -21 + (vocab / 256 + 64) * 2.0 ** -24 + 2.0 ** -22 * log_s
    allow = rel_s + 2.0 ** -23 * (far.abs().nan_to_num(posinf=0) + log_s)
    ok = lambda got, ref, room: bool((((got.double() - ref).abs() <= room) | (got.double() == ref)).all())   # noqa: E731
    assert ok(lp, want.gather(1, ids[:, None])[:, 0], allow.gather(1, ids[:, None])[:, 0])
    p = want.exp()
    spread = (p * far.nan_to_num(neginf=0).abs()).sum(-1)
    assert ok(ent, torch.special.entr(p).sum(-1),
              rel_s[:, 0] * (1 + 2 * spread) + 2.0 ** -21 * (p * far.nan_to_num(neginf=0) ** 2).sum(-1) + 2.0 ** -23 * (log_s[:, 0] + spread))
    order = x.float().sort(dim=-1, descending=True, stable=True).indices[:, :top]
    assert torch.equal(ti, order) and ok(tl, want.gather(1, order), allow.gather(1, order))


# (a warp, four warps, sixteen, a cluster for a row)
SIZES = [(5, 300, 7), (300, 3000, 20), (299, 20011, 8), (3, 32000, 5)]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows,vocab,top", SIZES, ids=[str(s[1]) for s in SIZES])
@pytest.mark.parametrize("at", [s * m for m in (2e9, 3.4e9, 1e10, 1e15, 1e30, 9e36, 1.1e37) for s in (1, -1)])
def test_rows_around_a_large_number(ops, rows, vocab, top, at, dtype):
    g = torch.Generator().manual_seed(vocab)
    x = torch.full((rows, vocab), at)
    x[1::4, ::3] = -math.inf                                                       # ruled out, beside it
    x[2::4, 1::2] = at * (1.25 if at < 0 else 0.5)                                 # and other numbers far below
    x[3::4, 1:] = torch.randn(rows, vocab - 1, generator=g)[3::4] * 3              # ordinary values: with one of 1e10, or all of them above one of -1e10
    _check(ops, x.to(dtype), top)


@pytest.mark.parametrize("rows,vocab,top", SIZES, ids=[str(s[1]) for s in SIZES])
@pytest.mark.parametrize("at", [3e4, 1e6, -1e6, 1.6e7, -1.6e7])
def test_differences_of_rows_far_from_zero(ops, rows, vocab, top, at):
    g = torch.Generator().manual_seed(vocab)
    _check(ops, (torch.randn(rows, vocab, generator=g) * 3 + at).float(), top)
