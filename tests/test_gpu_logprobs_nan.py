"""The likeliest tokens of rows with NaN: NaN first, the lowest id first, and every place of the lists written."""
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


# (a warp, four warps, sixteen, a cluster for a row; every token asked for)
@pytest.mark.parametrize("rows,vocab,top", [(6, 300, 7), (300, 3000, 20), (300, 20011, 8), (6, 32000, 5), (6, 12, 12), (6, 64, 64), (6, 1, 1)])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
def test_a_nan_at_the_first_token(ops, rows, vocab, top, dtype):
    x = torch.randn(rows, vocab, generator=torch.Generator().manual_seed(vocab)).to(dtype)
    x[0::6, 0] = math.nan
    x[1::6] = math.nan
    x[2::6, 0], x[2::6, vocab - 1] = -math.nan, math.nan
    x[3::6, 0] = math.inf
    x[4::6, 1:] = math.nan
    lp, ent, tl, ti = (t.cpu() for t in ops.token_logprobs(x.to(DEV), torch.zeros(rows, dtype=torch.int64, device=DEV), top))
    rank = torch.where(x.isnan(), torch.full((), math.inf, dtype=torch.float64), torch.where(x == math.inf, 1e300, x.double()))
    assert torch.equal(ti, rank.sort(dim=-1, descending=True, stable=True).indices[:, :top])
    bad = (x.isnan() | (x == math.inf)).any(-1)
    assert lp[bad].isnan().all() and ent[bad].isnan().all() and tl[bad].isnan().all() and lp[~bad].isfinite().all()
