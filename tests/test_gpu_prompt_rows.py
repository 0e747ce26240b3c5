"""Attention of many rows over a cache in pages: a row without a number among its scores leaves the rows beside it as they are, also where their largest scores climb by many powers
of two along the keys."""
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


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("T,H,KV,hd,slots,rise", [(90, 2, 2, 128, 320, 6.0), (300, 4, 1, 64, 320, 8.0), (90, 2, 1, 128, 4096, 24.0), (150, 4, 4, 64, 1600, 24.0)])
@pytest.mark.parametrize("spoil", ["nan", "inf", "-inf"])
def test_scores_that_climb_beside_a_row_of_none(ops, T, H, KV, hd, slots, rise, spoil, dtype):
    """q and k have values of one sign, so that a key's size is its score's: `rise` times sqrt(head_dim) more at the last key than at the first (16 powers of two and more within the first 128
    keys of the shortest), the rows of q up to 1.5 times apart."""
    page = 16
    g = torch.Generator().manual_seed(T)
    n = slots // page
    table = torch.randperm(n, generator=g).to(torch.int32)[None]
    size = torch.linspace(0, rise, slots)[:, None]
    keys = (size * (1 + 0.05 * torch.randn(slots, KV, hd, generator=g).transpose(0, 1).abs())).to(dtype)   # (KV, slots, hd)
    pool = torch.empty(n, KV, page, hd, dtype=dtype)
    pool[table[0].long()] = keys.view(KV, n, page, hd).transpose(0, 1)
    v = torch.randn(n, KV, page, hd, generator=g).to(dtype)
    cache = ops.PagedCache(pool.to(DEV), v.to(DEV), table.to(DEV))
    q = (1 + 0.5 * torch.rand(T, H, 1, generator=g)) * (1 + 0.1 * torch.rand(T, H, hd, generator=g))
    q = q.to(dtype)
    start = torch.tensor([slots - T], device=DEV)
    call = lambda q: ops.attention_paged(q.view(T, -1).to(DEV), cache, start).cpu().view(T, H, hd)   # noqa: E731
    sound = call(q)
    at = pool[table[0].long()].transpose(0, 1).reshape(KV, slots, hd).double()
    vals = v[table[0].long()].transpose(0, 1).reshape(KV, slots, hd).double()
    for h in range(H):   # (the rows are right: the weights to 2^-8 and the sums, results below 4)
        x = q[:, h].double() @ at[h // (H // KV)].T * hd ** -0.5
        x = x.masked_fill(torch.arange(slots) > slots - T + torch.arange(T)[:, None], -math.inf)
        want = torch.softmax(x, -1) @ vals[h // (H // KV)]
        assert (sound[:, h].double() - want).abs().max() <= 2.0 ** -5
    bad = q.clone()
    rows = [(0, 0), (5, H - 1), (37, 0), (T - 1, H - 1)]
    for t, h in rows:
        bad[t, h, 3] = float(spoil)
    got = call(bad)
    for t, h in rows:
        if spoil == "nan":
            assert got[t, h].isnan().all()
        got[t, h] = sound[t, h]
    assert torch.equal(got, sound)
