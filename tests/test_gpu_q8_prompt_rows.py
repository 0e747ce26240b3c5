"""Attention of many rows over the 8-bit cache: a row without a number among its scores leaves the rows beside it as they are, also where their largest scores climb by many powers of
two along the keys."""
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


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("code", [torch.int8, torch.float8_e4m3fn], ids=["int8", "e4m3"])
@pytest.mark.parametrize("T,H,KV,hd,slots,rise", [(90, 2, 2, 128, 320, 6.0), (300, 4, 1, 64, 320, 8.0), (90, 2, 1, 128, 4096, 24.0), (3100, 4, 4, 64, 3200, 30.0)])
@pytest.mark.parametrize("spoil", ["nan", "-inf"])
def test_scores_that_climb_beside_a_row_of_none(ops, T, H, KV, hd, slots, rise, spoil, code, dtype):
    """Codes and q have values of one sign, so that a key's scale is its score's size: it climbs along the blocks."""
    block = 16
    g = torch.Generator().manual_seed(T)
    top = 100.0
    codes = lambda: (top * (0.9 + 0.1 * torch.rand(1, KV, slots, hd, generator=g))).round().to(code)   # noqa: E731
    k, v = codes(), (torch.randn(1, KV, slots, hd, generator=g) * 30).round().to(code)
    ks = (torch.linspace(0, rise, slots // block) / top).expand(1, KV, -1).contiguous()
    vs = torch.full((1, KV, slots // block), 1 / 30)
    cache = ops.Q8Cache(*(t.to(DEV) for t in (k, v, ks, vs)), block)
    q = ((1 + 0.5 * torch.rand(T, H, 1, generator=g)) * (1 + 0.1 * torch.rand(T, H, hd, generator=g))).to(dtype)
    start = torch.tensor([slots - T], device=DEV)
    call = lambda q: ops.attention_q8(q.view(T, -1).to(DEV), cache, start).cpu().view(T, H, hd)   # noqa: E731
    sound = call(q)
    at, vals = (c.double().mul(s.double().repeat_interleave(block, -1)[..., None])[0] for c, s in ((k, ks), (v, vs)))
    for h in range(H):   # (the rows are right: the weights to 2^-11 and the sums, results below 5)
        x = q[:, h].double() @ at[h // (H // KV)].T * hd ** -0.5
        x = x.masked_fill(torch.arange(slots) > slots - T + torch.arange(T)[:, None], -math.inf)
        assert (sound[:, h].double() - torch.softmax(x, -1) @ vals[h // (H // KV)]).abs().max() <= 2.0 ** -5
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
