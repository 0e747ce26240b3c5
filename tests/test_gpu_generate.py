"""Generation from padded batches."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.fixture(scope="module")
def make():
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")
    from mem_efficient_blr_b200 import networks as nw
    shape = nw.LlamaShape(layers=2, d=512, heads=8, ffn=1024, vocab=384, b=16, rank_attn=64, rank_mlp=96)

    def f(batch=3, cache_len=64, **kw):
        return nw.LlamaDecoder(shape, "blast", batch=batch, cache_len=cache_len, device=DEV, dtype=torch.float16, seed=3, **kw)
    return f


def _ids(B, T, seed=1):
    return torch.randint(0, 384, (B, T), generator=torch.Generator().manual_seed(seed)).to(DEV)


def _u(B, N):
    return torch.rand(B, N, generator=torch.Generator().manual_seed(2)).to(DEV)


def _at(*p):
    return torch.tensor(p, device=DEV)


@pytest.mark.parametrize("kv", ["paged", "int8"])
def test_a_sequence_without_a_token_has_no_next_one(make, kv):
    ids, u = _ids(4, 9), _u(4, 5)
    m = make(batch=4, kv_cache=kv)
    got, lp = m.generate(ids, 5, u, 0.8, 50, 0.95, n_new=_at(9, 0, 4, -2))
    assert (got[1::2] == -1).all() and lp[1::2].isnan().all()
    want, want_lp = make(batch=4, kv_cache=kv).generate(ids, 5, u, 0.8, 50, 0.95, n_new=_at(9, 1, 4, 1))
    assert torch.equal(got[::2], want[::2]) and torch.equal(lp[::2], want_lp[::2]) and (got[::2] >= 0).all()
    got, lp = m.generate(ids, 1, u[:, :1], 0.0, n_new=_at(0, 0, 0, 3))
    assert (got[:3] == -1).all() and lp[:3].isnan().all() and got[3] >= 0 and lp[3] == 0
