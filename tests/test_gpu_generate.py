"""Generation from padded batches: sequences without a token, and pools that hold the batch and nothing more."""
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


@pytest.mark.parametrize("lens,N,pages", [((9, 9), 8, 2), ((9, 4), 8, 2), ((40, 3, 0), 9, 4), ((16, 1, 17), 1, 4), ((5, 33), 0, 4), ((62, 1), 20, 6)])
def test_a_pool_that_just_holds_the_batch(make, lens, N, pages):
    """A sequence of n tokens that goes on by N is appended to N - 1 times."""
    B, T = len(lens), max(lens)
    ids, u = _ids(B, T), _u(B, N)
    n = _at(*lens)
    m, ref = make(batch=B, kv_cache="paged", kv_pages=pages), make(batch=B, kv_cache="paged")
    got, want = (d.generate(ids, N, u, 0.9, 40, n_new=n) for d in (m, ref))
    assert torch.equal(got[0], want[0]) and all(torch.equal(a.isnan(), b.isnan()) and torch.equal(a.nan_to_num(), b.nan_to_num()) for a, b in ((got[1], want[1]),) if N)
    assert len(m._free) == 0
    if len(set(lens)) == 1:
        m = make(batch=B, kv_cache="paged", kv_pages=pages)
        assert torch.equal(m.generate(ids, N, u, 0.9, 40)[0], want[0])
    m = make(batch=B, kv_cache="paged", kv_pages=pages - 1)
    with pytest.raises(RuntimeError, match="1 more pages|are free"):
        m.generate(ids, N, u, 0.9, 40, n_new=n)
    assert len(m._free) == pages - 1


def test_generation_in_a_graph(make):
    """Where every sequence has its pages, nothing is read back on the host."""
    ids, u, n = _ids(2, 9), _u(2, 4), _at(9, 5)
    for pages in (None, 8):
        m = make(batch=2, kv_cache="paged", kv_pages=pages)
        want = m.generate(ids, 4, u, 0.9, 40, n_new=n)
        if pages:
            m.reserve([12, 12])
        st, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
        st.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(st):
            with torch.cuda.graph(graph, stream=st):
                got = m.generate(ids, 4, u, 0.9, 40, n_new=n)
            graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
