"""Tokens that do not fit a decoder's 8-bit cache: nobody on the host sees their positions, so the answers of their sequences, which would be made without them,
come out as NaN, and those of the other sequences as ever."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.fixture(scope="module")
def model():
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")
    from mem_efficient_blr_b200 import networks as nw
    shape = nw.LlamaShape(layers=2, d=512, heads=8, ffn=1024, vocab=384, b=16, rank_attn=64, rank_mlp=96)
    return lambda: nw.LlamaDecoder(shape, "blast", batch=3, cache_len=20, device=DEV, dtype=torch.float16, seed=3, kv_cache="int8")


def _ids(T):
    return torch.randint(0, 384, (3, T), generator=torch.Generator().manual_seed(T)).to(DEV)


def _at(*p):
    return torch.tensor(p, device=DEV)


@pytest.mark.parametrize("fused", [True, False])
def test_extend_past_the_end(model, fused):
    m, ref = model(), model()
    m.fused_decode = ref.fused_decode = fused
    for d in (m, ref):
        d.prefill(_ids(10))
    fits = ref.extend(_ids(4), _at(10, 10, 10))
    got = m.extend(_ids(4), _at(10, 17, 10))            # the second one's last token has no slot
    assert got[1].isnan().all() and torch.equal(got[[0, 2]], fits[[0, 2]])
    got = m.extend(_ids(4), _at(10, 17, -1), _at(4, 3, 4))   # three tokens fill it; a token ahead of the first slot
    assert got[:2].isfinite().all() and got[2].isnan().all() and torch.equal(got[0], fits[0])
    got = m.extend(_ids(4), _at(16, 16, 2 ** 62), _at(4, 4, 1))
    assert got[:2].isfinite().all() and got[2].isnan().all()


@pytest.mark.parametrize("fused", [True, False])
def test_decode_past_the_end(model, fused):
    from mem_efficient_blr_b200 import networks as nw
    m = model()
    m.fused_decode = fused
    m.prefill(_ids(20))
    assert m.decode_step(_ids(1), _at(19)).isfinite().all() and m.decode_step(_ids(1), _at(20)).isnan().all()
    got = m.decode_step(_ids(1), _at(19, 20, 0))
    assert got[[0, 2]].isfinite().all() and got[1].isnan().all()
    pos = _at(18)
    step = nw.GraphedCall(m.decode_step, _ids(1), pos)
    assert [bool(step(_ids(1), _at(p)).isnan().all()) for p in (18, 19, 20, 21, 3)] == [False, False, True, True, False]
