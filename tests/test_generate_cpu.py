"""What pages generation gives to the sequences of a padded batch, and what calls that fail leave behind.  No GPU: the calls end where a kernel would be launched."""
import pytest
import torch

from mem_efficient_blr_b200 import networks as nw

SHAPE = nw.LlamaShape(layers=2, d=128, heads=2, ffn=128, vocab=32, b=4, rank_attn=16, rank_mlp=16)


def _decoder(batch=3, cache_len=50, **kw):
    return nw.LlamaDecoder(SHAPE, "dense", batch=batch, cache_len=cache_len, device="cpu", dtype=torch.float16, kv_cache="paged", **kw)


def _held(m):
    return [len(p) for p in m._pages]


@pytest.mark.parametrize("lens,N,held", [(None, 8, [1, 1]), (None, 9, [2, 2]), ([9, 4], 9, [2, 1]), ([0, 9], 20, [0, 2]), ([-3, 30], 1, [0, 1]), ([1, 9], 0, [1, 1]), ([9, 2], 300, [4, 4])])
def test_pages_by_each_sequence_s_own_length(lens, N, held):
    m = _decoder(kv_pages=sum(held))
    n = None if lens is None else torch.tensor(lens)
    with pytest.raises(RuntimeError, match="CPU|CUDA"):
        m.generate(torch.zeros(2, 9, dtype=torch.int64), N, torch.zeros(2, N), n_new=n)
    assert _held(m) == held + [0]
    short = _decoder(kv_pages=sum(held) - 1)
    with pytest.raises(RuntimeError, match="are free"):
        short.generate(torch.zeros(2, 9, dtype=torch.int64), N, torch.zeros(2, N), n_new=n)
    assert not any(_held(short)) and len(short._free) == sum(held) - 1
