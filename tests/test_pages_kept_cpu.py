"""No page is lost by a call that fails: pages of a decoder's cache are either a sequence's, as the table has it, or free.  No GPU: nothing is computed."""
import pytest
import torch

from mem_efficient_blr_b200 import networks as nw

SHAPE = nw.LlamaShape(layers=1, d=128, heads=2, ffn=128, vocab=32, b=4, rank_attn=16, rank_mlp=16)


def _decoder():
    return nw.LlamaDecoder(SHAPE, "dense", batch=3, cache_len=50, device="cpu", dtype=torch.float16, kv_cache="paged", kv_pages=7)


def _same(m, pages, free):
    assert m._pages == pages and m._free == free and [[int(v) for v in row if v >= 0] for row in m.page_table] == pages


def test_a_table_that_cannot_be_written(monkeypatch):
    """As inside a stream capture, where a copy from the host is refused."""
    m = _decoder()
    m.reserve([17])
    pages, free = [list(p) for p in m._pages], list(m._free)

    def refused(*a, **k):
        raise RuntimeError("operation not permitted when stream is capturing")
    with monkeypatch.context() as patch:
        patch.setattr(torch, "tensor", refused)
        with pytest.raises(RuntimeError, match="capturing"):
            m.reserve([50, 20])
    _same(m, pages, free)
    m.reserve([50, 20, 1])
    assert [len(p) for p in m._pages] == [4, 2, 1] and not m._free


def test_a_release_with_a_sequence_that_is_none():
    m = _decoder()
    m.reserve([17, 30])
    pages, free = [list(p) for p in m._pages], list(m._free)
    for bad in ([0, 3], [1, -1], (b for b in (0, 1, 7))):
        with pytest.raises(ValueError, match="no sequence"):
            m.release(bad)
        _same(m, pages, free)
    m.release(b for b in (0, 0, 1))
    assert m._pages == [[], [], []] and sorted(m._free) == list(range(7))
