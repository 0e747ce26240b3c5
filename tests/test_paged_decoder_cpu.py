"""The pages of a decoder's cache: who has which, what is refused.  No GPU: nothing is computed."""
import pytest
import torch

from mem_efficient_blr_b200 import networks as nw

SHAPE = nw.LlamaShape(layers=2, d=128, heads=2, ffn=128, vocab=32, b=4, rank_attn=16, rank_mlp=16)


def _decoder(batch=3, cache_len=50, **kw):
    return nw.LlamaDecoder(SHAPE, "dense", batch=batch, cache_len=cache_len, device="cpu", dtype=torch.float16, kv_cache="paged", **kw)


def _held(m):
    """Pages of each sequence, as its row of the table has them: first the pages, then none."""
    rows = [[int(v) for v in row if v >= 0] for row in m.page_table]
    for row, pages in zip(m.page_table, rows):
        assert row[:len(pages)].tolist() == pages and (row[len(pages):] == -1).all()
    every = [p for r in rows for p in r]
    assert len(set(every)) == len(every) and all(0 <= p < m.kv_pages for p in every)
    assert sorted(every + m._free) == list(range(m.kv_pages))
    return rows


def test_every_sequence_has_its_pages_from_the_beginning():
    m = _decoder(kv_block=16)
    assert [len(r) for r in _held(m)] == [4, 4, 4] and not m._free
    assert m.paged[0].table is m.page_table and m.paged[1].table is m.page_table and m.paged[0].k.shape == (12, 2, 16, 64) and not m.kcache and m.q8cache is None


def test_pages_go_to_sequences_and_come_back():
    m = _decoder(kv_block=16, kv_pages=7)
    assert not any(_held(m))
    m.reserve([17, 0, 50])
    assert [len(r) for r in _held(m)] == [2, 0, 4]
    before = _held(m)
    m.reserve([16, 1])          # what a sequence has stays
    assert [len(r) for r in _held(m)] == [2, 1, 4] and _held(m)[0] == before[0]
    with pytest.raises(RuntimeError, match="1 more pages are needed, 0 are free"):
        m.reserve([33])
    assert [len(r) for r in _held(m)] == [2, 1, 4]
    m.release([2])
    m.reserve([33, 30])
    assert [len(r) for r in _held(m)] == [3, 2, 0]
    m.release(range(3))
    assert not any(_held(m)) and len(m._free) == 7


def test_what_is_refused():
    m = _decoder(kv_pages=2)
    for lengths in ([51], [-1], [1, 1, 1, 1]):
        with pytest.raises(ValueError, match="lengths"):
            m.reserve(lengths)
    with pytest.raises(ValueError, match="no sequence 3"):
        m.release([3])
    with pytest.raises(ValueError, match="kv_pages"):
        nw.LlamaDecoder(SHAPE, "dense", batch=1, cache_len=8, device="cpu", dtype=torch.float16, kv_cache="int8", kv_pages=3)
    with pytest.raises(AssertionError):
        _decoder(kv_block=24)
    plain = nw.LlamaDecoder(SHAPE, "dense", batch=1, cache_len=8, device="cpu", dtype=torch.float32)
    for call in (lambda: plain.reserve([1]), lambda: plain.release([0]), lambda: plain.generate(torch.zeros(1, 2, dtype=torch.int64), 2)):
        with pytest.raises(RuntimeError, match="paged"):
            call()
    with pytest.raises(ValueError, match="51 tokens"):
        m.prefill(torch.zeros(1, 51, dtype=torch.int64))
    with pytest.raises(RuntimeError, match="are free"):
        m.prefill(torch.zeros(1, 40, dtype=torch.int64))
    with pytest.raises(ValueError, match="uniform"):
        m.generate(torch.zeros(1, 4, dtype=torch.int64), 2, torch.zeros(1, 3))
