"""A decoder's cache of 16-bit values and tokens that do not fit it: refused where the host can see it, left out where only the device can."""
import pytest
import torch


def _decoder(device, dtype, **kw):
    from mem_efficient_blr_b200 import networks as nw
    shape = nw.LlamaShape(layers=1, d=128, heads=2, ffn=128, vocab=32, b=4, rank_attn=16, rank_mlp=16)
    return nw.LlamaDecoder(shape, "dense", batch=1, cache_len=8, device=device, dtype=dtype, **kw)


@pytest.mark.parametrize("cache", [None, "int8"])
def test_longer_texts_than_the_cache_are_refused(cache):
    m = _decoder("cpu", torch.float32 if cache is None else torch.float16, kv_cache=cache)
    ids = torch.zeros(1, 9, dtype=torch.int64)
    for call in (m.prefill, m.score, lambda x: m.decode_step(x, torch.zeros(1, dtype=torch.int64))):
        with pytest.raises(ValueError, match="9 tokens do not fit a cache of 8"):
            call(ids)
    if cache is None:
        assert m.prefill(ids[:, :8]).isfinite().all()


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_positions_outside_the_cache_write_nothing(dtype):
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")
    from mem_efficient_blr_b200 import ops
    dev, (B, H, slots, hd) = "cuda:0", (2, 3, 8, 64)
    x = torch.randn(3, B * 4, H * hd, generator=torch.Generator().manual_seed(1)).to(dtype).to(dev)
    cos, sin = torch.rand(2, slots, hd // 2, generator=torch.Generator().manual_seed(2)).to(dev)
    caches = torch.zeros(2, B, H, slots, hd, dtype=dtype, device=dev)
    sound = torch.zeros_like(caches)
    q = ops.rope_append(x[0].clone(), x[1], x[2], cos, sin, torch.tensor([3, slots, -1, 2 ** 40], device=dev), *caches, 4)
    first = [t.view(B, 4, -1)[:, 0].contiguous() for t in x]
    want = ops.rope_append(first[0], first[1], first[2], cos, sin, torch.tensor([3], device=dev), *sound, 1)
    assert torch.equal(caches, sound) and torch.equal(q.view(B, 4, -1)[:, 0], want) and torch.equal(q.view(B, 4, -1)[:, 1:], x[0].view(B, 4, -1)[:, 1:])
