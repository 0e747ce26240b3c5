"""Views whose memory is not what they show, handed to the 8-bit cache's operators."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def test_lazily_negated_views():
    """A view that is negated only where it is read (the imaginary part of a conjugate) holds the other sign in memory."""
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")
    from mem_efficient_blr_b200 import ops
    x = torch.randn(4, 128, generator=torch.Generator().manual_seed(1)).to(DEV).half()
    neg, plain = torch._neg_view(x), (-x).contiguous()
    tab, start = torch.ones(8, 32, device=DEV), torch.zeros(1, dtype=torch.int64, device=DEV)
    for a, b in ((neg, plain), (plain, neg)):
        c, d = (ops.q8_cache(1, 2, 8, 64, device=DEV) for _ in range(2))
        assert torch.equal(ops.rope_append_q8(a, b, a, tab, tab, start, c), ops.rope_append_q8(plain, plain, plain, tab, tab, start, d))
        assert all(torch.equal(s, t) for s, t in zip(c[:4], d[:4]))
        assert torch.equal(ops.attention_q8(a, c, start), ops.attention_q8(plain, d, start))
        for s, t in zip(ops.token_logprobs(a, start.expand(4), 3), ops.token_logprobs(plain, start.expand(4).contiguous(), 3)):
            assert torch.equal(s, t)
    with pytest.raises(AssertionError, match="negated"):
        ops.attention_q8(plain, ops.q8_cache(1, 2, 8, 64, device=DEV)._replace(k_scale=torch._neg_view(torch.zeros(1, 2, 1, device=DEV))), start)
