"""The 8-bit cache's operators inside a function that torch.compile takes apart: they run as they do without it, between the compiled pieces."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


@pytest.mark.filterwarnings("ignore")
@pytest.mark.parametrize("tokens", [4, 40])
def test_a_compiled_function_calls_them(tokens):
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")
    from mem_efficient_blr_b200 import ops
    x = torch.randn(tokens, 128, generator=torch.Generator().manual_seed(2)).half().to(DEV)
    tab, start = torch.ones(64, 32, device=DEV), torch.zeros(1, dtype=torch.int64, device=DEV)
    ids = torch.arange(tokens, device=DEV)

    def step(x, cache):
        q = ops.rope_append_q8(x * 2, x, x, tab, tab, start, cache, start + tokens)
        a = ops.attention_q8(q, cache, start, None, 0.5)
        k, v = ops.cache_read_q8(cache, torch.float16, start + tokens)
        return a * 2, k + v, ops.token_logprobs(a + 1, ids, 2)

    make = lambda: ops.q8_cache(1, 2, 64, 64, device=DEV)   # noqa: E731
    want = step(x, make())
    torch._dynamo.reset()
    compiled = torch.compile(step, backend="eager")
    for _ in range(2):
        got = compiled(x, make())
        for a, b in zip((*want[:2], *want[2]), (*got[:2], *got[2])):
            assert torch.equal(a, b)
