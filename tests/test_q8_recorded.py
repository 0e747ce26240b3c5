"""The operators around the 8-bit cache write into buffers that a recording of torch operators does not see: under a tracer they refuse, where a replay of
what was recorded would give back memory that nobody wrote.  So they do for tensors that carry a tangent, which would be lost."""
import pytest
import torch
import torch.autograd.forward_ad as fwd

CPU = "cpu"


def _calls(device):
    from mem_efficient_blr_b200 import ops
    cache = ops.q8_cache(1, 2, 32, 64, device=device)
    start, tab = torch.zeros(1, dtype=torch.int64, device=device), torch.zeros(32, 32, device=device)
    return {
        "append": lambda x: ops.rope_append_q8(x, x, x, tab, tab, start, cache),
        "append k": lambda x: ops.rope_append_q8(x.detach().clone(), x, x.detach().clone(), tab, tab, start, cache),
        "attention": lambda x: ops.attention_q8(x, cache, start),
        "read": lambda x: ops.cache_read_q8(cache, torch.float16, start)[0] + x[0, 0],
        "logprobs": lambda x: ops.token_logprobs(x, start)[0],
    }


CALLS = ["append", "append k", "attention", "read", "logprobs"]


def _x(device):
    return torch.randn(1, 128, generator=torch.Generator().manual_seed(1)).half().to(device)


def _trace(call, device):
    with pytest.raises(RuntimeError, match="record"):
        torch.jit.trace(call, (_x(device),), check_trace=False)


def _make_fx(call, device):
    from torch.fx.experimental.proxy_tensor import make_fx
    with pytest.raises(RuntimeError, match="record"):
        make_fx(call)(_x(device))


def _tangent(call, device):
    with fwd.dual_level():
        x = fwd.make_dual(_x(device), torch.ones(1, 128, dtype=torch.float16, device=device))
        with pytest.raises(RuntimeError, match="no derivative"):
            call(x)
        with torch.no_grad(), pytest.raises(RuntimeError, match="no derivative"):   # (forward mode has a switch of its own)
            call(x)


@pytest.mark.parametrize("name", CALLS)
@pytest.mark.parametrize("how", [_trace, _make_fx])
def test_what_records_is_refused(name, how):
    how(_calls(CPU)[name], CPU)


@pytest.mark.parametrize("name", [c for c in CALLS if c != "read"])
def test_a_tangent_is_refused(name):
    _tangent(_calls(CPU)[name], CPU)


@pytest.mark.gpu
@pytest.mark.parametrize("name", CALLS)
def test_on_the_device(name):
    call = _calls("cuda:0")[name]
    want = call(_x("cuda:0"))
    _trace(call, "cuda:0")
    _make_fx(call, "cuda:0")
    if name != "read":
        _tangent(call, "cuda:0")
        with fwd.dual_level():   # a level alone, or a tangent that the call does not see, is nothing to it
            fwd.make_dual(torch.ones(2, device="cuda:0"), torch.ones(2, device="cuda:0"))
            assert torch.equal(call(_x("cuda:0")), want)
    assert torch.equal(call(_x("cuda:0")), want)
