"""What the operators around the cache in pages and the choice of a token refuse, checked without a GPU: every check comes before the device is touched."""
import math

import pytest
import torch
import torch.autograd.forward_ad as fwd

ARG, SHAPE, UNSUPPORTED, WORKSPACE = -1, -2, -6, -4
P = 4096   # an aligned address that nothing reads


@pytest.fixture(scope="module")
def L():
    from mem_efficient_blr_b200 import build as b
    b.build()
    from mem_efficient_blr_b200 import _lib
    _lib.load()
    return _lib


def _desc(L, **kw):
    d = dict(k=P, v=P, k_strides=(2048, 1024, 64), v_strides=(2048, 1024, 64), table=P, ld_table=5, n_seq=2, pages=12, pages_per_seq=5, kv_heads=2, page=16, head_dim=64) | kw
    d["k_strides"], d["v_strides"] = ((L.C.c_int64 * 3)(*d[n]) for n in ("k_strides", "v_strides"))
    return L.PagedCacheDesc(*d.values())


def _append(L, desc, q=P, ldq=256, n_tok=1, heads=4, dtype=0, ldo=256, start=P, positions=80):
    return L.load().blr_rope_append_paged(q, ldq, P, 128, P, 128, P, P, positions, start, None, n_tok, heads, dtype, desc, P, ldo, None)


def _attend(L, desc, q=P, ldq=256, n_tok=1, heads=4, dtype=0, out=P, scratch=P, nbytes=1 << 30, start=P, scale=1.0):
    return L.load().blr_attention_paged(q, ldq, desc, start, None, n_tok, heads, scale, dtype, out, 256, scratch, nbytes, None, None)


@pytest.mark.parametrize("bad", [dict(head_dim=96), dict(head_dim=256), dict(page=8), dict(page=48), dict(page=256), dict(kv_heads=0), dict(pages_per_seq=0), dict(n_seq=-1),
                                 dict(pages=-1), dict(k=None), dict(table=None), dict(v=P + 8), dict(table=P + 2), dict(k_strides=(0, 1024, 64)), dict(v_strides=(2048, 1024, 60)),
                                 dict(k_strides=(2048, -1024, 64)), dict(ld_table=4), dict(pages_per_seq=1 << 28)])
def test_caches_that_are_none(L, bad):
    d = _desc(L, **bad)
    assert _append(L, d) < 0 and _attend(L, d) < 0
    assert L.load().blr_last_error()


def test_arguments_of_the_cache_operators(L):
    d, lib = _desc(L), L.load()
    assert _append(L, d, dtype=2) == ARG and _attend(L, d, dtype=2) == ARG
    assert _append(L, d, q=None) == ARG and _attend(L, d, q=None) == ARG and _attend(L, d, start=None) == ARG and _append(L, d, start=None) == ARG
    assert _append(L, d, q=P + 8) == ARG and _attend(L, d, out=P + 8) == ARG
    assert _append(L, d, ldq=252) == ARG and _append(L, d, ldo=252) == ARG and _attend(L, d, ldq=252) == ARG
    assert _append(L, d, n_tok=-1) == ARG and _append(L, d, heads=0) == ARG and _append(L, d, positions=-1) == ARG
    assert _attend(L, d, heads=3) == ARG and _attend(L, d, heads=0) == ARG and _attend(L, d, n_tok=-1) == SHAPE
    assert all(_attend(L, d, scale=s) == ARG for s in (0.0, -1.0, float("inf"), float("nan")))
    wide = _desc(L, n_seq=1, kv_heads=1, pages_per_seq=10000, head_dim=128)
    need = lib.blr_attention_paged_scratch_bytes(wide, 1, 1)
    assert need > 0 and _attend(L, wide, heads=1, nbytes=need - 1) == WORKSPACE and _attend(L, wide, heads=1, scratch=None) == WORKSPACE
    # nothing to do: no launch, no pointer looked at
    none = _desc(L, n_seq=0, k=None, v=None, table=None)
    assert _append(L, none, q=None) == 0 and _attend(L, none, q=None) == 0
    assert _append(L, d, n_tok=0, q=None) == 0 and _attend(L, d, n_tok=0, q=None) == 0


def test_arguments_of_the_choice(L):
    f = L.load().blr_sample

    def call(logits=P, ld=100, rows=2, vocab=100, kind=0, u=P, ids=P, **kw):
        s = dict(temperature=None, top_k=None, top_p=None, min_p=None, top_k_all=0, temperature_all=1.0, top_p_all=1.0, min_p_all=0.0) | kw
        return f(logits, ld, rows, vocab, kind, u, L.Sampling(*s.values()), ids, P, None)

    assert call(kind=3) == ARG and call(ld=99) == ARG and call(vocab=0) == ARG and call(rows=-1) == ARG
    assert call(vocab=2097153, ld=2097153) == UNSUPPORTED and call(vocab=1048577, ld=1048577, kind=2) == UNSUPPORTED and call(logits=P + 1) == ARG
    assert call(logits=None) == ARG and call(ids=None) == ARG and call(u=None) == ARG and f(P, 100, 2, 100, 0, P, None, P, P, None) == ARG
    assert call(temperature_all=-1.0) == ARG and call(temperature_all=math.nan) == ARG and call(top_p_all=math.nan) == ARG and call(min_p_all=math.nan) == ARG
    assert call(rows=0, logits=None) == 0


def _calls(device):
    from mem_efficient_blr_b200 import ops
    cache = ops.paged_cache(1, 2, 2, 2, 64, device=device)
    start, tab = torch.zeros(1, dtype=torch.int64, device=device), torch.zeros(32, 32, device=device)
    u = torch.zeros(1, device=device)
    return {
        "append": lambda x: ops.rope_append_paged(x, x, x, tab, tab, start, cache),
        "append v": lambda x: ops.rope_append_paged(x.detach().clone(), x.detach().clone(), x, tab, tab, start, cache),
        "attention": lambda x: ops.attention_paged(x, cache, start),
        "sample": lambda x: ops.sample(x, u, 0.9)[1],
    }


CALLS = ["append", "append v", "attention", "sample"]


def _x(device):
    return torch.randn(1, 128, generator=torch.Generator().manual_seed(1)).half().to(device)


def _recorded(call, device):
    from torch.fx.experimental.proxy_tensor import make_fx
    with pytest.raises(RuntimeError, match="record"):
        torch.jit.trace(call, (_x(device),), check_trace=False)
    with pytest.raises(RuntimeError, match="record"):
        make_fx(call)(_x(device))


def _derived(call, device):
    with pytest.raises(RuntimeError, match="no derivative"):
        call(_x(device).requires_grad_(True))
    with fwd.dual_level():
        x = fwd.make_dual(_x(device), torch.ones(1, 128, dtype=torch.float16, device=device))
        with torch.no_grad(), pytest.raises(RuntimeError, match="no derivative"):   # (forward mode has a switch of its own)
            call(x)


@pytest.mark.parametrize("name", CALLS)
def test_what_records_or_derives_is_refused(name):
    _recorded(_calls("cpu")[name], "cpu")
    _derived(_calls("cpu")[name], "cpu")
    with pytest.raises(RuntimeError, match="no CPU implementation"):
        _calls("cpu")[name](_x("cpu"))


@pytest.mark.gpu
@pytest.mark.parametrize("name", CALLS)
def test_on_the_device(name):
    call = _calls("cuda:0")[name]
    want = call(_x("cuda:0"))
    _recorded(call, "cuda:0")
    _derived(call, "cuda:0")
    with torch.no_grad():
        assert torch.equal(call(_x("cuda:0").requires_grad_(True)), want)


@pytest.mark.gpu
@pytest.mark.filterwarnings("ignore")
@pytest.mark.parametrize("tokens", [4, 40])
def test_a_compiled_function_calls_them(tokens):
    """Inside a function that torch.compile takes apart they run as they do without it, between the compiled pieces."""
    from mem_efficient_blr_b200 import ops
    dev = "cuda:0"
    x = torch.randn(tokens, 128, generator=torch.Generator().manual_seed(2)).half().to(dev)
    tab, start, u = torch.ones(64, 32, device=dev), torch.zeros(1, dtype=torch.int64, device=dev), torch.linspace(0, 0.99, tokens, device=dev)

    def step(x, cache):
        q = ops.rope_append_paged(x * 2, x, x, tab, tab, start, cache, start + tokens)
        a = ops.attention_paged(q, cache, start, None, 0.5)
        return (a * 2, *ops.sample(a + 1, u, u + 0.1, 30, 0.9))

    def make():
        c = ops.paged_cache(1, 2, 4, 4, 64, device=dev)
        c.table.copy_(torch.tensor([[2, 0, 3, 1]]))
        return c

    want = step(x, make())
    torch._dynamo.reset()
    compiled = torch.compile(step, backend="eager")
    for _ in range(2):
        for a, b in zip(want, compiled(x, make())):
            assert torch.equal(a, b)


def test_the_python_layer_refuses_caches_that_are_none():
    from mem_efficient_blr_b200 import ops
    for bad in (dict(head_dim=96), dict(page=24), dict(dtype=torch.float32)):
        with pytest.raises(AssertionError):
            ops.paged_cache(**(dict(n_seq=1, kv_heads=1, pages=2, pages_per_seq=2, head_dim=64, device="cpu") | bad))
