"""Append, attention and choice of the next token as a decoder uses them."""
import math

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

    def f(dtype=torch.float16, batch=3, cache_len=64, method="blast", **kw):
        return nw.LlamaDecoder(shape, method, batch=batch, cache_len=cache_len, device=DEV, dtype=dtype, seed=3, **kw)
    return f


def _ids(B, T, seed=1):
    return torch.randint(0, 384, (B, T), generator=torch.Generator().manual_seed(seed)).to(DEV)


def _at(*p):
    return torch.tensor(p, device=DEV)


def _rel(a, b):
    return float((a.double() - b.double()).norm() / b.double().norm())


@pytest.mark.parametrize("dtype,page", [(torch.float16, 16), (torch.bfloat16, 32)])
def test_decoder_on_pages(make, dtype, page):
    """Against the static cache's decoder (torch's attention), whole and in pieces.  Two layers of some ten roundings to 16 bits each, in both: within 30 half steps, relative to
    the logits' norm."""
    B, T = 3, 41
    tol = 30 * torch.finfo(dtype).eps / 2
    ids = _ids(B, T)
    m, slow, plain = make(dtype, kv_cache="paged", kv_block=page), make(dtype, kv_cache="paged", kv_block=page), make(dtype)
    slow.fused_decode = False
    a, c = m.prefill(ids[:, :T - 1]), plain.prefill(ids[:, :T - 1])
    assert _rel(a, c) < tol
    step = m.decode_step(ids[:, T - 1:], _at(T - 1))
    whole = make(dtype, cache_len=T).prefill(ids)
    assert _rel(step, whole) < tol
    # the same tokens in pieces, sequences at different positions and a padded batch, on pages that are given as they are needed
    n = _at(30, 17, 1)
    p = make(dtype, kv_cache="paged", kv_block=page, kv_pages=3 * -(-T // page) + 1)
    p.reserve([30, 17, 1])
    p.extend(ids[:, :30], torch.zeros(B, dtype=torch.int64, device=DEV), n)
    idx = (n[:, None] + torch.arange(T - 1, device=DEV)).clamp(max=T - 1)
    p.reserve([T] * 3)
    p.extend(ids.gather(1, idx), n, T - 1 - n)
    assert _rel(p.decode_step(ids[:, T - 1:], torch.full((B,), T - 1, device=DEV)), step) < tol
    slow.prefill(ids[:, :T - 1])
    assert _rel(slow.decode_step(ids[:, T - 1:], _at(T - 1)), step) < tol
    assert (plain.score(ids)[0] - m.score(ids)[0]).abs().mean() < 4 * tol   # (log probabilities of logits of size 1 or so, errors and their sum's: 4 times)


def test_tokens_without_a_place(make):
    m, ref = make(kv_cache="paged", kv_pages=5), make(kv_cache="paged")
    m.reserve([16, 32, 20])
    for d in (m, ref):
        d.extend(_ids(3, 10), _at(0, 0, 0))
    want = ref.extend(_ids(3, 8, 2), _at(10, 10, 10))
    got = m.extend(_ids(3, 8, 2), _at(10, 10, 10))          # slots 16 and 17 of the first sequence have no page
    assert got[0].isnan().all() and torch.equal(got[1:], want[1:])
    got = m.extend(_ids(3, 8, 2), _at(10, 60, 10), _at(6, 8, 8))   # six of them fit; beyond the last slot
    assert got[0].isfinite().all() and got[1].isnan().all() and torch.equal(got[2], want[2])
    assert m.decode_step(_ids(3, 1), _at(-1, 2 ** 62, 19))[:2].isnan().all()


def test_released_pages_serve_another_sequence(make):
    m, ref = make(kv_cache="paged", kv_pages=4), make(kv_cache="paged")
    m.reserve([64])
    m.extend(_ids(1, 60), _at(0))
    m.release([0])
    m.reserve([0, 0, 50])
    B3 = _ids(3, 50, 4)
    got = m.extend(B3, _at(0, 0, 0), _at(0, 0, 50))
    assert torch.equal(got[2], ref.extend(B3, _at(0, 0, 0), _at(0, 0, 50))[2])


def test_graphed_decode(make):
    from mem_efficient_blr_b200 import networks as nw
    ids = _ids(2, 40, 4)
    m = [make(batch=2, cache_len=48, method="blast_int8", kv_cache="paged") for _ in range(2)]
    for x in m:
        x.prefill(ids[:, :36])
    step = nw.GraphedCall(m[0].decode_step, ids[:, 36:37].clone(), _at(36))
    for i in range(36, 40):
        assert torch.equal(step(ids[:, i:i + 1], _at(i)), m[1].decode_step(ids[:, i:i + 1], _at(i)))


@pytest.mark.parametrize("kv", ["paged", "int8"])
def test_generate(make, kv):
    """Each token is the one that ops.sample takes from the logits of all tokens before it."""
    from mem_efficient_blr_b200 import ops
    B, T, N = 3, 9, 6
    ids, lens = _ids(B, T, 7), _at(9, 4, 1)
    u = torch.rand(B, N, generator=torch.Generator().manual_seed(2)).to(DEV)
    settings = (0.8, _at(40, 0, 5), torch.tensor([0.95, 0.9, 1.0], device=DEV), 0.01)
    m, ref = make(kv_cache=kv), make(kv_cache=kv)
    got, lp = m.generate(ids, N, u, *settings, n_new=lens)
    assert got.shape == lp.shape == (B, N) and (got >= 0).all() and (lp <= 0).all()
    logits, pos = ref.extend(ids, _at(0, 0, 0), lens), lens
    for i in range(N):
        token, p = ops.sample(logits, u[:, i].contiguous(), *settings)
        assert torch.equal(token, got[:, i]) and torch.equal(p, lp[:, i])
        logits = ref.decode_step(token[:, None], pos)
        pos = pos + 1
    greedy, glp = m.generate(ids, 3, None, 0.0, n_new=lens)
    assert (glp == 0).all()
    first = make(kv_cache=kv).extend(ids, _at(0, 0, 0), lens).float().argmax(-1)
    assert torch.equal(greedy[:, 0], first)
    assert m.generate(ids, 0)[0].shape == (B, 0)


def test_generate_past_the_end(make):
    """Sequences that fill the cache end there, the others go on."""
    m = make(cache_len=12, kv_cache="paged")
    ids = _ids(3, 9, 7)
    u = torch.rand(3, 8, generator=torch.Generator().manual_seed(2)).to(DEV)
    got, lp = m.generate(ids, 8, u, 1.0, 50, n_new=_at(9, 4, 1))
    # slots 9, 10, 11 take the first three tokens of the first sequence; the fourth, chosen from them, has no slot, and nothing follows it
    assert (got[0, :4] >= 0).all() and (got[0, 4:] == -1).all() and lp[0, 4:].isnan().all()
    assert (got[1:] >= 0).all() and not lp[1:].isnan().any()
    other = make(cache_len=32, kv_cache="paged").generate(ids, 8, u, 1.0, 50, n_new=_at(9, 4, 1))
    assert torch.equal(other[0][1:], got[1:]) and torch.equal(other[0][0, :4], got[0, :4])


def test_a_draw_from_the_whole_text(make):
    """Frequencies of the first token over many uniform numbers follow the model's own probabilities (token_logprobs)."""
    from mem_efficient_blr_b200 import ops
    m = make(batch=1, kv_cache="paged")
    logits = m.prefill(_ids(1, 5))
    n = 8192
    u = (torch.arange(n, device=DEV) + 0.5) / n     # an even grid: a token comes up its share of n, to one
    ids, lp = ops.sample(logits.expand(n, -1).contiguous(), u)
    seen = torch.bincount(ids, minlength=384)
    share = torch.softmax(logits[0].double(), 0) * n
    assert ((seen - share).abs() <= 1.001).all()
    want = ops.token_logprobs(logits.expand(n, -1).contiguous(), ids)[0]
    assert (lp - want).abs().max() <= 2.0 ** -19 * (1 + math.log(384))   # (the latter's fp32 sums)
