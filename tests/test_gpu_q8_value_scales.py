"""Value scales of very different size in one 8-bit cache.  A row's result is a matter of the keys that it sees: what later tokens bring changes no bit of it.
And what a row loses is measured by its own largest weighted value, not by the largest value in sight."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
I8, E4 = torch.int8, torch.float8_e4m3fn
TOP = {I8: 127.0, E4: 448.0}


@pytest.fixture(scope="module")
def ops():
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")
    from mem_efficient_blr_b200 import ops as o
    return o


def _parts(KV, slots, hd, block, code, g):
    nb = -(-slots // block)
    codes = lambda: (torch.randn(1, KV, slots, hd, generator=g) * (TOP[code] / 4)).round().clamp(-TOP[code], TOP[code]).to(code)   # noqa: E731
    scale = lambda: (torch.rand(1, KV, nb, generator=g) + 0.5) * 4 / TOP[code]   # noqa: E731
    return [codes(), codes(), scale(), scale()]


def _call(ops, q, parts, block, start, **kw):
    T, H, hd = q.shape
    out = ops.attention_q8(q.reshape(T, H * hd).to(DEV), ops.Q8Cache(*(t.to(DEV) for t in parts), block), torch.tensor([start], device=DEV), **kw)
    return out.view(T, H, hd)


def _check(got, q, parts, block, start, rows=None):
    """Against 64 bits, the given rows (None: all).  Allowed: the output's rounding; of each weight half a step of fp16 (2^-11) and 2^-15 for its exponent and the sums;
    half a step of fp16's smallest number (2^-25) of a weight whose largest, weighted with its block's scale, is held at 2^2 at least, so 2^-27 of that one times
    the largest code for each key; fp32 sums of products, 2^-23 for each step of 16 keys."""
    T, H, hd = q.shape
    KV, slots = parts[0].shape[1:3]
    dev = DEV
    k, v = ((c.to(dev).float().double() * s.to(dev).double().repeat_interleave(block, -1)[..., :slots, None])[0] for c, s in ((parts[0], parts[2]), (parts[1], parts[3])))
    room_of = parts[3].to(dev).double().repeat_interleave(block, -1)[0, :, :slots] * TOP[parts[0].dtype]
    rows = torch.arange(T) if rows is None else rows
    seen = (rows.to(dev) + start + 1).clamp(0, slots)
    half = torch.finfo(q.dtype).eps / 2
    tiny = torch.finfo(q.dtype).smallest_normal * torch.finfo(q.dtype).eps
    for h in range(H):
        kh, vh, most = k[h // (H // KV)], v[h // (H // KV)], room_of[h // (H // KV)]
        x = (q[rows, h].to(dev).double() @ kh.T * hd ** -0.5).masked_fill(torch.arange(slots, device=dev) >= seen[:, None], -torch.inf)
        p = (x - x.amax(1, keepdim=True)).exp()
        l = p.sum(1, keepdim=True)
        want, size = p @ vh / l, p @ vh.abs() / l
        heaviest = (p * most).amax(1, keepdim=True) / l
        room = (2.0 ** -11 + 2.0 ** -15 + (seen[:, None] / 16 + 16) * 2.0 ** -23) * size + seen[:, None] * 2.0 ** -27 * heaviest
        off = (got[rows, h].double() - want).abs()
        assert (off <= half * want.abs() * 1.001 + room + tiny).all(), float((off / (half * want.abs() + room + tiny)).max())


# Rows of a kv head: 8, 20 and 32 (mma.sync), 70 and 300 (tcgen05), 10400 (the same, codes widened ahead)
LATER = [(5, 2, 2, 128, 16), (5, 8, 2, 64, 16), (16, 2, 1, 128, 16), (70, 2, 2, 128, 16), (150, 4, 2, 64, 32), (2600, 4, 1, 64, 16), (2600, 4, 1, 128, 64)]


@pytest.mark.parametrize("code,dtype", [(I8, torch.bfloat16), (E4, torch.float16)], ids=["int8", "e4m3"])
@pytest.mark.parametrize("T,H,KV,hd,block", LATER, ids=[f"{c[0]}x{c[1]}on{c[2]}-{c[3]}" for c in LATER])
def test_later_values_change_nothing_in_earlier_rows(ops, T, H, KV, hd, block, code, dtype):
    g = torch.Generator().manual_seed(T + hd)
    start = block - 3 if T < 40 else 0     # (few tokens: the first three sit in a block of their own)
    parts = _parts(KV, start + T, hd, block, code, g)
    q = (torch.randn(T, H, hd, generator=g) * 2).to(dtype)
    for first in {1 if T < 40 else 2, parts[3].shape[2] - 1}:   # the first block that grows
        before = max(0, first * block - start)                   # rows that do not see it
        sound = _call(ops, q, parts, block, start)
        _check(sound, q, parts, block, start, torch.arange(before))
        for by in (2.0 ** 10, 2.0 ** 20, 2.0 ** 30, 1e30):
            grown = [t.clone() for t in parts]
            grown[3][:, :, first:] *= by
            got = _call(ops, q, grown, block, start)
            assert torch.equal(got[:before], sound[:before])
            if by < 1e30 and dtype == torch.bfloat16:
                _check(got, q, grown, block, start, torch.arange(0, T, max(1, T // 64)))


@pytest.mark.parametrize("code", [I8, E4], ids=["int8", "e4m3"])
@pytest.mark.parametrize("where", [0, 3, -2])
@pytest.mark.parametrize("T,H,KV,hd,slots", [(1, 2, 2, 128, 300), (1, 4, 1, 64, 5000), (5, 4, 2, 128, 700), (8, 4, 1, 128, 400), (60, 4, 2, 64, 900), (40, 4, 2, 128, 3000), (2600, 4, 1, 128, 2700)])
def test_a_block_of_large_values_and_little_weight(ops, T, H, KV, hd, slots, where, code):
    """Rows of q are positive, the keys of one block as negative as they get: its weights are some 2^-30 to 2^-60, its values 2^10 to 2^50 times the others'.  With the
    largest of these factors the block decides the result, with the smallest it has no part in it."""
    g = torch.Generator().manual_seed(slots)
    block = 16
    parts = _parts(KV, slots, hd, block, code, g)
    q = torch.randn(T, H, hd, generator=g).abs().bfloat16()
    at = where if where >= 0 else (slots - T) // block + where
    parts[0][:, :, at * block:(at + 1) * block] = torch.full((), -TOP[code]).to(code)
    parts[2][:, :, at] = 3.0 / TOP[code] * (1 if hd == 128 else 1.4)
    for by in (2.0 ** 10, 2.0 ** 25, 2.0 ** 40, 2.0 ** 50):
        grown = [t.clone() for t in parts]
        grown[3][:, :, at] *= by
        got = _call(ops, q, grown, block, slots - T)
        _check(got, q, grown, block, slots - T, torch.arange(0, T, max(1, T // 64)))


@pytest.mark.parametrize("T", [1, 6, 50])
def test_sizes_at_the_ends_of_fp32(ops, T):
    """Blocks without values ahead of ordinary ones, values of 1e-35 and of 1e34 beside each other."""
    g = torch.Generator().manual_seed(T)
    H, KV, hd, slots, block = 4, 2, 64, 640, 16
    q = torch.randn(T, H, hd, generator=g).bfloat16()
    for lead, rest in ((0.0, 1.0), (1e-35, 1.0), (1e34, 1.0), (1.0, 1e-35), (1.0, 1e34), (1e-35, 1e-35), (0.0, 1e-35), (1e-35, 1e34)):
        parts = _parts(KV, slots, hd, block, I8, g)
        parts[3][:, :, :20] *= lead
        parts[3][:, :, 20:] *= rest
        _check(_call(ops, q, parts, block, slots - T), q, parts, block, slots - T)
