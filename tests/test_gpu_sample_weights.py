"""Draws next to a border.  Rows of two tokens, 0 and the largest one, whose share of the whole lies within 2^-43.5 to 2^-40 (relative) of the row's uniform number: weights that are
exact to 2^-45 decide them as the definition does.  The wanted ids are those of 80-bit arithmetic."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = "cuda:0"

ROWS = [  # logit of token 0 (that of token 1 is 0), temperature, uniform number, id
    ("-0x1.5cbe92p+0", "0x1.7afadcp+0", "0x1.23c052p-2", 1),  # 2^-43.1
    ("-0x1.c27b00p-7", "0x1.48b6a0p+0", "0x1.fd4258p-2", 1),  # 2^-41.2
    ("-0x1.2df926p-1", "0x1.676bd0p+0", "0x1.96034cp-2", 1),  # 2^-42.2
    ("-0x1.bdf936p+0", "0x1.7f3458p-1", "0x1.6bfb56p-4", 1),  # 2^-40.3
    ("-0x1.4de176p-1", "0x1.04b536p+0", "0x1.617476p-2", 0),  # 2^-42.3
    ("-0x1.314b98p+0", "0x1.632e02p-1", "0x1.3744d0p-3", 1),  # 2^-42.2
    ("-0x1.db2ecap+0", "0x1.924ca0p+0", "0x1.e0f50cp-3", 0),  # 2^-41.7
    ("-0x1.1ffd5ap-2", "0x1.7c1370p-1", "0x1.a027f0p-2", 1),  # 2^-40.5
    ("-0x1.6925eep-2", "0x1.b74f6ap+0", "0x1.cb9240p-2", 1),  # 2^-41.5
    ("-0x1.d5c71cp+0", "0x1.e43c9ap-1", "0x1.014374p-3", 0),  # 2^-42.4
    ("-0x1.7b35dap-3", "0x1.622232p-1", "0x1.bbdfdap-2", 1),  # 2^-43.4
    ("-0x1.af6d66p+0", "0x1.ac2af0p+0", "0x1.11ddb2p-2", 0),  # 2^-40.5
    ("-0x1.69e9e4p-2", "0x1.8fb2c0p+0", "0x1.c64bdap-2", 1),  # 2^-41.6
    ("-0x1.8d36cep-3", "0x1.a559ccp+0", "0x1.e1de32p-2", 1),  # 2^-43.5
    ("-0x1.7893aap+0", "0x1.733e70p-1", "0x1.dc08c6p-4", 0),  # 2^-43.1
    ("-0x1.60c7aap-3", "0x1.40e8bcp+0", "0x1.dce090p-2", 1),  # 2^-43.5
    ("-0x1.1c4000p-6", "0x1.6481b8p+0", "0x1.fccf8ep-2", 0),  # 2^-43.2
    ("-0x1.0c7076p-1", "0x1.acaf72p+0", "0x1.b07ef0p-2", 1),  # 2^-43.3
    ("-0x1.f10b74p+0", "0x1.034eb6p+0", "0x1.0696a6p-3", 1),  # 2^-42.8
    ("-0x1.84d5b2p+0", "0x1.c3201ap-1", "0x1.360508p-3", 0),  # 2^-41.8
    ("-0x1.6203d4p-4", "0x1.bed752p-1", "0x1.e6ab18p-2", 0),  # 2^-42.7
    ("-0x1.9de008p-2", "0x1.9f4cf2p+0", "0x1.c08c2cp-2", 0),  # 2^-40.5
    ("-0x1.ac9f24p+0", "0x1.263890p-1", "0x1.a5c434p-5", 0),  # 2^-41.3
    ("-0x1.673930p-1", "0x1.eeb1f2p-1", "0x1.4ddd68p-2", 0),  # 2^-43.4
]


@pytest.mark.parametrize("vocab", [2, 1000, 40000])
def test_draws_next_to_a_border(vocab):
    from mem_efficient_blr_b200 import ops
    n = len(ROWS)
    number = lambda i: torch.tensor([float.fromhex(r[i]) for r in ROWS], dtype=torch.float64).float()   # noqa: E731
    x = torch.full((n, vocab), -torch.inf)
    x[:, vocab // 2 - 1], x[:, vocab - 1] = number(0), 0.0
    u, T = number(2), number(1)
    want = torch.tensor([(vocab - 1) if r[3] else vocab // 2 - 1 for r in ROWS])
    # the same border by the other settings that leave both tokens
    for k, p, mp in ((0, 1.0, 0.0), (2, 1.0, 0.0), (0, 1.0, 0.01), (2, 1 - 2.0 ** -24, 0.0)):
        ids, lp = (t.cpu() for t in ops.sample(x.to(DEV), u.to(DEV), T.to(DEV), k, p, mp))
        assert torch.equal(ids, want)
        w = torch.exp(number(0).double() / T.double())
        lp_want = torch.log(torch.where(want == vocab - 1, 1.0, w) / (1 + w))
        assert ((lp.double() - lp_want).abs() <= 2.0 ** -23 * lp_want.abs()).all()
