"""The projection with a 4-bit weight on sums that are exact in FP32 whatever their order: small integers in x (times a power of two of each row's own), block scales of 1/2, 1 and 2. A product is a
multiple of 1/4 (in the row's unit) and at most 48; a row of 12,736 sums to at most 2.4 million quarters, less than 2^24. So a logit has one rounding, to BF16, and is compared bit for bit, at vocabularies
where a block has full passes of several tiles, tiles left over, or both."""
import pytest
import torch

import lithos_metal_b200 as lm

pytestmark = pytest.mark.gpu

E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
G = 0.125


def make_weight(gen, vocab, hidden, g=G):
    """An Nvfp4Weight and its values over g in binary64 (by a table, without the framework)."""
    codes = torch.randint(0, 256, (vocab, hidden // 2), dtype=torch.uint8, device="cuda", generator=gen)
    powers = torch.randint(0, 3, (vocab, hidden // 16), device="cuda", generator=gen)
    scales = (0x30 + 8 * powers).to(torch.uint8)                              # e4m3 of 1/2, 1, 2
    table = torch.tensor(E2M1 + tuple(-v for v in E2M1), dtype=torch.float64, device="cuda")
    values = torch.stack((table[(codes & 15).long()], table[(codes >> 4).long()]), dim=-1).view(vocab, hidden // 16, 16)
    values = (values * torch.ldexp(torch.ones_like(powers, dtype=torch.float64), powers - 1).unsqueeze(-1)).view(vocab, hidden)
    return lm.Nvfp4Weight(codes, scales, torch.full((1,), g, device="cuda")), values


def make_x(gen, rows, hidden, low, high):
    """Integers of -4 .. 4 times 2^low .. 2^high, another power for every row."""
    e = torch.randint(low, high + 1, (rows, 1), device="cuda", generator=gen)
    whole = torch.randint(-4, 5, (rows, hidden), device="cuda", generator=gen)
    return torch.ldexp(whole.double(), e).bfloat16()


def rounded(values):
    """binary64 values of at most 24 bits, rounded once to BF16."""
    assert torch.equal(values.float().double(), values)
    return values.float().bfloat16()


@pytest.mark.parametrize("rows", [17, 33, 70, 130, 256, 300])
@pytest.mark.parametrize("hidden,vocab", [(192, 200_003), (512, 45_001), (1024, 300)])
def test_every_row_by_its_own_factor(rows, hidden, vocab):
    gen = torch.Generator(device="cuda").manual_seed(rows + hidden)
    w, values = make_weight(gen, vocab, hidden)
    x = make_x(gen, rows, hidden, -50, 50)
    want = rounded((x.double() @ values.T) * G)
    for _ in range(3):
        assert torch.equal(lm.lm_head(x, w), want)


@pytest.mark.parametrize("rows", [1, 8, 16, 17, 40, 130, 256])
@pytest.mark.parametrize("hidden,vocab", [(192, 200_003), (512, 45_001), (1024, 300)])
def test_factors_beyond_the_ordinary_range(rows, hidden, vocab):
    """Logits that are scaled in binary64 because g times a row's power of two leaves the range where binary32 is safe: in every pass and for every accumulator of one."""
    gen = torch.Generator(device="cuda").manual_seed(rows + hidden + 1)
    g = 2.0 ** -100
    w, values = make_weight(gen, vocab, hidden, g)
    x = make_x(gen, rows, hidden, 0, 40)
    assert torch.equal(lm.lm_head(x, w), rounded((x.double() @ values.T) * g))


@pytest.mark.parametrize("rows", [1, 3, 8, 9, 16, 17, 70, 256])
@pytest.mark.parametrize("hidden", [64, 320, 4096, 6400, 12736])
@pytest.mark.parametrize("vocab", [300, 40_003])
def test_every_column_counts(rows, hidden, vocab):
    """Quarters of a row in four warps (few rows, the tiles left over), last steps that are not whole, x in as many pieces as the longest row has."""
    gen = torch.Generator(device="cuda").manual_seed(rows + hidden)
    w, values = make_weight(gen, vocab, hidden)
    x = make_x(gen, rows, hidden, -6, 6)
    assert torch.equal(lm.lm_head(x, w), rounded((x.double() @ values.T) * G))


@pytest.mark.parametrize("rows", [3, 8, 16, 17, 40, 130, 256, 300])
@pytest.mark.parametrize("hidden,vocab", [(192, 200_003), (512, 45_001), (1024, 300)])
def test_rows_that_are_done_over(rows, hidden, vocab):
    """Rows of x whose elements lie too far apart for binary16, or are infinite or NaN, in the middle of rows that are not: in every pass, for every tile of one, behind full rounds. Their sums are
    binary64's (here exact: 2^16 down to 2^-32 are 48 bits), rounded to binary32 and then to BF16."""
    gen = torch.Generator(device="cuda").manual_seed(rows + hidden + 2)
    w, values = make_weight(gen, vocab, hidden)
    x = make_x(gen, rows, hidden, -6, 6)
    far = [0, rows // 2] if rows > 3 else [0]
    x[far] = 0.0
    x[far, 5] = 2.0 ** 10
    x[far, 140] = -(2.0 ** -30)
    x[1, 17] = float("inf")
    x[rows - 1, 33] = float("nan")
    got = lm.lm_head(x, w)
    exact = (x.double() @ values.T) * G
    want = exact.float().bfloat16()
    assert (values[:, 5] == 0).any() and (want[0][values[:, 5] == 0].abs() < 1e-6).all()          # (the small element is all that is left)
    assert torch.isnan(got[rows - 1]).all()
    assert torch.equal(torch.isnan(got), torch.isnan(want)) and torch.equal(got.nan_to_num(nan=1.0), want.nan_to_num(nan=1.0))
    alone = [r for r in range(rows) if r not in (*far, 1, rows - 1)]
    assert torch.equal(want[alone], rounded(exact[alone]))
