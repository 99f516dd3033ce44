"""How exactly ``mx4_moe`` holds activations: as sums of eight MXFP4 terms.

A first term leaves at most its scale (5 lies between 4 and 6), and at most half of it where the block's largest value is
below 4.5 times the scale; each further one an eighth of that.  So n terms leave at most 8^(1 - n) / 4.5 of the largest value
(a fifth for n = 1), eight less than 2^-23, or 2^-129 (half the smallest code times the smallest scale) where that is more;
and what they leave of a value is a whole number of its last places, so a bf16 value of 2^-15 of the largest is exact.  Layers of selecting weights (0, 1 and -1 times powers of two, which MXFP4 holds exactly) let the difference of two
copies of a value through, one beside a value far larger and one not: in exact arithmetic the output is zero, here it is
what the terms leave, times known factors.  The gate is 24 for every token: 1 + exp(-24) is 1 in fp32, so silu(24) is 24.
"""
import pytest
import torch

from oracle import mx4 as ref

DEV = torch.device("cuda:0")
LEFT = 2.0 ** -23


def terms(v, count):
    """What `count` terms hold of v [..., 32], in 64 bits."""
    grid = torch.tensor(ref.E2M1, dtype=torch.float64)
    even = torch.arange(8) % 2 == 0
    left, held = v.double().clone(), torch.zeros(v.shape, dtype=torch.float64)
    for _ in range(count):
        mantissa, e = torch.frexp(left.abs().amax(-1, keepdim=True))           # mantissa in [0.5, 1)
        s = torch.exp2((e - 3 + (mantissa > 0.75)).clamp_min(-127).double())
        d = ((left / s).abs().unsqueeze(-1) - grid).abs()
        near = d == d.amin(-1, keepdim=True)
        code = torch.where(near.sum(-1) == 1, near.int().argmax(-1), (near & even).int().argmax(-1))
        q = grid[code] * torch.sign(left) * s
        held, left = held + q, left - q
    return held


def blocks(count, ratio, seed, size=1.0):
    """bf16 blocks of 32: the first value some `ratio` times the others, which lie between size / 4 and 2 size."""
    g = torch.Generator().manual_seed(seed)
    v = (1 + torch.rand(count, 32, generator=g)) * torch.where(torch.rand(count, 32, generator=g) < 0.5, -1.0, 1.0)
    v *= torch.exp2(-torch.randint(0, 3, (count, 32), generator=g).float())
    v[:, 0] = (v[:, 0].sign() * (1 + torch.rand(count, generator=g))) * ratio
    return (v * size).bfloat16()


RATIOS = [1, 2 ** 6, 1000, 2 ** 11, 2 ** 12, 2 ** 15]


@pytest.mark.parametrize("ratio", RATIOS)
def test_what_terms_leave(ratio):
    """The statement itself, and that fewer terms break it."""
    v = blocks(4000, ratio, ratio).double()
    top = v.abs().amax(-1, keepdim=True)
    left = (v - terms(v, 8)).abs()
    assert bool((left <= LEFT * top).all())
    exact = v.abs() >= top * 2.0 ** -15
    assert not left[exact].any()
    assert ratio > 2 ** 11 or bool(exact.all())
    for fewer, least in ((3, 1), (4, 2 ** 6), (6, 1000)):
        if least <= ratio <= 2 ** 12:
            assert bool((v - terms(v, fewer))[exact].any()), fewer
    # values of 24 bits, ties among them
    g = torch.Generator().manual_seed(ratio)
    w = torch.randn(4000, 32, generator=g)
    w[:, 1] = w[:, 0] * 5 / 6
    w[:, 2:6] = w[:, :1] * (4 + torch.rand(4000, 4, generator=g)) / 6
    w[:, 0] *= ratio
    top = w.double().abs().amax(-1, keepdim=True)
    for count in range(1, 9):
        most = 0.2 if count == 1 else 8.0 ** (1 - count) / 4.5
        left = (w - terms(w, count)).abs()
        assert bool((left <= most * top).all())
        assert ratio > 2 ** 12 or bool((left <= LEFT * top).all()) == (count == 8)


@pytest.mark.parametrize("exponent", [-100, -110, -117, -122, -126])
def test_what_terms_leave_of_tiny_values(exponent):
    v = blocks(2000, 4, 7, 2.0 ** exponent).double()
    left = (v - terms(v, 8)).abs()
    assert bool((left <= (LEFT * v.abs().amax(-1, keepdim=True)).clamp_min(2.0 ** -129)).all())


def selecting(rows, cols, ones):
    """An MXFP4 matrix [1, rows, cols] of the (row, column, value) triples."""
    from wisp_b200.mx4 import mx4_dequantize, mx4_quantize
    m = torch.zeros(1, rows, cols)
    for r, c, v in ones:
        m[0, r, c] = v
    q = mx4_quantize(m.to(DEV))
    assert torch.equal(mx4_dequantize(q, torch.float32).cpu(), m)              # held exactly
    return q


def run(x, w13, w2):
    from wisp_b200.mx4 import mx4_moe
    ids = torch.zeros(x.shape[0], 1, dtype=torch.int32, device=DEV)
    return mx4_moe(x.to(DEV), w13, w2, topk_weights=torch.ones(x.shape[0], 1, device=DEV), topk_ids=ids).double().cpu()


def gate(inter, column):
    return [(j, column, 24.0) for j in range(inter)]


@pytest.mark.gpu
@pytest.mark.parametrize("ratio", RATIOS)
def test_inputs(ratio):
    """x = [a block with a large value, the block without it, 1 0 0 ..]; u_j = x_j - x_(32 + j)."""
    big = blocks(64, ratio, ratio + 1)
    small = big.clone()
    small[:, 0] = 0
    one = torch.zeros(64, 32, dtype=torch.bfloat16)
    one[:, 0] = 1
    up = [(32 + j, j, 1.0) for j in range(1, 32)] + [(32 + j, 32 + j, -1.0) for j in range(1, 32)]
    out = run(torch.cat((big, small, one), 1), selecting(64, 96, gate(32, 64) + up),
              selecting(96, 32, [(j, j, 1.0) for j in range(32)]))
    top = big.double().abs().amax(-1, keepdim=True)
    exact = big.double().abs() >= top * 2.0 ** -15
    off = out[:, :32].abs()
    assert not off[exact].any()
    # what is left of x, carried by 24 and through terms and a rounding of its own
    assert bool((off <= 24 * LEFT * top * (1 + 2.0 ** -7)).all())


@pytest.mark.gpu
@pytest.mark.parametrize("ratio", [2.0 ** e for e in (0, 4, 7, 10, 13)])
def test_products_of_gate_and_up(ratio):
    """silu(g) u: a block with a large value, the same block without it; the output is their difference.  24 x_j has 10
    bits, so it is held exactly down to 2^-13 of the block's largest."""
    v = blocks(64, 1, int(ratio) + 2)
    one = torch.zeros(64, 32, dtype=torch.bfloat16)
    one[:, 0] = 1
    up = [(64, 0, ratio)] + [(64 + j, j, 1.0) for j in range(1, 32)] + [(96 + j, j, 1.0) for j in range(1, 32)]
    down = [(j, j, 1.0) for j in range(1, 32)] + [(j, 32 + j, -1.0) for j in range(1, 32)]
    out = run(torch.cat((v, one), 1), selecting(128, 64, gate(64, 32) + up), selecting(64, 64, down))
    a = 24 * v.double()
    top = torch.maximum(a.abs().amax(-1), ratio * a[:, 0].abs()).unsqueeze(-1)
    off = out[:, 1:32].abs()
    exact = a[:, 1:].abs() >= top * 2.0 ** -13
    assert not off[exact].any()
    assert ratio > 2 ** 9 or bool(exact.all())
    # what is left of either copy; the difference is rounded to bf16
    assert bool((off <= 2 * LEFT * top * (1 + 2.0 ** -7)).all())
    assert not out[:, 0].any() and not out[:, 32:].any()


@pytest.mark.gpu
@pytest.mark.parametrize("exponent", [-100, -110, -117, -122, -126])
def test_tiny_inputs(exponent):
    """Blocks near the smallest scale, brought back by weights of 2^100: u_j = 2^100 x_j."""
    v = blocks(64, 4, exponent + 200, 2.0 ** exponent)
    one = torch.zeros(64, 32, dtype=torch.bfloat16)
    one[:, 0] = 1
    up = [(32 + j, j, 2.0 ** 100) for j in range(32)]
    out = run(torch.cat((v, one), 1), selecting(64, 64, gate(32, 32) + up),
              selecting(64, 32, [(j, j, 1.0) for j in range(32)]))[:, :32]
    want = 24 * 2.0 ** 100 * v.double()
    left = 24 * 2.0 ** 100 * (LEFT * v.double().abs().amax(-1, keepdim=True)).clamp_min(2.0 ** -129)
    bound = left + LEFT * want.abs().amax(-1, keepdim=True) + want.abs() * (2.0 ** -8 + 2.0 ** -20)
    assert bool(((out - want).abs() <= bound * (1 + 2.0 ** -8)).all())
    assert bool(want.abs().amax() > 0) and bool(out.any(-1).all())
