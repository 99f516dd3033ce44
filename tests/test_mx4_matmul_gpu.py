"""``mx4_matmul`` against the 64-bit oracle over the dequantised operands.

Tolerance, element by element: products of E2M1 values and powers of two are
exact, the fp32 accumulation adds at most one part in 2^23 of the magnitudes
that meet in an output for each of K / 32 + 32 additions (32 products meet in
one step of the unit), and the result is rounded to bf16 once (2^-8)."""
import pytest
import torch

from oracle import mx4 as ref

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")


def random_mx4(shape, seed, spread=3):
    """Codes of every value, scales that differ from block to block."""
    from wisp_b200.mx4 import Mx4Tensor
    g = torch.Generator(device=DEV).manual_seed(seed)
    codes = torch.randint(0, 256, (*shape[:-1], shape[-1] // 2), generator=g, device=DEV, dtype=torch.uint8)
    scales = torch.randint(127 - spread, 128 + spread, (*shape[:-1], shape[-1] // 32), generator=g, device=DEV,
                           dtype=torch.uint8)
    return Mx4Tensor(codes, scales)


def expected(a, w, offsets):
    av, wv = ref.values(a.codes, a.scales), ref.values(w.codes, w.scales)
    n = wv.shape[-2]
    out = torch.full((av.shape[0], n), float("nan"), dtype=torch.float64, device=DEV)
    size = torch.zeros_like(out)
    if offsets is None:
        wv, offsets = wv.reshape(1, n, -1), [0, av.shape[0]]
    for g, (p, q) in enumerate(zip(offsets[:-1], offsets[1:])):
        out[p:q], size[p:q] = av[p:q] @ wv[g].T, av[p:q].abs() @ wv[g].abs().T
    return out, size


def check(out, a, w, offsets=None):
    want, size = expected(a, w, offsets)
    k = a.shape[1]
    bound = want.abs() * 2.0 ** -8 + size * (k / 32 + 32) * 2.0 ** -23 * (1 + 2.0 ** -8)
    done = ~torch.isnan(want)
    off = (out.double() - want).abs()
    assert bool((off <= bound)[done].all()), float((off / bound)[done].max())
    return done


@pytest.mark.parametrize("m,n,k", [
    (128, 192, 256), (1, 192, 256), (128, 192, 64), (128, 192, 128), (1, 8, 32), (1, 1, 32), (16, 4096, 4096), (127, 191, 288), (129, 193, 544),
    (300, 1000, 2048), (5, 7, 96), (1000, 24, 1120), (64, 2048, 768), (2, 40000, 160),
])
def test_one_matrix(m, n, k):
    from wisp_b200.mx4 import mx4_matmul, mx4_synchronize
    a, w = random_mx4((m, k), m + k), random_mx4((n, k), n)
    out = mx4_matmul(a, w)
    mx4_synchronize()
    assert out.shape == (m, n) and bool(check(out, a, w).all())
    assert torch.equal(out, mx4_matmul(a, w))


@pytest.mark.parametrize("counts,n,k", [
    ([3, 0, 130, 1, 0, 0, 257], 200, 320), ([0, 0, 5], 64, 64), ([128, 128], 192, 256), ([0], 96, 128), ([1] * 70, 48, 96),
    ([40] * 128, 512, 512), ([0] * 1000 + [7] + [0] * 23, 16, 32),
])
@pytest.mark.parametrize("rest", [0, 3])
def test_groups(counts, n, k, rest):
    """Ragged and empty groups; rows behind the last group stay as they were."""
    from wisp_b200.mx4 import mx4_matmul, mx4_synchronize
    m = sum(counts) + rest
    a, w = random_mx4((max(m, 1), k), 1)[:m], random_mx4((len(counts), n, k), 2)
    offsets = [0]
    for c in counts:
        offsets.append(offsets[-1] + c)
    out = torch.full((m, n), 7.0, dtype=torch.bfloat16, device=DEV)
    mx4_matmul(a, w, torch.tensor(offsets, dtype=torch.int32, device=DEV), out=out)
    mx4_synchronize()
    if m:
        done = check(out, a, w, offsets)
        assert bool((out[~done] == 7.0).all()) and int((~done).sum()) == rest * n


def moved(q, offset):
    """The same matrix with its scale bytes `offset` bytes behind a 256-byte boundary, between bytes of another value."""
    from wisp_b200.mx4 import Mx4Tensor
    n = q.scales.numel()
    buffer = torch.full((n + 512,), 255, dtype=torch.uint8, device=DEV)
    scales = buffer[256 + offset:256 + offset + n].view(q.scales.shape)
    scales.copy_(q.scales)
    return Mx4Tensor(q.codes, scales)


@pytest.mark.parametrize("k", [32, 96, 256, 288, 1120, 2048])
@pytest.mark.parametrize("offset", [1, 2, 3, 4, 7, 8, 16])
def test_scale_rows_of_any_alignment(k, offset):
    from wisp_b200.mx4 import mx4_matmul, mx4_synchronize
    a, w = random_mx4((150, k), 3), random_mx4((210, k), 4)
    want = mx4_matmul(a, w)
    check(want, a, w)
    for x, y in ((moved(a, offset), w), (a, moved(w, offset)), (moved(a, offset), moved(w, 3))):
        assert torch.equal(mx4_matmul(x, y), want)
    mx4_synchronize()


@pytest.mark.parametrize("n,k", [(500, 672), (64, 32), (1000, 2048)])
def test_bits_do_not_depend_on_the_rows_beside(n, k):
    """Few rows go through narrow tiles, many through wide ones: the same sums in the same order."""
    from wisp_b200.mx4 import mx4_matmul
    a, w = random_mx4((20000, k), 5), random_mx4((n, k), 6)
    few, many = mx4_matmul(a[300:333], w), mx4_matmul(a, w)
    assert torch.equal(few, many[300:333])


def test_special_scales():
    """Scales at both ends, a NaN scale in one row of each operand, rows of zeros."""
    from wisp_b200.mx4 import mx4_matmul
    a, w = random_mx4((40, 256), 5), random_mx4((56, 256), 6)
    a.scales[0], a.scales[1] = 1, 250
    a.codes[2] = 0
    a.scales[3, 2] = 255
    w.scales[5, 7] = 255
    w.scales[6] = 0
    out = mx4_matmul(a, w).double()
    want, size = expected(a, w, None)
    nan = torch.isnan(want)
    assert bool(torch.isnan(out[3]).all()) and bool(torch.isnan(out[:, 5]).all())
    assert torch.equal(torch.isnan(out), nan)
    tiny = 2.0 ** -125                                  # what fp32 sums of subnormal products may lose
    bound = want.abs() * 2.0 ** -8 + size * 40 * 2.0 ** -23 + tiny
    # a partial sum is at most `size`, so below 2^127 it is finite in fp32 and the result in bf16; above, either may
    # pass the types' largest value (2^128), and an infinity is the right rounding
    fits = (size < 2.0 ** 127) & ~nan
    assert bool(((out - want).abs() <= bound)[fits].all()) and not out[2, :5].any()
    assert bool(((out - want).abs() <= bound)[~nan & ~fits].logical_or(~torch.isfinite(out[~nan & ~fits])).all())
    assert int((~fits & ~nan).sum()) < 56 and int(torch.isinf(out[1]).sum()) > 0


def test_quantised_layer_matches_float_layer():
    """quantise -> product, as a layer uses them: the error of the product is the quantisation's alone."""
    from wisp_b200.mx4 import mx4_matmul, mx4_quantize
    g = torch.Generator(device=DEV).manual_seed(0)
    x = torch.randn(70, 512, generator=g, device=DEV).bfloat16()
    w = (torch.randn(300, 512, generator=g, device=DEV) * 0.05).bfloat16()
    qx, qw = mx4_quantize(x), mx4_quantize(w)
    out = mx4_matmul(qx, qw)
    check(out, qx, qw)
    want = x.double() @ w.double().T
    assert float((out.double() - want).norm() / want.norm()) < 0.25


def test_out_of_order_offsets_stay_in_bounds():
    """Offsets that descend or point outside the matrix give empty or shorter groups."""
    from wisp_b200.mx4 import mx4_matmul, mx4_synchronize
    a, w = random_mx4((100, 64), 1), random_mx4((4, 32, 64), 2)
    out = torch.full((100, 32), 7.0, dtype=torch.bfloat16, device=DEV)
    mx4_matmul(a, w, torch.tensor([-5, 40, 20, 20, 1000], dtype=torch.int32, device=DEV), out=out)
    mx4_synchronize()
    # rows 0 .. 40 of group 0, group 1 empty, group 2 empty, group 3 rows 20 .. 100 (written by two groups: 20 .. 40)
    one, _ = expected(a, w[0], None)
    four, _ = expected(a, w[3], None)
    for rows, want in ((slice(0, 20), one), (slice(40, 100), four)):
        assert float((out[rows].double() - want[rows]).norm() / want[rows].norm()) < 1e-2


def test_graph_and_streams():
    from wisp_b200.mx4 import mx4_matmul
    a, w = random_mx4((200, 256), 1), random_mx4((3, 100, 256), 2)
    offsets = torch.tensor([0, 50, 50, 200], dtype=torch.int32, device=DEV)
    out = torch.empty(200, 100, dtype=torch.bfloat16, device=DEV)
    mx4_matmul(a, w, offsets)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        mx4_matmul(a, w, offsets, out=out)
    a.codes.copy_(a.codes.flip(0))
    offsets.copy_(torch.tensor([0, 10, 150, 200], dtype=torch.int32))
    graph.replay()
    torch.cuda.synchronize()
    check(out, a, w, [0, 10, 150, 200])
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        other = mx4_matmul(a, w, offsets)
    side.synchronize()
    assert torch.equal(out, other)
