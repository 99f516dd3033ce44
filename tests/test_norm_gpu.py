"""``block_norm`` against the 64-bit oracle.

Tolerance: each output is rounded once (half a step, eps / 2 relative; the
smallest subnormal's half below that), and the fp32 arithmetic before it adds
a few fp32 steps of the values that meet in the sum: r' = residual + g z takes
one product chain of five roundings on |g z| and one on the sum; n multiplies
r' by a reciprocal root (its sum of squares over at most 16384 terms, pairwise
over threads and then in a row of at most 64: 100 roundings at the outside, each
2^-24 relative, halved by the root) and a weight.  So 2^-24 * 8 * (|r'| + |g z|)
for r', and for n 2^-24 * 64 * |n| plus r's error times n / r'.
"""
import pytest
import torch

from oracle.mx4 import block_norm as ref_norm

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
BF, HF, FP = torch.bfloat16, torch.float16, torch.float32


def inputs(rows, cols, dtype, rdtype, wdtype, post, gate, seed=0):
    g = torch.Generator().manual_seed(seed + rows * 7 + cols)
    y = (torch.randn(rows, cols, generator=g) * 0.3).to(dtype)
    r = (torch.randn(rows, cols, generator=g) * 2).to(rdtype)
    w = (1 + 0.1 * torch.randn(cols, generator=g)).to(wdtype)
    p = (1 + 0.1 * torch.randn(cols, generator=g)).to(wdtype) if post else None
    shape = {"none": None, "channel": (cols,), "token": (rows, 1), "full": (rows, cols)}[gate]
    gt = None if shape is None else torch.tanh(torch.randn(*shape, generator=g)).to(dtype)
    return y, r, w, p, gt


def compare(got, y, r, w, p, gt, scale, eps):
    n, rn = (t.cpu() for t in got)
    en, er = ref_norm(y, r, w, p, gt, scale, eps)
    gz = (er - r.double()).abs()
    u = 2.0 ** -24
    r32 = 8 * u * (er.abs() + gz)                        # r' before it is rounded
    rt, nt = torch.finfo(rn.dtype), torch.finfo(n.dtype)
    bound_r = r32 + er.abs() * rt.eps / 2 * (1 + 1e-3) + rt.smallest_normal * rt.eps
    assert bool(((rn.double() - er).abs() <= bound_r).all())
    factor = (en / er).abs().nan_to_num(0.0, 0.0, 0.0)
    n32 = 64 * u * en.abs() + r32 * factor
    bound_n = n32 + (en.abs() + n32) * nt.eps / 2 * (1 + 1e-3) + nt.smallest_normal * nt.eps
    assert bool(((n.double() - en).abs() <= bound_n).all())
    assert n.dtype == y.dtype and rn.dtype == r.dtype


def run(y, r, w, p, gt, scale=0.5, eps=1e-6):
    from wisp_b200.norm import block_norm
    d = [None if t is None else t.to(DEV) for t in (y, r, w, p, gt)]
    compare(block_norm(d[0], d[1], d[2], post_weight=d[3], gate=d[4], scale=scale, eps=eps), y, r, w, p, gt, scale, eps)


@pytest.mark.parametrize("gate", ["none", "channel", "token", "full"])
@pytest.mark.parametrize("post", [False, True])
@pytest.mark.parametrize("rows,cols", [(1, 2048), (7, 2050), (301, 4096), (1200, 63), (3, 1), (2, 16384), (5, 16383),
                                       (4, 8192), (3, 5122), (300, 5120), (300, 8192), (200, 12288)])
def test_matches_oracle(rows, cols, post, gate):
    run(*inputs(rows, cols, BF, BF, BF, post, gate))


@pytest.mark.parametrize("dtype,rdtype,wdtype", [(BF, FP, BF), (BF, BF, FP), (BF, FP, FP), (HF, HF, HF), (HF, FP, FP),
                                                 (HF, HF, FP), (HF, FP, HF), (FP, FP, FP)])
@pytest.mark.parametrize("cols", [2048, 2050, 4096, 4094, 4099, 16384])
def test_types(dtype, rdtype, wdtype, cols):
    run(*inputs(9, cols, dtype, rdtype, wdtype, True, "full"))


@pytest.mark.parametrize("dtype,rdtype,wdtype", [(BF, BF, BF), (HF, FP, HF), (FP, FP, FP)])
@pytest.mark.parametrize("gate,post", [("full", True), ("channel", False), ("token", True)])
@pytest.mark.parametrize("cols", [2, 5, 8, 9, 131, 255, 257, 513, 770, 1025, 2047, 2049, 2562, 3329, 4097, 8191, 8194, 11001,
                                  14001, 16383])
def test_widths(cols, gate, post, dtype, rdtype, wdtype):
    """Rows that begin anywhere in a 16-byte granule, of every length class."""
    run(*inputs(11, cols, dtype, rdtype, wdtype, post, gate))


@pytest.mark.parametrize("rows", [1, 3, 4, 5, 700, 20000])
@pytest.mark.parametrize("cols", [33, 301, 801, 1203])
def test_many_short_rows(rows, cols):
    run(*inputs(rows, cols, BF, BF, BF, True, "none"))


def test_outputs_leave_their_neighbours_alone():
    """Outputs in the middle of a buffer, each beginning at an odd value: nothing beside them changes."""
    from wisp_b200.norm import block_norm
    for cols in (7, 301, 2803):
        y, res = torch.randn(5, cols, device=DEV).bfloat16(), torch.randn(5, cols, device=DEV).bfloat16()
        w = torch.randn(cols, device=DEV).bfloat16()
        n = 5 * cols
        buffer = torch.full((2 * n + 64,), 7.0, dtype=torch.bfloat16, device=DEV)
        out, res_out = buffer[13:13 + n].view(5, cols), buffer[n + 29:2 * n + 29].view(5, cols)
        block_norm(y, res, w, out=out, residual_out=res_out)
        want, want_res = block_norm(y, res, w)
        assert torch.equal(out, want) and torch.equal(res_out, want_res)
        beside = torch.cat((buffer[:13], buffer[13 + n:n + 29], buffer[2 * n + 29:]))
        assert bool((beside == 7.0).all())


def test_zero_rows_and_row_of_zeros():
    from wisp_b200.norm import block_norm
    y, r, w, p, gt = inputs(4, 256, BF, BF, BF, True, "token")
    y[1], r[1], y[2] = 0, 0, 0
    run(y, r, w, p, gt)
    n, rn = block_norm(y[:0].to(DEV), r[:0].to(DEV), w.to(DEV))
    assert n.shape == rn.shape == (0, 256)


def test_strides_dims_and_unaligned():
    from wisp_b200.norm import block_norm
    y, r, w, p, gt = inputs(24, 512, BF, FP, BF, True, "full")
    big = [torch.zeros(24, 1040, dtype=t.dtype, device=DEV) for t in (y, r, gt)]
    for at in (8, 1):                                   # aligned to 16 bytes, and not
        views = [b[:, at:at + 512] for b in big]
        for v, t in zip(views, (y, r, gt)):
            v.copy_(t)
        got = block_norm(views[0], views[1], w.to(DEV), post_weight=p.to(DEV), gate=views[2], scale=0.5)
        compare(got, y, r, w, p, gt, 0.5, 1e-6)
    a = block_norm(y.view(2, 12, 512).to(DEV), r.view(2, 12, 512).to(DEV), w.to(DEV), gate=gt.view(2, 12, 512).to(DEV))
    b = block_norm(y.to(DEV), r.to(DEV), w.to(DEV), gate=gt.to(DEV))
    assert a[0].shape == (2, 12, 512) and all(torch.equal(s.view(24, 512), t) for s, t in zip(a, b))
    t3 = gt[:, :1].contiguous()
    c = block_norm(y.view(2, 12, 512).to(DEV), r.view(2, 12, 512).to(DEV), w.to(DEV), gate=t3.view(2, 12, 1).to(DEV))
    compare([s.view(24, 512) for s in c], y, r, w, None, t3, 1.0, 1e-6)
    t2 = gt.to(DEV)[:, 3:4]                             # a column of a wider matrix: strided token gate
    compare(block_norm(y.to(DEV), r.to(DEV), w.to(DEV), gate=t2), y, r, w, None, gt[:, 3:4], 1.0, 1e-6)
    v = block_norm(y[0].to(DEV), r[0].to(DEV), w.to(DEV))
    compare(v, y[0], r[0], w, None, None, 1.0, 1e-6)


@pytest.mark.parametrize("cols", [33, 301, 1147, 2803, 4104, 6144, 7168])
def test_in_place_rows_of_any_width(cols):
    """Rows share 16-byte granules with their neighbours, which other CTAs overwrite."""
    from wisp_b200.norm import block_norm
    y, r, w, p, gt = (None if t is None else t.to(DEV) for t in inputs(3000, cols, BF, BF, BF, True, "full"))
    n, rn = block_norm(y, r, w, post_weight=p, gate=gt)
    n2, rn2 = block_norm(y, r, w, post_weight=p, gate=gt, out=y, residual_out=r)
    assert n2.data_ptr() == y.data_ptr() and torch.equal(n2, n) and torch.equal(rn2, rn)


def test_in_place_and_deterministic():
    from wisp_b200.norm import block_norm
    y, r, w, p, gt = (None if t is None else t.to(DEV) for t in inputs(3000, 2048, BF, BF, BF, True, "channel"))
    n1, r1 = block_norm(y, r, w, post_weight=p, gate=gt)
    n2, r2 = block_norm(y, r, w, post_weight=p, gate=gt)
    assert torch.equal(n1, n2) and torch.equal(r1, r2)
    rr, yy = r.clone(), y.clone()
    n3, r3 = block_norm(yy, rr, w, post_weight=p, gate=gt, out=yy, residual_out=rr)
    assert r3 is rr and n3 is yy and torch.equal(rr, r1) and torch.equal(yy, n1)


def test_nan_stays_in_its_row():
    from wisp_b200.norm import block_norm
    y, r, w, p, gt = inputs(6, 1024, BF, BF, BF, True, "none")
    n0, r0 = block_norm(y.to(DEV), r.to(DEV), w.to(DEV), post_weight=p.to(DEV))
    y[2, 77] = float("nan")
    n1, r1 = block_norm(y.to(DEV), r.to(DEV), w.to(DEV), post_weight=p.to(DEV))
    rest = [0, 1, 3, 4, 5]
    assert torch.equal(n0[rest], n1[rest]) and torch.equal(r0[rest], r1[rest]) and bool(torch.isnan(n1[2]).all())


def test_graph():
    from wisp_b200.norm import block_norm
    y, r, w, p, gt = (t.to(DEV) for t in inputs(33, 2048, BF, BF, BF, True, "token"))
    out, ro = torch.empty_like(y), torch.empty_like(r)
    block_norm(y, r, w, post_weight=p, gate=gt, out=out, residual_out=ro)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        block_norm(y, r, w, post_weight=p, gate=gt, out=out, residual_out=ro)
    y.mul_(2)
    graph.replay()
    torch.cuda.synchronize()
    compare((out, ro), *(t.cpu() for t in (y, r, w, p, gt)), 1.0, 1e-6)
