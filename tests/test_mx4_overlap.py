"""Outputs of the 4-bit operators over their own inputs: refused, since a block is written while another is read.  The
refusals come before anything runs, so addresses are numbers here and no GPU is needed (nor wanted: a call that was not
refused must not run)."""
import pytest
import torch

pytestmark = pytest.mark.skipif(torch.cuda.is_available(), reason="a call that is not refused must not run")
AT = 1 << 20


def refused(name, *args):
    from wisp_b200 import _lib
    L = _lib.lib()
    rc = getattr(L, name)(*args)
    return rc == _lib.WISP_ERR_INVALID and b"overlap" in L.wisp_last_error()


@pytest.mark.parametrize("dtype,size", [(0, 2), (1, 2), (2, 4)])
def test_quantize_and_back(dtype, size):
    rows, cols = 6, 64
    codes, scales, x = rows * cols // 2, rows * cols // 32, rows * cols * size
    far, other = AT + (1 << 16), AT + (1 << 17)

    def quantize(at, c, s, stride=cols):
        return refused("wisp_mx4_quantize", at, dtype, rows, cols, stride, c, s, None)
    assert quantize(AT, AT, other) and quantize(AT, AT + x - 4, other) and quantize(AT, AT - codes + 4, other)
    assert quantize(AT, other, AT) and quantize(AT, other, AT + x - 1) and quantize(AT, other, AT - scales + 1)
    assert quantize(AT, other, other) and quantize(AT, other, other + codes - 1)
    assert quantize(AT, AT + 5 * 16 * cols * size, far, 16 * cols)       # the last row of rows that lie apart

    def dequantize(c, s, out):
        return refused("wisp_mx4_dequantize", c, s, rows, cols, out, dtype, None)
    assert dequantize(AT, other, AT) and dequantize(AT + x - 4, other, AT) and dequantize(AT - codes + 4, other, AT)
    assert dequantize(other, AT, AT) and dequantize(other, AT + x - 1, AT) and dequantize(other, AT - scales + 1, AT)


def test_matmul():
    rows, groups, n, k = 5, 3, 24, 64
    sizes = [rows * k // 2, rows * k // 32, groups * n * k // 2, groups * n * k // 32, 4 * (groups + 1)]
    out_bytes = rows * n * 2

    def matmul(a, sa, w, sw, offsets, out):
        return refused("wisp_mx4_matmul", a, sa, rows, w, sw, groups, n, k, offsets, out, None)
    apart = [AT + (i << 16) for i in range(1, 6)]
    for i, size in enumerate(sizes):
        for at in (apart[i], apart[i] + size - 2, apart[i] - out_bytes + 2):
            assert matmul(*apart, at), (i, at)


def test_what_meets():
    """Edges that only touch, and gaps between rows, are no overlap: these calls get as far as the missing GPU."""
    rows, cols = 6, 64
    for c in (AT + rows * cols * 2, AT - rows * cols // 2):
        assert not refused("wisp_mx4_quantize", AT, 0, rows, cols, cols, c, AT + (1 << 17), None)
    assert not refused("wisp_mx4_quantize", AT, 0, rows, cols, 16 * cols, AT + 2 * cols, AT + (1 << 17), None)
    assert refused("wisp_mx4_quantize", AT, 0, rows, cols, 16 * cols, AT + 2 * cols - 4, AT + (1 << 17), None)
    assert not refused("wisp_mx4_dequantize", AT, AT + (1 << 17), rows, cols, AT + rows * cols // 2, 0, None)
