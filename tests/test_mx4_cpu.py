"""What the 4-bit operators and the block norm refuse (no GPU needed): the C entry points return
WISP_ERR_INVALID with a message before they touch the device, the Python functions raise."""
import pytest
import torch

from oracle import mx4 as ref
from wisp_b200 import _lib
from wisp_b200.mx4 import Mx4Tensor, mx4_dequantize, mx4_quantize
from wisp_b200.norm import block_norm

P = 1 << 20         # an aligned address that no refused call reads


def refused(rc, word):
    assert rc == _lib.WISP_ERR_INVALID and word in _lib.lib().wisp_last_error().decode()


def test_quantize_refusals():
    q = _lib.lib().wisp_mx4_quantize
    refused(q(P, 3, 1, 32, 32, P, P, None), "dtype")
    refused(q(P, 0, 1, 33, 33, P, P, None), "multiple of 32")
    refused(q(P, 0, 1, 0, 0, P, P, None), "multiple of 32")
    refused(q(P, 0, -1, 32, 32, P, P, None), "rows")
    refused(q(P, 0, 1 << 40, 32, 32, P, P, None), "2^38")
    refused(q(None, 0, 1, 32, 32, P, P, None), "NULL")
    refused(q(P + 2, 0, 1, 32, 32, P, P, None), "16-byte")
    refused(q(P, 0, 2, 64, 32, P, P, None), "overlap")
    refused(q(P, 0, 2, 32, 33, P, P, None), "16-byte")
    assert q(None, 0, 0, 32, 32, None, None, None) == _lib.WISP_OK
    d = _lib.lib().wisp_mx4_dequantize
    refused(d(P, P, 1, 32, P, 7, None), "dtype")
    refused(d(P, P, 1, 16, P, 0, None), "multiple of 32")
    refused(d(P, None, 1, 32, P, 0, None), "NULL")
    refused(d(P + 1, P, 1, 32, P, 0, None), "aligned")
    refused(d(P, P, 1, 32, P + 8, 0, None), "aligned")


def test_block_norm_refusals():
    n = _lib.lib().wisp_block_norm

    def call(dtype=0, rdtype=0, wdtype=0, rows=1, cols=64, gate=None, kind=0, y=P, stride=64):
        return n(y, stride, P, 64, P, None, gate, kind, 0, dtype, rdtype, wdtype, rows, cols, 1.0, 1e-6, P, P, None)
    refused(call(dtype=5), "type")
    refused(call(rdtype=1), "type")
    refused(call(wdtype=1), "type")
    refused(call(cols=0), "columns")
    refused(call(cols=16385), "columns")
    refused(call(rows=-1), "rows")
    refused(call(gate=P), "gate_kind")
    refused(call(kind=2), "gate_kind")
    refused(call(kind=4, gate=P), "gate_kind")
    refused(call(y=None), "NULL")
    refused(call(rows=2, stride=-64), "stride")
    refused(call(y=P + 1), "aligned")
    refused(call(gate=P + 1, kind=2), "aligned")
    refused(call(y=P + 2, dtype=2, rdtype=2, wdtype=2), "aligned")
    assert call(rows=0) == _lib.WISP_OK


def test_python_refusals():
    x = torch.zeros(2, 64)
    with pytest.raises(ValueError, match="CUDA"):
        mx4_quantize(x)
    with pytest.raises(TypeError, match="Tensor"):
        mx4_quantize([1.0])
    codes, scales = ref.quantize(x)
    with pytest.raises(ValueError, match="CUDA"):
        mx4_dequantize(Mx4Tensor(codes, scales))
    with pytest.raises(TypeError, match="uint8"):
        Mx4Tensor(codes.int(), scales)
    with pytest.raises(ValueError, match="match"):
        Mx4Tensor(codes, scales[:, :1])
    with pytest.raises(ValueError, match="match"):
        Mx4Tensor(codes[:1], scales)
    with pytest.raises(ValueError, match="contiguous"):
        Mx4Tensor(codes.t().contiguous().t(), scales)
    blob = torch.zeros(3, 70, dtype=torch.uint8)         # a stack whose matrices lie apart
    assert Mx4Tensor(blob[:, :64].view(3, 2, 32), torch.zeros(3, 2, 2, dtype=torch.uint8)).shape == (3, 2, 64)
    with pytest.raises(ValueError, match="CUDA"):
        block_norm(x, x, x[0])


def test_mx4_tensor():
    codes, scales = ref.quantize(torch.randn(3, 4, 64))
    t = Mx4Tensor(codes, scales.view(torch.float8_e8m0fnu))
    assert t.shape == (3, 4, 64) and t.scales.dtype == torch.uint8 and t[1].shape == (4, 64)
    assert torch.equal(t[1].codes, codes[1]) and t[0, 2].shape == (64,)
    with pytest.raises(IndexError):
        t[0, 0, 0]


def test_oracle_quantizer_is_the_nearest_value():
    """The oracle against its own definition: no E2M1 value lies nearer than the one it chose."""
    x = torch.randn(64, 96, dtype=torch.float64, generator=torch.Generator().manual_seed(0)) * 10
    codes, scales = ref.quantize(x)
    v = ref.values(codes, scales)
    s = torch.exp2(scales.double() - 127).repeat_interleave(32, -1)
    grid = torch.tensor(ref.E2M1 + [-a for a in ref.E2M1], dtype=torch.float64)
    best = (x.unsqueeze(-1) - s.unsqueeze(-1) * grid).abs().amin(-1)
    assert torch.equal((x - v).abs(), best)
    assert torch.equal(ref.values(*ref.quantize(v)), v) or bool((v.abs() / s <= 6).all())


def test_moe_refusals():
    import ctypes
    f = _lib.lib().wisp_mx4_moe

    def call(T=1, E=4, k=2, H=64, I=32, slots=4, x=P, router=P, ids=None, w=None, emap=None, c13=P, ws=P,
             nbytes=1 << 30, stride=64, out=P, strides=None):
        strides = strides and (ctypes.c_int64 * 4)(*strides)
        return f(x, stride, router, ids, 0, w, emap, c13, P, P, P, strides, slots, T, E, k, H, I, 1, ws, nbytes, out, None)
    refused(call(T=65), "64 tokens")
    refused(call(T=-1), "64 tokens")
    refused(call(E=1025), "1024 experts")
    refused(call(k=0), "top_k")
    refused(call(k=5), "top_k")
    refused(call(k=17, E=64, slots=64), "top_k")
    refused(call(slots=0), "top_k")
    refused(call(H=48), "multiples of 32")
    refused(call(I=16), "multiples of 32")
    refused(call(H=65536), "at most")
    refused(call(x=None), "NULL")
    refused(call(ws=None), "NULL")
    refused(call(router=None), "either")
    refused(call(ids=P, w=P), "either")
    refused(call(router=None, ids=P), "either")
    refused(call(slots=3), "slots")
    refused(call(c13=P + 8), "aligned")
    refused(call(out=P + 8), "aligned")
    refused(call(ws=P + 4), "aligned")
    good = [64 * 32, 64 * 2, 64 * 16, 64]               # slots of H 64, I 32 that follow one another
    for i, bad in ((0, 64 * 32 - 32), (0, 64 * 32 + 16), (1, 64), (2, 0), (3, 48)):
        refused(call(strides=good[:i] + [bad] + good[i + 1:]), "whole rows")
    refused(call(slots=1 << 26, I=32), "rows")
    refused(call(T=2, stride=32), "overlap")
    refused(call(T=2, stride=68), "16-byte")
    refused(call(nbytes=64), "workspace")
    assert call(T=0) == _lib.WISP_OK
    n = ctypes.c_int64()
    refused(_lib.lib().wisp_mx4_moe_workspace(65, 4, 2, 64, 32, ctypes.byref(n)), "64 tokens")
    refused(_lib.lib().wisp_mx4_moe_workspace(4, 4, 2, 64, 32, None), "NULL")
    assert _lib.lib().wisp_mx4_moe_workspace(4, 4, 2, 64, 32, ctypes.byref(n)) == 0 and n.value >= 4 * 64 * 2


def test_matmul_refusals():
    f = _lib.lib().wisp_mx4_matmul

    def call(rows=1, groups=1, n=8, k=32, a=P, s=P, w=P, offsets=None, out=P):
        return f(a, s, rows, w, P, groups, n, k, offsets, out, None)
    refused(call(rows=-1), "rows")
    refused(call(rows=(1 << 30) + 1), "rows")
    refused(call(groups=0), "groups")
    refused(call(groups=1025, offsets=P), "groups")
    refused(call(n=0), "n >= 1")
    refused(call(k=48), "multiple of 32")
    refused(call(k=0), "multiple of 32")
    refused(call(groups=1024, n=1 << 22, offsets=P), "too large")
    refused(call(groups=2), "offsets")
    refused(call(a=None), "NULL")
    refused(call(out=None), "NULL")
    refused(call(a=P + 8), "aligned")
    refused(call(w=P + 4), "aligned")
    refused(call(out=P + 1), "out")
    assert call(rows=0) == _lib.WISP_OK
