"""Waits inside the 4-bit kernels that run out.  A test fault makes a launch wait for something that never comes, with
a short limit: every role gives up, the copies and products in flight end before the kernel does, the status is
reported, and the next launch is as if nothing had been."""
import contextlib
import time

import pytest
import torch

from tests.test_mx4_moe_gpu import DEV, layer, tokens

pytestmark = pytest.mark.gpu


@contextlib.contextmanager
def in_vain(what):
    from wisp_b200 import _lib
    L = _lib.lib()
    torch.cuda.synchronize()
    _lib.check(L.wisp_mx4_config(_lib.MX4_TRIES, 1024))
    _lib.check(L.wisp_mx4_config(_lib.MX4_DROP, what))
    try:
        yield
    finally:
        torch.cuda.synchronize()
        _lib.check(L.wisp_mx4_config(_lib.MX4_DROP, _lib.MX4_DROP_NONE))
        _lib.check(L.wisp_mx4_config(_lib.MX4_TRIES, _lib.MX4_DEFAULT_TRIES))


def timed_out():
    from wisp_b200 import _lib
    from wisp_b200.mx4 import mx4_synchronize
    with pytest.raises(_lib.WispError, match="ran out") as e:
        mx4_synchronize()
    return e.value.code == _lib.WISP_ERR_TIMEOUT


@pytest.mark.parametrize("rows,n,k", [(16, 256, 96), (20, 2080, 1056), (700, 4224, 1056), (5000, 8192, 2048)])
def test_product_gives_up(rows, n, k):
    """Both tile widths; as many steps along K as the ring has stages, and more."""
    from wisp_b200 import _lib
    from wisp_b200.mx4 import mx4_matmul, mx4_quantize, mx4_synchronize
    g = torch.Generator(device=DEV).manual_seed(rows)
    a, w = (mx4_quantize(torch.randn(m, k, generator=g, device=DEV)) for m in (rows, n))
    want = mx4_matmul(a, w)
    mx4_synchronize()
    start = time.monotonic()
    with in_vain(_lib.MX4_DROP_SCALES):
        mx4_matmul(a, w)
        assert timed_out()
    assert time.monotonic() - start < 5
    for _ in range(3):
        assert torch.equal(mx4_matmul(a, w), want)
    mx4_synchronize()


@pytest.mark.parametrize("what", ["scales", "terms"])
@pytest.mark.parametrize("T,E,k,H,I", [(1, 4, 2, 64, 32), (5, 16, 4, 256, 128), (16, 128, 8, 2048, 768),
                                       (40, 12, 3, 512, 4160)])
def test_moe_layer_gives_up(T, E, k, H, I, what):
    from wisp_b200 import _lib
    from wisp_b200.mx4 import mx4_moe, mx4_synchronize
    w13, w2, router = layer(E, H, I)
    x = tokens(T, H)
    want = mx4_moe(x, w13, w2, k, router=router)
    mx4_synchronize()
    start = time.monotonic()
    with in_vain({"scales": _lib.MX4_DROP_SCALES, "terms": _lib.MX4_DROP_TERMS}[what]):
        mx4_moe(x, w13, w2, k, router=router)
        assert timed_out()
    assert time.monotonic() - start < 5
    for _ in range(3):
        assert torch.equal(mx4_moe(x, w13, w2, k, router=router), want)
    mx4_synchronize()


def test_unknown_keys_and_values_are_refused():
    from wisp_b200 import _lib
    L = _lib.lib()
    for key, value in ((0, 0), (3, 0), (_lib.MX4_DROP, 3), (_lib.MX4_DROP, -1), (_lib.MX4_TRIES, 0),
                       (_lib.MX4_TRIES, 1 << 32)):
        assert L.wisp_mx4_config(key, value) == _lib.WISP_ERR_INVALID
