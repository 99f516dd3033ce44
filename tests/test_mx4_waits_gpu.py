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


def test_every_stream_is_told():
    """The streams of other calls, asked first, do not take the report from the stream of the call that gave up."""
    from wisp_b200 import _lib
    from wisp_b200.mx4 import mx4_moe, mx4_synchronize
    w13, w2, router = layer(4, 64, 32)
    x = tokens(2, 64)
    streams = [torch.cuda.Stream() for _ in range(3)]
    with in_vain(_lib.MX4_DROP_TERMS):
        with torch.cuda.stream(streams[0]):
            mx4_moe(x, w13, w2, 2, router=router)
        torch.cuda.synchronize()
        for s in (streams[1], streams[2], streams[0], torch.cuda.current_stream()):
            with torch.cuda.stream(s):
                assert timed_out()
    for s in (*streams, torch.cuda.current_stream()):
        with torch.cuda.stream(s):
            mx4_synchronize()


def test_every_layer_is_told():
    from wisp_b200 import _lib
    from wisp_b200.integrations.vllm import WispMoEStateMX4
    from wisp_b200.mx4 import mx4_synchronize
    w13, w2, _ = layer(4, 64, 32)
    x, w = tokens(2, 64), torch.ones(2, 2, device=DEV)
    ids = torch.tensor([[0, 1], [1, 0]], device=DEV)
    a, b = (WispMoEStateMX4(w13, w2, 2, DEV, i) for i in range(2))
    with in_vain(_lib.MX4_DROP_TERMS):
        a.forward(x, w, ids)
        torch.cuda.synchronize()
        for st in (b, a):
            with pytest.raises(_lib.WispError, match="ran out") as e:
                st.synchronize()
            assert e.value.code == _lib.WISP_ERR_TIMEOUT
        assert timed_out()
    want = b.forward(x, w, ids)
    late = WispMoEStateMX4(w13, w2, 2, DEV, 2)
    assert torch.equal(a.forward(x, w, ids), want) and torch.equal(late.forward(x, w, ids), want)
    for st in (a, b, late):
        st.synchronize()
        st.close()
    mx4_synchronize()
