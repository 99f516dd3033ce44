"""The compiled binding beside other Python threads."""
import threading
import time

import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")


def test_synchronize_lets_other_threads_run():
    from wisp_b200.mx4 import mx4_synchronize
    mx4_synchronize(DEV)
    ticks, stop = [], threading.Event()

    def tick():
        while not stop.is_set():
            ticks.append(time.monotonic())
            time.sleep(0.005)
    other = threading.Thread(target=tick)
    other.start()
    torch.cuda._sleep(800_000_000)                          # some 0.4 s or more on the stream
    start = time.monotonic()
    mx4_synchronize(DEV)
    end = time.monotonic()
    stop.set()
    other.join()
    assert end - start > 0.2
    within = sum(start + 0.02 < t < end - 0.02 for t in ticks)
    assert within > 5, (within, end - start)


def test_errors_reach_the_caller_as_before():
    from wisp_b200 import _lib
    from wisp_b200.mx4 import mx4_quantize
    from wisp_b200.norm import block_norm
    x = torch.zeros(2, 64, device=DEV)
    with pytest.raises(ValueError, match="multiple of 32"):
        mx4_quantize(x[:, :33])
    with pytest.raises(TypeError, match="fp32"):
        mx4_quantize(x.double())
    with pytest.raises(_lib.WispError, match="columns") as e:
        block_norm(torch.zeros(1, 16385, device=DEV), torch.zeros(1, 16385, device=DEV), torch.zeros(16385, device=DEV))
    assert e.value.code == _lib.WISP_ERR_INVALID


def test_operators_in_threads():
    """Each thread on a stream of its own, the results as in one thread."""
    from wisp_b200.mx4 import mx4_dequantize, mx4_matmul, mx4_moe, mx4_quantize
    from wisp_b200.norm import block_norm
    g = torch.Generator(device=DEV).manual_seed(0)
    x = torch.randn(12, 256, generator=g, device=DEV).bfloat16()
    w13, w2 = (mx4_quantize(torch.randn(6, *s, generator=g, device=DEV) * 0.05) for s in ((128, 256), (256, 64)))
    router = torch.randn(6, 256, generator=g, device=DEV).bfloat16()
    weight = torch.ones(256, device=DEV, dtype=torch.bfloat16)

    def step(x):
        n, r = block_norm(x, x, weight)
        y = mx4_moe(n, w13, w2, 2, router=router)
        q = mx4_quantize(y)
        return (n, r, y, mx4_dequantize(q), mx4_matmul(q, w13[0]))
    inputs = [x * 2.0 ** i for i in range(4)]
    want = [step(v) for v in inputs]
    torch.cuda.synchronize()
    got, errors = [None] * 4, []

    def work(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(200):
                    got[i] = step(inputs[i])
        except Exception as e:                              # noqa: BLE001  (reported below)
            errors.append(e)
    threads = [threading.Thread(target=work, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert not errors, errors
    for a, b in zip(got, want):
        assert all(torch.equal(u, v) for u, v in zip(a, b))
