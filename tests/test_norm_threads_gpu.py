"""block_norm from several host threads at once, through the C entry point (which no lock of the interpreter guards)."""
import threading

import pytest
import torch

from tests.test_norm_gpu import compare

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")


def test_threads_with_rows_of_different_lengths():
    """Widths that take the same kernel with different amounts of shared memory, most of them above 48 KB."""
    from wisp_b200 import _lib
    L = _lib.lib()
    widths, rows, calls = (6659, 8191, 7013, 7655), 3, 1500
    jobs, errors = [], []
    for n, cols in enumerate(widths):
        g = torch.Generator(device=DEV).manual_seed(n)
        y, r = (torch.randn(rows, cols, generator=g, device=DEV).bfloat16() for _ in range(2))
        w = torch.randn(cols, generator=g, device=DEV).bfloat16()
        jobs.append((cols, y, r, w, torch.empty_like(y), torch.empty_like(y), torch.cuda.Stream()))
    torch.cuda.synchronize()
    start = threading.Barrier(len(jobs))

    def work(cols, y, r, w, out, res, stream):
        torch.cuda.set_device(DEV)
        start.wait()
        for _ in range(calls):
            rc = L.wisp_block_norm(y.data_ptr(), cols, r.data_ptr(), cols, w.data_ptr(), None, None, 0, 0, 0, 0, 0, rows,
                                   cols, 1.0, 1e-6, out.data_ptr(), res.data_ptr(), _lib.stream_ptr(stream))
            if rc:
                errors.append((cols, rc, L.wisp_last_error()))
                return
    threads = [threading.Thread(target=work, args=job) for job in jobs]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert not errors, errors
    for _, y, r, w, out, res, _ in jobs:
        compare((out, res), y.cpu(), r.cpu(), w.cpu(), None, None, 1.0, 1e-6)
