"""Outputs of ``block_norm`` in the memory of its inputs: row by row in place gives the same bits, anything else is
refused (a row would be written while another that lies there is still to be read)."""
import ctypes

import pytest
import torch

DEV = torch.device("cuda:0")
COLS = [256, 2050, 131, 1]                              # 16-byte pieces, pairs, granules, less than a granule


@pytest.mark.skipif(torch.cuda.is_available(), reason="addresses are numbers here: a call that is not refused must not run")
def test_refusals_of_the_entry_point():
    """No memory is touched."""
    from wisp_b200 import _lib
    L = _lib.lib()
    rows, cols, at = 8, 64, 1 << 20

    def call(y=at, ys=cols, r=at + (1 << 16), rs=cols, w=at + (1 << 17), post=None, gate=None, kind=0, gs=0,
             out=at + (1 << 18), res=at + (1 << 19), dtype=0, rdtype=0):
        rc = L.wisp_block_norm(y, ys, r, rs, w, post, gate, kind, gs, dtype, rdtype, 0, rows, cols, 1.0, 1e-6, out, res, None)
        return rc == _lib.WISP_ERR_INVALID and b"overlap" in L.wisp_last_error()
    size = rows * cols * 2
    assert call(out=at + 2) and call(out=at + size - 2) and call(res=at + 2 * cols) and call(out=at - size + 2)
    assert call(r=at, rs=0, res=at)                     # every row reads the one that is written first
    assert call(y=at, ys=2 * cols, out=at) and call(y=at, ys=cols - 2, out=at)
    assert call(y=at, ys=8 * cols, out=at + 2 * 8 * cols - 2) and call(y=at, ys=8 * cols, out=at + 2 * 57 * cols - 2)
    assert call(res=at + (1 << 18)) and call(res=at + (1 << 18) + 2 * cols) and call(out=at + (1 << 19) + 2)
    assert call(w=at + (1 << 18)) and call(post=at + (1 << 19) + 2 * size - 2 - size)
    gate = at + (1 << 21)
    assert call(gate=gate, kind=1, gs=cols, out=gate) and call(gate=gate, kind=2, out=gate)
    assert call(gate=gate, kind=3, gs=cols, out=gate + 2) and call(gate=gate, kind=3, gs=0, out=gate)
    assert call(y=at, res=at, rdtype=2)                 # rows of another length in bytes


def tensors(rows, cols, gate):
    g = torch.Generator(device=DEV).manual_seed(cols)
    y, r = (torch.randn(rows, cols, generator=g, device=DEV).bfloat16() for _ in range(2))
    w = torch.randn(cols, generator=g, device=DEV).bfloat16()
    return y, r, w, torch.randn(rows, cols, generator=g, device=DEV).bfloat16() if gate else None


@pytest.mark.gpu
@pytest.mark.parametrize("cols", COLS)
@pytest.mark.parametrize("post", [False, True])
def test_in_the_place_of_any_input(cols, post):
    from wisp_b200.norm import block_norm
    rows = 700
    for out_at, res_at in (("y", "r"), ("r", "y"), ("g", "y"), ("r", "g"), ("y", None), (None, "y"), ("r", None), (None, "g")):
        y, r, w, g = tensors(rows, cols, True)
        p = w if post else None
        want = block_norm(y, r, w, post_weight=p, gate=g)
        at = {"y": y, "r": r, "g": g, None: None}
        got = block_norm(y, r, w, post_weight=p, gate=g, out=at[out_at], residual_out=at[res_at])
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]), (out_at, res_at)


@pytest.mark.gpu
@pytest.mark.parametrize("cols", COLS)
def test_same_tensor_twice_and_gaps(cols):
    from wisp_b200.norm import block_norm
    y, _, w, _ = tensors(300, cols, False)
    want = block_norm(y, y, w)
    got = block_norm(y, y, w, residual_out=y)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    # outputs in the gaps between the rows of an input
    y, r, w, _ = tensors(2, cols, False)
    flat = torch.zeros(2, 10 * cols, dtype=torch.bfloat16, device=DEV)
    flat[:, :cols] = y
    want = block_norm(y, r, w)
    out, res = (flat.flatten()[k * cols:(k + 2) * cols].view(2, cols) for k in (3, 6))
    got = block_norm(flat[:, :cols], r, w, out=out, residual_out=res)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]) and torch.equal(flat[:, :cols], y)


@pytest.mark.gpu
def test_refusals():
    from wisp_b200 import _lib
    from wisp_b200.norm import block_norm
    buf = torch.zeros(9, 64, dtype=torch.bfloat16, device=DEV)
    y, w = torch.zeros(8, 64, dtype=torch.bfloat16, device=DEV), torch.ones(64, dtype=torch.bfloat16, device=DEV)
    for kwargs in (dict(residual=buf[:8], residual_out=buf[1:]), dict(residual=buf[:1].expand(8, 64), residual_out=buf[:8]),
                   dict(residual=y, out=buf[:8], residual_out=buf[:8]), dict(residual=y, out=buf[1:], residual_out=buf[:8]),
                   dict(residual=y, gate=buf[2], out=buf[:8]), dict(residual=y, gate=buf[:8, 3:4], out=buf[:8])):
        with pytest.raises(_lib.WispError, match="overlaps"):
            block_norm(y, weight=w, **kwargs)


@pytest.mark.gpu
@pytest.mark.parametrize("cols", COLS)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_in_place_with_a_fp32_residual(cols, dtype):
    """y and the residual updated where they lie, rows of different lengths in bytes; replayed from a graph as well."""
    from wisp_b200.norm import block_norm
    y, r, w, g = tensors(900, cols, True)
    y, r, w, g = y.to(dtype), r.float(), w.float(), g.to(dtype)
    first = block_norm(y, r, w, post_weight=w, gate=g)
    second = block_norm(*first, w, post_weight=w, gate=g)
    ys, rs = y.clone(), r.clone()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        block_norm(ys, rs, w, post_weight=w, gate=g, out=ys, residual_out=rs)
    for want in (first, second):
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(ys, want[0]) and torch.equal(rs, want[1])
