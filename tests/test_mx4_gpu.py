"""MXFP4 quantisation (``mx4_quantize`` / ``mx4_dequantize``) against the 64-bit oracle: codes and scale bytes are
exact whole numbers (every product by a power of two is exact), values read back are exact in bf16 and fp32."""
import pytest
import torch

from oracle import mx4 as ref

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")
DTYPES = [torch.bfloat16, torch.float16, torch.float32]


def sample(rows, cols, dtype, seed):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, cols, generator=g) * torch.exp(2 * torch.randn(rows, cols // 32, generator=g)
                                                         ).repeat_interleave(32, 1)
    return x.to(dtype)


def check(x):
    from wisp_b200.mx4 import mx4_dequantize, mx4_quantize
    q = mx4_quantize(x)
    codes, scales = ref.quantize(x.cpu())
    assert torch.equal(q.scales.cpu(), scales)
    # a value that rounds to zero keeps its sign: codes 0 and 8 stand for the same value
    got, want = ref.values(q.codes.cpu(), q.scales.cpu()), ref.values(codes, scales)
    assert torch.equal(got.nan_to_num(7e77), want.nan_to_num(7e77))
    for dtype in (torch.bfloat16, torch.float32):
        back = mx4_dequantize(q, dtype)
        assert back.dtype == dtype and back.shape == x.shape
        assert torch.equal(back.cpu().double().nan_to_num(7e77), want.nan_to_num(7e77))
    half = mx4_dequantize(q, torch.float16).cpu()
    assert torch.equal(half.nan_to_num(7.0, 8.0, -8.0), want.to(torch.float16).nan_to_num(7.0, 8.0, -8.0))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,cols", [(1, 32), (1, 2048), (3, 96), (257, 800), (1021, 4096), (5, 32 * 1000)])
def test_quantize_matches_oracle(rows, cols, dtype):
    check(sample(rows, cols, dtype, rows + cols).to(DEV))


@pytest.mark.parametrize("dtype", DTYPES)
def test_every_code_and_tie(dtype):
    """All E2M1 values, the midpoints between them and their neighbours, under several scales."""
    mids = [0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0]
    eps = 2.0 ** -7
    v = ref.E2M1 + mids + [m * (1 + eps) for m in mids] + [m * (1 - eps) for m in mids]
    v = v + [7.0, 7.96875] + [0.0] * (31 - (len(v) + 2) % 32) + [4.0]
    x = torch.tensor(v, dtype=torch.float64).reshape(-1, 32)
    x[:, -1] = 4.0                                      # the block's scale is 1
    x = torch.cat([x, -x])
    scales = [1.0, 2.0 ** -10, 2.0 ** 10] + ([] if dtype == torch.float16 else [2.0 ** -100, 2.0 ** 100])
    check(torch.cat([x * s for s in scales]).to(dtype).to(DEV))


@pytest.mark.parametrize("dtype", DTYPES)
def test_extremes(dtype):
    """Zeros, subnormals, the type's largest values, infinities and NaN, each in a block of its own."""
    info = torch.finfo(dtype)
    rows = [torch.zeros(32), torch.full((32,), -0.0), torch.full((32,), info.smallest_normal),
            torch.full((32,), info.smallest_normal * info.eps), torch.full((32,), info.max),
            torch.full((32,), -info.max)]
    for bad in (float("inf"), float("-inf"), float("nan")):
        r = torch.linspace(-3, 3, 32)
        r[17] = bad
        rows.append(r)
    rows.append(torch.linspace(-3, 3, 32))
    check(torch.stack(rows).to(dtype).to(DEV))


def test_strided_and_unaligned_rows():
    from wisp_b200.mx4 import mx4_quantize
    x = sample(40, 256, torch.bfloat16, 1).to(DEV)
    for view in (x[:, 64:192], x[::3], x[5:, 1:129], x.t()[:64, :32], x[1:2, 32:64], x.view(4, 10, 256)[:, 2]):
        check(view)
    q = mx4_quantize(x.view(2, 4, 5, 256))
    assert q.shape == (2, 4, 5, 256) and torch.equal(q.codes.view(40, 128), mx4_quantize(x).codes)
    assert mx4_quantize(x[:0]).shape == (0, 256)


def test_large_offsets():
    """More than 2^32 values: offsets pass 32 bits."""
    from wisp_b200.mx4 import mx4_dequantize, mx4_quantize
    rows, cols = 131_073, 32_768
    x = torch.zeros(rows, cols, dtype=torch.bfloat16, device=DEV)
    x[-2:] = sample(2, cols, torch.bfloat16, 3).to(DEV)
    q = mx4_quantize(x)
    del x
    codes, scales = ref.quantize(sample(2, cols, torch.bfloat16, 3))
    assert torch.equal(q.scales[-2:].cpu(), scales) and int(q.scales[:-2].max()) == 0
    back = mx4_dequantize(q)
    assert torch.equal(back[-2:].cpu().double(), ref.values(codes, scales)) and not back[:-2].any()


def test_graph_and_stream():
    from wisp_b200.mx4 import Mx4Tensor, mx4_dequantize, mx4_quantize
    x = sample(64, 512, torch.bfloat16, 4).to(DEV)
    side = torch.cuda.Stream()
    q = Mx4Tensor(torch.zeros(64, 256, dtype=torch.uint8, device=DEV), torch.zeros(64, 16, dtype=torch.uint8, device=DEV))
    out = torch.empty_like(x)
    mx4_dequantize(mx4_quantize(x))                     # the kernels' code is on the device
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        mx4_dequantize(mx4_quantize(x, out=q), out=out)
    for seed in (5, 6):
        x.copy_(sample(64, 512, torch.bfloat16, seed))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out.cpu().double(), ref.values(*ref.quantize(x.cpu())))
