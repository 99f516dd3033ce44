"""``mx4_moe`` against the 64-bit oracle over the dequantised experts.

Tolerance, element by element.  The output is rounded to bf16 once: 2^-8 of
it.  x and silu(g) u go into the products as six MXFP4 terms, which leave at
most 2^-12 of the largest value of a block of 32 (a term leaves less than a
quarter); 2^-8 of ``size``, the sum of the terms' magnitudes, is what one
rounding of silu(g) u to bf16 could cost, and holds the kernel to that.  The
exponential and the quotient
add less than 2^-18 of it, the routing weights (softmax of fp32 logits: the
error of a logit is at most (H / 256 + 8) 2^-24 of the magnitudes that meet in
it, here below 64) less than 2^-14, and the fp32 sums of the down product at
most one part in 2^23 an addition, (I / 16 + 64) of them.  g and u carry one
part in 2^23 of the magnitudes that meet in them an addition, H / 16 + 64
additions at most (blocks of 32 on the matrix unit, then one multiply-add a
block), which ``slack`` carries to the output."""
import pytest
import torch

from oracle import mx4 as ref

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")


def weights(experts, rows, cols, seed, std=0.02):
    g = torch.Generator(device=DEV).manual_seed(seed)
    w = torch.randn(experts, rows, cols, generator=g, device=DEV) * std
    w = w * torch.exp2(torch.randint(-2, 3, (experts, rows, cols // 32), generator=g, device=DEV).float()
                       ).repeat_interleave(32, -1)
    from wisp_b200.mx4 import mx4_quantize
    return mx4_quantize(w)


def layer(experts, hidden, inter, seed=0):
    w13, w2 = weights(experts, 2 * inter, hidden, seed), weights(experts, hidden, inter, seed + 1)
    g = torch.Generator(device=DEV).manual_seed(seed + 2)
    router = (torch.randn(experts, hidden, generator=g, device=DEV) / hidden ** 0.5).bfloat16()
    return w13, w2, router


def tokens(count, hidden, seed=3):
    g = torch.Generator(device=DEV).manual_seed(seed + count)
    return torch.randn(count, hidden, generator=g, device=DEV).bfloat16()


def check(out, x, w13, w2, w, ids, expert_map=None):
    d13, d2 = ref.values(w13.codes, w13.scales), ref.values(w2.codes, w2.scales)
    want, size, slack = ref.moe(x, d13, d2, w, ids, expert_map)
    inter, hidden = d2.shape[2], d2.shape[1]
    bound = (want.abs() * 2.0 ** -8 + size * (2.0 ** -8 + 2.0 ** -14 + 2.0 ** -18 + (inter / 16 + 64) * 2.0 ** -23)
             + slack * (hidden / 16 + 64) * 2.0 ** -23)
    bound = bound * (1 + 2.0 ** -8) + 1e-30
    off = (out.double() - want).abs()
    assert out.dtype == torch.bfloat16 and bool((off <= bound).all()), float((off / bound).max())
    # and as a whole: the roundings are independent, so far below their bound
    assert float(off.norm() / want.norm().clamp_min(1e-30)) < 4e-3


@pytest.mark.parametrize("T,E,k,H,I", [
    (1, 128, 8, 2048, 768), (2, 8, 2, 1024, 896), (5, 16, 4, 256, 128), (16, 128, 8, 512, 256), (64, 12, 3, 256, 160),
    (33, 4, 4, 128, 64), (64, 3, 1, 64, 32), (7, 5, 2, 96, 32), (3, 40, 16, 32, 96), (12, 300, 8, 160, 64),
    (4, 1024, 2, 64, 64), (9, 6, 2, 2080, 1056), (64, 64, 16, 128, 96), (1, 1, 1, 64, 64),
])
@pytest.mark.parametrize("renormalize", [True, False])
def test_router_and_experts(T, E, k, H, I, renormalize):
    from wisp_b200.mx4 import mx4_moe
    w13, w2, router = layer(E, H, I)
    x = tokens(T, H)
    out = mx4_moe(x, w13, w2, k, router=router, renormalize=renormalize)
    w, ids = ref.route(x, router, k, renormalize)
    check(out, x, w13, w2, w, ids)
    assert torch.equal(out, mx4_moe(x, w13, w2, k, router=router, renormalize=renormalize))


@pytest.mark.parametrize("ids_dtype", [torch.int32, torch.int64])
def test_given_routing_slots_and_missing_experts(ids_dtype):
    """Slots in any order, experts without one, ids out of range, an expert named twice."""
    from wisp_b200.mx4 import Mx4Tensor, mx4_moe
    E, S, k, H, I, T = 20, 9, 5, 192, 96, 11
    w13, w2, _ = layer(S, H, I)
    g = torch.Generator().manual_seed(1)
    expert_map = torch.full((E,), -1, dtype=torch.int32)
    expert_map[torch.randperm(E, generator=g)[:S]] = torch.randperm(S, generator=g).int()
    expert_map[3] = S                                   # a slot that is not there
    ids = torch.stack([torch.randperm(E, generator=g)[:k] for _ in range(T)]).to(ids_dtype)
    ids[0, 1] = ids[0, 3]                               # the same expert twice
    ids[1, 0], ids[2, 4] = -1, E
    ids[5] = torch.tensor([e for e in range(E) if not 0 <= expert_map[e] < S][:1] * k)   # nothing to read
    w = torch.rand(T, k, generator=g)
    x = tokens(T, H)
    out = mx4_moe(x, w13, w2, topk_weights=w.to(DEV), topk_ids=ids.to(DEV), expert_map=expert_map.to(DEV))
    check(out, x, w13, w2, w, ids, expert_map.tolist())
    assert not out[5].any()
    # the same experts in other slots: the same bits
    order = torch.randperm(S, generator=g)
    moved = expert_map.clone()
    for e in range(E):
        if 0 <= expert_map[e] < S:
            moved[e] = int((order == int(expert_map[e])).nonzero())
    at = order.to(DEV)
    again = mx4_moe(x, Mx4Tensor(w13.codes[at], w13.scales[at]), Mx4Tensor(w2.codes[at], w2.scales[at]),
                    topk_weights=w.to(DEV), topk_ids=ids.to(DEV), expert_map=moved.to(DEV))
    assert torch.equal(out, again)


def test_no_routed_expert_and_no_tokens():
    from wisp_b200.mx4 import mx4_moe
    w13, w2, router = layer(4, 64, 32)
    x = tokens(3, 64)
    ids, w = torch.full((3, 2), -1, dtype=torch.int32, device=DEV), torch.ones(3, 2, device=DEV)
    assert not mx4_moe(x, w13, w2, topk_weights=w, topk_ids=ids, out=torch.ones_like(x)).any()
    assert mx4_moe(x[:0], w13, w2, 2, router=router).shape == (0, 64)


@pytest.mark.parametrize("size", [2.0 ** -60, 2.0 ** -8, 2.0 ** 20, 2.0 ** 60])
def test_activations_of_any_size(size):
    """fp16 operands hold bf16 activations of every size: x is scaled row by row, silu(g) u pair by pair."""
    from wisp_b200.mx4 import mx4_moe
    w13, w2, _ = layer(6, 256, 128)
    x = tokens(4, 256) * size
    x[1] *= 2.0 ** -10
    x[2, :8] = 0
    g = torch.Generator().manual_seed(2)
    ids = torch.stack([torch.randperm(6, generator=g)[:2] for _ in range(4)])
    w = torch.rand(4, 2, generator=g)
    out = mx4_moe(x, w13, w2, topk_weights=w.to(DEV), topk_ids=ids.to(DEV))
    want, _, _ = ref.moe(x, ref.values(w13.codes, w13.scales), ref.values(w2.codes, w2.scales), w, ids)
    if float(want.abs().max()) < 2.0 ** -120:           # g u is below what fp32 holds: silu(g) u is 0 or nearly
        assert float(out.abs().max()) < 2.0 ** -110
    else:
        check(out, x, w13, w2, w, ids)


@pytest.mark.parametrize("H,I", [(96, 32), (288, 160), (1056, 544), (512, 256)])
@pytest.mark.parametrize("offset", [1, 2, 4, 8])
def test_scale_rows_of_any_alignment(H, I, offset):
    """Scale bytes that begin anywhere, between bytes of NaN: the same bits."""
    from wisp_b200.mx4 import Mx4Tensor, mx4_moe, mx4_synchronize
    w13, w2, router = layer(6, H, I, seed=9)
    x = tokens(5, H)
    want = mx4_moe(x, w13, w2, 3, router=router)

    def moved(q):
        buffer = torch.full((q.scales.numel() + 512,), 255, dtype=torch.uint8, device=DEV)
        scales = buffer[256 + offset:256 + offset + q.scales.numel()].view(q.scales.shape)
        return Mx4Tensor(q.codes, scales.copy_(q.scales))

    assert torch.equal(mx4_moe(x, moved(w13), w2, 3, router=router), want)
    assert torch.equal(mx4_moe(x, moved(w13), moved(w2), 3, router=router), want)
    mx4_synchronize()


def test_zero_token_and_non_finite_token_stay_apart():
    from wisp_b200.mx4 import mx4_moe
    w13, w2, router = layer(8, 128, 64)
    x = tokens(6, 128)
    x[4] = 0
    clean = mx4_moe(x, w13, w2, 2, router=router)
    assert not clean[4].any()
    for bad in (float("nan"), float("inf")):
        y = x.clone()
        y[2, 5] = bad
        out = mx4_moe(y, w13, w2, 2, router=router)
        assert not torch.isfinite(out[2]).any()
        keep = [0, 1, 3, 4, 5]
        want, _, _ = ref.moe(x, ref.values(w13.codes, w13.scales), ref.values(w2.codes, w2.scales),
                             *ref.route(x, router, 2))
        assert float((out[keep].double() - want[keep]).norm() / want[keep].norm()) < 4e-3


def test_nan_scale_makes_nan():
    from wisp_b200.mx4 import mx4_moe
    w13, w2, _ = layer(2, 64, 64)
    w2.scales[1, 7, 1] = 255
    x = tokens(2, 64)
    ids = torch.tensor([[0], [1]], device=DEV)
    out = mx4_moe(x, w13, w2, topk_weights=torch.ones(2, 1, device=DEV), topk_ids=ids)
    assert bool(torch.isfinite(out[0]).all()) and bool(torch.isnan(out[1, 7])) and int(torch.isnan(out[1]).sum()) == 1


def test_ties_take_the_lower_id():
    from wisp_b200.mx4 import mx4_moe
    w13, w2, router = layer(8, 64, 32)
    router[:] = router[:1]                              # every logit the same
    x = tokens(3, 64)
    out = mx4_moe(x, w13, w2, 3, router=router)
    ids, w = torch.arange(3).repeat(3, 1), torch.full((3, 3), 1 / 3)
    check(out, x, w13, w2, w, ids)


def test_strided_x_streams_and_graphs():
    from wisp_b200.mx4 import mx4_moe
    w13, w2, router = layer(16, 256, 128)
    wide = torch.zeros(10, 512, dtype=torch.bfloat16, device=DEV)
    x = tokens(10, 256)
    want = mx4_moe(x, w13, w2, 4, router=router)
    for at in (64, 1):
        wide[:, at:at + 256] = x
        assert torch.equal(mx4_moe(wide[:, at:at + 256], w13, w2, 4, router=router), want)
    torch.cuda.synchronize()
    # two captured calls, each with a workspace of its own
    runs = []
    for seed in (1, 2):
        xs, out = tokens(10, 256, seed), torch.empty(10, 256, dtype=torch.bfloat16, device=DEV)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            mx4_moe(xs, w13, w2, 4, router=router, out=out)
        runs.append((xs, out, graph))
    for _ in range(3):
        for xs, out, graph in runs:
            xs.mul_(-0.5)
            graph.replay()
    torch.cuda.synchronize()
    for xs, out, _ in runs:
        assert torch.equal(out, mx4_moe(xs, w13, w2, 4, router=router))
