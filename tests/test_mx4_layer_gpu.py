"""Paged layers of 4-bit experts (``WispMoEStateMX4``): pager state against the oracle pager, outputs byte-identical to
``mx4_moe`` over all experts whatever the cap; and the operators as a decoder layer uses them, one after the other."""
import numpy as np
import pytest
import torch

from oracle import mx4 as ref
from oracle.pager import PagerOracle, first_fit_groups

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda:0")


def experts(E, H, I, seed=0):
    from wisp_b200.mx4 import mx4_quantize
    g = torch.Generator(device=DEV).manual_seed(seed)
    return (mx4_quantize(torch.randn(E, 2 * I, H, generator=g, device=DEV) * 0.05),
            mx4_quantize(torch.randn(E, H, I, generator=g, device=DEV) * 0.05))


def routing(T, E, k, seed):
    g = torch.Generator().manual_seed(seed)
    ids = torch.stack([torch.randperm(E, generator=g)[:k] for _ in range(T)])
    w = torch.rand(T, k, generator=g)
    return (w / w.sum(1, keepdim=True)).to(DEV), ids.to(torch.int32).to(DEV)


def tokens(T, H, seed):
    return torch.randn(T, H, generator=torch.Generator().manual_seed(seed)).bfloat16().to(DEV)


@pytest.mark.parametrize("H,I", [(256, 128), (96, 32), (512, 288)])
def test_paged_layer(H, I):
    from wisp_b200.integrations.vllm import WispMoEStateMX4
    from wisp_b200.mx4 import mx4_moe
    E, k = 12, 3
    w13, w2 = experts(E, H, I)
    for cap in (3, 5, 12):
        st, oracle = WispMoEStateMX4(w13, w2, cap, DEV, 0), PagerOracle(E, cap)
        for n, T in enumerate((1, 4, 9, 1, 70)):
            x = tokens(T, H, n)
            w, ids = routing(T, E, k, 10 * n + T)
            out = st.forward(x, w, ids)
            st.synchronize()
            want = torch.cat([mx4_moe(x[i:i + 64], w13, w2, topk_weights=w[i:i + 64], topk_ids=ids[i:i + 64])
                              for i in range(0, T, 64)])
            assert torch.equal(out, want), (cap, T)
            rows = ids.cpu().numpy()
            if cap < E:                                   # 64 tokens are never the limit here
                for a, b in first_fit_groups(rows, cap):
                    oracle.ensure_resident(rows[a:b])
                s2e, tick, clock, stats = st._read()
                assert (s2e, tick, clock) == (oracle.slot_to_expert, oracle.lru_tick, oracle.lru_clock)
                assert stats[1:] == oracle.stats()[1:]
        st.close()


def test_resident_layer_and_errors():
    from wisp_b200 import _lib
    from wisp_b200.integrations.vllm import WispMoEStateMX4
    from wisp_b200.mx4 import mx4_moe
    E, H, I, k = 8, 128, 64, 4
    w13, w2 = experts(E, H, I)
    x = tokens(5, H, 1)
    w, ids = routing(5, E, k, 2)
    st = WispMoEStateMX4(w13, w2, E, DEV, 0, mode="resident")
    with pytest.raises(_lib.WispError, match="prime_identity"):
        st.forward(x, w, ids)
    st.prime_identity()
    assert torch.equal(st.forward(x, w, ids), mx4_moe(x, w13, w2, topk_weights=w, topk_ids=ids))
    router = tokens(E, H, 3)
    assert torch.equal(st.forward_router(x, router, k), mx4_moe(x, w13, w2, k, router=router))
    logits = x.float() @ router.float().t()
    assert st.forward_logits(x, logits, k).shape == (5, H)
    st.close()
    st = WispMoEStateMX4(w13, w2, 2, DEV, 0)
    with pytest.raises(RuntimeError, match="sub-batch"):
        st.forward(x, w, ids)
    with pytest.raises(ValueError, match="resident"):
        st.forward_router(x, router, k)
    st.resize_cap(6)
    assert torch.equal(st.forward(x, w, ids), mx4_moe(x, w13, w2, topk_weights=w, topk_ids=ids))
    bad = ids.clone()
    bad[2, 1] = E
    with pytest.raises(_lib.WispError, match="outside"):
        st.forward(x, w, bad)
    assert st.forward(x[:0], w[:0], ids[:0]).shape == (0, H)
    with pytest.raises(ValueError):
        st.forward(x[:, :64], w, ids)
    with pytest.raises(ValueError, match="do not match"):
        WispMoEStateMX4(w2, w13, 2, DEV, 0)
    st.close()


@pytest.mark.parametrize("mode,cap", [("paged", 3), ("resident", 6)])
def test_routing_of_other_lengths_is_refused(mode, cap):
    """Fewer rows of routing than tokens would leave rows of the result unwritten."""
    from wisp_b200.integrations.vllm import WispMoEStateMX4
    st = WispMoEStateMX4(*experts(6, 64, 32), cap, DEV, 0, mode=mode)
    if mode == "resident":
        st.prime_identity()
    x = tokens(5, 64, 1)
    for rows in (4, 6):
        w, ids = routing(rows, 6, 2, rows)
        with pytest.raises(ValueError, match="topk_weights"):
            st.forward(x, w, ids)
    w, ids = routing(5, 6, 2, 5)
    with pytest.raises(ValueError, match="topk_weights"):
        st.forward(x, w[:, :1], ids)
    assert st.forward(x, w, ids).shape == (5, 64)
    st.synchronize()
    st.close()


def test_a_token_does_not_depend_on_the_others():
    from wisp_b200.mx4 import mx4_moe
    w13, w2 = experts(20, 384, 4160)                      # several pieces of the intermediate size
    x = tokens(40, 384, 5)
    w, ids = routing(40, 20, 6, 6)
    out = mx4_moe(x, w13, w2, topk_weights=w, topk_ids=ids)
    for a, b in ((0, 1), (7, 9), (20, 40), (39, 40)):
        assert torch.equal(out[a:b], mx4_moe(x[a:b], w13, w2, topk_weights=w[a:b], topk_ids=ids[a:b]))


def test_decoder_layer_runs_them_together():
    """norm -> experts -> norm for a decode batch, then the same experts as quantised products for a prompt.  The
    whole against 64 bits: each step rounds once to bf16 (2^-9 of a value on average, at most 2^-8), four such steps,
    and the norms and sums carry them on without growth."""
    from wisp_b200.mx4 import mx4_dequantize, mx4_matmul, mx4_moe, mx4_quantize
    from wisp_b200.norm import block_norm
    E, H, I, k, T = 16, 512, 256, 4, 24
    w13, w2 = experts(E, H, I, 3)
    d13, d2 = ref.values(w13.codes, w13.scales), ref.values(w2.codes, w2.scales)
    router = tokens(E, H, 4)
    attn, residual = tokens(T, H, 5), tokens(T, H, 6).float()
    pre, post, after = (1 + 0.1 * tokens(1, H, s)[0] for s in (7, 8, 9))
    x, r = block_norm(attn, residual, pre.float(), post_weight=post.float(), scale=0.5)
    y = mx4_moe(x, w13, w2, k, router=router)
    n, r2 = block_norm(y, r, after.float(), scale=0.5)
    ex, er = ref.block_norm(attn, residual, pre, post, scale=0.5)
    weights, ids = ref.route(x, router, k)
    ey, _, _ = ref.moe(x, d13, d2, weights, ids)
    en, er2 = ref.block_norm(ey, er, after, scale=0.5)
    for got, want in ((x, ex), (r, er), (y, ey), (r2, er2), (n, en)):
        assert float((got.double() - want).norm() / want.norm()) < 2.0 ** -8
    # the prompt form: rows sorted by expert, quantised activations, grouped products
    flat = torch.sort(ids.flatten(), stable=True)
    offsets = torch.cat((torch.zeros(1, device=DEV), torch.bincount(ids.flatten(), minlength=E).cumsum(0))).int()
    rows = x[flat.indices // k]
    q = mx4_quantize(rows)
    h = mx4_matmul(q, w13, offsets)
    g, u = h.float().chunk(2, -1)
    a = mx4_quantize((g / (1 + torch.exp(-g)) * u).bfloat16())
    z = mx4_matmul(a, w2, offsets)
    for i in (0, 17, T * k - 1):
        e = int(flat.values[i])
        want = d13[e] @ mx4_dequantize(q[i:i + 1], torch.float32)[0].double()
        assert float((h[i].double() - want).norm() / want.norm()) < 2.0 ** -8
        want = d2[e] @ mx4_dequantize(a[i:i + 1], torch.float32)[0].double()
        assert float((z[i].double() - want).norm() / want.norm()) < 2.0 ** -8
