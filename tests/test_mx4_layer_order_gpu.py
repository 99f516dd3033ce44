"""What else is asked of a layer of 4-bit experts while a forward's kernels are still queued: prefetches, forwards on
other streams, other threads.  A kernel is held up by a spin on its stream, put between a forward's admission and its
launch, so that whatever does not wait for it comes first."""
import threading

import pytest
import torch

from oracle.pager import PagerOracle
from tests.test_mx4_layer_gpu import DEV, experts, routing, tokens

pytestmark = pytest.mark.gpu
E, H, I = 12, 256, 128


@pytest.fixture()
def held_up(monkeypatch):
    """mx4_moe as the layer calls it, behind a spin of some 30 ms on its stream."""
    from wisp_b200.integrations.vllm import fused_moe_mx4 as m
    real = m.mx4_moe

    def late(x, *args, **kwargs):
        torch.cuda._sleep(50_000_000)
        return real(x, *args, **kwargs)
    monkeypatch.setattr(m, "mx4_moe", late)
    return real


def route_to(sets, seed=0):
    """(weights, ids) of one token for each set of experts."""
    ids = torch.tensor([list(s) for s in sets], dtype=torch.int32, device=DEV)
    w = torch.rand(ids.shape, generator=torch.Generator().manual_seed(seed)).to(DEV)
    return w, ids


def test_prefetch_waits_for_a_queued_forward_and_spares_its_experts(held_up):
    from wisp_b200.integrations.vllm import WispMoEStateMX4
    w13, w2 = experts(E, H, I)
    st, oracle = WispMoEStateMX4(w13, w2, 6, DEV, 0), PagerOracle(E, 6)
    x = tokens(2, H, 1)
    assert st.last_unique_experts == set()
    for step, (sets, predicted) in enumerate([
            (((0, 1, 2), (1, 2, 3)), {8, 9, 10, 11}),      # 4 in use, 2 free: the prediction is cut to 2
            (((4, 5, 0), (5, 0, 1)), {6, 7}),              # those of the forward are no victims
            (((4, 5, 0), (3, 2, 1)), {8, 9, 10}),          # every slot in use: nothing is loaded
    ]):
        w, ids = route_to(sets, step)
        out = st.forward(x, w, ids)
        done = torch.cuda.Event()
        done.record()
        st.prefetch_async(predicted)
        assert done.query(), "the prefetch did not wait for the forward"
        st.synchronize()
        assert torch.equal(out, held_up(x, w13, w2, topk_weights=w, topk_ids=ids))
        used = set().union(*sets)
        assert st.last_unique_experts == used
        oracle.ensure_resident(ids.cpu().numpy())
        oracle.prefetch_async(predicted, used)
        s2e, tick, clock, stats = st._read()
        assert (s2e, tick, clock) == (oracle.slot_to_expert, oracle.lru_tick, oracle.lru_clock)
        assert stats[1:] == oracle.stats()[1:]
    st.close()


def test_forwards_on_two_streams_wait_for_one_another(held_up):
    """Each evicts every expert of the one before it."""
    from wisp_b200.integrations.vllm import WispMoEStateMX4
    w13, w2 = experts(E, H, I, 1)
    st = WispMoEStateMX4(w13, w2, 4, DEV, 0)
    x = tokens(1, H, 2)
    jobs = []
    for n in range(6):
        w, ids = route_to([[4 * (n % 3) + j for j in range(4)]], n)
        jobs.append((torch.cuda.Stream(), w, ids))
    torch.cuda.synchronize()
    outs = []
    for stream, w, ids in jobs:
        with torch.cuda.stream(stream):
            outs.append(st.forward(x, w, ids))
    torch.cuda.synchronize()
    for out, (_, w, ids) in zip(outs, jobs):
        assert torch.equal(out, held_up(x, w13, w2, topk_weights=w, topk_ids=ids))
    st.close()


def test_threads_share_a_layer(held_up):
    """Forwards and prefetches of two threads: an admission and its kernels belong together."""
    from wisp_b200.integrations.vllm import WispMoEStateMX4
    w13, w2 = experts(E, H, I, 2)
    st = WispMoEStateMX4(w13, w2, 4, DEV, 0)
    x = tokens(3, H, 3)
    jobs = [route_to([[(5 * n + 3 * t + j) % E for j in range(3)] for t in range(3)], n) for n in range(12)]
    torch.cuda.synchronize()
    outs, errors = [None] * len(jobs), []

    def work(first):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for n in range(first, len(jobs), 2):
                    outs[n] = st.forward(x, *jobs[n])
                    st.prefetch_async({(7 * n + j) % E for j in range(4)})
        except Exception as e:                              # noqa: BLE001  (reported below)
            errors.append(e)
    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert not errors
    for out, (w, ids) in zip(outs, jobs):
        assert torch.equal(out, held_up(x, w13, w2, topk_weights=w, topk_ids=ids))
    st.close()


def test_a_failed_forward_leaves_its_first_groups_covered(held_up):
    from wisp_b200 import _lib
    from wisp_b200.integrations.vllm import WispMoEStateMX4
    st = WispMoEStateMX4(*experts(E, H, I, 3), 3, DEV, 0)
    x = tokens(2, H, 4)
    w, ids = route_to([(0, 1, 2), (3, 4, E)])
    out = torch.empty_like(x)
    with pytest.raises(_lib.WispError, match="outside"):
        st.forward(x, w, ids, out=out)
    assert st.last_unique_experts == {0, 1, 2}
    st.synchronize()
    st.close()


def test_primed_experts_are_there_for_every_stream():
    from wisp_b200.integrations.vllm import WispMoEStateMX4
    from wisp_b200.mx4 import mx4_moe
    w13, w2 = experts(48, 1024, 1024, 4)                    # 80 MB: the copy takes more than a millisecond
    x = tokens(4, 1024, 5)
    w, ids = routing(4, 48, 8, 6)
    want = mx4_moe(x, w13, w2, topk_weights=w, topk_ids=ids)
    torch.cuda.synchronize()
    st = WispMoEStateMX4(w13, w2, 48, DEV, 0, mode="resident")
    st.prime_identity()
    with torch.cuda.stream(torch.cuda.Stream()):
        out = st.forward(x, w, ids)
    torch.cuda.synchronize()
    assert torch.equal(out, want)
    st.close()


def test_used_refuses_what_it_cannot_cover():
    import ctypes

    from wisp_b200 import _lib
    from wisp_b200.integrations.vllm import WispMoEStateMX4
    L = _lib.lib()
    st = WispMoEStateMX4(*experts(4, 64, 32), 2, DEV, 0)
    ids = (ctypes.c_int32 * 2)(1, 4)
    assert L.wisp_layer_used(None, ids, 1, None) == _lib.WISP_ERR_INVALID
    assert L.wisp_layer_used(st._h, None, 1, None) == _lib.WISP_ERR_INVALID
    assert L.wisp_layer_used(st._h, ids, -1, None) == _lib.WISP_ERR_INVALID
    assert L.wisp_layer_used(st._h, ids, 2, None) == _lib.WISP_ERR_BAD_EXPERT
    assert L.wisp_layer_used(st._h, ids, 1, None) == _lib.WISP_OK and st.last_unique_experts == {1}
    st.close()
    st = WispMoEStateMX4(*experts(4, 64, 32), 4, DEV, 0, mode="resident")
    assert L.wisp_layer_used(st._h, ids, 1, None) == _lib.WISP_ERR_INVALID
    st.close()


@pytest.mark.parametrize("mode,cap", [("paged", 3), ("resident", E)])
def test_arguments_are_refused_before_anything_is_paged_in(mode, cap):
    from wisp_b200.integrations.vllm import WispMoEStateMX4
    st = WispMoEStateMX4(*experts(E, H, I, 5), cap, DEV, 0, mode=mode)
    if mode == "resident":
        st.prime_identity()
    x = tokens(3, H, 1)
    w, ids = routing(3, E, 2, 1)
    before = st._read()
    wide = torch.empty(3, 2 * H, dtype=torch.bfloat16, device=DEV)
    for error, args, out in [
            (TypeError, (x.half(), w, ids), None), (TypeError, (x, w, ids.to(torch.int16)), None),
            (ValueError, (x.cpu(), w, ids), None), (ValueError, (x, w.cpu(), ids), None),
            (ValueError, (x, w, ids.cpu()), None), (ValueError, (x, w, ids), torch.empty_like(x).cpu()),
            (ValueError, (x, w, ids), torch.empty(4, H, dtype=torch.bfloat16, device=DEV)),
            (ValueError, (x, w, ids), torch.empty(2, H, dtype=torch.bfloat16, device=DEV)),
            (ValueError, (x, w, ids), torch.empty(3, H, device=DEV)), (ValueError, (x, w, ids), wide[:, :H])]:
        with pytest.raises(error):
            st.forward(*args, out=out)
    assert st._read() == before
    st.close()


@pytest.mark.parametrize("mode,cap,T", [("paged", 3, 9), ("paged", E, 100), ("resident", E, 150)])
def test_result_in_the_memory_of_the_tokens(mode, cap, T):
    """In their place, and a row further on, where a group's rows are the next one's tokens."""
    from wisp_b200.integrations.vllm import WispMoEStateMX4
    st = WispMoEStateMX4(*experts(E, H, I, 6), cap, DEV, 0, mode=mode)
    if mode == "resident":
        st.prime_identity()
    w, ids = routing(T, E, 2, 3)
    buf = tokens(T + 1, H, 2)
    keep = buf.clone()
    for a, b in ((0, 0), (0, 1), (1, 0)):
        buf.copy_(keep)
        want = st.forward(buf[a:a + T].clone(), w, ids)
        assert torch.equal(st.forward(buf[a:a + T], w, ids, out=buf[b:b + T]), want), (a, b)
    st.synchronize()
    st.close()


@pytest.mark.parametrize("mode,cap", [("paged", 4), ("resident", E)])
def test_synchronize_waits_for_forwards_on_any_stream(held_up, mode, cap):
    from wisp_b200.integrations.vllm import WispMoEStateMX4
    st = WispMoEStateMX4(*experts(E, H, I, 7), cap, DEV, 0, mode=mode)
    if mode == "resident":
        st.prime_identity()
    x = tokens(1, H, 1)
    w, ids = routing(1, E, 2, 1)
    torch.cuda.synchronize()
    done = torch.cuda.Event()
    with torch.cuda.stream(torch.cuda.Stream()):
        st.forward(x, w, ids)
        done.record()
    st.synchronize()
    assert done.query()
    st.close()


@pytest.mark.parametrize("T", [1, 70])
def test_resident_forward_in_a_graph(T):
    """One launch, and two of them; between replays the layer is used as usual."""
    from wisp_b200.integrations.vllm import WispMoEStateMX4
    st = WispMoEStateMX4(*experts(E, H, I, 8), E, DEV, 0, mode="resident")
    st.prime_identity()
    x, out = tokens(T, H, 9), torch.empty(T, H, dtype=torch.bfloat16, device=DEV)
    w, ids = routing(T, E, 3, 10)
    st.forward(x, w, ids)
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        st.forward(x, w, ids, out=out)
    for _ in range(3):
        x.mul_(-0.75)
        graph.replay()
        assert torch.equal(out, st.forward(x, w, ids))
        st.synchronize()
    st.close()
