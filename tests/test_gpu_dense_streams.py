"""What the objects hold for their kernels stays theirs until a stream that they were used on is done, also when the object is dropped
first."""

import pytest
import torch

from tests.test_gpu_dense_attention import i32, paged_case, prompt_case, randn
from interattn_b200 import dense_attention, ops, page_cache

pytestmark = pytest.mark.gpu


def reused(address, size, side, use, drop):
    """Whether memory of `size` bytes that this stream allocates can be the one at `address` while `side` still works on it."""
    del [torch.empty((size,), dtype=torch.uint8, device="cuda") for _ in range(400)][:]      # so that the allocator has some
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        torch.cuda._sleep(1_000_000_000)
        use()
    drop()
    taken = [torch.empty((size,), dtype=torch.uint8, device="cuda") for _ in range(420)]
    busy = not side.query()
    again = any(t.data_ptr() <= address < t.data_ptr() + size for t in taken)
    torch.cuda.synchronize()
    return busy, again


def test_a_dropped_plan_is_not_overwritten():
    q, k, v, plan = prompt_case(8, 2, 64, torch.bfloat16, [200, 31], [200, 31], seed=1)
    want, out = plan.run(q, k, v), []
    box = [plan]
    address, size = plan._plan.data_ptr(), plan._plan.numel() * 4
    del plan
    assert reused(address, size, torch.cuda.Stream(), lambda: out.append(box[0].run(q, k, v)), box.clear) == (True, False)
    assert torch.equal(out[0], want) and ops.device_status() == 0


def test_a_dropped_step_is_not_overwritten():
    q, kv, _ = paged_case(8, 2, 64, torch.float32, [2, 1], [48, 0], [60, 49, 33], seed=2)
    box = [dense_attention.SharedPrefixAttention(kv, [2, 1], i32([48, 0]), 8)]
    want, out = box[0].step(q), []
    address, size = box[0]._plan.data_ptr(), box[0]._plan.numel() * 4
    assert reused(address, size, torch.cuda.Stream(), lambda: out.append(box[0].step(q)), box.clear) == (True, False)
    assert torch.equal(out[0], want) and ops.device_status() == 0


@pytest.mark.parametrize("what", ["_scratch", "_addresses"])
def test_a_dropped_cache_is_not_overwritten(what):
    pools = [(randn((9, 2, 16, 64), torch.bfloat16, 3), randn((9, 2, 16, 64), torch.bfloat16, 4))]
    table, lens, refs = torch.full((3, 4), -1, dtype=torch.int32, device="cuda"), i32([0] * 3), i32([0] * 9)
    box = [page_cache.PageCache(pools, table, lens, refs)]
    rows, n, child = i32([0]), i32([20]), i32([1])

    def use():
        box[0].extend(rows, n)
        box[0].fork(rows, child)

    other = page_cache.PageCache.empty(1, 9, 2, 64, 3, 4)      # a kernel's first launch waits for the GPU: not the ones below
    other.extend(rows, n), other.fork(rows, child)
    held = getattr(box[0], what)
    address, size = held.data_ptr(), held.numel() * held.element_size()
    del held
    assert reused(address, size, torch.cuda.Stream(), use, box.clear) == (True, False)
    assert table[:2, :2].tolist() == [[0, 1], [0, 2]] and lens.tolist() == [20, 20, 0] and ops.device_status() == 0


def test_a_new_cache_is_ready_for_any_stream():
    other = page_cache.PageCache.empty(1, 9, 2, 64, 3, 4)
    pools, state = other.pools, (other.block_table, other.seq_lens, other.refs)
    rows, n, starts, k = i32([0]), i32([16]), i32([0, 16]), randn((16, 2, 64), torch.bfloat16, 6)
    torch.full((1 << 20,), 255, dtype=torch.uint8, device="cuda")      # what the scratch may be made of
    torch.cuda.synchronize()
    torch.cuda._sleep(200_000_000)
    cache = page_cache.PageCache(pools, *state)
    with torch.cuda.stream(torch.cuda.Stream()):
        cache.extend(rows, n)
        cache.write(0, rows, starts, k, k)
    torch.cuda.synchronize()
    assert torch.equal(pools[0][0][0].transpose(0, 1), k) and ops.device_status() == 0


def test_one_object_on_two_streams_and_captured():
    """The streams' use of the object does not get into a capture's way."""
    q, k, v, plan = prompt_case(8, 2, 64, torch.bfloat16, [5, 60], [7000, 2000], seed=5)
    want = plan.run(q, k, v)
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = plan.run(q, k, v)
        graphs.append((graph, y))
    for graph, y in graphs:
        y.zero_()
        graph.replay()
        assert torch.equal(y, want)
    del graphs
