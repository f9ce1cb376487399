"""The page cache on the GPU against its rules on Python lists."""

import random

import pytest
import torch

from tests.dense_util import PAGE, PagesModel
from interattn_b200 import _lib, ops, page_cache

pytestmark = pytest.mark.gpu


def i32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def make(n_pages, n_rows, max_pages, layers=2, hkv=2, d=64, dtype=torch.bfloat16, strided=False):
    """A cache whose page p holds numbers that name (layer, k or v, page, head, token)."""
    pools = []
    for layer in range(layers):
        pair = []
        for which in range(2):
            shape = (n_pages, hkv, PAGE, d)
            if strided:   # heads outermost, as a static cache addressed in place has them
                x = torch.zeros((hkv, n_pages, PAGE, d), dtype=dtype, device="cuda").transpose(0, 1)
            else:
                x = torch.zeros(shape, dtype=dtype, device="cuda")
            g = torch.Generator(device="cuda").manual_seed(2 * layer + which)
            x.copy_(torch.randn(shape, generator=g, device="cuda", dtype=torch.float32).to(dtype))
            pair.append(x)
        pools.append(tuple(pair))
    cache = page_cache.PageCache(pools, torch.full((n_rows, max_pages), -1, dtype=torch.int32, device="cuda"),
                                 torch.zeros((n_rows,), dtype=torch.int32, device="cuda"),
                                 torch.zeros((n_pages,), dtype=torch.int32, device="cuda"))
    return cache, PagesModel(n_pages, n_rows, max_pages), [(k.clone(), v.clone()) for k, v in pools]


def same(cache, model, pools=None):
    assert cache.seq_lens.tolist() == model.lens
    assert cache.refs.tolist() == model.refs
    table = cache.block_table.tolist()
    for row, pages in zip(table, model.rows):
        assert row[:len(pages)] == pages
    if pools is not None:
        live = torch.tensor([p for p, r in enumerate(model.refs) if r], dtype=torch.long, device="cuda")
        came_from = torch.tensor(model.contents, device="cuda")[live]
        for pair, before in zip(cache.pools, pools):
            for x, y in zip(pair, before):
                assert torch.equal(x[live], y[came_from])


@pytest.mark.parametrize("strided", [False, True])
@pytest.mark.parametrize("dtype,d", [(torch.bfloat16, 128), (torch.bfloat16, 64), (torch.float32, 64), (torch.float32, 128)])
def test_extend_fork_free_compact(dtype, d, strided):
    cache, model, pools = make(61, 9, 12, d=d, dtype=dtype, strided=strided)
    cache.extend(i32([3, 0, 5, 1]), i32([1, 33, 0, 160])), model.extend([3, 0, 5, 1], [1, 33, 0, 160])
    same(cache, model, pools)
    cache.fork(i32([0, 1, 0, 3, 5]), i32([2, 4, 6, 7, 8])), model.fork([0, 1, 0, 3, 5], [2, 4, 6, 7, 8], True)
    same(cache, model, pools)
    cache.free(i32([1, 5, 6])), model.free([1, 5, 6])
    same(cache, model, pools)
    cache.fork(i32([4, 2]), i32([1, 6]), share=False), model.fork([4, 2], [1, 6], False)
    same(cache, model, pools)
    cache.free(i32([4, 0])), model.free([4, 0])
    cache.compact(), model.compact()
    same(cache, model, pools)
    cache.compact(), model.compact()     # nothing left to move
    same(cache, model, pools)
    cache.extend(i32([1]), i32([16])), model.extend([1], [16])
    same(cache, model, pools)
    assert ops.device_status() == 0


@pytest.mark.parametrize("seed", range(6))
def test_random_calls(seed):
    rng = random.Random(seed)
    n_pages, n_rows, max_pages = rng.choice([(40, 6, 9), (300, 40, 30), (9000, 100, 200), (70000, 30, 4000)])
    cache, model, pools = make(n_pages, n_rows, max_pages, layers=1, hkv=1)
    for _ in range(30):
        what = rng.choice(["extend", "extend", "fork", "copy", "free", "compact"])
        some = rng.sample(range(n_rows), rng.randint(1, n_rows))
        if what == "extend":
            counts = [rng.choice([0, 1, 15, 16, 17, rng.randint(0, max_pages * 4)]) for _ in some]
            cache.extend(i32(some), i32(counts)), model.extend(some, counts)
        elif what in ("fork", "copy"):
            parents = [rng.randrange(n_rows) for _ in some]
            cache.fork(i32(parents), i32(some), share=what == "fork"), model.fork(parents, some, what == "fork")
        elif what == "free":
            cache.free(i32(some)), model.free(some)
        else:
            cache.compact(), model.compact()
        same(cache, model, pools)
    status = ops.device_status()
    assert bool(status & _lib.IA_DEV_STATUS_BAD_INDEX) == model.bad and bool(status & _lib.IA_DEV_STATUS_NO_PAGES) == model.full


@pytest.mark.parametrize("aligned", [True, False])
@pytest.mark.parametrize("n_pages,n_rows", [(1, 3), (127, 5), (129, 256), (4099, 257), (16384, 30), (16385, 30), (32768, 256), (32769, 7),
                                            (70001, 40)])
def test_pools_and_lists_around_the_plans_sizes(n_pages, n_rows, aligned):
    """Free pages scattered over the whole pool, also where the counts begin between 16-byte boundaries."""
    rng = random.Random(n_pages + n_rows)
    max_pages = max(1, 2 * n_pages // n_rows)
    pool = torch.arange(n_pages, device="cuda", dtype=torch.float32).view(-1, 1, 1, 1).expand(n_pages, 1, PAGE, 64).contiguous()
    refs = torch.zeros((n_pages + 1,), dtype=torch.int32, device="cuda")[0 if aligned else 1:][:n_pages]
    cache = page_cache.PageCache([(pool, pool.clone())], torch.full((n_rows, max_pages), -1, dtype=torch.int32, device="cuda"),
                                 i32([0] * n_rows), refs)
    model = PagesModel(n_pages, n_rows, max_pages)
    rows = list(range(n_rows))
    for _ in range(2):
        counts = [rng.randint(0, max(1, n_pages // n_rows) * 14) for _ in rows]
        counts = [min(c, max_pages * PAGE - n) for c, n in zip(counts, model.lens)]
        cache.extend(i32(rows), i32(counts)), model.extend(rows, counts)
        gone = rng.sample(rows, n_rows // 2)
        cache.free(i32(gone)), model.free(gone)
        same(cache, model)
    parents = [rng.choice([r for r in rows if r not in gone]) for _ in gone]
    share = n_rows % 2 == 0
    cache.fork(i32(parents), i32(gone), share=share), model.fork(parents, gone, share)
    same(cache, model)
    gone = rng.sample(rows, n_rows // 3)
    cache.free(i32(gone)), model.free(gone)
    cache.compact(), model.compact()
    same(cache, model)
    live = [p for p, r in enumerate(model.refs) if r]
    want = torch.tensor(model.contents, device="cuda")[live].float()
    assert all(torch.equal(x[live, 0, 0, 0], want) and torch.equal(x[live, 0, 15, 63], want) for x in cache.pools[0])
    assert bool(ops.device_status() & _lib.IA_DEV_STATUS_NO_PAGES) == model.full and not model.bad


def test_refused_entries_change_nothing():
    cache, model, pools = make(20, 6, 8)
    cache.extend(i32([0, 1]), i32([20, 40])), model.extend([0, 1], [20, 40])
    before = cache.block_table.clone()
    assert ops.device_status() == 0
    rows, counts = [0, 9, -1, 0, 1, 2], [-1, 5, 5, 3, 8 * PAGE - 39, 2 ** 31 - 1]
    cache.extend(i32(rows), i32(counts)), model.extend(rows, counts)     # nothing of this is served: 0 is named first with -1
    same(cache, model, pools)
    assert torch.equal(cache.block_table, before) and ops.device_status() == _lib.IA_DEV_STATUS_BAD_INDEX
    parents, children = [0, 0, 6, 1, 0, 0], [0, 1, 2, -3, 3, 3]     # itself, occupied, no such parent, no such child, twice
    cache.fork(i32(parents), i32(children)), model.fork(parents, children, True)
    same(cache, model, pools)
    assert model.lens[3] == 20 and ops.device_status() == _lib.IA_DEV_STATUS_BAD_INDEX
    cache.free(i32([7, 3, 3, 5])), model.free([7, 3, 3, 5])
    same(cache, model, pools)
    assert ops.device_status() == _lib.IA_DEV_STATUS_BAD_INDEX


def test_out_of_pages_keeps_the_rest_as_it_was():
    cache, model, pools = make(10, 5, 8)
    cache.extend(i32([0, 1, 2, 3]), i32([48, 80, 48, 0])), model.extend([0, 1, 2, 3], [48, 80, 48, 0])
    same(cache, model, pools)
    assert model.lens[:4] == [48, 80, 0, 0] and ops.device_status() == _lib.IA_DEV_STATUS_NO_PAGES
    cache.fork(i32([0, 1]), i32([2, 3]), share=False), model.fork([0, 1], [2, 3], False)
    same(cache, model, pools)
    assert ops.device_status() == _lib.IA_DEV_STATUS_NO_PAGES
    cache.fork(i32([0, 1]), i32([2, 3])), model.fork([0, 1], [2, 3], True)     # whole pages need no page
    same(cache, model, pools)
    assert ops.device_status() == 0


@pytest.mark.parametrize("dtype,hkv,d", [(torch.bfloat16, 8, 128), (torch.float32, 2, 64), (torch.bfloat16, 3, 64),
                                         (torch.float32, 1, 128)])
def test_write(dtype, hkv, d):
    cache, model, _ = make(40, 5, 10, hkv=hkv, d=d, dtype=dtype)
    lens = [37, 0, 1, 16]
    rows = [4, 0, 2, 1]
    cache.extend(i32(rows), i32(lens)), model.extend(rows, lens)
    want = [(k.clone(), v.clone()) for k, v in cache.pools]
    total = sum(lens)
    fused = torch.randn((total + 3, 2, hkv + 1, d), device="cuda").to(dtype)      # strided views; three tokens nobody names
    k, v = fused[:, 0, :hkv], fused[:, 1, 1:]
    starts, at = [0], 0
    for row, n in zip(rows, lens):
        for t in range(n):
            page, slot = model.rows[row][t // PAGE], t % PAGE
            want[1][0][page, :, slot] = k[at + t]
            want[1][1][page, :, slot] = v[at + t]
        at += n
        starts.append(at)
    cache.write(1, i32(rows), i32(starts), k, v)
    for got, exp in zip(cache.pools, want):
        assert torch.equal(got[0], exp[0]) and torch.equal(got[1], exp[1])
    # one more token each, at the end of what is there
    cache.extend(i32([4, 2]), i32([1, 1])), model.extend([4, 2], [1, 1])
    cache.write(0, i32([4, 2]), i32([0, 1, 2]), k[:2], v[:2])
    for i, (row, pos) in enumerate([(4, 37), (2, 1)]):
        assert torch.equal(cache.pools[0][0][model.rows[row][pos // PAGE], :, pos % PAGE], k[i])
        assert torch.equal(cache.pools[0][1][model.rows[row][pos // PAGE], :, pos % PAGE], v[i])
    assert ops.device_status() == 0


def test_write_refuses_what_does_not_fit():
    cache, model, _ = make(10, 3, 4)
    cache.extend(i32([0, 1]), i32([5, 5]))
    want = [(k.clone(), v.clone()) for k, v in cache.pools]
    k = torch.ones((30, 2, 64), device="cuda", dtype=torch.bfloat16)
    cache.write(0, i32([0, 3, 2]), i32([0, 6, 8, 10]), k, k)      # longer than the row, no such row, an empty row
    assert ops.device_status() == _lib.IA_DEV_STATUS_BAD_INDEX
    for got, exp in zip(cache.pools, want):
        assert torch.equal(got[0], exp[0]) and torch.equal(got[1], exp[1])
    cache.write(0, i32([0, 0]), i32([0, 2, 4]), k, 2 * k)         # a row named twice: the first counts
    assert ops.device_status() == _lib.IA_DEV_STATUS_BAD_INDEX
    page = int(cache.block_table[0, 0])
    assert float(cache.pools[0][0][page, :, 3:5].float().sum()) == 2 * 2 * 64
    page = int(cache.block_table[1, 0])
    assert torch.equal(cache.pools[0][0][page], want[0][0][page])
    before = [(k.clone(), v.clone()) for k, v in cache.pools]
    for starts in ([0, 31], [-1, 3], [-(2 ** 31), 2 ** 31 - 1], [5, 2], [2 ** 31 - 5, 2 ** 31 - 1]):      # not these tokens
        cache.write(0, i32([0]), i32(starts), k, k)
        ops.device_status()
    for got, exp in zip(cache.pools, before):
        assert torch.equal(got[0], exp[0]) and torch.equal(got[1], exp[1])


def test_captured_and_on_another_stream():
    cache, model, pools = make(64, 8, 6)
    rows, counts, parents, children = i32([0, 1]), i32([40, 17]), i32([0, 1, 0]), i32([2, 3, 4])
    everyone = i32([0, 1, 2, 3, 4])

    def cycle():
        cache.free(everyone)
        cache.extend(rows, counts)
        cache.fork(parents, children)
        cache.compact()

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        cycle()
    torch.cuda.current_stream().wait_stream(side)
    model.extend([0, 1], [40, 17]), model.fork([0, 1, 0], [2, 3, 4], True), model.compact()
    same(cache, model)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        cycle()
    counts.copy_(i32([3, 90]))
    for _ in range(3):
        graph.replay()
    model.free([0, 1, 2, 3, 4]), model.extend([0, 1], [3, 90]), model.fork([0, 1, 0], [2, 3, 4], True), model.compact()
    same(cache, model)
    assert ops.device_status() == 0
