"""What a write may not touch: rows whose tokens were refused, and pages that other rows read too."""

import pytest
import torch

from tests.dense_util import PAGE
from interattn_b200 import _lib, ops, page_cache

pytestmark = pytest.mark.gpu
FULL, BAD = _lib.IA_DEV_STATUS_NO_PAGES, _lib.IA_DEV_STATUS_BAD_INDEX


def i32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def make(n_pages, n_rows, max_pages, taken=0, layers=2, hkv=2, d=64):
    """A cache of random pools whose last `taken` pages someone else holds."""
    g = torch.Generator(device="cuda").manual_seed(n_pages)
    pools = [tuple(torch.randn((n_pages, hkv, PAGE, d), generator=g, device="cuda").bfloat16() for _ in range(2)) for _ in range(layers)]
    return page_cache.PageCache(pools, torch.full((n_rows, max_pages), -1, dtype=torch.int32, device="cuda"), i32([0] * n_rows),
                                i32([0] * (n_pages - taken) + [1] * taken))


def tokens(n, hkv=2, d=64, seed=0):
    g = torch.Generator(device="cuda").manual_seed(1000 + seed)
    return [torch.randn((n, hkv, d), generator=g, device="cuda").bfloat16() for _ in range(2)]


def copies(cache):
    return [(k.clone(), v.clone()) for k, v in cache.pools]


def put(pools, cache, row, pos, k, v):
    """The token at `pos` of `row` in the expected contents of every layer."""
    page = int(cache.block_table[row, pos // PAGE])
    for kp, vp in pools:
        kp[page, :, pos % PAGE], vp[page, :, pos % PAGE] = k, v


def unchanged(cache, want):
    for got, exp in zip(cache.pools, want):
        assert torch.equal(got[0], exp[0]) and torch.equal(got[1], exp[1])


def write_all(cache, rows, starts, k, v):
    for layer in range(len(cache.pools)):
        cache.write(layer, i32(rows), i32(starts), k, v)


SIZES = [40, 33000]     # both forms of the plan


@pytest.mark.parametrize("n_pages", SIZES)
def test_write_after_extend_ran_out_of_pages(n_pages):
    """Parent and child of a sharing fork both want a page and there is one: the refused one must not write into the shared page."""
    cache = make(n_pages, 4, 8, taken=n_pages - 4)
    cache.extend(i32([0, 2]), i32([32, 16]))
    k, v = tokens(48)
    write_all(cache, [0, 2], [0, 32, 48], k, v)
    cache.fork(i32([0]), i32([1]))
    want = copies(cache)
    assert ops.device_status() == 0
    cache.extend(i32([0, 1]), i32([1, 1]))
    k, v = tokens(2, seed=1)
    write_all(cache, [0, 1], [0, 1, 2], k, v)
    assert cache.seq_lens.tolist() == [33, 32, 16, 0] and ops.device_status() == FULL | BAD
    put(want, cache, 0, 32, k[0], v[0])
    unchanged(cache, want)
    write_all(cache, [1], [0, 1], k[1:], v[1:])                # and again, and after nothing was asked for
    cache.extend(i32([1]), i32([0]))
    write_all(cache, [1], [0, 1], k[1:], v[1:])
    assert ops.device_status() == BAD
    unchanged(cache, want)
    cache.free(i32([2]))
    cache.extend(i32([1]), i32([1]))                           # the retry
    write_all(cache, [1], [0, 1], k[1:], v[1:])
    put(want, cache, 1, 32, k[1], v[1])
    unchanged(cache, want)
    assert ops.device_status() == 0


@pytest.mark.parametrize("n_pages", SIZES)
@pytest.mark.parametrize("length", [64, 63])
def test_write_after_extend_met_the_table_s_end(n_pages, length):
    cache = make(n_pages, 3, 4)
    cache.extend(i32([0]), i32([length]))
    k, v = tokens(length)
    write_all(cache, [0], [0, length], k, v)
    cache.fork(i32([0]), i32([1]))
    want = copies(cache)
    n = 65 - length
    k, v = tokens(2 * n, seed=1)
    cache.extend(i32([0, 1]), i32([n, n]))
    write_all(cache, [0, 1], [0, n, 2 * n], k, v)
    assert ops.device_status() == BAD and cache.seq_lens.tolist() == [length, length, 0]
    unchanged(cache, want)


@pytest.mark.parametrize("n_pages", SIZES)
def test_write_after_extend_was_refused_behind_another(n_pages):
    """A row that wants no page itself is refused with those behind the first that does not fit; bad rows and second mentions are not
    what decides about a row's own entry."""
    cache = make(n_pages, 6, 8, taken=n_pages - 4)
    cache.extend(i32([0, 1, 2]), i32([16, 20, 5]))
    want = copies(cache)
    k, v = tokens(5)
    cache.extend(i32([2, 0, 1, 9, 2]), i32([1, 1, 1, 1, 1]))
    assert cache.seq_lens.tolist() == [16, 20, 6, 0, 0, 0] and ops.device_status() == FULL | BAD
    write_all(cache, [2, 0, 1], [0, 1, 2, 3], k, v)
    put(want, cache, 2, 5, k[0], v[0])
    unchanged(cache, want)
    assert ops.device_status() == BAD
    cache.free(i32([0, 1]))
    cache.extend(i32([1, 0]), i32([2, 1]))                     # new sequences in the same rows
    write_all(cache, [1, 0], [0, 2, 3], k, v)
    put(want, cache, 1, 0, k[0], v[0]), put(want, cache, 1, 1, k[1], v[1]), put(want, cache, 0, 0, k[2], v[2])
    unchanged(cache, want)
    assert ops.device_status() == 0


@pytest.mark.parametrize("n_pages", SIZES)
def test_a_row_that_asked_for_nothing_is_not_refused_its_write(n_pages):
    cache = make(n_pages, 3, 8, taken=n_pages - 2)
    cache.extend(i32([0, 1]), i32([16, 5]))
    cache.extend(i32([0, 1]), i32([1, 0]))                     # row 1 stands behind one that does not fit
    assert ops.device_status() == FULL
    want = copies(cache)
    k, v = tokens(5)
    write_all(cache, [1], [0, 5], k, v)
    for t in range(5):
        put(want, cache, 1, t, k[t], v[t])
    unchanged(cache, want)
    assert ops.device_status() == 0


@pytest.mark.parametrize("n_pages", SIZES)
def test_write_into_pages_that_others_read(n_pages):
    """More tokens than were appended since the fork: refused while another row holds the page, whoever of them writes."""
    cache = make(n_pages, 5, 8)
    cache.extend(i32([0]), i32([40]))
    k, v = tokens(40)
    write_all(cache, [0], [0, 40], k, v)
    cache.fork(i32([0, 0]), i32([1, 2]))
    cache.fork(i32([1]), i32([3]), share=False)
    want = copies(cache)
    k, v = tokens(10, seed=1)
    for row in (0, 1):
        write_all(cache, [row], [0, 9], k, v)                  # 8 tokens of the last page are the row's own, the ninth is not
        assert ops.device_status() == BAD
        unchanged(cache, want)
    cache.extend(i32([2]), i32([9]))
    for n in (9, 17):                                          # what was appended, and the copy of the partly filled page
        k, v = tokens(n, seed=n)
        write_all(cache, [2], [0, n], k, v)
        for t in range(n):
            put(want, cache, 2, 49 - n + t, k[t], v[t])
        unchanged(cache, want)
    write_all(cache, [2], [0, 18], *tokens(18, seed=3))
    assert ops.device_status() == BAD
    unchanged(cache, want)
    for row in (3, 1):                                         # the copy shares nothing; the last of them does not any more
        if row == 1:
            cache.free(i32([0, 2]))
        k, v = tokens(30, seed=4 + row)
        write_all(cache, [row], [0, 30], k, v)
        for t in range(30):
            put(want, cache, row, 10 + t, k[t], v[t])
        unchanged(cache, want)
    assert ops.device_status() == 0


def test_pages_that_the_caller_holds_can_be_filled_up():
    """A count of the caller's own on a partly filled page does not keep its row from growing."""
    cache = make(40, 3, 8)
    cache.extend(i32([0]), i32([20]))
    cache.refs[cache.block_table[0, :2].long()] += 1
    want = copies(cache)
    cache.extend(i32([0]), i32([1]))
    k, v = tokens(1)
    write_all(cache, [0], [0, 1], k, v)
    put(want, cache, 0, 20, k[0], v[0])
    unchanged(cache, want)
    assert ops.device_status() == 0


def test_captured_loop_with_a_refused_row():
    """The same captured step, refused for one row, later served."""
    cache = make(12, 4, 8, taken=4)
    cache.extend(i32([0, 2]), i32([32, 64]))
    cache.fork(i32([0]), i32([1]))
    rows, ones, starts = i32([0, 1]), i32([1, 1]), i32([0, 1, 2])
    k, v = tokens(2, seed=1)
    want = copies(cache)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        cache.extend(rows, ones)
        for layer in range(2):
            cache.write(layer, rows, starts, k, v)
    assert ops.device_status() == 0
    cache.refs[7] = 1                                          # one page is left
    graph.replay()
    put(want, cache, 0, 32, k[0], v[0])
    unchanged(cache, want)
    assert ops.device_status() == FULL | BAD
    cache.refs[7] = 0
    graph.replay()
    put(want, cache, 0, 33, k[0], v[0]), put(want, cache, 1, 32, k[1], v[1])
    unchanged(cache, want)
    assert cache.seq_lens.tolist() == [34, 33, 64, 0] and ops.device_status() == 0


TOP = 2 ** 31 - 1


@pytest.mark.parametrize("starts", [[0, 40, 20, 60], [0, 10, 5, 60], [5, 2, 2, 2], [60, 60, 60, 59], [0, 0, -5, 10], [0, 60, 0, 60],
                                    [TOP, -TOP - 1, 0, 60]])
def test_starts_that_fall_are_refused_as_a_whole(starts):
    """Which tokens such a list means cannot be said: nothing is written, and it is reported."""
    cache = make(40, 4, 8)
    cache.extend(i32([0, 1, 2]), i32([40, 40, 40]))
    want = copies(cache)
    write_all(cache, [0, 1, 2], starts, *tokens(60))
    assert ops.device_status() == BAD
    unchanged(cache, want)


@pytest.mark.parametrize("starts,good", [([0, 20, 40, 61], 2), ([-1, 20, 40, 60], [1, 2]), ([0, 30, 60, TOP], 2), ([61, 61, 61, 61], []),
                                         ([TOP - 5, TOP - 3, TOP - 1, TOP], []), ([-TOP - 1, -9, -9, 20], [])])
def test_starts_outside_the_tokens_are_reported(starts, good):
    """Also where no token belongs to such an entry; the others are written."""
    good = list(range(good)) if isinstance(good, int) else good
    cache = make(40, 4, 8)
    cache.extend(i32([0, 1, 2]), i32([40, 40, 40]))
    want = copies(cache)
    k, v = tokens(60)
    write_all(cache, [0, 1, 2], starts, k, v)
    assert ops.device_status() == BAD
    for i in good:
        for t in range(starts[i], starts[i + 1]):
            put(want, cache, i, 40 - starts[i + 1] + t, k[t], v[t])
    unchanged(cache, want)


def test_tokens_before_the_first_and_behind_the_last_start_are_left_out():
    n = 700                                                    # more entries than a CTA has threads
    cache = make(1500, n, 2)
    cache.extend(i32(range(n)), i32([3] * n))
    want = copies(cache)
    k, v = tokens(2 * n + 9)
    starts = [4 + 2 * i for i in range(n + 1)]
    write_all(cache, list(range(n)), starts, k, v)
    for kp, vp in want:
        for pool, x in ((kp, k), (vp, v)):
            pages = cache.block_table[:, 0].long()
            pool[pages, :, 1], pool[pages, :, 2] = x[4:4 + 2 * n:2], x[5:5 + 2 * n:2]
    unchanged(cache, want)
    assert ops.device_status() == 0
    starts[650] = starts[649] - 1
    write_all(cache, list(range(n)), starts, v, k)
    assert ops.device_status() == BAD
    unchanged(cache, want)
