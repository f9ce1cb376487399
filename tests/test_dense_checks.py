"""Host-side behaviour of the dense operators and the page cache, without a GPU: plans, refusals, and what can only be read
from the kernels' sources."""

import ctypes
import os
import re
import struct

import pytest
import torch
from torch._subclasses.fake_tensor import FakeTensorMode

from interattn_b200 import _lib, build, dense_attention, ops, page_cache

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "interattn_b200", "csrc")


@pytest.fixture(scope="module")
def lib():
    build.build()
    return _lib.load()


def ints(values):
    return (ctypes.c_int32 * max(len(values), 1))(*values)


def prompt_plan(lib, q_lens, kv_lens, hkv, group, d, dtype):
    args = (ints(q_lens), ints(kv_lens), len(q_lens), hkv, group, d, dtype)
    words = lib.ia_prompt_plan_ints(*args)
    assert words > 0, lib.ia_last_error_string()
    plan = (ctypes.c_int32 * words)()
    _lib.check(lib.ia_prompt_plan(*args, plan, words))
    return list(plan)


@pytest.mark.parametrize("dtype", [_lib.IA_F32, _lib.IA_BF16])
@pytest.mark.parametrize("hkv,group", [(2, 4), (1, 1), (3, 3), (1, 16), (8, 5)])
@pytest.mark.parametrize("q_lens,kv_lens", [([1], [1]), ([], []), ([0, 5, 0], [7, 5, 0]), ([1000, 3, 64, 129], [1000, 300, 10, 129]),
                                            ([5000] * 7, [9000] * 7), ([3], [20000]), ([40, 1, 0], [5000, 9001, 77]),
                                            ([70], [200])])
def test_prompt_plan_holds_every_token_and_head_once(lib, dtype, hkv, group, q_lens, kv_lens):
    plan = prompt_plan(lib, q_lens, kv_lens, hkv, group, 128, dtype)
    n_items, ctas, _, first = plan[:4]
    begin = plan[8:8 + ctas + 1]
    assert begin[0] == 0 and begin[-1] == n_items and all(a <= b for a, b in zip(begin, begin[1:]))
    items = [plan[first + 8 * i:first + 8 * i + 7] for i in range(n_items)]
    if plan[2] >= 2:    # keys are cut: put the parts of every piece together again
        parts, items = {it[6]: it for it in items}, []
        assert sorted(parts) == list(range(n_items))
        for i in range(plan[2] // 2):
            q_tok, n_tok, head, slot, n, *_ = plan[first + 8 * (n_items + i):first + 8 * (n_items + i) + 8]
            mine = [parts[slot + k] for k in range(n)]
            for a, b in zip(mine, mine[1:]):
                assert a[2] + a[4] == b[2] and a[3] - a[4] == b[3] and a[4] % 128 == 0
            assert all((it[0], it[1], it[5]) == (q_tok, n_tok, head) for it in mine)
            assert all(min(it[3] + n_tok - 1, it[4]) > 0 for it in mine[1:])
            _, _, kv_tok, limit0, *_ = mine[0]
            whole = sum(it[4] for it in mine)
            seq = next(s for s in range(len(q_lens)) if sum(q_lens[:s]) <= q_tok < sum(q_lens[:s + 1]))
            assert whole >= min(kv_lens[seq], limit0 + n_tok - 1) and whole <= kv_lens[seq]
            items.append([q_tok, n_tok, kv_tok, limit0, kv_lens[seq], head])
    seen = set()
    for q_tok, n_tok, kv_tok, limit0, kv_len, head, *_ in items:
        seq = next(s for s in range(len(q_lens)) if sum(q_lens[:s]) <= q_tok < sum(q_lens[:s + 1]))
        assert 0 < n_tok * group <= 256 and kv_tok == sum(kv_lens[:seq]) and kv_len == kv_lens[seq]
        assert limit0 == kv_lens[seq] - q_lens[seq] + (q_tok - sum(q_lens[:seq])) + 1
        assert q_tok + n_tok <= sum(q_lens[:seq + 1])
        for t in range(q_tok, q_tok + n_tok):
            assert (t, head) not in seen
            seen.add((t, head))
    assert len(seen) == sum(q_lens) * hkv


def test_prompt_plan_of_the_longest_sequence(lib):
    """2^30 keys for each of 300 small pieces: what would be an SM's share of them is past 32 bits."""
    plan = prompt_plan(lib, [300], [1 << 30], 30, 4, 128, _lib.IA_BF16)
    items = [plan[plan[3] + 8 * i:plan[3] + 8 * i + 6] for i in range(plan[0])]
    assert all(0 < it[4] <= 1 << 30 and 0 <= it[2] < 1 << 30 and it[3] > 0 for it in items)
    assert sum(it[1] * it[4] for it in items) == 300 * 30 << 30


def test_prompt_plan_shares_the_work_evenly(lib):
    lens = [32768, 100, 5000, 17]
    plan = prompt_plan(lib, lens, lens, 8, 4, 128, _lib.IA_BF16)
    n_items, ctas, _, first = plan[:4]
    keys = [max(0, min(plan[first + 8 * i + 3] + plan[first + 8 * i + 1] - 1, plan[first + 8 * i + 4])) for i in range(n_items)]
    loads = [sum(keys[a:b]) for a, b in zip(plan[8:8 + ctas], plan[9:9 + ctas])]
    assert max(loads) <= 1.02 * sum(loads) / ctas + 256


@pytest.mark.parametrize("dtype,lens,small", [
    (_lib.IA_F32, [130], True), (_lib.IA_F32, [1000], False), (_lib.IA_F32, [300] * 4, False),
    (_lib.IA_BF16, [600], True), (_lib.IA_BF16, [1000], True), (_lib.IA_BF16, [700] * 3, False), (_lib.IA_BF16, [9000], False),
    (_lib.IA_F32, [300, 200, 100, 50], True), (_lib.IA_BF16, [300, 200, 100, 50], True)])
def test_prompt_plan_takes_small_pieces_where_the_busiest_sm_then_ends_first(lib, dtype, lens, small):
    """32 / 8 heads of 128 on 148 SMs; each of the two was timed."""
    plan = prompt_plan(lib, lens, lens, 8, 4, 128, dtype)
    rows = 4 * max(plan[plan[3] + 8 * i + 1] for i in range(plan[0]))
    full = 128 if dtype == _lib.IA_F32 else 256
    assert plan[2] == small and (rows <= full // 2) == small


@pytest.mark.parametrize("dtype,lens,prior,cut", [
    (_lib.IA_F32, [1], [16000], True), (_lib.IA_BF16, [1], [16000], True), (_lib.IA_F32, [100], [8000], True),
    (_lib.IA_BF16, [100], [2000], True), (_lib.IA_F32, [600], [0], True), (_lib.IA_BF16, [4] * 8, [3000] * 8, True),
    (_lib.IA_F32, [1000], [0], False), (_lib.IA_BF16, [600], [0], False), (_lib.IA_BF16, [500], [16000], False),
    (_lib.IA_F32, [500], [16000], False), (_lib.IA_BF16, [64] * 8, [1000] * 8, False)])
def test_prompt_plan_cuts_keys_where_few_pieces_have_many(lib, dtype, lens, prior, cut):
    """32 / 8 heads of 128 on 148 SMs; both sides were timed."""
    plan = prompt_plan(lib, lens, [a + b for a, b in zip(lens, prior)], 8, 4, 128, dtype)
    assert (plan[2] >= 2) == cut and (lib.ia_prompt_workspace_bytes(ints(plan[:8])) > 0) == cut


def busiest_and_mean(plan):
    n_items, ctas, _, first = plan[:4]
    keys = [max(0, min(plan[first + 8 * i + 3] + plan[first + 8 * i + 1] - 1, plan[first + 8 * i + 4])) for i in range(n_items)]
    return max(sum(keys[a:b]) for a, b in zip(plan[8:8 + ctas], plan[9:9 + ctas])), sum(keys) / 148, max(keys)


@pytest.mark.parametrize("n", [73, 74, 75, 150, 400])
def test_prompt_plan_of_one_long_sequence_among_many(lib, n):
    """One token each, one behind 100000 keys: no SM walks them alone, on either side of four pieces an SM."""
    for dtype in (_lib.IA_BF16, _lib.IA_F32):
        plan = prompt_plan(lib, [1] * n, [100000] + [500] * (n - 1), 8, 4, 128, dtype)
        busiest, mean, longest = busiest_and_mean(plan)
        assert plan[2] >= 2 and plan[2] & 1 and longest < 100000
        assert max(busiest if dtype == _lib.IA_BF16 else longest, mean) <= 1.4 * mean
    plan = prompt_plan(lib, [1] * 40, [16000] + [500] * 39, 16, 4, 128, _lib.IA_BF16)
    busiest, mean, _ = busiest_and_mean(plan)
    assert busiest <= 1.4 * mean


@pytest.mark.parametrize("n", [73, 74, 300, 2000])
def test_prompt_plan_takes_small_pieces_for_few_rows_however_many_there_are(lib, n):
    """A single token's four rows never get a tile of 128 in fp32, nor two of them in bf16."""
    for dtype in (_lib.IA_F32, _lib.IA_BF16):
        assert prompt_plan(lib, [1] * n, [500] * n, 8, 4, 128, dtype)[2] & 1


@pytest.mark.parametrize("dtype,q_lens,prior,small,cut", [
    (_lib.IA_F32, [10] * 150, [0] * 150, True, False), (_lib.IA_F32, [20] * 150, [0] * 150, False, False),
    (_lib.IA_F32, [70] * 100, [0] * 100, False, False), (_lib.IA_BF16, [70] * 100, [0] * 100, False, False),
    (_lib.IA_BF16, [40] * 150, [1000] * 150, False, False), (_lib.IA_BF16, [2000] + [30] * 100, [0] * 101, False, False),
    (_lib.IA_BF16, [512] * 12, [16000] + [188] * 11, True, False), (_lib.IA_BF16, [64] * 100, [30000] + [200] * 99, True, True)])
def test_prompt_plan_where_there_are_many_pieces(lib, dtype, q_lens, prior, small, cut):
    """32 / 8 heads of 128 on 148 SMs; both sides were timed."""
    plan = prompt_plan(lib, q_lens, [a + b for a, b in zip(q_lens, prior)], 8, 4, 128, dtype)
    assert bool(plan[2] & 1) == small and (plan[2] >= 2) == cut
    assert lib.ia_prompt_workspace_bytes(ints(plan[:8])) <= 32 * 148 * 128 * 129 * 4


@pytest.mark.parametrize("change,word", [
    (dict(hkv=0), b"kv heads"), (dict(group=17), b"group size"), (dict(d=96), b"head_dim"), (dict(dtype=7), b"dtype"),
    (dict(q=[4, -1]), b"sequence 1"), (dict(kv=[4, -2]), b"sequence 1"), (dict(q=[1 << 30, 1]), b"tokens"),
    (dict(hkv=4096, group=16), b"query heads")])
def test_prompt_plan_refusals(lib, change, word):
    a = dict(q=[4, 4], kv=[4, 4], hkv=2, group=4, d=64, dtype=_lib.IA_BF16)
    a.update(change)
    assert lib.ia_prompt_plan_ints(ints(a["q"]), ints(a["kv"]), 2, a["hkv"], a["group"], a["d"], a["dtype"]) == -1
    assert word in lib.ia_last_error_string()


def tensors(**kw):
    a = dict(q=16, k=16, v=16, out=16, lse=None, q_tok_stride=512, q_head_stride=64, k_tok_stride=128, k_head_stride=64,
             v_tok_stride=128, v_head_stride=64, n_q_tokens=8, n_kv_tokens=8, n_kv_heads=2, group_size=4, head_dim=64,
             dtype=_lib.IA_BF16)
    a.update(kw)
    return bytes(_lib.PromptTensors(**a))


@pytest.mark.parametrize("change,word", [
    (dict(n_kv_heads=4), b"other heads"), (dict(head_dim=128), b"other heads"), (dict(dtype=_lib.IA_F32), b"other heads"),
    (dict(n_q_tokens=7), b"the plan has"), (dict(n_kv_tokens=9), b"the plan has"), (dict(q=None), b"null"), (dict(k=None), b"null"),
    (dict(out=8), b"aligned"), (dict(v=20), b"aligned"), (dict(q_tok_stride=33), b"strides"), (dict(k_head_stride=32), b"strides"),
    (dict(v_tok_stride=130), b"strides"), (dict(), b"overlap"), (dict(q=1 << 20, k=16 + 8 * 8 * 64 * 2 - 16, v=1 << 20), b"overlap"),
    (dict(q=1 << 20, k=1 << 20, v=(1 << 20) - 7 * 256 - 2 * 64 * 2, out=(1 << 20) - 128), b"overlap")])
def test_prompt_call_refusals(lib, change, word):
    plan = prompt_plan(lib, [4, 4], [4, 4], 2, 4, 64, _lib.IA_BF16)
    host = ints(plan[:8])
    assert lib.ia_prompt_attention(tensors(**change), host, 16, None, 0, None) < 0
    assert word in lib.ia_last_error_string()
    assert lib.ia_prompt_attention(tensors(), host, None, None, 0, None) < 0
    plan = prompt_plan(lib, [4, 4], [9000, 9000], 2, 4, 64, _lib.IA_BF16)     # few queries, many keys: cut
    host, fit = ints(plan[:8]), tensors(out=1 << 30, k=1 << 20, v=1 << 20, n_kv_tokens=18000)
    need = lib.ia_prompt_workspace_bytes(host)
    assert need > 0 and lib.ia_prompt_workspace_bytes(None) == -1
    for ws, size in ((None, need), (16, need - 1), (24, need)):
        assert lib.ia_prompt_attention(fit, host, 16, ws, size, None) < 0
        assert b"workspace" in lib.ia_last_error_string()


def test_strides_that_nothing_steps_by_are_not_looked_at(lib):
    """Of one token or one head: torch gives such a dimension any stride.  The call gets past the checks, as far as the next one."""
    plan = prompt_plan(lib, [1], [1], 2, 4, 64, _lib.IA_BF16)
    odd = dict(n_q_tokens=1, n_kv_tokens=1, q_tok_stride=1, k_tok_stride=7, v_tok_stride=0)
    assert lib.ia_prompt_attention(tensors(**odd), ints(plan[:8]), 16, None, 0, None) < 0
    assert b"overlap" in lib.ia_last_error_string()
    plan = prompt_plan(lib, [8], [8], 1, 1, 64, _lib.IA_BF16)
    odd = dict(n_kv_heads=1, group_size=1, q_head_stride=1, k_head_stride=3, v_head_stride=0)
    assert lib.ia_prompt_attention(tensors(**odd), ints(plan[:8]), 16, None, 0, None) < 0
    assert b"overlap" in lib.ia_last_error_string()
    plan = prompt_plan(lib, [8], [8], 1, 4, 64, _lib.IA_BF16)     # one kv head, but four query heads
    assert lib.ia_prompt_attention(tensors(**{**odd, "group_size": 4}), ints(plan[:8]), 16, None, 0, None) < 0
    assert b"strides" in lib.ia_last_error_string()
    for cache, strides, n in ((cache_state(n_kv_heads=1), (1, 64, 128, 64), 4), (cache_state(), (128, 1, 128, 64), 1)):
        assert lib.ia_pages_write(cache, 16, 16, 1, 16, 16, *strides, n, 16, 16, None) < 0
        assert b"strides" in lib.ia_last_error_string()


def test_packed_arguments_match_the_struct():
    assert len(dense_attention._PROMPT_TENSORS(*range(17))) == struct.calcsize("=5Q6q6i") == ctypes.sizeof(_lib.PromptTensors)
    p = _lib.PromptTensors.from_buffer_copy(dense_attention._PROMPT_TENSORS(*range(17)))
    assert [getattr(p, name) or 0 for name, _ in _lib.PromptTensors._fields_] == list(range(17))


def geom(**kw):
    a = dict(batch=5, n_kv_heads=2, group_size=4, head_dim=64, page_size=16, block_size=16, max_pages=8, max_blocks=1,
             dtype=_lib.IA_BF16, n_pool_pages=64, pool_page_stride=2048, pool_head_stride=1024)
    a.update(kw)
    return _lib.Geom(**a)


@pytest.mark.parametrize("dtype", [_lib.IA_F32, _lib.IA_BF16])
@pytest.mark.parametrize("groups,group", [([5], 4), ([1] * 9, 1), ([100, 1, 33], 4), ([70], 16), ([300], 1), ([43, 2], 3)])
def test_shared_plan_puts_every_sequence_into_one_shared_part(lib, dtype, groups, group):
    batch = sum(groups)
    g = geom(batch=batch, group_size=group, dtype=dtype)
    words = lib.ia_shared_prefix_plan_ints(ints(groups), len(groups), ctypes.byref(g))
    plan = (ctypes.c_int32 * words)()
    _lib.check(lib.ia_shared_prefix_plan(ints(groups), len(groups), ctypes.byref(g), plan, words))
    plan = list(plan)
    n = plan[0]
    entities = [plan[8 + 8 * e:16 + 8 * e] for e in range(n + batch)]
    info = plan[8 + 8 * (n + batch):]
    seq = 0
    for e, (first, count, group_first, group_n, which, *_) in enumerate(entities[:n]):
        assert first == seq and 0 < count * group <= 256 and group_first <= first and first + count <= group_first + group_n
        assert (group_first, group_n) == (sum(groups[:which]), groups[which])
        for i in range(count):
            assert info[2 * (first + i):2 * (first + i) + 2] == [e, i]
        seq += count
    assert seq == batch
    for b, ent in enumerate(entities[n:]):
        assert ent[:4] == [b, 1, b, 1]
    assert lib.ia_shared_prefix_workspace_bytes(n, ctypes.byref(g)) > 0


def test_shared_plan_fp32_units_follow_the_rows(lib):
    """Keys of a unit: 64 where all entities are of few rows, longer for the few among many."""
    def units(groups, group):
        g = geom(batch=sum(groups), group_size=group, dtype=_lib.IA_F32)
        words = lib.ia_shared_prefix_plan_ints(ints(groups), len(groups), ctypes.byref(g))
        plan = (ctypes.c_int32 * words)()
        _lib.check(lib.ia_shared_prefix_plan(ints(groups), len(groups), ctypes.byref(g), plan, words))
        return {(plan[8 * e + 9] * group, plan[8 * e + 13]) for e in range(plan[0] + sum(groups))}
    assert units([4, 1, 3], 4) == {(4, 64), (12, 64), (16, 64)}
    assert units([1, 8, 16, 32, 40], 4) == {(4, 512), (32, 128), (64, 64), (128, 64)}


def test_shared_refusals(lib):
    for groups in ([4], [3, 3], [5, 0], [6, -1]):
        assert lib.ia_shared_prefix_plan_ints(ints(groups), len(groups), ctypes.byref(geom())) == -1
    assert lib.ia_shared_prefix_plan_ints(ints([5]), 1, ctypes.byref(geom(max_pages=1 << 27))) == -1
    assert lib.ia_shared_prefix_plan_ints(ints([5]), 1, ctypes.byref(geom(head_dim=80))) == -1
    short = (ctypes.c_int32 * 4)()
    assert lib.ia_shared_prefix_plan(ints([5]), 1, ctypes.byref(geom()), short, 4) < 0
    assert lib.ia_shared_prefix_workspace_bytes(6, ctypes.byref(geom())) == -1
    need = lib.ia_shared_prefix_workspace_bytes(1, ctypes.byref(geom()))

    def call(q=16, ws=256, size=need, lens=16, out=16, **kw):
        g = geom(**kw)
        return lib.ia_shared_prefix_decode(q, 16, 16, 16, lens, 16, 16, 1, ctypes.byref(g), ws, size, out, None)

    for bad in (dict(q=None), dict(q=24), dict(ws=None), dict(size=need - 1), dict(lens=None), dict(out=4), dict(page_size=32)):
        assert call(**bad) < 0
    assert call(batch=0, q=None) == 0


def cache_state(**kw):
    a = dict(block_table=16, seq_lens=16, refs=16, pools=16, scratch=256, scratch_bytes=1 << 30, page_stride=2048, head_stride=1024,
             n_rows=4, max_pages=8, n_pages=64, n_pools=2, n_kv_heads=2, head_dim=64, dtype=_lib.IA_BF16, reserved=0)
    a.update(kw)
    return ctypes.byref(_lib.PageCacheState(**a))


@pytest.mark.parametrize("change", [dict(block_table=None), dict(refs=None), dict(scratch=None), dict(scratch=128), dict(scratch_bytes=64),
                                    dict(n_rows=0), dict(max_pages=0), dict(n_pages=-1), dict(head_dim=72), dict(dtype=3), dict(reserved=1),
                                    dict(page_stride=512), dict(head_stride=1023), dict(n_rows=1 << 20, max_pages=1 << 12), dict(pools=None)])
def test_page_cache_refusals(lib, change):
    bad = cache_state(**change)
    assert lib.ia_pages_extend(bad, 16, 16, 1, None) < 0
    assert lib.ia_pages_fork(bad, 16, 16, 1, 1, None) < 0
    assert lib.ia_pages_free(bad, 16, 1, None) < 0
    assert lib.ia_pages_compact(bad, None) < 0
    assert lib.ia_pages_write(bad, 16, 16, 1, 16, 16, 128, 64, 128, 64, 4, 16, 16, None) < 0


def test_page_cache_list_refusals(lib):
    good = cache_state()
    for n in (-1, 5):
        assert lib.ia_pages_extend(good, 16, 16, n, None) < 0 and lib.ia_pages_free(good, 16, n, None) < 0
        assert lib.ia_pages_fork(good, 16, 16, n, 0, None) < 0
    assert lib.ia_pages_extend(good, None, 16, 1, None) < 0 and lib.ia_pages_fork(good, 16, None, 1, 0, None) < 0
    assert lib.ia_pages_write(good, 16, 16, 1, 16, 16, 128, 63, 128, 64, 4, 16, 16, None) < 0
    assert lib.ia_pages_write(good, 16, 16, 1, 24, 16, 128, 64, 128, 64, 4, 16, 16, None) < 0
    assert lib.ia_pages_write(good, 16, 16, 1, 16, 16, 128, 64, 128, 64, -1, 16, 16, None) < 0
    for nothing in (lib.ia_pages_extend(good, None, None, 0, None), lib.ia_pages_free(good, None, 0, None),
                    lib.ia_pages_fork(good, None, None, 0, 1, None),
                    lib.ia_pages_write(good, None, None, 0, None, None, 0, 0, 0, 0, 0, None, None, None)):
        assert nothing == 0
    assert lib.ia_pages_scratch_bytes(0, 5) == -1 and lib.ia_pages_scratch_bytes(5, 0) == -1


def test_python_refusals():
    with pytest.raises(ValueError, match="CUDA"):
        dense_attention.PromptAttention([4], 8, 2, 64, device="cpu")
    with pytest.raises(ValueError, match="multiple"):
        dense_attention.PromptAttention([4], 8, 3, 64)
    with pytest.raises(ValueError, match="float16"):
        dense_attention.PromptAttention([4], 8, 2, 64, dtype=torch.float16)
    with pytest.raises(ValueError, match="lengths"):
        dense_attention.PromptAttention([4, -4], 8, 2, 64)
    with pytest.raises(ValueError, match="same sequences"):
        dense_attention.PromptAttention([4], 8, 2, 64, kv_lens=[4, 4])
    with FakeTensorMode():
        new = lambda *shape, dtype=torch.bfloat16, device="cuda:0": torch.empty(shape, dtype=dtype, device=device)  # noqa: E731
        i32 = lambda *shape, **kw: new(*shape, dtype=torch.int32, **kw)  # noqa: E731
        kv = ops.PagedKV(new(9, 2, 16, 64), new(9, 2, 16, 64), i32(3, 4), i32(3), i32(3))
        for shared in (i32(2), i32(1, device="cuda:1"), new(1, dtype=torch.int64), i32(2, 2)[:, 0]):
            with pytest.raises(ValueError, match="shared_lens"):
                dense_attention.SharedPrefixAttention(kv, [3], shared, 8)
        with pytest.raises(ValueError, match="multiple"):
            dense_attention.SharedPrefixAttention(kv, [3], i32(1), 7)
        good = dict(pools=[(new(9, 2, 16, 64), new(9, 2, 16, 64))], block_table=i32(3, 4), seq_lens=i32(3), refs=i32(9))
        for change in (dict(pools=[]), dict(pools=[(new(9, 2, 8, 64), new(9, 2, 8, 64))]), dict(block_table=i32(12)), dict(seq_lens=i32(4)),
                       dict(refs=i32(8)), dict(refs=new(9)), dict(seq_lens=i32(3, device="cuda:1")),
                       dict(pools=[(new(9, 2, 16, 64), new(8, 2, 16, 64))]), dict(block_table=i32(4, 3).t())):
            with pytest.raises(ValueError):
                page_cache.PageCache(**{**good, **change})


@pytest.mark.parametrize("lens", [[4.5], [4.0, 2.25], torch.tensor([3.0, float("nan")]), [float("inf")], [[4]], 4, torch.tensor([1 << 31]), [-0.5]])
def test_lengths_are_whole_numbers(lens):
    """Nothing is rounded on the way in."""
    with pytest.raises(ValueError, match="lengths"):
        dense_attention.PromptAttention(lens, 8, 2, 64)
    with pytest.raises(ValueError, match="lengths"):
        dense_attention.PromptAttention([4], 8, 2, 64, kv_lens=lens)
    assert dense_attention._host_lens("x", []).shape == (0,)
    for good in ((3, 0), torch.tensor([3, 0], dtype=torch.int16), [3.0, 0.0], torch.tensor([3, 0]).double()):
        got = dense_attention._host_lens("x", good)
        assert got.dtype == torch.int32 and got.tolist() == [3, 0]


# ---- read from the sources: a GPU test would see the lack of these by hanging ------------------------------------------

def source(name):
    with open(os.path.join(CSRC, name)) as f:
        return re.sub(r"//[^\n]*", "", f.read())


def test_every_wait_of_the_tensor_core_kernel_is_bounded():
    text = source("dense_attention_tc.cu")
    body = text[text.index("bool mbar_wait_slow("):text.index("bool mbar_wait(")]
    assert "global_timer_ns() - start < kWaitNs" in body
    assert len(re.findall(r"mbarrier\.(?:try|test)_wait", text)) == 2      # in mbar_try and mbar_test, nowhere else
    assert "bar.sync" not in text                                          # sets meet at mbarriers only


def test_tensor_core_kernel_leaves_nothing_in_flight():
    text = source("dense_attention_tc.cu")
    copy = text[text.index("struct CopyRole"):text.index("struct MmaRole")]
    assert re.search(r"if \(!alive\) \{\s*for \(uint32_t i = it > C::stages.*?full\[i % C::stages\].*?q_full\[i & 1\]", copy, re.S)
    mma = text[text.index("struct MmaRole"):text.index("softmax_role(")]
    assert re.search(r"umma_commit\(&bars->drain\).*?wait\(&bars->drain, 0\)", mma, re.S)


def test_page_plan_waits_for_the_cluster_before_it_reads_a_peer():
    text = source("page_cache.cu")
    for kernel in ("pages_plan_kernel(const PlanParams", "pages_compact_plan_kernel(const CompactParams"):
        body = text[text.index(kernel):]
        assert 0 < body.index("if constexpr (CTAS > 1) sync_all<CTAS>()") < body.index("scan<CTAS>(")
    scan = text[text.index("Sums scan("):]
    assert scan.index("sync_all<CTAS>()") < scan.index("peer_word(")


def test_shared_workspace_does_not_grow_with_the_group_sizes(lib):
    """Partial rows: one per query row and part, and one block per SM - also for many groups of one."""
    for dtype in (_lib.IA_F32, _lib.IA_BF16):
        g = geom(batch=2048, n_kv_heads=8, dtype=dtype)
        for n_shared in (8, 2048):
            rows = 2 * 2048 * 32 + 160 * 256
            assert lib.ia_shared_prefix_workspace_bytes(n_shared, ctypes.byref(g)) <= rows * 65 * 4 + 8 * 4200 + 1024
