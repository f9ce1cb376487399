"""Prompt attention and the shared-prefix decode step against the formula in float64."""

import pytest
import torch

from tests.dense_util import PAGE, decode_reference, prompt_reference
from interattn_b200 import _lib, dense_attention, ops, page_cache

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32
GEOMETRIES = [(8, 2, 64, BF16), (8, 2, 128, BF16), (8, 2, 64, F32), (4, 1, 128, F32), (3, 3, 64, BF16), (6, 2, 128, BF16),
              (16, 1, 128, BF16), (14, 2, 64, BF16), (5, 1, 64, F32), (16, 1, 64, F32), (2, 2, 128, BF16)]


def randn(shape, dtype, seed, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * scale).to(dtype).cuda()


def i32(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def prompt_case(hq, hkv, d, dtype, q_lens, kv_lens, seed=0):
    q = randn((sum(q_lens), hq, d), dtype, seed, 1.5)
    k, v = randn((sum(kv_lens), hkv, d), dtype, seed + 1), randn((sum(kv_lens), hkv, d), dtype, seed + 2)
    plan = dense_attention.PromptAttention(q_lens, hq, hkv, d, kv_lens=kv_lens, dtype=dtype)
    return q, k, v, plan


@pytest.mark.parametrize("hq,hkv,d,dtype", GEOMETRIES)
@pytest.mark.parametrize("q_lens,kv_lens", [
    ([1], [1]), ([0, 3, 0], [0, 3, 0]), ([127, 1, 128, 129], None), ([300, 17], None),
    ([5, 64, 1, 2], [200, 64, 129, 257]),          # continued prompts
    ([40, 3, 7], [10, 0, 6]),                      # rows that see nothing
])
def test_prompt(hq, hkv, d, dtype, q_lens, kv_lens):
    kv_lens = q_lens if kv_lens is None else kv_lens
    q, k, v, plan = prompt_case(hq, hkv, d, dtype, q_lens, kv_lens)
    ref = prompt_reference(q, k, v, q_lens, kv_lens)
    out, lse = plan.run(q, k, v, return_lse=True)
    assert ops.device_status() == 0
    ref.check(out, dtype)
    ref.check_lse(lse)
    assert torch.equal(plan.run(q, k, v), out)      # the same bits again, and without the log-sum-exp


@pytest.mark.parametrize("hq,hkv,d,dtype", GEOMETRIES)
@pytest.mark.parametrize("q_lens,kv_lens", [
    ([3], [9000]), ([1, 17, 0], [5000, 3001, 64]), ([64, 5], [2100, 4000]), ([100, 1], [2600, 4099]),
    ([4, 9], [3, 6000]),                           # one whose first query sees nothing
])
def test_prompt_few_queries_many_keys(hq, hkv, d, dtype, q_lens, kv_lens):
    """The keys of a piece are cut and the parts merged."""
    q, k, v, plan = prompt_case(hq, hkv, d, dtype, q_lens, kv_lens, seed=40)
    assert plan._ws_bytes > 0
    k = (k.float() * torch.linspace(0.05, 3.0, k.shape[0], device="cuda")[:, None, None]).to(dtype)
    ref = prompt_reference(q, k, v, q_lens, kv_lens)
    out, lse = plan.run(q, k, v, return_lse=True)
    assert ops.device_status() == 0
    ref.check(out, dtype)
    ref.check_lse(lse)
    assert torch.equal(plan.run(q, k, v), out)


@pytest.mark.parametrize("dtype,d", [(BF16, 128), (BF16, 64), (F32, 64)])
@pytest.mark.parametrize("poison", [float("nan"), float("inf"), float("-inf")])
@pytest.mark.parametrize("back", [1, 3, 40])
def test_prompt_cut_keys_bad_places(dtype, d, poison, back):
    """A bad value that only the last `back` queries see, and a neighbour's keys behind the end."""
    q_lens, kv_lens = [50, 2], [6000, 3000]
    q, k, v, plan = prompt_case(4, 2, d, dtype, q_lens, kv_lens, seed=41)
    want = plan.run(q, k, v)
    v[6000 - back, 1, 5] = poison
    k[6000:], v[6000:] = poison, poison
    out = plan.run(q, k, v)
    assert plan._ws_bytes > 0 and ops.device_status() == 0
    bad = ~torch.isfinite(out[:50])
    assert bad[50 - back:, 2:, 5].all() and int(bad.sum()) == back * 2
    ref = want[:50].float()
    assert torch.equal(out[:50 - back], want[:50 - back]) or torch.allclose(out[:50 - back].float(), ref[:50 - back], rtol=2 ** -7, atol=2 ** -9)


def test_prompt_cut_keys_captured_and_on_two_streams():
    q_lens, kv_lens = [5, 60], [7000, 2000]
    q, k, v, plan = prompt_case(8, 2, 128, BF16, q_lens, kv_lens, seed=42)
    assert plan._ws_bytes > 0
    want, q2 = plan.run(q, k, v), torch.randn_like(q)
    want2 = plan.run(q2, k, v)
    inputs = [q.clone(), q.clone()]
    graphs = []
    for x in inputs:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            y = plan.run(x, k, v)
        graphs.append((g, y))
    inputs[1].copy_(q2)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(20):
        for (g, _y), s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    assert torch.equal(graphs[0][1], want) and torch.equal(graphs[1][1], want2)


@pytest.mark.parametrize("hq,hkv,d,dtype", [(8, 2, 128, BF16), (8, 2, 64, BF16), (4, 4, 64, F32)])
def test_prompt_of_many_tiles(hq, hkv, d, dtype):
    """Enough pieces that a CTA takes several, with a rising score that moves the running maximum often."""
    q_lens, kv_lens = [900, 1, 450, 513], [900, 1, 1450, 513]
    q, k, v, plan = prompt_case(hq, hkv, d, dtype, q_lens, kv_lens, seed=5)
    k = (k.float() * torch.linspace(0.05, 6.0, k.shape[0], device="cuda")[:, None, None]).to(dtype)
    ref = prompt_reference(q, k, v, q_lens, kv_lens)
    out = plan.run(q, k, v)
    assert ops.device_status() == 0
    ref.check(out, dtype)


@pytest.mark.parametrize("dtype,d", [(BF16, 128), (F32, 64)])
def test_prompt_strided_views(dtype, d):
    """Queries, keys and values as views of one fused projection."""
    hq, hkv, lens = 8, 2, [70, 33]
    fused = randn((sum(lens), (hq + 2 * hkv) * d), dtype, 3).view(sum(lens), hq + 2 * hkv, d)
    q, k, v = fused[:, :hq], fused[:, hq:hq + hkv], fused[:, hq + hkv:]
    plan = dense_attention.PromptAttention(lens, hq, hkv, d, dtype=dtype)
    out = plan.run(q, k, v)
    assert torch.equal(out, plan.run(q.contiguous(), k.contiguous(), v.contiguous()))
    prompt_reference(q, k, v, lens, lens).check(out, dtype)
    heads_first = q.transpose(0, 1).contiguous().transpose(0, 1)
    assert torch.equal(out, plan.run(heads_first, k, v))


def test_prompt_output_may_not_overlap_what_is_read():
    q, k, v, plan = prompt_case(2, 2, 64, BF16, [5, 9], [5, 9], seed=4)
    for out in (q, k, v):
        with pytest.raises(ValueError, match="overlap"):
            plan.run(q, k, v, out=out)
    both = torch.stack([q, q])
    assert torch.equal(plan.run(both[0], k, v, out=both[1]), plan.run(q, k, v))


@pytest.mark.parametrize("dtype,d,hq,hkv", [(BF16, 128, 8, 2), (BF16, 64, 2, 2), (F32, 64, 4, 2), (F32, 128, 2, 2)])
@pytest.mark.parametrize("poison", [float("nan"), float("inf"), float("-inf"), 3.0e38])
def test_prompt_rows_do_not_see_the_future_or_the_neighbour(dtype, d, hq, hkv, poison):
    lens = [150, 20, 1, 140]
    q, k, v, plan = prompt_case(hq, hkv, d, dtype, lens, lens, seed=11)
    clean, clean_lse = plan.run(q, k, v, return_lse=True)
    at = 100                                          # a token of the first sequence, and the whole second one
    k2, v2 = k.clone(), v.clone()
    k2[at], v2[at] = poison, poison
    k2[150:170], v2[150:170] = poison, poison
    out, lse = plan.run(q, k2, v2, return_lse=True)
    assert ops.device_status() == 0
    keep = list(range(at)) + list(range(170, sum(lens)))
    ref = prompt_reference(q, k, v, lens, lens)
    got = clean.clone()
    got[keep] = out[keep]
    ref.check(got, dtype)
    got_lse = clean_lse.clone()
    got_lse[keep] = lse[keep]
    ref.check_lse(got_lse)
    if poison != poison:
        assert bool(torch.isnan(out[at:170].float()).all())


@pytest.mark.parametrize("dtype,d", [(BF16, 128), (BF16, 64), (F32, 64)])
@pytest.mark.parametrize("poison", [float("nan"), float("inf")])
@pytest.mark.parametrize("at", [0, 15, 24, 31, 63, 100, 127, 129, 158])
def test_prompt_a_bad_key_spoils_exactly_the_rows_that_see_it(dtype, d, poison, at):
    """Wherever in a tile the key lies; a logit of +infinity gives NaN too (infinity minus infinity), one of -infinity does
    not, so the key's sign is taken from the query."""
    lens = [160]
    q, k, v, plan = prompt_case(2, 1, d, dtype, lens, lens, seed=17)
    q = q.abs()
    k[at] = 0
    k[at, :, 0] = poison
    out = plan.run(q, k, v).float()
    bad = torch.isnan(out).flatten(1).all(dim=1).cpu()
    assert ops.device_status() == 0
    assert not bool(torch.isnan(out[:at]).any()) and bool(bad[at:].all())


def test_prompt_graph_streams_and_threads():
    q_lens = [200, 31]
    q, k, v, plan = prompt_case(8, 2, 128, BF16, q_lens, q_lens, seed=7)
    want = plan.run(q, k, v)
    q2 = torch.randn_like(q)
    want2 = plan.run(q2, k, v)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        a = plan.run(q, k, v)
    b = plan.run(q2, k, v)                            # at the same time on this stream
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(a, want) and torch.equal(b, want2)
    graph, buf, out = torch.cuda.CUDAGraph(), q.clone(), torch.empty_like(q)
    with torch.cuda.graph(graph):
        plan.run(buf, k, v, out=out)
    buf.copy_(q2)
    graph.replay()
    assert torch.equal(out, want2)
    buf.copy_(q)
    graph.replay()
    assert torch.equal(out, want)


# ---- the decode step ------------------------------------------------------------------------------------------------

def paged_case(hq, hkv, d, dtype, groups, shared, lens, seed=0, spare=3):
    """Random pages; the sequences of a group have the same leading pages, and a prefix that ends inside a page is copied."""
    g = torch.Generator().manual_seed(seed)
    rows, n_pages, b, copies = [], 0, 0, []
    for n, s in zip(groups, shared):
        full = s // PAGE
        base = n_pages
        n_pages += full
        for i in range(n):
            pages = -(-lens[b] // PAGE)
            own = max(0, pages - full)
            rows.append(list(range(base, base + full))[:max(pages, 0)] + list(range(n_pages, n_pages + own)))
            if s % PAGE and own:
                copies.append((b, n, full, s % PAGE))
            n_pages += own
            b += 1
    total = n_pages + spare
    perm = torch.randperm(total, generator=g)
    width = max([len(r) for r in rows] + [1]) + 2
    table = torch.full((len(rows), width), -1, dtype=torch.int32)
    for i, r in enumerate(rows):
        table[i, :len(r)] = perm[torch.tensor(r, dtype=torch.long)].int()
    k_pool, v_pool = randn((total, hkv, PAGE, d), dtype, seed + 1), randn((total, hkv, PAGE, d), dtype, seed + 2)
    lead = 0
    for n, s in zip(groups, shared):
        if s % PAGE:
            have = [i for i in range(lead, lead + n) if lens[i] > s // PAGE * PAGE]
            for i in have[1:]:
                for pool in (k_pool, v_pool):
                    pool[table[i, s // PAGE].long(), :, :s % PAGE] = pool[table[have[0], s // PAGE].long(), :, :s % PAGE]
        lead += n
    kv = ops.PagedKV(k_pool, v_pool, table.cuda(), i32(lens), i32(lens))
    q = randn((len(rows), hq, d), dtype, seed + 3, 1.5)
    return q, kv, table


DECODES = [
    ([1], [0], [1]), ([2], [16], [17, 16]), ([3], [40], [41, 40, 100]), ([1, 4, 2], [0, 300, 129], [77, 301, 300, 420, 555, 129, 130]),
    ([5], [1000], [1000, 1001, 1016, 0, 1500]),      # one row is idle
    ([40], [256], [256 + i for i in range(40)]),     # more rows than one block holds
    ([2, 2], [64, 0], [30, 70, 5, 0]),               # a member shorter than what the others share
    ([3, 2], [200, 50], [0, 210, 333, 0, 0]),        # the first members have left; a whole group has
    ([3], [100], [40, 70, 20]),                      # nobody holds all of it
]


@pytest.mark.parametrize("hq,hkv,d,dtype", GEOMETRIES)
@pytest.mark.parametrize("groups,shared,lens", DECODES)
def test_shared_prefix(hq, hkv, d, dtype, groups, shared, lens):
    q, kv, table = paged_case(hq, hkv, d, dtype, groups, shared, lens)
    step = dense_attention.SharedPrefixAttention(kv, groups, i32(shared), hq)
    out = step.step(q)
    assert ops.device_status() == 0
    decode_reference(q, kv.k_pool, kv.v_pool, table, lens).check(out, dtype)
    assert torch.equal(step.step(q), out)
    alone = dense_attention.SharedPrefixAttention(kv, [1] * len(lens), i32([0] * len(lens)), hq)
    decode_reference(q, kv.k_pool, kv.v_pool, table, lens).check(alone.step(q), dtype)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("group", [1, 4, 5])
@pytest.mark.parametrize("groups", [[1, 2, 3], [4, 1], [8, 5], [13, 1, 16], [17], [31, 3], [32, 1], [33]])
def test_shared_prefix_fp32_row_counts(d, group, groups):
    """Both sides of every row count at which the fp32 step changes its form; members of different lengths, one idle, one
    inside the shared part, own parts from nothing to several units of the longest kind."""
    n = sum(groups)
    shared = [150 + 97 * g for g in range(len(groups))]
    lens, first = [], 0
    for size, split in zip(groups, shared):
        lens += [[split + 41 * i, split, 1200 + i, split // 2, 0][(i + size) % 5] for i in range(size)]
        first += size
    q, kv, table = paged_case(2 * group, 2, d, F32, groups, shared, lens, seed=30)
    step = dense_attention.SharedPrefixAttention(kv, groups, i32(shared), 2 * group)
    out = step.step(q)
    assert ops.device_status() == 0 and out.shape[0] == n
    decode_reference(q, kv.k_pool, kv.v_pool, table, lens).check(out, F32)
    assert torch.equal(step.step(q), out)


@pytest.mark.parametrize("poison", [float("nan"), float("inf"), float("-inf")])
@pytest.mark.parametrize("dtype,hq,groups", [(F32, 4, [1, 1]), (F32, 8, [1, 1]), (F32, 16, [1, 1]), (F32, 8, [5, 1]), (BF16, 8, [1, 1])])
def test_shared_prefix_a_bad_value_spoils_exactly_the_rows_that_see_it(dtype, hq, groups, poison):
    n = sum(groups)
    shared, lens = [0] * len(groups), [100 + 13 * i for i in range(n)]
    q, kv, table = paged_case(hq, 1, 64, dtype, groups, shared, lens, seed=31)
    at = lens[0] - 1  # the first sequence's last token, and the place behind it
    kv.v_pool[table[0, at // 16].long(), :, at % 16, 7] = poison
    kv.v_pool[table[n - 1, lens[n - 1] // 16].long(), :, lens[n - 1] % 16:, 9] = poison
    out = dense_attention.SharedPrefixAttention(kv, groups, i32(shared), hq).step(q)
    bad = ~torch.isfinite(out)
    assert bad[0, :, 7].all() and int(bad.sum()) == hq


@pytest.mark.parametrize("hq,hkv,d,dtype", [(32, 8, 128, BF16), (8, 2, 64, F32)])
def test_shared_prefix_long(hq, hkv, d, dtype):
    """Cut over all SMs; lengths that end inside tiles."""
    groups, shared = [3, 1, 6], [9001, 0, 4444]
    lens = [9001 + 5, 9001 + 700, 9001, 2777, 4444 + 1, 4444 + 16, 4445 + 31, 4444 + 333, 5000, 4460]
    q, kv, table = paged_case(hq, hkv, d, dtype, groups, shared, lens, seed=3)
    step = dense_attention.SharedPrefixAttention(kv, groups, i32(shared), hq)
    out = step.step(q)
    assert ops.device_status() == 0
    decode_reference(q, kv.k_pool, kv.v_pool, table, lens).check(out, dtype)


@pytest.mark.parametrize("dtype,d", [(BF16, 128), (BF16, 64), (F32, 64)])
@pytest.mark.parametrize("poison", [float("nan"), float("inf")])
def test_shared_prefix_unwritten_places_do_not_count(dtype, d, poison):
    """Fresh cache memory behind the last token, and whole pages that no sequence holds, may hold anything."""
    groups, shared, lens = [3, 1], [150, 0], [151, 150, 200, 33]
    q, kv, table = paged_case(8, 2, d, dtype, groups, shared, lens, seed=9)
    want = decode_reference(q, kv.k_pool, kv.v_pool, table, lens)
    seen = torch.zeros(kv.k_pool.shape[:1] + (PAGE,), dtype=torch.bool)
    for b, n in enumerate(lens):
        for t in range(n):
            seen[int(table[b, t // PAGE]), t % PAGE] = True
    for pool in (kv.k_pool, kv.v_pool):
        pool.transpose(1, 2)[~seen.cuda()] = poison
    out = dense_attention.SharedPrefixAttention(kv, groups, i32(shared), 8).step(q)
    assert ops.device_status() == 0
    want.check(out, dtype)


@pytest.mark.parametrize("dtype,d", [(BF16, 128), (F32, 64)])
def test_shared_prefix_shorter_member_next_to_poison(dtype, d):
    """A member that ends inside the shared part must not see what the longer ones see there."""
    groups, shared, lens = [3], [160], [170, 70, 161]
    q, kv, table = paged_case(8, 2, d, dtype, groups, shared, lens, seed=10)
    want = decode_reference(q, kv.k_pool, kv.v_pool, table, lens)
    kv.v_pool[table[0, 6].long(), :, 3] = float("nan")
    out = dense_attention.SharedPrefixAttention(kv, groups, i32(shared), 8).step(q)
    assert bool(torch.isnan(out[[0, 2]].float()).all())
    want.out[[0, 2]], want.mean_abs[[0, 2]] = 0, 0
    out[[0, 2]] = 0
    want.check(out, dtype)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_shared_prefix_in_place_and_with_the_cache_s_fields_replaced(dtype):
    groups, shared, lens = [3, 1], [64, 0], [70, 99, 64, 200]
    q, kv, table = paged_case(8, 2, 64, dtype, groups, shared, lens, seed=33)
    step = dense_attention.SharedPrefixAttention(kv, groups, i32(shared), 8)
    want = step.step(q)
    shape = kv.block_table.shape
    kv.block_table, kv.seq_lens = None, None        # the step holds what it was given
    other = torch.full(shape, 1 << 20, dtype=torch.int32, device="cuda")
    assert step.step(q, out=q) is q and torch.equal(q, want)
    assert ops.device_status() == 0 and other.shape == shape


def test_shared_prefix_bad_entries_are_reported():
    groups, shared, lens = [2], [64], [100, 90]
    for dtype in (BF16, F32):
        for bad in (-1, 10 ** 6):
            for at in (1, 5, 6):                       # a shared page, an own page, the last page of the first sequence
                q, kv, table = paged_case(8, 2, 64, dtype, groups, shared, lens, seed=12)
                kv.block_table[0, at] = bad
                dense_attention.SharedPrefixAttention(kv, groups, i32(shared), 8).step(q)
                assert ops.device_status() == _lib.IA_DEV_STATUS_BAD_INDEX
                if at >= 4:                            # the other sequence is not concerned
                    got = dense_attention.SharedPrefixAttention(kv, groups, i32(shared), 8).step(q)
                    ref = decode_reference(q, kv.k_pool, kv.v_pool, table, lens)
                    ref.out[0], ref.mean_abs[0] = 0, 0
                    got[0] = 0
                    ref.check(got, dtype)
                    ops.device_status()


def test_shared_prefix_captured_steps_follow_the_lengths():
    groups, shared, lens = [2, 1], [48, 0], [60, 49, 33]
    q, kv, table = paged_case(8, 2, 128, BF16, groups, shared, lens, seed=13)
    step = dense_attention.SharedPrefixAttention(kv, groups, i32(shared), 8)
    out = torch.empty_like(q)
    step.step(q, out=out)
    graphs = []
    for _ in range(2):                                 # two graphs of one object on two streams
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = step.step(q)
        graphs.append((graph, y))
    shorter = [50, 48, 20]
    kv.seq_lens.copy_(i32(shorter))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    for _ in range(3):
        graphs[0][0].replay()
        with torch.cuda.stream(side):
            graphs[1][0].replay()
    torch.cuda.current_stream().wait_stream(side)
    ref = decode_reference(q, kv.k_pool, kv.v_pool, table, shorter)
    for _, y in graphs:
        ref.check(y, BF16)
    assert ops.device_status() == 0


# ---- together -------------------------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype,hq,hkv,d", [(BF16, 8, 2, 128), (F32, 8, 2, 64)])
def test_prompts_forks_and_steps_together(dtype, hq, hkv, d):
    """Two prompts are read and written into pages, answered several times each; an answer leaves, the pages close up."""
    layers, lens, answers = 2, [75, 32], [3, 2]
    cache = page_cache.PageCache.empty(layers, 64, hkv, d, 5, 12, dtype=dtype)
    total, leaders = sum(lens), [0, 3]
    starts = i32([0, lens[0], total])
    plan = dense_attention.PromptAttention(lens, hq, hkv, d, dtype=dtype)
    history = [[[], []] for _ in range(5)]            # keys and values of every row, layer 1
    cache.extend(i32(leaders), i32(lens))
    for layer in range(layers):
        q, k, v = randn((total, hq, d), dtype, 20 + layer), randn((total, hkv, d), dtype, 30 + layer), randn((total, hkv, d), dtype, 40 + layer)
        out = plan.run(q, k, v)
        prompt_reference(q, k, v, lens, lens).check(out, dtype)
        cache.write(layer, i32(leaders), starts, k, v)
    cache.fork(i32([0, 0, 3]), i32([1, 2, 4]))
    for row in range(5):
        s = slice(0, lens[0]) if row < 3 else slice(lens[0], total)
        history[row] = [[k[s]], [v[s]]]
    kv = cache.kv(1)
    shared = i32(lens)
    step = dense_attention.SharedPrefixAttention(kv, answers, shared, hq)
    everyone, ones, each = i32([0, 1, 2, 3, 4]), i32([1] * 5), i32(list(range(6)))

    def token(seed):
        cache.extend(everyone, ones)
        k, v = randn((5, hkv, d), dtype, seed), randn((5, hkv, d), dtype, seed + 1)
        for layer in range(layers):
            cache.write(layer, everyone, each, k, v)
        for row in range(5):
            history[row][0].append(k[row:row + 1])
            history[row][1].append(v[row:row + 1])
        q = randn((5, hq, d), dtype, seed + 2)
        out = step.step(q)
        keys, values = [torch.cat(h[0]) for h in history], [torch.cat(h[1]) for h in history]
        n = [len(x) for x in keys]
        ref = prompt_reference(q, torch.cat(keys), torch.cat(values), [1] * 5, n)
        ref.check(out, dtype)

    for i in range(20):
        token(100 + 3 * i)
    cache.free(i32([1]))
    cache.compact()
    cache.fork(i32([2]), i32([1]))
    history[1] = [list(history[2][0]), list(history[2][1])]
    for i in range(3):
        token(200 + 3 * i)
    assert int((cache.refs > 0).sum()) == len(set(cache.block_table.flatten().tolist()) - {-1})
    # and the block-sparse step of the framework reads the same pages
    summ = ops.build_summaries(cache.kv(1), 64, max_blocks=3)
    sparse = ops.DecodeAttention(cache.kv(1), summ, hq, top_k=3)
    q = randn((5, hq, d), dtype, 300)
    keys, values = [torch.cat(h[0]) for h in history], [torch.cat(h[1]) for h in history]
    prompt_reference(q, torch.cat(keys), torch.cat(values), [1] * 5, [len(x) for x in keys])
    torch.testing.assert_close(sparse.step(q).float(), step.step(q).float(), rtol=2e-2, atol=2e-2)
    assert ops.device_status() == 0


# ---- the ends of the ranges -------------------------------------------------------------------------------------------

@pytest.mark.parametrize("dtype,d", [(BF16, 128), (BF16, 64), (F32, 64)])
def test_nothing_to_do(dtype, d):
    plan = dense_attention.PromptAttention([], 8, 2, d, dtype=dtype)
    none_q, none_k = torch.empty((0, 8, d), dtype=dtype, device="cuda"), torch.empty((0, 2, d), dtype=dtype, device="cuda")
    assert plan.run(none_q, none_k, none_k).shape == (0, 8, d)
    plan = dense_attention.PromptAttention([3, 0], 8, 2, d, kv_lens=[0, 0], dtype=dtype)     # queries, but no key anywhere
    out, lse = plan.run(randn((3, 8, d), dtype, 0), none_k, none_k, return_lse=True)
    assert not out.any() and bool((lse == float("-inf")).all())
    pool = torch.zeros((1, 2, PAGE, d), dtype=dtype, device="cuda")
    kv = ops.PagedKV(pool, pool, torch.zeros((0, 1), dtype=torch.int32, device="cuda"), i32([]), i32([]))
    assert dense_attention.SharedPrefixAttention(kv, [], i32([]), 8).step(none_q).shape == (0, 8, d)
    kv = ops.PagedKV(pool, pool, torch.full((2, 1), -1, dtype=torch.int32, device="cuda"), i32([0, 0]), i32([0, 0]))
    out = dense_attention.SharedPrefixAttention(kv, [2], i32([16]), 8).step(randn((2, 8, d), dtype, 1))
    assert not out.any() and ops.device_status() == 0


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_offsets_past_32_bits(dtype):
    """Tokens and pages far apart in large tensors: element offsets beyond 2^32, byte offsets beyond 2^33."""
    hq, hkv, d, n = 4, 2, 64, 70
    gap = 1 << 26                                            # elements between tokens, and between pages
    flat = torch.empty((n * gap,), dtype=dtype, device="cuda")
    far = lambda heads, at: flat[at:].as_strided((n, heads, d), (gap, d, 1))  # noqa: E731
    q, k, v = far(hq, 0), far(hkv, hq * d), far(hkv, (hq + hkv) * d)
    for i, t in enumerate((q, k, v)):
        t.copy_(randn(t.shape, dtype, 50 + i))
    lens = [n - 3, 3]
    plan = dense_attention.PromptAttention(lens, hq, hkv, d, dtype=dtype)
    prompt_reference(q, k, v, lens, lens).check(plan.run(q, k, v), dtype)
    pages = n - 1
    pools = [flat[at:].as_strided((pages, hkv, PAGE, d), (gap, PAGE * d, d, 1)) for at in (4096, 16384)]
    for i, t in enumerate(pools):
        t.copy_(randn(t.shape, dtype, 60 + i))
    table = torch.arange(pages - 1, -1, -1, dtype=torch.int32).view(3, -1)
    seq = [300, 301, 368]
    kv = ops.PagedKV(*pools, table.cuda(), i32(seq), i32(seq))
    q = randn((3, hq, d), dtype, 70)
    out = dense_attention.SharedPrefixAttention(kv, [1, 1, 1], i32([100, 0, 368]), hq).step(q)
    decode_reference(q, *pools, table, seq).check(out, dtype)
    cache = page_cache.PageCache([tuple(pools)], torch.full((4, 30), -1, dtype=torch.int32, device="cuda"), i32([0] * 4),
                                 i32([1] * 40 + [0] * (pages - 40)))
    cache.extend(i32([0]), i32([40]))
    kk, vv = randn((40, hkv, d), dtype, 71), randn((40, hkv, d), dtype, 72)
    cache.write(0, i32([0]), i32([0, 40]), kk, vv)
    cache.fork(i32([0]), i32([1]), share=False)
    assert cache.block_table[:2, :3].tolist() == [[40, 41, 42], [43, 44, 45]]
    got = pools[1][43:46].transpose(1, 2).reshape(48, hkv, d)[:40]
    assert torch.equal(got, vv) and ops.device_status() == 0


@pytest.mark.parametrize("seed", range(8))
def test_random_batches(seed):
    """Lengths, groups and heads as they come."""
    import random
    rng = random.Random(seed)
    hq, hkv, d = rng.choice([(8, 2, 128), (6, 6, 64), (15, 3, 64), (16, 1, 128), (9, 1, 64)])
    dtype = BF16 if seed % 4 else F32
    n = rng.randint(1, 9)
    q_lens = [rng.choice([0, 1, rng.randint(1, 40), rng.randint(1, 300)]) for _ in range(n)]
    kv_lens = [max(0, x + rng.choice([0, 0, -2, rng.randint(0, 400)])) for x in q_lens]
    if sum(q_lens) == 0:
        q_lens[0], kv_lens[0] = 3, 5
    q, k, v, plan = prompt_case(hq, hkv, d, dtype, q_lens, kv_lens, seed=seed)
    prompt_reference(q, k, v, q_lens, kv_lens).check(plan.run(q, k, v), dtype)
    groups = [rng.choice([1, 2, rng.randint(1, 40)]) for _ in range(rng.randint(1, 5))]
    shared = [rng.choice([0, 15, 16, rng.randint(0, 900)]) for _ in groups]
    lens = [max(0, s + rng.choice([0, 1, rng.randint(0, 300), -rng.randint(0, 900)])) for g, s in zip(groups, shared) for _ in range(g)]
    q, kv, table = paged_case(hq, hkv, d, dtype, groups, shared, lens, seed=seed)
    step = dense_attention.SharedPrefixAttention(kv, groups, i32(shared), hq)
    decode_reference(q, kv.k_pool, kv.v_pool, table, lens).check(step.step(q), dtype)
    assert ops.device_status() == 0
