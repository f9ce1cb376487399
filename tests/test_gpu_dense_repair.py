"""Rows that are done again because a bad value lies in their tiles but not before them: behind long prefixes, many at once, with
more work for the same SM after them."""

import pytest
import torch

from tests.dense_util import Reference, decode_reference
from tests.test_gpu_dense_attention import i32, paged_case, randn
from interattn_b200 import dense_attention, ops

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32


def on_gpu(shape, dtype, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randn(shape, generator=g, device="cuda").to(dtype)


def rows_reference(q, k, v, rows, seen):
    """Rows of one sequence over its first seen[i] keys, in float64 on the GPU."""
    hkv = k.shape[1]
    ref = Reference(len(rows), q.shape[1], q.shape[2])
    k, v = k.double().transpose(0, 1), v.double().transpose(0, 1)
    for i, (r, n) in enumerate(zip(rows, seen)):
        ref.row(i, q[r].double().view(hkv, -1, q.shape[2]), k[:, :n], v[:, :n])
    return ref


@pytest.mark.parametrize("poison", [float("inf"), float("nan")])
@pytest.mark.parametrize("dtype,prior,n,seqs,hkv", [(BF16, 150000, 4800, 4, 2), (F32, 20000, 300, 6, 2)])
def test_prompt_rows_behind_a_long_prefix(dtype, prior, n, seqs, hkv, poison):
    """The last token's value is bad: all queries of its piece but the last are done again, each over more than `prior` keys."""
    hq, d = 4 * hkv, 64
    q = on_gpu((seqs * n, hq, d), dtype, 1)
    k, v = on_gpu((seqs * (prior + n), hkv, d), dtype, 2), on_gpu((seqs * (prior + n), hkv, d), dtype, 3)
    plan = dense_attention.PromptAttention([n] * seqs, hq, hkv, d, kv_lens=[prior + n] * seqs, dtype=dtype)
    clean = plan.run(q, k, v)
    for s in range(seqs):
        v[(s + 1) * (prior + n) - 1] = poison
    out = plan.run(q, k, v)
    assert ops.device_status() == 0
    for s in range(seqs):
        first, k0 = s * n, s * (prior + n)
        assert not torch.isfinite(out[first + n - 1].float()).any()
        assert torch.equal(out[first:first + n - 64], clean[first:first + n - 64])
        assert bool(torch.isfinite(out[first + n - 64:first + n - 1].float()).all())
        rows = [n - 64, n - 40, n - 17, n - 3, n - 2]
        ref = rows_reference(q[first:first + n], k[k0:k0 + prior + n], v[k0:k0 + prior + n], rows, [prior + r + 1 for r in rows])
        ref.check(out[[first + r for r in rows]], dtype)


@pytest.mark.parametrize("hq,hkv,d", [(8, 2, 64), (3, 1, 128), (16, 1, 128), (2, 2, 128), (14, 2, 64)])
def test_prompt_with_a_bad_value_in_every_piece(hq, hkv, d):
    """A row before each bad token is clean, the row at it and all behind it are not: columns of their own tell them apart."""
    lens = [700, 33, 1, 400]
    q, k, v = on_gpu((sum(lens), hq, d), BF16, 4), on_gpu((sum(lens), hkv, d), BF16, 5), on_gpu((sum(lens), hkv, d), BF16, 6)
    plan = dense_attention.PromptAttention(lens, hq, hkv, d)
    at = [(t, c) for c, t in enumerate(range(3, 700, 61))]            # token t spoils column c
    refs = [rows_reference(q, k, v, list(range(700)), [r + 1 for r in range(700)])]
    for t, c in at:
        v[t, :, c] = float("nan")
    v[700] = float("inf")                                            # the neighbour's first token
    out = plan.run(q, k, v)
    assert ops.device_status() == 0
    want = torch.zeros((700, d), dtype=torch.bool)
    for t, c in at:
        want[t:, c] = True
    got = torch.isnan(out[:700].float()).cpu()
    assert torch.equal(got, want[:, None].expand_as(got))
    refs[0].out[got], refs[0].mean_abs[got] = 0, 0
    refs[0].check(torch.where(got.cuda(), 0, out[:700]), BF16)
    assert bool(torch.isfinite(out[733:].float()).all())


@pytest.mark.parametrize("dtype,d", [(BF16, 128), (BF16, 64), (F32, 64)])
@pytest.mark.parametrize("groups,hq", [([2, 1], 8), ([36, 3], 8), ([70, 1], 4)])
def test_shared_prefix_short_members_beside_long_ones(dtype, d, groups, hq):
    """Members end everywhere inside a long shared part in which values behind them are bad."""
    shared = [9000, 500]
    lens = [9000 - 257 * i % 8000 for i in range(groups[0])] + [900 + i for i in range(groups[1])]
    q, kv, table = paged_case(hq, 2, d, dtype, groups, shared, lens, seed=6)
    want = decode_reference(q, kv.k_pool, kv.v_pool, table, lens)
    for pos in (8950, 8800, 5003):
        kv.v_pool[table[0, pos // 16].long(), :, pos % 16] = float("nan")
    out = dense_attention.SharedPrefixAttention(kv, groups, i32(shared), hq).step(q)
    assert ops.device_status() == 0
    bad = torch.tensor([b < groups[0] and n > 5003 for b, n in enumerate(lens)])
    assert bool(torch.isnan(out[bad.cuda()].float()).all())
    want.out[bad], want.mean_abs[bad] = 0, 0
    out[bad.cuda()] = 0
    want.check(out, dtype)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_cut_keys_with_a_bad_value_in_every_part(dtype):
    q_lens, kv_lens = [60, 4], [9000, 4000]
    q, k, v = randn((64, 8, 64), dtype, 7), randn((13000, 2, 64), dtype, 8), randn((13000, 2, 64), dtype, 9)
    plan = dense_attention.PromptAttention(q_lens, 8, 2, 64, kv_lens=kv_lens, dtype=dtype)
    assert plan._ws_bytes > 0
    ref = rows_reference(q[:60], k[:9000], v[:9000], list(range(60)), [8941 + r for r in range(60)])
    v[8950:9000:7, :, 3] = float("inf")
    v[64:8900:100, :, 5] = float("nan")
    out = plan.run(q, k, v)
    bad = ~torch.isfinite(out[:60].float()).cpu()
    want = torch.zeros((60, 64), dtype=torch.bool)
    want[10:, 3], want[:, 5] = True, True
    assert torch.equal(bad, want[:, None].expand_as(bad)) and ops.device_status() == 0
    ref.out[bad], ref.mean_abs[bad] = 0, 0
    ref.check(torch.where(bad.cuda(), 0, out[:60]), dtype)


@pytest.mark.parametrize("dtype,d", [(BF16, 128), (BF16, 64), (F32, 64), (F32, 128)])
@pytest.mark.parametrize("q_lens,kv_lens", [([160], [160]), ([20], [9000]), ([900, 30], [900, 200])])
def test_log_sum_exps_do_not_depend_on_the_values(dtype, d, q_lens, kv_lens):
    """Rows that are NaN throughout, beside a bad value that they do not see: done again or not, their log-sum-exps are the keys'."""
    q, k, v = on_gpu((sum(q_lens), 4, d), dtype, 10), on_gpu((sum(kv_lens), 2, d), dtype, 11), on_gpu((sum(kv_lens), 2, d), dtype, 12)
    plan = dense_attention.PromptAttention(q_lens, 4, 2, d, kv_lens=kv_lens, dtype=dtype)
    n, m = q_lens[0], kv_lens[0]
    v[10], v[m - 1] = float("nan"), float("inf")
    out, lse = plan.run(q, k, v, return_lse=True)
    ref = rows_reference(q[:n], k[:m], v[:m].nan_to_num(0, 0, 0), list(range(n)), [m - n + r + 1 for r in range(n)])
    ref.check_lse(lse[:n])
    sees = torch.tensor([m - n + r + 1 > 10 for r in range(n)], device="cuda")
    assert bool(torch.isnan(out[:n][sees].float()).all()) and bool(torch.isfinite(out[:n][~sees].float()).all())
    assert bool(torch.isfinite(lse).all()) and ops.device_status() == 0
