"""Keys whose logits are -infinity weigh nothing, however the keys are cut; a row that sees no other key is NaN, as the formula
has it (infinity minus infinity)."""

import pytest
import torch

from tests.dense_util import decode_reference, prompt_reference
from tests.test_gpu_dense_attention import i32, paged_case, randn
from interattn_b200 import dense_attention, ops

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32
NEG = float("-inf")


def all_nan(x):
    return bool(torch.isnan(x.float()).all())


@pytest.mark.parametrize("dtype,hq,hkv,d", [(BF16, 8, 2, 128), (BF16, 4, 2, 64), (F32, 8, 2, 64), (F32, 4, 1, 128)])
@pytest.mark.parametrize("q_lens,kv_lens,bad", [([3], [9000], 4000), ([1], [16000], 15990), ([40, 2], [6000, 3000], 5500)])
def test_prompt_parts_of_minus_infinity(dtype, hq, hkv, d, q_lens, kv_lens, bad):
    q = randn((sum(q_lens), hq, d), dtype, 1).abs() + 0.01
    k, v = randn((sum(kv_lens), hkv, d), dtype, 2), randn((sum(kv_lens), hkv, d), dtype, 3)
    k[:bad], k[:bad, :, 0] = 0, NEG
    plan = dense_attention.PromptAttention(q_lens, hq, hkv, d, kv_lens=kv_lens, dtype=dtype)
    assert plan._ws_bytes > 0
    out, lse = plan.run(q, k, v, return_lse=True)
    ref = prompt_reference(q, k[bad:], v[bad:], q_lens, [kv_lens[0] - bad] + kv_lens[1:])
    ref.check(out, dtype)
    ref.check_lse(lse)
    k[:kv_lens[0]], k[:kv_lens[0], :, 0] = 0, NEG
    out, lse = plan.run(q, k, v, return_lse=True)
    assert all_nan(out[:q_lens[0]]) and bool((lse[:q_lens[0]] == NEG).all()) and ops.device_status() == 0
    assert bool(torch.isfinite(out[q_lens[0]:].float()).all())


@pytest.mark.parametrize("dtype,d", [(BF16, 128), (BF16, 64), (F32, 64), (F32, 128)])
@pytest.mark.parametrize("groups,hq", [([1, 1], 4), ([2, 1], 8), ([4, 1], 8), ([5, 1], 8), ([9, 1], 8), ([20, 1], 8), ([40, 1], 8)])
def test_shared_prefix_parts_of_minus_infinity(dtype, d, groups, hq):
    """The own part of the first sequence, the shared part of the first group, everything of the last sequence."""
    n = sum(groups)
    shared, lens = [320, 64], [321 + 7 * i for i in range(n - 1)] + [90]
    q, kv, table = paged_case(hq, 2, d, dtype, groups, shared, lens, seed=3)
    q = q.abs() + 0.01

    def spoil(pages, slots=slice(None)):
        for page in pages:
            kv.k_pool[page, :, slots] = 0
            kv.k_pool[page, :, slots, 0] = NEG

    spoil([int(table[0, 20])])                              # sequence 0: its one own token
    spoil([int(x) for x in table[n - 1, :6]])
    step = dense_attention.SharedPrefixAttention(kv, groups, i32(shared), hq)
    out = step.step(q)
    assert all_nan(out[n - 1])
    seen = [320] + lens[1:n - 1] + [0]
    out[n - 1] = 0
    decode_reference(q, kv.k_pool, kv.v_pool, table, seen).check(out, dtype)
    spoil([int(x) for x in table[0, :20]])                  # the shared part: sequence 0 has nothing left
    out = step.step(q)
    assert all_nan(out[0]) and all_nan(out[n - 1]) and ops.device_status() == 0
    out[0], out[n - 1] = 0, 0
    own = table.clone()
    own[:, :table.shape[1] - 20] = table[:, 20:]
    decode_reference(q, kv.k_pool, kv.v_pool, own, [0] + [x - 320 for x in lens[1:n - 1]] + [0]).check(out, dtype)


def test_idle_rows_beside_them_are_zeros():
    for dtype in (BF16, F32):
        q, kv, table = paged_case(8, 2, 64, dtype, [3], [64], [0, 70, 65], seed=4)
        kv.k_pool.zero_()
        kv.k_pool[..., 0] = NEG
        out = dense_attention.SharedPrefixAttention(kv, [3], i32([64]), 8).step(q.abs() + 0.01)
        assert not out[0].any() and all_nan(out[1:]) and ops.device_status() == 0


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_log_sum_exp_merge_of_such_a_row(dtype):
    """Two runs over the halves of the keys, merged by their log-sum-exps: the half that weighs nothing does not spoil the other."""
    q = randn((5, 8, 64), dtype, 7).abs() + 0.01
    k, v = randn((60, 2, 64), dtype, 8), randn((60, 2, 64), dtype, 9)
    k[:30], k[:30, :, 0] = 0, NEG
    plan = dense_attention.PromptAttention([5], 8, 2, 64, kv_lens=[34], dtype=dtype)      # 30 to 34 keys
    a, la = plan.run(q, torch.cat([k[:30], k[:4]]), torch.cat([v[:30], v[:4]]), return_lse=True)
    b, lb = plan.run(q, k[26:], v[26:], return_lse=True)
    assert all_nan(a) and bool((la == NEG).all())
    merged = ops.finalize(torch.stack([a, b], 2).float(), torch.stack([la, lb], 2), out_dtype=F32)
    torch.testing.assert_close(merged.view(5, 8, 64), b.float(), rtol=1e-6, atol=1e-6)
