"""Batches of many pieces whose plan is not large and whole pieces: results do not depend on the plan."""

import pytest
import torch

from tests.dense_util import prompt_reference
from tests.test_gpu_dense_attention import prompt_case
from interattn_b200 import ops

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("hq,hkv,d,q_lens,kv_lens,cut", [
    (32, 8, 64, [1] * 80, [9000] + [60] * 79, True), (16, 8, 128, [3, 1] * 60, [40, 7000] + [33, 2] * 59, True),
    (32, 8, 64, [2, 1] * 60, [70, 10] * 60, False), (64, 16, 64, [5] * 45, [5] * 45, False)])
def test_many_pieces(dtype, hq, hkv, d, q_lens, kv_lens, cut):
    q, k, v, plan = prompt_case(hq, hkv, d, dtype, q_lens, kv_lens, seed=60)
    assert (plan._ws_bytes > 0) == cut
    ref = prompt_reference(q, k, v, q_lens, kv_lens)
    out, lse = plan.run(q, k, v, return_lse=True)
    assert ops.device_status() == 0
    ref.check(out, dtype)
    ref.check_lse(lse)
    assert torch.equal(plan.run(q, k, v), out)
