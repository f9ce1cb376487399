"""Dimensions of one element, whose stride means nothing and is whatever its maker left there."""

import pytest
import torch

from tests.test_gpu_dense_attention import i32, prompt_case, randn
from interattn_b200 import dense_attention, ops, page_cache

pytestmark = pytest.mark.gpu


def loose(t, dim, stride):
    """The same elements, with another stride for a dimension of one."""
    strides = list(t.stride())
    assert t.shape[dim] == 1
    strides[dim] = stride
    return t.as_strided(t.shape, strides)


@pytest.mark.parametrize("dtype,d", [(torch.bfloat16, 128), (torch.bfloat16, 64), (torch.float32, 64)])
@pytest.mark.parametrize("stride", [0, 1, 7, 1 << 41])
def test_one_token_and_one_head(dtype, d, stride):
    q, k, v, plan = prompt_case(8, 2, d, dtype, [1], [1], seed=1)
    want = plan.run(q, k, v)
    assert torch.equal(plan.run(loose(q, 0, stride), loose(k, 0, stride), loose(v, 0, stride)), want)
    q, k, v, plan = prompt_case(1, 1, d, dtype, [70], [90], seed=2)
    want = plan.run(q, k, v)
    assert torch.equal(plan.run(loose(q, 1, stride), loose(k, 1, stride), loose(v, 1, stride)), want)
    q, k, v, plan = prompt_case(4, 1, d, dtype, [3], [5000], seed=3)
    want = plan.run(q, k, v)
    assert plan._ws_bytes > 0 and torch.equal(plan.run(q, loose(k, 1, stride), loose(v, 1, stride)), want)
    for hkv, n, dim in ((2, 1, 0), (1, 5, 1)):
        cache = page_cache.PageCache.empty(1, 4, hkv, d, 2, 2, dtype=dtype)
        cache.extend(i32([0]), i32([n]))
        x, y = randn((n, hkv, d), dtype, 4), randn((n, hkv, d), dtype, 5)
        cache.write(0, i32([0]), i32([0, n]), loose(x, dim, stride), loose(y, dim, stride))
        assert torch.equal(cache.pools[0][0][0, :, :n].transpose(0, 1), x) and torch.equal(cache.pools[0][1][0, :, :n].transpose(0, 1), y)
    assert ops.device_status() == 0


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_no_tokens_at_all(dtype):
    """An expanded tensor of no tokens is contiguous to torch, whatever its strides."""
    none = torch.zeros((0, 1, 1), dtype=dtype, device="cuda").expand(0, 2, 64)
    assert none.is_contiguous() and none.stride(2) == 0
    plan = dense_attention.PromptAttention([3], 4, 2, 64, kv_lens=[0], dtype=dtype)
    assert not plan.run(randn((3, 4, 64), dtype, 1), none, none).any()
    plan = dense_attention.PromptAttention([0], 2, 2, 64, kv_lens=[5], dtype=dtype)
    assert plan.run(none, randn((5, 2, 64), dtype, 2), randn((5, 2, 64), dtype, 3)).shape == (0, 2, 64)
    cache = page_cache.PageCache.empty(1, 4, 2, 64, 2, 2, dtype=dtype)
    cache.extend(i32([0, 1]), i32([0, 0]))
    cache.write(0, i32([0, 1]), i32([0, 0, 0]), none, none)
    assert ops.device_status() == 0
