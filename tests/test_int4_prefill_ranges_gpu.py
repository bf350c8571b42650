"""Prefill over a 4-bit cache against bounds of the operands that each unit runs with:
fp16 ones where the cache's scales allow it, bf16 weights and values where they do not."""

import numpy as np
import pytest
import torch

from conftest import dtype_name, storage
from int4_cases import Case, assert_near, assert_within, prefill_bound
from my_vllm_b200 import ops
from oracle import int4

pytestmark = pytest.mark.gpu
TYPES = [torch.bfloat16, torch.float16]


def _prefill(c, dev, status=None):
    q = c.q.to(dev)
    out = torch.full_like(q, float("nan"))
    return ops.paged_prefill(q, c.k.to(dev), c.v.to(dev), c.tables.to(dev), c.lens.to(dev),
                             c.starts.to(dev), out, max(c.q_lens), c.scale, status=status)


def _check(c, dev, wide=False, carried=128):
    out = _prefill(c, dev)
    ref, bounds = c.reference()
    assert_within(out, ref, prefill_bound(ref, bounds, c.dtype, wide))
    assert_near(out, ref, c.dtype, wide, carried)


def _rewrite(c, key=None, value=None, dtype=None):
    """Append the case's rows again with other keys or values, of ``dtype`` (the case's)."""
    dtype = dtype or c.dtype
    key = (c.key if key is None else key).to(dtype)
    value = (c.value if value is None else value).to(dtype)
    int4.kv_append_int4(storage(key), storage(value), c.k.numpy(), c.v.numpy(),
                        c.all_slots.numpy(), dtype_name(key))


def _groups(*exponents):
    return torch.repeat_interleave(2.0 ** torch.tensor(exponents, dtype=torch.float64), 32)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("large", [2.0 ** 14, 2.0 ** 17, 2.0 ** 60, 2.0 ** 120])
@pytest.mark.parametrize("q,kv,hq,hkv", [([70, 20], [150, 20], 8, 2), ([40], [3000], 4, 1)])
def test_one_large_value_group(cuda_device, dtype, large, q, kv, hq, hkv):
    """Rows in front of the token must not see it: 0 times a value that overflows is NaN."""
    c = Case(q, kv, hq, hkv, 16, dtype, seed=4)
    token = kv[0] - q[0] // 2  # the first half of the rows stands in front of it
    page, row = divmod(c.slots[0][token], 16)
    bits = int(np.float32(large).view(np.uint32) >> 16)
    int4.Pages(c.v.numpy()).scales[page, hkv - 1, row].view(np.uint16)[1] = bits
    out = _prefill(c, cuda_device)
    ref, bounds = c.reference()
    first = q[0] - q[0] // 2
    assert out[:first].isfinite().all()
    # a row that sees it holds values beyond fp16 there
    fits = np.abs(ref) < torch.finfo(dtype).max
    tol = prefill_bound(ref, bounds, dtype, wide=True)
    assert_within(out.double().cpu().masked_fill(torch.tensor(~fits), 0.0),
                  np.where(fits, ref, 0.0), np.where(fits, tol, 0.0))
    assert fits[:first].all()
    assert_near(out[:first], ref[:first], dtype, wide=True)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("factor", [2.0 ** 16, 2.0 ** 60, 2.0 ** -20, 2.0 ** -60])
def test_keys_beyond_fp16(cuda_device, dtype, factor):
    # keys appended in bf16, and a softmax_scale that brings their scores back
    c = Case([60, 20, 1], [60, 300, 2000], 4, 1, 16, dtype, seed=9)
    _rewrite(c, key=c.key.double() * factor, value=c.value, dtype=torch.bfloat16)
    c.scale = c.scale / factor
    _check(c, cuda_device, wide=True)


@pytest.mark.parametrize("dtype", TYPES)
def test_one_key_beyond_fp16(cuda_device, dtype):
    # scores of 2^14 and more against one token; rows that see it give it everything, or nothing
    c = Case([40], [300], 4, 1, 16, dtype, seed=7)
    key = c.key.double()
    key[280] *= 2.0 ** 18
    _rewrite(c, key=key, dtype=torch.bfloat16)
    c.scale = 2.0 ** -7
    _check(c, cuda_device, wide=True)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("exponents", [(0, 8, -8, 0), (-14, 0, 0, 12), (0, 40, -40, 0)])
def test_groups_far_apart(cuda_device, dtype, exponents):
    if dtype == torch.float16 and max(exponents) > 15:
        pytest.skip("values beyond the type")
    c = Case([60, 20], [60, 1200], 8, 2, 16, dtype, seed=6)
    _rewrite(c, value=c.value.double() * _groups(*exponents))
    _check(c, cuda_device, wide=max(exponents) > 12 or min(exponents) < -12, carried=32)
