"""Prefill over a 4-bit cache against bounds of the operands that each unit runs with:
fp16 ones where the cache's scales allow it, bf16 weights and values where they do not."""

import numpy as np
import pytest
import torch

from conftest import dtype_name, storage
from int4_cases import Case, assert_near, assert_within, prefill_bound
from my_vllm_b200 import _native, ops
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


# few units of many tiles (parts, joins), whole ones, ragged ones
SHAPES = [([1], [5000], 4, 1), ([200], [3000], 5, 1), ([600], [4000], 2, 2), ([30], [2500], 4, 2),
          ([60, 20, 1], [60, 300, 2000], 4, 1), ([300, 129], [300, 640], 8, 2)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("q,kv,hq,hkv", SHAPES)
def test_long_contexts(cuda_device, dtype, q, kv, hq, hkv):
    _check(Case(q, kv, hq, hkv, 16, dtype, seed=kv[0]), cuda_device)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("spread,v_spread", [(4.0, 1.0), (1.0, 0.02), (0.05, 50.0)])
def test_scales_within_fp16(cuda_device, dtype, spread, v_spread):
    c = Case([60, 20, 200], [60, 300, 1500], 8, 2, 32, dtype, seed=3, spread=spread,
             v_spread=v_spread)
    _check(c, cuda_device)


@pytest.mark.parametrize("exponent", [-100, -30, 20, 100])
def test_queries_of_any_magnitude(cuda_device, exponent):
    c = Case([40, 3], [60, 2500], 8, 2, 16, torch.bfloat16, seed=2)
    c.q = (c.q.float() * 2.0 ** exponent * torch.linspace(1, 2 ** 10, 43)[:, None, None]).bfloat16()
    c.q[5] = 0
    c.scale = c.scale * 2.0 ** -exponent / 2 ** 10
    _check(c, cuda_device)


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
@pytest.mark.parametrize("apart", [20, 30, 40, 90, 120])
@pytest.mark.parametrize("q,kv", [(20, 400), (20, 3000)])
def test_a_key_far_above_the_others_that_no_row_wants(cuda_device, dtype, apart, q, kv):
    # its scores are far below every other, whose keys it must not cost anything
    c = Case([q], [kv], 4, 1, 16, dtype, seed=apart)
    c.q[:] = c.q[:1, :1].clone()
    direction = c.q[0, 0].double() / c.q[0, 0].double().square().sum() / c.scale
    key = c.key.double()
    key[30] = -direction * 2.0 ** apart
    _rewrite(c, key, dtype=torch.bfloat16)
    out = _prefill(c, cuda_device)
    # the same with a key that is just low enough, and the bound of the keys that count
    key[30] = -200 * direction
    _rewrite(c, key, dtype=torch.bfloat16)
    ref, bounds = c.reference()
    key[30] = 0
    _rewrite(c, key, dtype=torch.bfloat16)
    others = c.reference()[1]
    bounds.update(keys=others["keys"], terms=others["terms"])
    assert_within(out, ref, prefill_bound(ref, bounds, dtype, wide=True, bf16_keys=True))


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
@pytest.mark.parametrize("apart", [12, 16, 20, 26])
def test_one_token_above_the_others_with_a_low_score(cuda_device, dtype, apart):
    # its weight is some 2^-apart of the largest one's, its values 2^apart times theirs
    if dtype == torch.float16 and apart > 24:
        pytest.skip("values beyond the type")
    c = Case([20], [400], 4, 1, 16, dtype, seed=apart)
    key, value = torch.zeros_like(c.key).double(), c.value.double() * 2.0 ** (2 - apart / 2)
    c.q[:] = c.q[:1, :1].clone()  # one query for all rows and heads
    direction = c.q[0, 0].double() / c.q[0, 0].double().square().sum() / c.scale
    key[30] = -apart * np.log(2.0) * direction
    value[30] *= 2.0 ** apart
    key[31] = 4 * direction  # the row's largest weight, without a value
    value[31] = 0
    _rewrite(c, key, value)
    _check(c, cuda_device, wide=apart > 18)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("exponents", [(0, 8, -8, 0), (-14, 0, 0, 12), (0, 40, -40, 0)])
def test_groups_far_apart(cuda_device, dtype, exponents):
    if dtype == torch.float16 and max(exponents) > 15:
        pytest.skip("values beyond the type")
    c = Case([60, 20], [60, 1200], 8, 2, 16, dtype, seed=6)
    _rewrite(c, value=c.value.double() * _groups(*exponents))
    _check(c, cuda_device, wide=max(exponents) > 12 or min(exponents) < -12, carried=32)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("column", [1, 2, 5, 6])
@pytest.mark.parametrize("bad", [-1, 1 << 30])
def test_a_bad_page_counts_as_rows_of_zeros(cuda_device, dtype, column, bad):
    q, kv = [20, 20], [130, 20]
    c = Case(q, kv, 4, 2, 16, dtype, seed=1)
    status = torch.zeros(1, dtype=torch.int32, device=cuda_device)
    keep = c.tables.clone()
    c.tables[0, column] = bad
    out = _prefill(c, cuda_device, status=status)
    assert int(status) == _native.STATUS_PAGE_OUT_OF_RANGE
    c.tables = keep
    for slot in c.slots[0][16 * column: 16 * column + 16]:
        for cache in (c.k, c.v):
            int4.Pages(cache.numpy()).put(slot, np.full((2, 128), 8, np.uint8), np.zeros((2, 4)))
    ref, bounds = c.reference()
    assert_within(out, ref, prefill_bound(ref, bounds, dtype))


@pytest.mark.parametrize("dtype", TYPES)
def test_tokens_past_the_table_count_as_rows_of_zeros(cuda_device, dtype):
    c = Case([20, 20], [96, 20], 4, 2, 16, dtype, seed=1)
    status = torch.zeros(1, dtype=torch.int32, device=cuda_device)
    q, k, v, lens, starts = (x.to(cuda_device) for x in (c.q, c.k, c.v, c.lens, c.starts))
    short = c.tables[:, :5].contiguous().to(cuda_device)  # 80 of the 96 tokens
    out = torch.full_like(q, float("nan"))
    ops.paged_prefill(q, k, v, short, lens, starts, out, 20, c.scale, status=status)
    assert int(status) == _native.STATUS_PAGE_OUT_OF_RANGE
    for slot in c.slots[0][80:]:
        for cache in (c.k, c.v):
            int4.Pages(cache.numpy()).put(slot, np.full((2, 128), 8, np.uint8), np.zeros((2, 4)))
    ref, bounds = c.reference()
    assert_within(out, ref, prefill_bound(ref, bounds, dtype))
