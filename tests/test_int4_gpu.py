"""The 4-bit cache's operators on the GPU: append and read-back bit for bit
against the oracle's format, decode and prefill against attention in 64 bits."""

import numpy as np
import pytest
import torch

from conftest import dtype_name, storage
from int4_cases import Case, assert_within, decode_tolerance, prefill_tolerance
from my_vllm_b200 import _native, ops
from oracle import int4

pytestmark = pytest.mark.gpu
TYPES = [torch.bfloat16, torch.float16]
PAGE_BIT = _native.STATUS_PAGE_OUT_OF_RANGE


def _status(dev):
    return torch.zeros(1, dtype=torch.int32, device=dev)


# ------------------------------------------------------- append, read back --
def _hard_rows(hkv, dtype, g):
    """Rows where the format can go wrong: ties, zeros, range ends, no numbers."""
    x = torch.randn(40, hkv, 128, generator=g)
    x[1] *= 1e-3
    x[2] *= 1e4 if dtype == torch.float16 else 1e30
    x[3] = 0
    x[4] = torch.randint(-14, 15, (hkv, 128), generator=g) / 2  # a = 7: every half a tie
    x[4, :, ::32] = 7
    x[5, 0, 3], x[6, 0, 40], x[7, 0, 127] = float("nan"), float("inf"), float("-inf")
    x[8] = torch.finfo(dtype).max
    x[9] = torch.finfo(dtype).tiny
    x[10] = x[10].sign() * torch.finfo(dtype).smallest_normal / 64
    x[11] = 2.0 ** -126 * 3 if dtype == torch.bfloat16 else 0
    x[12, :, 1:] = 0  # one value a row
    x[13] = -x[13].abs()
    x[14] = 21 * torch.randint(-1, 2, (hkv, 128), generator=g) / 7
    return x.to(dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("hkv,bs,wide", [(1, 16, False), (3, 48, False), (8, 256, True)])
def test_append_and_read_back_bit_exact(cuda_device, dtype, hkv, bs, wide):
    g = torch.Generator().manual_seed(11)
    key, value = _hard_rows(hkv, dtype, g), _hard_rows(hkv, dtype, g)
    n, blocks = key.size(0), 300 // bs + 2
    shape = ops.int4_cache_shape(blocks, bs, hkv)
    k = torch.randint(0, 256, shape, generator=g, dtype=torch.uint8)
    v = torch.randint(0, 256, shape, generator=g, dtype=torch.uint8)
    slots = torch.randperm(blocks * bs, generator=g)[:n]
    slots[17] = slots[n - 1] = -1
    slots = slots.to(torch.int64 if wide else torch.int32)
    # rows strided in a fused projection, pools whose pages are apart
    qkv = torch.cat([key.flatten(1), torch.zeros(n, 128, dtype=dtype), value.flatten(1)], 1)
    qkv = qkv.to(cuda_device)
    pool = torch.stack([k, v], 1).to(cuda_device)
    k_ref, v_ref = k.numpy().copy(), v.numpy().copy()
    int4.kv_append_int4(storage(key), storage(value), k_ref, v_ref, slots.numpy(),
                        dtype_name(key))
    status = _status(cuda_device)
    ops.store_kvcache_int4(qkv[:, : hkv * 128].unflatten(1, (hkv, 128)),
                           qkv[:, (hkv + 1) * 128:].unflatten(1, (hkv, 128)),
                           pool[:, 0], pool[:, 1], slots.to(cuda_device), status=status)
    assert np.array_equal(pool[:, 0].cpu().numpy(), k_ref)  # the slots, and nothing else
    assert np.array_equal(pool[:, 1].cpu().numpy(), v_ref)

    out = torch.full((n, 3 * hkv * 128), 5.0, dtype=dtype, device=cuda_device)
    k_out = out[:, : hkv * 128].unflatten(1, (hkv, 128))
    v_out = out[:, 2 * hkv * 128:].unflatten(1, (hkv, 128))
    ops.load_kvcache_int4(pool[:, 0], pool[:, 1], slots.to(cuda_device), k_out, v_out,
                          status=status)
    live = slots >= 0
    for got, cache in ((k_out, k_ref), (v_out, v_ref)):
        want = torch.full((n, hkv, 128), 5.0, dtype=dtype)
        # s (c - 8) has 11 bits: exact in fp32, then one rounding
        want[live] = torch.tensor(int4.kv_load_int4(cache, slots[live].numpy())).float().to(dtype)
        assert torch.equal(got.cpu().isnan(), want.isnan())
        assert torch.equal(got.cpu().nan_to_num(0.5), want.nan_to_num(0.5))
    assert (out[:, hkv * 128: 2 * hkv * 128] == 5).all()
    assert int(status) == 0


@pytest.mark.parametrize("shift,gap", [(8, 0), (0, 8), (16, 16)])
def test_rows_aligned_to_16_bytes_only(cuda_device, shift, gap):
    g = torch.Generator().manual_seed(7)
    row = 2 * 128 + gap
    flat = torch.randn(20 * row + shift, generator=g).half().to(cuda_device)
    x = flat[shift:].view(20, row)[:, :256].unflatten(1, (2, 128))
    k = torch.zeros(ops.int4_cache_shape(2, 16, 2), dtype=torch.uint8, device=cuda_device)
    v = torch.zeros_like(k)
    slots = torch.arange(20, device=cuda_device) + 3
    ops.store_kvcache_int4(x, x, k, v, slots)
    assert torch.equal(k, v)
    out = torch.full_like(flat, 9.0)
    back = out[shift:].view(20, row)[:, :256].unflatten(1, (2, 128))
    ops.load_kvcache_int4(k, v, slots, back, torch.empty_like(x.contiguous()))
    want = int4.kv_load_int4(k.cpu().numpy(), slots.cpu().numpy())
    assert torch.equal(back.cpu(), torch.tensor(want).half())
    assert (out[shift:].view(20, row)[:, 256:] == 9).all() and (out[:shift] == 9).all()
    ref = np.zeros(k.shape, np.uint8)
    int4.kv_append_int4(storage(x), storage(x), ref, ref.copy(), slots.cpu().numpy(), "float16")
    assert np.array_equal(k.cpu().numpy(), ref)


def test_append_dispatches_on_the_cache_type(cuda_device):
    g = torch.Generator().manual_seed(5)
    x = torch.randn(4, 2, 128, generator=g).bfloat16().to(cuda_device)
    caches = [torch.zeros(ops.int4_cache_shape(2, 16, 2), dtype=torch.uint8, device=cuda_device)
              for _ in range(4)]
    slots = torch.arange(4, dtype=torch.int32, device=cuda_device)
    ops.store_kvcache(x, -x, caches[0], caches[1], slots)
    ops.store_kvcache_int4(x, -x, caches[2], caches[3], slots)
    assert torch.equal(caches[0], caches[2]) and torch.equal(caches[1], caches[3])
    assert caches[0].any()


def test_slots_out_of_range_are_skipped_and_reported(cuda_device):
    x = torch.ones(3, 2, 128, dtype=torch.float16, device=cuda_device)
    cache = torch.zeros(ops.int4_cache_shape(2, 16, 2), dtype=torch.uint8, device=cuda_device)
    status = _status(cuda_device)
    for slots in ([0, 32, 1], [0, -2, 1]):
        s = torch.tensor(slots, dtype=torch.int32, device=cuda_device)
        ops.store_kvcache_int4(x, x, cache, cache.clone(), s, status=status)
        assert int(status) == _native.STATUS_SLOT_OUT_OF_RANGE
        status.zero_()
        out = torch.full_like(x, 3.0)
        ops.load_kvcache_int4(cache, cache, s, out, torch.empty_like(out), status=status)
        assert int(status) == _native.STATUS_SLOT_OUT_OF_RANGE
        status.zero_()
        # a row of ones: s = bf16(1 / 7) = 73 / 512, read back as 7 s = 511 / 512
        assert (out[1] == 3).all() and (out[::2] == 511 / 512).all()


# ------------------------------------------------------------------- decode --
def _decode(c, dev, parts=0, q=None, out=None, status=None, plan=None):
    q = c.q.to(dev) if q is None else q
    out = torch.full_like(q, float("nan")) if out is None else out
    if plan is None:
        plan = ops.plan_decode(len(c.kv_lens), c.hq, c.hkv, 128, c.bs, max(c.kv_lens),
                               force_num_parts=parts, total_kv_tokens=sum(c.kv_lens),
                               kv_int4=True)
    ws = torch.full((plan.workspace_bytes,), 255, dtype=torch.uint8, device=dev)
    ops.paged_decode(q, c.k.to(dev), c.v.to(dev), c.tables.to(dev), c.lens.to(dev), out, plan,
                     c.scale, ws, status=status)
    return out


def _check_decode(c, dev, **more):
    status = _status(dev)
    out = _decode(c, dev, status=status, **more)
    ref, bounds = c.reference()
    assert_within(out, ref, decode_tolerance(ref, bounds, c.dtype))
    assert int(status) == 0
    return out


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("hq,hkv", [(1, 1), (4, 2), (8, 2), (5, 1), (7, 1), (8, 1), (9, 1),
                                    (32, 2), (24, 3)])
def test_decode_groups(cuda_device, dtype, hq, hkv):
    lens = [1, 2, 15, 16, 17, 31, 32, 33, 64, 100, 129, 300]
    _check_decode(Case([1] * len(lens), lens, hq, hkv, 16, dtype, seed=hq), cuda_device)


@pytest.mark.parametrize("bs", [16, 32, 48, 64, 256])
@pytest.mark.parametrize("parts", [0, 1, 3, 20, 600])
def test_decode_pages_and_splits(cuda_device, bs, parts):
    lens = [1, 47, 48, 49, 255, 256, 257, 700, 1025]
    c = Case([1] * len(lens), lens, 8, 2, bs, torch.bfloat16, seed=bs + parts)
    _check_decode(c, cuda_device, parts=parts)


@pytest.mark.parametrize("lens", [[1, 1, 1, 1], [3000, 1, 40, 2900], [0, 0, 0, 0], [64, 0, 0, 2000],
                                  [0, 2000, 17, 0], [1500, 1500, 1500, 1500]])
def test_decode_one_plan_for_any_lengths(cuda_device, lens):
    # the shares are dealt on the device: a captured graph's plan serves them all
    plan = ops.plan_decode(4, 16, 4, 128, 32, 64, force_num_parts=13, kv_int4=True)
    full = [max(n, 1) for n in lens]
    c = Case([1] * 4, full, 16, 4, 32, torch.float16, seed=4)
    c.kv_lens = lens
    c.lens = torch.tensor(lens, dtype=torch.int32)
    _check_decode(c, cuda_device, plan=plan)


@pytest.mark.parametrize("lens", [[1, 0, 512, 40], [700, 3, 0, 33]])
def test_decode_one_plan_of_whole_sequences(cuda_device, lens):
    # planned for short sequences, which no CTA shares; longer ones are still right
    plan = ops.plan_decode(4, 16, 2, 128, 32, 512, kv_int4=True)
    assert plan.part_tokens == 0
    c = Case([1] * 4, [max(n, 1) for n in lens], 16, 2, 32, torch.float16, seed=4)
    c.kv_lens = lens
    c.lens = torch.tensor(lens, dtype=torch.int32)
    _check_decode(c, cuda_device, plan=plan)


def test_decode_many_sequences(cuda_device):
    # more sequences than a CTA has threads, most of them without tokens
    lens = [0] * 700
    for i in (3, 4, 130, 131, 132, 300, 511, 698):
        lens[i] = 30 + 37 * (i % 11)
    c = Case([1] * 700, [max(n, 1) for n in lens], 2, 1, 16, torch.bfloat16, seed=14)
    c.kv_lens = lens
    c.lens = torch.tensor(lens, dtype=torch.int32)
    for parts in (1, 7, 0):
        _check_decode(c, cuda_device, parts=parts)


def test_decode_refuses_a_plan_for_another_cache(cuda_device):
    c = Case([1], [40], 4, 2, 16, torch.float16)
    with pytest.raises(ValueError, match="4-bit"):
        _decode(c, cuda_device, plan=ops.plan_decode(1, 4, 2, 128, 16, 40))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("spread,v_spread", [(8.0, 1.0), (1.0, 1e-3), (0.01, 100.0)])
def test_decode_ranges(cuda_device, dtype, spread, v_spread):
    lens = [40, 513, 1000]
    c = Case([1] * 3, lens, 8, 2, 16, dtype, seed=9, spread=spread, v_spread=v_spread)
    _check_decode(c, cuda_device)


def _rewrite_values(c, scale_of_token):
    """Scale token t of every sequence's values by scale_of_token(t), in the cache."""
    factors = torch.tensor([scale_of_token(t) for n in c.kv_lens for t in range(n)])
    value = (c.value.float() * factors[:, None, None]).to(c.dtype)
    int4.kv_append_int4(storage(c.key), storage(value), c.k.numpy(), c.v.numpy(),
                        c.all_slots.numpy(), dtype_name(c.key))


@pytest.mark.parametrize("order", ["growing", "falling"])
@pytest.mark.parametrize("parts", [1, 2])
def test_decode_values_of_many_magnitudes(cuda_device, order, parts):
    # value scales from 2^-20 to 2^20 along the sequence, bf16's range used in earnest
    n = 400
    c = Case([1] * 2, [n, n], 4, 1, 16, torch.bfloat16, seed=3)
    _rewrite_values(c, lambda t: 2.0 ** ((t if order == "growing" else n - 1 - t) / n * 40 - 20))
    _check_decode(c, cuda_device, parts=parts)


@pytest.mark.parametrize("exponent", [-60, 60])
def test_decode_extreme_values(cuda_device, exponent):
    c = Case([1] * 2, [5, 130], 4, 1, 16, torch.bfloat16, seed=8)
    _rewrite_values(c, lambda t: 2.0 ** exponent)
    _check_decode(c, cuda_device)


@pytest.mark.parametrize("exponent", [-40, 20])
def test_decode_query_magnitudes(cuda_device, exponent):
    # q far from 1: the softmax is flat, or one key takes it all
    c = Case([1] * 2, [33, 70], 4, 1, 16, torch.bfloat16, seed=8)
    c.q = (c.q.float() * 2.0 ** exponent).to(c.dtype)
    if exponent > 0:  # keys whose best two are apart by more than their error
        c.scale *= 2.0 ** -14
    _check_decode(c, cuda_device)


def test_decode_nan_stays_in_its_group(cuda_device):
    c = Case([1] * 2, [50, 70], 8, 2, 16, torch.bfloat16, seed=2)
    pages = int4.Pages(c.v.numpy())
    page, row = divmod(c.slots[0][20], 16)
    pages.scales[page, 1, row].view(np.uint16)[2] = 0x7FC0  # sequence 0, head 1, group 2
    out = _decode(c, cuda_device).cpu().double()
    ref, bounds = c.reference()
    bad = torch.zeros(2, 8, 128, dtype=torch.bool)
    bad[0, 4:, 64:96] = True
    assert torch.equal(out.isnan(), bad)
    assert np.array_equal(np.isnan(ref), bad.numpy())
    tol = np.nan_to_num(decode_tolerance(ref, bounds, c.dtype))
    assert_within(out.masked_fill(bad, 0.0), np.nan_to_num(ref), tol)
    # in a key, every output of the heads that read it
    c = Case([1] * 2, [50, 70], 8, 2, 16, torch.bfloat16, seed=2)
    pages = int4.Pages(c.k.numpy())
    page, row = divmod(c.slots[1][69], 16)
    pages.scales[page, 0, row].view(np.uint16)[0] = 0x7FC0
    out = _decode(c, cuda_device).cpu()
    assert out[1, :4].isnan().all() and out[1, 4:].isfinite().all() and out[0].isfinite().all()


def test_decode_empty_sequences_and_rows_behind(cuda_device):
    for parts in (1, 2):
        c = Case([1] * 3, [64, 40, 64], 4, 2, 16, torch.bfloat16, seed=6)
        c.lens[1] = c.kv_lens[1] = 0
        # a padded graph's output: rows behind the batch stay as they are
        whole = torch.full((5, 6, 256), 7.0, dtype=torch.bfloat16, device=cuda_device)
        out = whole[:3, 1:5, 64:192]
        _check_decode(c, cuda_device, parts=parts, out=out)
        assert (out[1] == 0).all()
        mine = torch.zeros_like(whole, dtype=torch.bool)
        mine[:3, 1:5, 64:192] = True
        assert (whole[~mine] == 7).all()


def test_decode_strided_queries(cuda_device):
    c = Case([1] * 4, [9, 90, 33, 200], 8, 4, 32, torch.float16, seed=13)
    whole = torch.randn(4, 14, 130, device=cuda_device).half()
    q = whole[:, 3:11, :128]
    q.copy_(c.q)
    assert q.stride(1) % 2 == 0 and q.data_ptr() % 16 == 12
    _check_decode(c, cuda_device, q=q, out=torch.empty(4, 8, 128, dtype=torch.float16,
                                                       device=cuda_device))


def test_decode_bad_pages_are_reported(cuda_device):
    c = Case([1] * 2, [40, 40], 4, 2, 16, torch.bfloat16, seed=1)
    for bad in (-1, c.k.size(0), 1 << 30):
        status = _status(cuda_device)
        keep = c.tables.clone()
        c.tables[0, 1] = bad
        out = _decode(c, cuda_device, status=status)
        assert int(status) == PAGE_BIT
        c.tables = keep
        assert out.isfinite().all()
        ref, bounds = c.reference()
        tol = decode_tolerance(ref, bounds, c.dtype)
        assert_within(out[1:], ref[1:], tol[1:])
        # the lost page counts as rows of zeros
        lost = Case([1] * 2, [40, 40], 4, 2, 16, torch.bfloat16, seed=1)
        for slot in lost.slots[0][16:32]:
            for pages in (int4.Pages(lost.k.numpy()), int4.Pages(lost.v.numpy())):
                pages.put(slot, np.full((2, 128), 8, np.uint8), np.zeros((2, 4)))
        ref, bounds = lost.reference()
        assert_within(out, ref, decode_tolerance(ref, bounds, c.dtype))
    # a sequence longer than its table row of three pages (and than its 40 rows, so
    # that its own result means nothing)
    status = _status(cuda_device)
    c.lens[0] = 64
    out = _decode(c, cuda_device, status=status)
    assert int(status) == PAGE_BIT
    assert_within(out[1:], ref[1:], tol[1:])


# ------------------------------------------------------------------ prefill --
def _prefill(c, dev, q=None, out=None, status=None, **more):
    q = c.q.to(dev) if q is None else q
    out = torch.full_like(q, float("nan")) if out is None else out
    return ops.paged_prefill(q, c.k.to(dev), c.v.to(dev), c.tables.to(dev), c.lens.to(dev),
                             c.starts.to(dev), out, max(c.q_lens), c.scale, status=status, **more)


def _check_prefill(c, dev, **more):
    status = _status(dev)
    out = _prefill(c, dev, status=status, **more)
    ref, bounds = c.reference()
    assert_within(out[: len(ref)], ref, prefill_tolerance(ref, bounds, c.dtype))
    assert int(status) == 0
    return out


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("hq,hkv,bs", [(1, 1, 16), (4, 2, 32), (8, 2, 16), (5, 1, 48), (7, 1, 16),
                                       (16, 2, 256), (32, 2, 16), (24, 3, 64)])
def test_prefill_groups(cuda_device, dtype, hq, hkv, bs):
    c = Case([1, 33, 70, 5], [1, 33, 200, 133], hq, hkv, bs, dtype, seed=hq)
    _check_prefill(c, cuda_device)


@pytest.mark.parametrize("dtype", TYPES)
def test_prefill_lengths(cuda_device, dtype):
    q = [1, 2, 31, 64, 65, 128, 200, 300]
    kv = [1, 129, 31, 128, 257, 640, 201, 555]
    _check_prefill(Case(q, kv, 8, 2, 16, dtype, seed=21), cuda_device)


@pytest.mark.parametrize("spread,v_spread", [(8.0, 1.0), (1.0, 1e-3), (0.01, 100.0)])
@pytest.mark.parametrize("dtype", TYPES)
def test_prefill_ranges(cuda_device, dtype, spread, v_spread):
    c = Case([60, 20], [60, 300], 4, 1, 16, dtype, seed=9, spread=spread, v_spread=v_spread)
    _check_prefill(c, cuda_device)


# bf16 scales that leave fp16's range: all of them, or one value or key of one head
@pytest.mark.parametrize("spread,v_spread", [(1.0, 2.0 ** 60), (1.0, 2.0 ** -60), (2.0 ** -60, 1.0),
                                             (2.0 ** 18, 1.0), (1.0, 1e-6), (1e-6, 1e-6)])
def test_prefill_wide_ranges(cuda_device, spread, v_spread):
    c = Case([60, 20, 1], [60, 300, 2000], 4, 1, 16, torch.bfloat16, seed=9, spread=spread,
             v_spread=v_spread)
    c.scale = c.scale / max(spread, 1.0)
    _check_prefill(c, cuda_device)


@pytest.mark.parametrize("wide", [2.0 ** -40, 2.0 ** 17])
@pytest.mark.parametrize("q,kv,hq,hkv", [([70, 20, 9], [150, 20, 300], 8, 2), ([40], [3000], 4, 1),
                                         ([1] * 200, [130] * 200, 8, 8)])
def test_prefill_one_wide_group(cuda_device, wide, q, kv, hq, hkv):
    c = Case(q, kv, hq, hkv, 16, torch.bfloat16, seed=4)
    token = c.slots[0][kv[0] - q[0]]
    pages = int4.Pages(c.v.numpy())
    page, row = divmod(token, 16)
    bits = pages.scales[page, hkv - 1, row].view(np.uint16)
    bits[1] = int(np.float32(wide).view(np.uint32) >> 16)
    # and behind the end of the sequence, where it does not matter
    for cache in (c.k, c.v):
        last, used = divmod(c.slots[0][-1], 16)
        if used < 15:
            int4.Pages(cache.numpy()).scales[last, 0, 15].view(np.uint16)[:] = 0x7000
    _check_prefill(c, cuda_device)


@pytest.mark.parametrize("exponent", [-100, -40, 20, 100])
def test_prefill_query_magnitudes(cuda_device, exponent):
    c = Case([40, 3], [60, 500], 8, 2, 16, torch.bfloat16, seed=2)
    c.q = (c.q.float() * 2.0 ** exponent).bfloat16()
    c.q[5] = 0
    c.scale = c.scale * 2.0 ** -exponent
    _check_prefill(c, cuda_device)


@pytest.mark.parametrize("hq,hkv", [(8, 2), (5, 1)])
def test_prefill_leaves_other_rows(cuda_device, hq, hkv):
    # a sequence without new tokens in the middle, rows behind the last sequence
    c = Case([20, 0, 40], [50, 30, 40], hq, hkv, 16, torch.bfloat16, seed=17)
    q = torch.randn(70, hq, 128, device=cuda_device).bfloat16()
    q[:60] = c.q.to(cuda_device)
    out = torch.full_like(q, 7.0)
    _check_prefill(c, cuda_device, q=q, out=out)
    assert (out[60:] == 7).all()
    # the first two sequences alone
    out = torch.full_like(q, 7.0)
    _prefill(c, cuda_device, q=q, out=out, num_seqs=2)
    assert (out[20:] == 7).all() and (out[:20] != 7).any()


def test_prefill_strided(cuda_device):
    c = Case([30, 17], [64, 17], 4, 2, 16, torch.float16, seed=23)
    whole = torch.zeros(47, 6, 144, dtype=torch.float16, device=cuda_device)
    q = whole[:, 1:5, 8:136]
    q.copy_(c.q)
    held = torch.full((47, 5, 136), 7.0, dtype=torch.float16, device=cuda_device)
    _check_prefill(c, cuda_device, q=q, out=held[:, :4, :128])
    assert (held[:, 4] == 7).all() and (held[:, :, 128:] == 7).all()


def test_prefill_bad_pages_are_reported(cuda_device):
    c = Case([20, 20], [60, 20], 4, 2, 16, torch.bfloat16, seed=1)
    ref, bounds = c.reference()
    tol = prefill_tolerance(ref, bounds, c.dtype)
    for bad in (-1, c.k.size(0), 1 << 30):
        keep = c.tables.clone()
        c.tables[0, 1] = bad
        status = _status(cuda_device)
        out = _prefill(c, cuda_device, status=status)
        assert int(status) == PAGE_BIT
        c.tables = keep
        assert_within(out[20:], ref[20:], tol[20:])
    status = _status(cuda_device)
    c.lens[0] = 80  # past its table row
    out = _prefill(c, cuda_device, status=status)
    assert int(status) & PAGE_BIT
    assert_within(out[20:], ref[20:], tol[20:])


@pytest.mark.parametrize("dtype", TYPES)
def test_prefill_nan_reaches_the_rows_that_see_it(cuda_device, dtype):
    c = Case([90, 20], [150, 20], 8, 2, 16, dtype, seed=2)
    ref, bounds = c.reference()
    token = 100  # of sequence 0: rows 40 and up see it
    for cache, group in ((c.v, 1), (c.k, 3)):
        pages = int4.Pages(cache.numpy())
        page, row = divmod(c.slots[0][token], 16)
        held = pages.scales[page, 1, row].copy()
        pages.scales[page, 1, row].view(np.uint16)[group] = 0x7FC0
        out = _prefill(c, cuda_device).cpu().double()
        bad = torch.zeros(out.shape, dtype=torch.bool)
        if cache is c.v:  # its group of columns; the other columns as if nothing were there
            bad[40:90, 4:, 32:64] = True
            clean = bad
        else:
            bad[40:90, 4:] = True
        assert torch.equal(out.isnan(), bad)
        good = out.masked_fill(bad, 0.0)
        want = np.where(bad.numpy(), 0.0, ref)
        assert_within(good, want, prefill_tolerance(ref, bounds, dtype))
        pages.scales[page, 1, row] = held
    assert clean.any()


@pytest.mark.parametrize("hq,hkv", [(8, 2), (5, 1)])
def test_prefill_rows_that_see_nothing(cuda_device, hq, hkv):
    # more query rows than keys: the first rows stand before every key
    c = Case([150, 40, 3], [100, 40, 16], hq, hkv, 16, torch.bfloat16, seed=12)
    c.lens[2] = c.kv_lens[2] = 0
    out = _check_prefill(c, cuda_device)
    assert (out[:50] == 0).all() and (out[50] != 0).any() and (out[190:] == 0).all()


# (few units of many tiles, cut among SMs: parts, joins, cuts near a unit's ends)
@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("q,kv,hq,hkv", [([1], [5000], 4, 1), ([3, 70], [2100, 1500], 8, 2),
                                         ([200], [3000], 5, 1), ([600], [4000], 2, 2)])
def test_prefill_cut_units(cuda_device, dtype, q, kv, hq, hkv):
    c = Case(q, kv, hq, hkv, 16, dtype, seed=len(kv))
    out = _check_prefill(c, cuda_device)
    assert torch.equal(out, _prefill(c, cuda_device))  # parts are joined in order


@pytest.mark.parametrize("tokens", [896, 897, 1023, 1024, 1025])  # 7, 8 and 9 tiles
def test_prefill_shortest_cut_units(cuda_device, tokens):
    _check_prefill(Case([2], [tokens], 4, 1, 16, torch.float16, seed=tokens), cuda_device)


def test_prefill_on_two_streams(cuda_device):
    dev = cuda_device
    c = Case([30], [2500], 4, 2, 16, torch.bfloat16, seed=5)
    want = _check_prefill(c, dev)
    args = [x.to(dev) for x in (c.q, c.k, c.v, c.tables, c.lens, c.starts)]
    outs = [torch.empty_like(args[0]) for _ in range(8)]
    streams = [torch.cuda.Stream(dev) for _ in range(2)]
    torch.cuda.synchronize()
    for i, out in enumerate(outs):
        with torch.cuda.stream(streams[i & 1]):
            ops.paged_prefill(*args, out, 30, c.scale)
    torch.cuda.synchronize()
    assert all(torch.equal(out, want) for out in outs)


def test_prefill_nan_in_one_part_of_a_cut_unit(cuda_device):
    c = Case([40], [3000], 4, 1, 16, torch.bfloat16, seed=3)
    ref, bounds = c.reference()
    pages = int4.Pages(c.v.numpy())
    for token, first in ((1000, 0), (2975, 15)):  # seen by every row, by rows 15 and up
        page, row = divmod(c.slots[0][token], 16)
        held = pages.scales[page, 0, row].copy()
        pages.scales[page, 0, row].view(np.uint16)[2] = 0x7FC0
        out = _prefill(c, cuda_device).cpu().double()
        bad = torch.zeros(out.shape, dtype=torch.bool)
        bad[first:, :, 64:96] = True
        assert torch.equal(out.isnan(), bad)
        assert_within(out.masked_fill(bad, 0.0), np.where(bad.numpy(), 0.0, ref),
                      prefill_tolerance(ref, bounds, c.dtype))
        pages.scales[page, 0, row] = held


# (more than 128 blocks of rows, more units than a list of a CTA holds)
@pytest.mark.parametrize("hq,hkv,n", [(8, 8, 330), (4, 1, 130), (20, 10, 250)])
def test_prefill_many_sequences(cuda_device, hq, hkv, n):
    q = [1 + (i % 3 == 0) - (i % 50 == 7) for i in range(n)]
    kv = [max(q[i], (37 * i) % 150) for i in range(n)]
    _check_prefill(Case(q, kv, hq, hkv, 16, torch.bfloat16, seed=n), cuda_device)


# (units much shorter than a CTA's share, dealt whole; more blocks than are ranked)
@pytest.mark.parametrize("q,kv,hq,hkv", [([1100, 900], [1100, 1000], 64, 4), ([700], [700], 96, 1)])
def test_prefill_many_blocks(cuda_device, q, kv, hq, hkv):
    _check_prefill(Case(q, kv, hq, hkv, 16, torch.bfloat16, seed=hq), cuda_device)


def test_prefill_workspaces(cuda_device):
    dev = cuda_device
    c = Case([30], [2500], 4, 2, 16, torch.float16, seed=5)
    want = _check_prefill(c, dev)
    ws = torch.full((ops.prefill_workspace_bytes(kv_int4=True),), 255, dtype=torch.uint8, device=dev)
    assert torch.equal(_prefill(c, dev, workspace=ws), want)
    with pytest.raises(ValueError, match="workspace"):
        _prefill(c, dev, workspace=ws[:4096])
    with pytest.raises(ValueError, match="workspace"):
        _prefill(c, dev, workspace=ws[8:])
    with pytest.raises(ValueError, match="one device"):
        _prefill(c, dev, workspace=ws.cpu())
    # none at all, from C: whole units
    q, k, v, tables, lens, starts = (x.to(dev) for x in (c.q, c.k, c.v, c.tables, c.lens, c.starts))
    out = torch.full_like(q, float("nan"))
    cache = _native.Int4Cache(k.data_ptr(), v.data_ptr(), k.size(0), 16, 2, k.stride(0))
    rc = _native.load_library().b200_paged_prefill_int4(
        q.data_ptr(), q.stride(0), q.stride(1), 0, cache, tables.data_ptr(), tables.stride(0),
        tables.size(1), lens.data_ptr(), starts.data_ptr(), 1, 30, 30, 4, out.data_ptr(),
        out.stride(0), out.stride(1), c.scale, None, 0, None,
        torch.cuda.current_stream().cuda_stream)
    assert rc == _native.B200_OK
    ref, bounds = c.reference()
    assert_within(out, ref, prefill_tolerance(ref, bounds, c.dtype))


@pytest.mark.parametrize("shared", [True, False])
def test_prefill_graphs(cuda_device, shared):
    # with one workspace, and with one that each graph takes from its own pool
    dev = cuda_device
    ws = torch.empty(ops.prefill_workspace_bytes(kv_int4=True), dtype=torch.uint8, device=dev)
    ws = ws if shared else None
    cases = [Case([30], [2500], 4, 2, 16, torch.bfloat16, seed=5),
             Case([2, 3], [900, 1700], 4, 2, 32, torch.bfloat16, seed=6)]
    wants = [_check_prefill(c, dev) for c in cases]
    graphs = []
    for c in cases:
        q, k, v, tables, lens, starts = (x.to(dev) for x in (c.q, c.k, c.v, c.tables, c.lens,
                                                             c.starts))
        out = torch.empty_like(q)
        args = (q, k, v, tables, lens, starts, out, max(c.q_lens), c.scale)
        ops.paged_prefill(*args, workspace=ws)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            ops.paged_prefill(*args, workspace=ws)
        graphs.append((graph, out, args))
    for _ in range(3):
        for (graph, out, _args), want in zip(graphs, wants):
            out.fill_(9.0)
            graph.replay()
            assert torch.equal(out, want)


# ----------------------------------------------------------- used together --
@pytest.mark.parametrize("dtype", TYPES)
def test_a_prompt_then_steps_of_decoding(cuda_device, dtype):
    """Prefill of two prompts, then five captured decode steps on a side stream:
    append, attend, read back, against the oracle's cache and attention."""
    dev, hq, hkv, bs, steps = cuda_device, 8, 2, 16, 5
    prompts, g = [37, 90], torch.Generator().manual_seed(40)
    caches = [torch.randint(0, 256, ops.int4_cache_shape(16, bs, hkv), generator=g,
                            dtype=torch.uint8) for _ in range(2)]
    k, v = (x.to(dev) for x in caches)
    tables = torch.randperm(16, generator=g).to(torch.int32).view(2, 8)
    tokens = [[torch.randn(n + steps, hkv, 128, generator=g).to(dtype) for n in prompts]
              for _ in range(2)]

    def slots(s, t):
        return int(tables[s, t // bs]) * bs + t % bs

    # the prompts
    new = torch.tensor([slots(s, t) for s, n in enumerate(prompts) for t in range(n)],
                       dtype=torch.int32)
    key, value = (torch.cat([x[:n] for x, n in zip(side, prompts)]) for side in tokens)
    ops.store_kvcache(key.to(dev), value.to(dev), k, v, new.to(dev))
    int4.kv_append_int4(storage(key), storage(value), *(x.numpy() for x in caches), new.numpy(),
                        dtype_name(key))
    starts = torch.tensor([0, 37, 127], dtype=torch.int32)
    q = torch.randn(127, hq, 128, generator=g).to(dtype)
    out = torch.empty_like(q, device=dev)
    lens = torch.tensor(prompts, dtype=torch.int32, device=dev)
    ops.paged_prefill(q.to(dev), k, v, tables.to(dev), lens, starts.to(dev), out, 90, 0.09)
    ref, bounds = int4.attention(q.double().numpy(), *(x.numpy() for x in caches), tables.numpy(),
                                 prompts, starts.numpy(), 0.09)
    assert_within(out, ref, prefill_tolerance(ref, bounds, dtype))

    # one decode step, captured once, replayed for each token
    plan = ops.plan_decode(2, hq, hkv, 128, bs, 128, force_num_parts=3, kv_int4=True)
    ws = torch.empty(plan.workspace_bytes, dtype=torch.uint8, device=dev)
    status = _status(dev)
    slot = torch.full((3,), -1, dtype=torch.int32, device=dev)  # one row of padding
    rows = [torch.zeros(3, hkv, 128, dtype=dtype, device=dev) for _ in range(2)]
    qd = torch.zeros(2, hq, 128, dtype=dtype, device=dev)
    od, lens = torch.zeros_like(qd), torch.ones(2, dtype=torch.int32, device=dev)
    back = [torch.zeros(3, hkv, 128, dtype=dtype, device=dev) for _ in range(2)]
    tables_d = tables.to(dev)

    def step():
        ops.store_kvcache(rows[0], rows[1], k, v, slot, status=status)
        ops.paged_decode(qd, k, v, tables_d, lens, od, plan, 0.09, ws, status=status)
        ops.load_kvcache_int4(k, v, slot, back[0], back[1], status=status)

    stream = torch.cuda.Stream(dev)
    stream.wait_stream(torch.cuda.current_stream(dev))
    with torch.cuda.stream(stream):
        step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        step()
    with torch.cuda.stream(stream):
        for i in range(steps):
            at = [n + i for n in prompts]
            host = torch.tensor([slots(0, at[0]), slots(1, at[1]), -1], dtype=torch.int32)
            q = torch.randn(2, hq, 128, generator=g).to(dtype)
            slot.copy_(host)
            lens.copy_(torch.tensor(at, dtype=torch.int32) + 1)
            qd.copy_(q)
            for side, row in zip(tokens, rows):
                row[:2] = torch.stack([side[s][at[s]] for s in range(2)]).to(dev)
            graph.replay()
            stream.synchronize()
            key, value = (torch.stack([side[s][at[s]] for s in range(2)]) for side in tokens)
            int4.kv_append_int4(storage(key), storage(value), *(x.numpy() for x in caches),
                                host[:2].numpy(), dtype_name(key))
            ref, bounds = int4.attention(q.double().numpy(), *(x.numpy() for x in caches),
                                         tables.numpy(), [n + 1 for n in at], [0, 1, 2], 0.09)
            assert_within(od, ref, decode_tolerance(ref, bounds, dtype))
            want = int4.kv_load_int4(caches[0].numpy(), host[:2].numpy())
            assert torch.equal(back[0][:2].cpu(), torch.tensor(want).float().to(dtype))
            assert (back[0][2] == 0).all()
    assert int(status) == 0
    assert np.array_equal(k.cpu().numpy(), caches[0].numpy())
    assert np.array_equal(v.cpu().numpy(), caches[1].numpy())


def test_queries_written_just_before_decode(cuda_device):
    """Decode starts while the kernel before it still runs: it must not read q,
    lengths or tables that kernel writes."""
    c = Case([1] * 64, [200] * 64, 8, 2, 16, torch.bfloat16, seed=30)
    dev = cuda_device
    k, v, tables, lens = (x.to(dev) for x in (c.k, c.v, c.tables, c.lens))
    good, plan = c.q.to(dev), ops.plan_decode(64, 8, 2, 128, 16, 200, kv_int4=True)
    ws = torch.empty(plan.workspace_bytes, dtype=torch.uint8, device=dev)
    want = ops.paged_decode(good, k, v, tables, lens, torch.empty_like(good), plan, c.scale, ws)
    q, n, t = torch.empty_like(good), torch.empty_like(lens), torch.empty_like(tables)
    for _ in range(20):
        q.fill_(9.0)
        n.fill_(1)
        t.fill_(0)
        t.copy_(tables)
        n.copy_(lens)
        q.copy_(good)
        out = ops.paged_decode(q, k, v, t, n, torch.empty_like(q), plan, c.scale, ws)
        assert torch.equal(out, want)
    # and the same call gives the same bits


def test_opcheck(cuda_device):
    dev = cuda_device
    c = Case([1] * 2, [20, 30], 4, 2, 16, torch.bfloat16)
    k, v, tables, lens, q = (x.to(dev) for x in (c.k, c.v, c.tables, c.lens, c.q))
    x = c.key[:2].contiguous().to(dev)
    slots = torch.arange(2, dtype=torch.int32, device=dev)
    b200 = _native.load_torch_ops()
    utils = ("test_schema", "test_faketensor")
    starts = torch.arange(3, dtype=torch.int32, device=dev)
    for op, args in ((b200.kv_append_int4, (x, x, k, v, slots)),
                     (b200.kv_load_int4, (k, v, slots, x, x.clone())),
                     (b200.paged_decode_int4, (q, k, v, tables, lens, torch.empty_like(q), 1, 32,
                                               0.1, torch.empty(1 << 16, dtype=torch.uint8,
                                                                device=dev))),
                     (b200.paged_prefill_int4, (q, k, v, tables, lens, starts,
                                                torch.empty_like(q), 1, 0.1, 2))):
        torch.library.opcheck(op.default, args, test_utils=utils)
