"""The 4-bit cache without a GPU: the oracle's format against hand-made rows, and
the operators' refusals (through fake CUDA tensors and the C ABI)."""

import numpy as np
import pytest
import torch

import my_vllm_b200
from conftest import storage
from my_vllm_b200 import _native, ops
from oracle import int4


def _row(values, dtype=torch.bfloat16):
    x = torch.zeros(1, 128)
    x[0, : len(values)] = torch.tensor(values)
    return storage(x.to(dtype))


def test_codes_of_a_hand_made_group():
    # a = 7: the scale is 1 and halves are ties, which go to the even code
    codes, scales = int4.quantize(_row([7, -7, 0.5, 1.5, 2.5, -0.5, -1.5, 3.25]))
    assert scales[0].tolist() == [1, 0, 0, 0]
    assert codes[0, :8].tolist() == [15, 1, 8, 10, 10, 8, 6, 11]
    assert codes[0, 8:].tolist() == [8] * 120
    back = int4.dequantize(codes, scales)
    assert back[0, :8].tolist() == [7, -7, 0, 2, 2, 0, -2, 3]


def test_scales_round_to_bf16_and_stay_in_range():
    rng = np.random.default_rng(3)
    for dtype in (torch.bfloat16, torch.float16):
        x = torch.tensor(rng.standard_normal((64, 128)) * 10.0 ** rng.integers(-3, 4, (64, 1)))
        codes, scales = int4.quantize(storage(x.to(dtype)), str(dtype)[6:])
        a = x.to(dtype).double().abs().reshape(64, 4, 32).amax(-1)
        assert torch.equal(torch.tensor(scales), (a / 7).float().bfloat16().double())
        assert codes.min() >= 1 and codes.max() <= 15
        err = np.abs(int4.dequantize(codes, scales) - x.to(dtype).double().numpy())
        # half a step, and a largest value whose scale rounded down
        assert (err <= np.repeat(scales, 32, -1) * (0.5 + 7 * 2.0 ** -8)).all()
    codes, scales = int4.quantize(_row([65504.0], torch.float16), "float16")
    assert scales[0, 0] == 9344.0 and codes[0, 0] == 15  # 7 s = 65408 is finite in fp16


def test_groups_without_a_finite_scale():
    codes, scales = int4.quantize(_row([float("nan"), 3.0]))
    assert np.isnan(scales[0, 0]) and (codes == 8).all() and scales[0, 1] == 0
    codes, scales = int4.quantize(_row([float("-inf")]))
    assert np.isnan(scales[0, 0]) and (codes == 8).all()
    codes, scales = int4.quantize(_row([2.0 ** -125]))  # a / 7 is not normal
    assert scales[0, 0] == 0 and (codes == 8).all()


def test_page_layout():
    cache = np.zeros((2, 16, 3, 72), np.uint8)
    key = storage(torch.arange(3 * 128).reshape(1, 3, 128).float().bfloat16())
    int4.kv_append_int4(key, key, cache, cache.copy(), [16 + 5])
    codes, scales = int4.quantize(key)
    page = cache[1].reshape(-1)
    head, row = 2, 5
    at = (head * 16 + row) * 64
    assert page[at] == codes[0, head, 0] | codes[0, head, 1] << 4
    at = 3 * 16 * 64 + (head * 16 + row) * 8
    assert page[at: at + 8].view(np.uint16).tolist() == int4._scale_bits(scales[0, head]).tolist()
    assert not cache[0].any()
    np.testing.assert_array_equal(int4.kv_load_int4(cache, [21])[0],
                                  int4.dequantize(codes, scales)[0])


def test_public_names_and_shape():
    assert my_vllm_b200.int4_cache_shape(10, 32, 4) == (10, 32, 4, 72)
    for bad in ((10, 8, 4), (0, 16, 4), (10, 16, 0)):
        with pytest.raises(ValueError):
            ops.int4_cache_shape(*bad)
    with pytest.raises(ValueError, match="head_dim"):
        ops.int4_cache_shape(10, 16, 4, 64)
    for name in ("store_kvcache_int4", "load_kvcache_int4"):
        assert getattr(my_vllm_b200, name) is getattr(ops, name)


def test_cpu_tensors_are_refused():
    x = torch.zeros(2, 2, 128, dtype=torch.bfloat16)
    cache = torch.zeros(ops.int4_cache_shape(2, 16, 2), dtype=torch.uint8)
    slots = torch.zeros(2, dtype=torch.int32)
    for call in (ops.store_kvcache, ops.store_kvcache_int4):
        with pytest.raises(ValueError, match="CUDA"):
            call(x, x, cache, cache, slots)
    with pytest.raises(ValueError, match="CUDA"):
        ops.load_kvcache_int4(cache, cache, slots, x, x)


@pytest.fixture
def fake():
    from torch._subclasses.fake_tensor import FakeTensorMode

    with FakeTensorMode():
        yield lambda *shape, dtype=torch.bfloat16: torch.empty(*shape, dtype=dtype, device="cuda")


def _i32(fake, *shape):
    return fake(*shape, dtype=torch.int32)


def test_append_and_read_back_refusals(fake):
    x, slots = fake(3, 2, 128), _i32(fake, 3)
    cache = fake(4, 16, 2, 72, dtype=torch.uint8)
    both = (lambda k, v, kc, vc, s: ops.store_kvcache_int4(k, v, kc, vc, s),
            lambda k, v, kc, vc, s: ops.load_kvcache_int4(kc, vc, s, k, v))
    for call in both:
        call(x, x, cache, cache, slots)  # the Meta kernel: traced, not run
        call(x, x, cache, cache, fake(3, dtype=torch.int64))
        call(fake(0, 2, 128), fake(0, 2, 128), cache, cache, _i32(fake, 0))
        with pytest.raises(TypeError, match="float16/bfloat16"):
            call(x.float(), x.float(), cache, cache, slots)
        with pytest.raises(TypeError, match="float16/bfloat16"):
            call(x, x.half(), cache, cache, slots)
        with pytest.raises(TypeError, match="uint8"):
            call(x, x, cache, fake(4, 16, 2, 72, dtype=torch.int8), slots)
        with pytest.raises(ValueError, match="72"):
            call(x, x, fake(4, 16, 2, 64, dtype=torch.uint8),
                 fake(4, 16, 2, 64, dtype=torch.uint8), slots)
        with pytest.raises(ValueError, match="strides"):
            call(x, x, cache, fake(4, 2, 16, 2, 72, dtype=torch.uint8)[:, 0], slots)
        other = fake(4, 2, 16, 72, dtype=torch.uint8).transpose(1, 2)
        with pytest.raises(ValueError, match="packed"):
            call(x, x, other, other, slots)
        with pytest.raises(ValueError, match="num_kv_heads"):
            call(fake(3, 4, 128), fake(3, 4, 128), cache, cache, slots)
        with pytest.raises(ValueError, match="num_kv_heads"):
            call(fake(3, 2, 64), fake(3, 2, 64), cache, cache, slots)
        gap = fake(3, 2, 256)[:, :, :128]
        with pytest.raises(ValueError, match="packed"):
            call(gap, gap, cache, cache, slots)
        with pytest.raises(TypeError, match="int32 or int64"):
            call(x, x, cache, cache, fake(3, dtype=torch.int16))
        for bad in (_i32(fake, 4), _i32(fake, 6)[::2], _i32(fake, 3, 1)):
            with pytest.raises(ValueError, match="one slot per token"):
                call(x, x, cache, cache, bad)


def test_attention_refusals(fake):
    cache = fake(8, 16, 2, 72, dtype=torch.uint8)
    q, out = fake(3, 8, 128), fake(3, 8, 128)
    tables, lens, starts = _i32(fake, 3, 2), _i32(fake, 3), _i32(fake, 4)
    plan, room = ops.DecodePlan(1, 32, 8192), fake(8192, dtype=torch.uint8)

    def decode(q=q, cache=cache, out=out, workspace=room, **more):
        return ops.paged_decode(q, cache, cache, tables, lens, out, plan, 0.1, workspace, **more)

    def prefill(q=q, cache=cache, out=out, **more):
        return ops.paged_prefill(q, cache, cache, tables, lens, starts, out, 1, 0.1, **more)

    for call in (decode, prefill):
        call()
        with pytest.raises(TypeError, match="float16/bfloat16"):
            call(q=fake(3, 8, 128, dtype=torch.float32), out=fake(3, 8, 128, dtype=torch.float32))
        with pytest.raises(ValueError, match="one dtype"):
            call(out=fake(3, 8, 128, dtype=torch.float16))
        with pytest.raises(ValueError, match="72"):
            call(cache=fake(8, 16, 2, 128, dtype=torch.uint8))
        with pytest.raises(ValueError, match="divisible"):
            call(q=fake(3, 7, 128), out=fake(3, 7, 128))
        with pytest.raises(ValueError, match="head_dim"):
            call(q=fake(3, 8, 64), out=fake(3, 8, 64))
        with pytest.raises(ValueError, match="FP8"):
            call(k_scale=fake(1, dtype=torch.float32))
    with pytest.raises(ValueError, match="workspace"):
        decode(workspace=None)
    with pytest.raises(ValueError, match="contiguous"):
        decode(workspace=fake(16384, dtype=torch.uint8)[::2])


def test_plan_for_a_4bit_cache():
    # CTAs that share the batch: three per SM of 148, fewer where each would have
    # under four tiles of 32 tokens (groups of more than 8 heads read theirs twice)
    plan = ops.plan_decode(4, 32, 8, 128, 16, 32768, kv_int4=True)
    assert plan.num_parts == 444 and plan.part_tokens == 32
    assert plan.workspace_bytes >= 2 * 444 * 4 * 129 * 4 + 32 * 16
    assert ops.plan_decode(1, 16, 1, 128, 16, 640, kv_int4=True).num_parts == 10
    # up to 512 tokens a sequence, in one wave: nothing is cut (part_tokens 0)
    for batch, tokens in ((1, 1), (55, 512)):
        plan = ops.plan_decode(batch, 8, 8, 128, 16, tokens, kv_int4=True)
        assert (plan.num_parts, plan.part_tokens) == (1, 0)
    for batch, tokens in ((56, 512), (55, 513)):
        assert ops.plan_decode(batch, 8, 8, 128, 16, tokens, kv_int4=True).part_tokens == 32
    assert ops.plan_decode(9, 8, 1, 128, 16, 32768, total_kv_tokens=6400,
                           kv_int4=True).num_parts == 52
    assert ops.plan_decode(4, 8, 2, 128, 16, 1000, force_num_parts=5, kv_int4=True).num_parts == 5
    with pytest.raises(ValueError, match="either"):
        ops.plan_decode(4, 8, 2, 128, 16, 1000, kv_int4=True, kv_fp8=True)
    with pytest.raises(ValueError, match="head_dim"):
        ops.plan_decode(4, 8, 2, 64, 16, 1000, kv_int4=True)
    with pytest.raises(RuntimeError, match="block_size"):
        ops.plan_decode(4, 8, 2, 128, 8, 1000, kv_int4=True)
    with pytest.raises(ValueError, match="divisible"):
        ops.plan_decode(4, 9, 2, 128, 16, 1000, kv_int4=True)
    with pytest.raises(RuntimeError, match="16 q heads"):
        ops.plan_decode(4, 34, 2, 128, 16, 1000, kv_int4=True)


BF16 = _native.DTYPE_BFLOAT16


def _cache(**change):
    given = dict(k_cache=0x1000, v_cache=0x2000, num_blocks=16, block_size=16, num_kv_heads=2,
                 block_stride_bytes=16 * 2 * 72)
    given.update(change)
    return _native.Int4Cache(*(given[n] for n, _ in _native.Int4Cache._fields_))


BAD_CACHES = [
    (dict(k_cache=None), _native.B200_ERR_INVALID_ARGUMENT, b"both be present"),
    (dict(v_cache=0x2008), _native.B200_ERR_INVALID_ARGUMENT, b"16-byte aligned"),
    (dict(num_blocks=0), _native.B200_ERR_INVALID_ARGUMENT, b"positive"),
    (dict(num_blocks=1 << 31), _native.B200_ERR_UNSUPPORTED, b"int32"),
    (dict(block_size=24), _native.B200_ERR_UNSUPPORTED, b"multiple of 16"),
    (dict(num_kv_heads=0), _native.B200_ERR_INVALID_ARGUMENT, b"positive"),
    (dict(block_stride_bytes=16 * 2 * 72 - 16), _native.B200_ERR_INVALID_ARGUMENT, b"cover"),
    (dict(block_stride_bytes=16 * 2 * 72 + 64), _native.B200_ERR_INVALID_ARGUMENT, b"128 bytes"),
    (dict(block_stride_bytes=1 << 35), _native.B200_ERR_UNSUPPORTED, b"256 GiB"),
]


@pytest.mark.parametrize("change,code,text", BAD_CACHES)
def test_c_abi_refuses_bad_caches(change, code, text):
    lib, bad = _native.load_library(), _cache(**change)
    plan = _native.DecodePlan(1, 32, 0)
    calls = (
        lambda: lib.b200_store_kvcache_int4(0x3000, 256, 0x4000, 256, BF16, bad, 0x5000, 0, 4,
                                            None, None),
        lambda: lib.b200_load_kvcache_int4(bad, 0x5000, 0, 4, 0x3000, 256, 0x4000, 256, BF16,
                                           None, None),
        lambda: lib.b200_paged_decode_int4(0x3000, 1024, 128, BF16, bad, 0x4000, 8, 8, 0x5000, 4,
                                           8, 0x6000, 1024, 128, 0.1, plan, 0x8000, 1 << 20, None,
                                           None),
        lambda: lib.b200_paged_prefill_int4(0x3000, 1024, 128, BF16, bad, 0x4000, 8, 8, 0x5000,
                                            0x7000, 4, 8, 2, 8, 0x6000, 1024, 128, 0.1, None,
                                            0, None, None),
    )
    for call in calls:
        assert call() == code
        assert text in lib.b200_last_error()


def test_c_abi_refuses_bad_rows_and_sizes():
    lib, c = _native.load_library(), _cache()

    def store(key=0x3000, stride=256, dtype=BF16, n=4, slots=0x5000):
        return lib.b200_store_kvcache_int4(key, stride, 0x4000, 256, dtype, c, slots, 0, n, None,
                                           None)

    assert store(dtype=7) == _native.B200_ERR_UNSUPPORTED
    assert store(n=-1) == _native.B200_ERR_INVALID_ARGUMENT
    assert store(key=0x3008) == _native.B200_ERR_INVALID_ARGUMENT
    assert store(stride=260) == _native.B200_ERR_INVALID_ARGUMENT
    assert store(stride=128) == _native.B200_ERR_INVALID_ARGUMENT
    assert store(slots=None) == _native.B200_ERR_INVALID_ARGUMENT
    assert store(n=0, key=None) == _native.B200_OK

    def decode(hq=8, q=0x3000, plan=_native.DecodePlan(2, 32, 0), ws=0x8000, nbytes=1 << 20, n=4):
        return lib.b200_paged_decode_int4(q, 1024, 128, BF16, c, 0x4000, 8, 8, 0x5000, n, hq,
                                          0x6000, 1024, 128, 0.1, plan, ws, nbytes, None, None)

    assert decode(hq=9) == _native.B200_ERR_INVALID_ARGUMENT
    assert decode(hq=34) == _native.B200_ERR_UNSUPPORTED  # 17 heads per KV head
    assert decode(q=0x3002) == _native.B200_ERR_INVALID_ARGUMENT
    assert decode(q=None) == _native.B200_ERR_INVALID_ARGUMENT
    assert decode(plan=None) == _native.B200_ERR_INVALID_ARGUMENT
    for bad in (_native.DecodePlan(0, 32, 0), _native.DecodePlan(1, 4096, 0)):
        assert decode(plan=bad) == _native.B200_ERR_INVALID_ARGUMENT
        assert b"4-bit" in lib.b200_last_error()
    assert decode(ws=None) == _native.B200_ERR_INVALID_ARGUMENT
    assert b"workspace" in lib.b200_last_error()
    assert decode(nbytes=4096) == _native.B200_ERR_INVALID_ARGUMENT
    assert decode(ws=0x8010) == _native.B200_ERR_INVALID_ARGUMENT
    assert decode(n=0, q=None) == _native.B200_OK

    def prefill(hq=8, q=0x3000, rows=8, most=2, scale=0.1, n=4, ws=None, nbytes=0):
        return lib.b200_paged_prefill_int4(q, 1024, 128, BF16, c, 0x4000, 8, 8, 0x5000, 0x7000, n,
                                           rows, most, hq, 0x6000, 1024, 128, scale, ws, nbytes,
                                           None, None)

    assert prefill(hq=9) == _native.B200_ERR_INVALID_ARGUMENT
    assert prefill(hq=2 * 129) == _native.B200_ERR_UNSUPPORTED
    assert prefill(q=0x3008) == _native.B200_ERR_INVALID_ARGUMENT
    assert prefill(most=0) == _native.B200_ERR_INVALID_ARGUMENT
    assert prefill(scale=0.0) == _native.B200_ERR_INVALID_ARGUMENT
    assert prefill(scale=float("nan")) == _native.B200_ERR_INVALID_ARGUMENT
    assert prefill(rows=-1) == _native.B200_ERR_INVALID_ARGUMENT
    assert prefill(ws=0x8010, nbytes=1 << 30) == _native.B200_ERR_INVALID_ARGUMENT
    assert prefill(ws=0x8000, nbytes=4096) == _native.B200_ERR_INVALID_ARGUMENT
    assert b"workspace" in lib.b200_last_error()
    assert prefill(rows=0, q=None) == _native.B200_OK


@pytest.mark.parametrize("scale", [0.0, -0.1, float("nan"), float("-inf")])
def test_attention_refuses_a_scale_that_is_not_positive(scale):
    lib, c, plan = _native.load_library(), _cache(), _native.DecodePlan(2, 32, 0)
    calls = (
        lambda: lib.b200_paged_decode_int4(0x3000, 1024, 128, BF16, c, 0x4000, 8, 8, 0x5000, 4, 8,
                                           0x6000, 1024, 128, scale, plan, 0x8000, 1 << 20, None,
                                           None),
        lambda: lib.b200_paged_prefill_int4(0x3000, 1024, 128, BF16, c, 0x4000, 8, 8, 0x5000,
                                            0x7000, 4, 8, 2, 8, 0x6000, 1024, 128, scale, None, 0,
                                            None, None),
    )
    for call in calls:
        assert call() == _native.B200_ERR_INVALID_ARGUMENT
        assert b"softmax_scale" in lib.b200_last_error()
