"""Decode over a 4-bit cache whose value scales lie far apart: between groups of a
head, between tokens, between the tokens that the heads of a group attend to, and
near the ends of the scales' range."""

import numpy as np
import pytest
import torch

from conftest import dtype_name, storage
from int4_cases import Case, assert_within, decode_tolerance
from my_vllm_b200 import ops
from oracle import int4

pytestmark = pytest.mark.gpu


def _rewrite(c, key=None, value=None):
    """Append the case's rows again, with other keys or values ([tokens, heads, 128])."""
    key = c.key if key is None else key.to(c.dtype)
    value = c.value if value is None else value.to(c.dtype)
    int4.kv_append_int4(storage(key), storage(value), c.k.numpy(), c.v.numpy(),
                        c.all_slots.numpy(), dtype_name(key))


def _decode(c, dev, parts=0):
    q = c.q.to(dev)
    out = torch.full_like(q, float("nan"))
    plan = ops.plan_decode(len(c.kv_lens), c.hq, c.hkv, 128, c.bs, max(c.kv_lens),
                           force_num_parts=parts, total_kv_tokens=sum(c.kv_lens), kv_int4=True)
    ws = torch.full((plan.workspace_bytes,), 255, dtype=torch.uint8, device=dev)
    ops.paged_decode(q, c.k.to(dev), c.v.to(dev), c.tables.to(dev), c.lens.to(dev), out, plan,
                     c.scale, ws)
    return out


def _check(c, dev, parts=0):
    out = _decode(c, dev, parts)
    ref, bounds = c.reference()
    assert_within(out, ref, decode_tolerance(ref, bounds, c.dtype))
    return out, ref


def _groups(*exponents):
    """Factors 2^exponent for the four groups of a row."""
    return torch.repeat_interleave(2.0 ** torch.tensor(exponents, dtype=torch.float64), 32)


def _tokens(c):
    """Position of each of the case's rows in its sequence, and its length."""
    return (torch.cat([torch.arange(n) for n in c.kv_lens]),
            torch.cat([torch.full((n,), n) for n in c.kv_lens]))


HEADS = [(4, 1), (8, 1), (3, 3), (16, 1)]


@pytest.mark.parametrize("parts", [1, 3])
@pytest.mark.parametrize("hq,hkv", HEADS)
@pytest.mark.parametrize("apart", [16, 24, 40, 90])
def test_one_group_above_the_others(cuda_device, apart, hq, hkv, parts):
    c = Case([1] * 3, [33, 400, 1500], hq, hkv, 16, torch.bfloat16, seed=apart)
    _rewrite(c, value=c.value.double() * _groups(0, 0, apart, -5))
    _check(c, cuda_device, parts)


def test_one_group_above_the_others_fp16(cuda_device):
    c = Case([1] * 3, [33, 400, 1500], 8, 2, 16, torch.float16, seed=1)
    _rewrite(c, value=c.value.double() * _groups(-8, 10, -10, 0))
    _check(c, cuda_device)


def _push(c, seq, token, scores):
    """The key that gives the heads of a KV head these scores (nats) against one token of a
    sequence, before it is quantised; [heads, 128]."""
    group = c.hq // c.hkv
    key = torch.zeros(c.hkv, 128, dtype=torch.float64)
    for h in range(c.hkv):
        q = c.q[seq, h * group:(h + 1) * group].double()
        key[h] = torch.linalg.lstsq(q, torch.tensor(scores, dtype=torch.float64) / c.scale).solution
    return key


@pytest.mark.parametrize("parts", [1, 2])
@pytest.mark.parametrize("hq,hkv", HEADS[:3])
@pytest.mark.parametrize("token", [0, 37, 399])
def test_one_token_above_the_others_with_a_low_score(cuda_device, token, hq, hkv, parts):
    # its weight is some 2^-23 of the others', its values 2^24 times theirs
    c = Case([1], [400], hq, hkv, 16, torch.bfloat16, seed=token + hq)
    key, value = c.key.double(), c.value.double()
    key[token] = _push(c, 0, token, [-16.0] * (hq // hkv))
    value[token] *= 2.0 ** 24
    _rewrite(c, key, value)
    _check(c, cuda_device, parts)


@pytest.mark.parametrize("hq,hkv", [(4, 1), (8, 1)])
@pytest.mark.parametrize("token", [2, 200])
def test_one_token_that_one_head_attends_to(cuda_device, token, hq, hkv):
    # the first head gives the large token most of its weight, the others next to none
    c = Case([1], [300], hq, hkv, 16, torch.bfloat16, seed=token)
    key, value = c.key.double(), c.value.double()
    key[token] = _push(c, 0, token, [8.0] + [-16.0] * (hq - 1))
    value[token] *= 2.0 ** 24
    _rewrite(c, key, value)
    _check(c, cuda_device, 1)


@pytest.mark.parametrize("hq,hkv", [(4, 1), (8, 1)])
def test_a_group_that_only_early_low_scores_have(cuda_device, hq, hkv):
    # group 1 holds values among the first 100 tokens alone, whose scores are 40 below the
    # rest, group 3 from token 300 on
    c = Case([1], [500], hq, hkv, 16, torch.bfloat16, seed=5)
    key, value = c.key.double(), c.value.double()
    at = torch.arange(500)
    key[at < 100] += _push(c, 0, 0, [-40.0] * (hq // hkv))
    value[at >= 100, :, 32:64] = 0
    value[at < 300, :, 96:] = 0
    _rewrite(c, key, value)
    out, ref = _check(c, cuda_device, 1)
    assert (out[:, :, 32:64] != 0).any() and (out[:, :, 96:] != 0).any()


@pytest.mark.parametrize("parts", [1, 2])
def test_groups_that_drift_apart(cuda_device, parts):
    c = Case([1] * 2, [700, 90], 8, 1, 16, torch.bfloat16, seed=6)
    at, n = _tokens(c)
    value = c.value.double().unflatten(2, (4, 32))
    drift = (at / n)[:, None] * torch.tensor([40.0, -40.0, 80.0, 0.0])
    _rewrite(c, value=(value * (2.0 ** drift)[:, None, :, None]).flatten(2))
    _check(c, cuda_device, parts)


@pytest.mark.parametrize("parts", [1, 3])
@pytest.mark.parametrize("exponent", [-110, -95, 116, 120])
def test_values_near_the_ends_of_the_range(cuda_device, exponent, parts):
    c = Case([1] * 3, [5, 130, 1000], 8, 2, 16, torch.bfloat16, seed=8, spread=4.0)
    _rewrite(c, value=c.value.double() * 2.0 ** exponent)
    _check(c, cuda_device, parts)


def test_zero_values(cuda_device):
    c = Case([1] * 2, [40, 300], 8, 2, 16, torch.float16, seed=3)
    _rewrite(c, value=torch.zeros_like(c.value))
    assert (_decode(c, cuda_device) == 0).all()


def test_a_token_without_a_finite_scale_beside_large_ones(cuda_device):
    c = Case([1], [200], 8, 1, 16, torch.bfloat16, seed=4)
    _rewrite(c, value=c.value.double() * _groups(0, 30, 0, -30))
    page, row = divmod(c.slots[0][50], 16)
    int4.Pages(c.v.numpy()).scales[page, 0, row].view(np.uint16)[2] = 0x7FC0
    out = _decode(c, cuda_device).cpu().double()
    ref, bounds = c.reference()
    bad = torch.zeros(out.shape, dtype=torch.bool)
    bad[:, :, 64:96] = True
    assert torch.equal(out.isnan(), bad)
    assert_within(out.masked_fill(bad, 0.0), np.nan_to_num(ref),
                  np.nan_to_num(decode_tolerance(ref, bounds, c.dtype)))


@pytest.mark.parametrize("n,parts", [(2048, 1), (32768, 1), (32768, 0), (131072, 1)])
def test_flat_softmax_over_long_sequences(cuda_device, n, parts):
    """Against 64 bits by norm. The weights' roundings (2^-11 of each, of either sign) add up
    like the values themselves, so they stay 2^-11 of the result; its own is another 2^-11.
    What grows with the length would be a bias of the sums, of which 2^-10 is left."""
    c = Case([1], [n], 4, 1, 16, torch.float16, seed=n, spread=0.01)
    out = _decode(c, cuda_device, parts).cpu().double().numpy()
    ref, _ = c.reference()
    err = np.linalg.norm(out - ref, axis=-1) / np.linalg.norm(ref, axis=-1)
    assert err.max() <= 2.0 ** -9


@pytest.mark.parametrize("scale", [1e-3, 1e-30, 1e-44])
def test_small_softmax_scales(cuda_device, scale):
    # scores that vanish: means of the values, over partial tiles too
    c = Case([1] * 2, [40, 33], 8, 2, 16, torch.float16, seed=2)
    c.q[0] *= 2.0 ** -10
    c.scale = scale
    _check(c, cuda_device)


@pytest.mark.parametrize("parts", [1, 3])
@pytest.mark.parametrize("hq,hkv", [(4, 1), (8, 1)])
def test_scores_of_minus_infinity_in_front(cuda_device, hq, hkv, parts):
    # scores below fp32's range against the first 13 pages, and some -3000 behind them
    c = Case([1], [500], hq, hkv, 16, torch.bfloat16, seed=5)
    key = c.key.double() + _push(c, 0, 0, [-400.0] * hq)
    key[:208] = _push(c, 0, 0, [-1.0] * hq) * 2.0 ** 126
    _rewrite(c, key)
    c.scale *= 8
    out = _decode(c, cuda_device, parts)
    # as if those pages were not there
    ref, bounds = int4.attention(c.q.double().numpy(), c.k.numpy(), c.v.numpy(),
                                 c.tables.numpy()[:, 13:], [292], [0, 1], c.scale)
    assert_within(out, ref, decode_tolerance(ref, bounds, c.dtype))
