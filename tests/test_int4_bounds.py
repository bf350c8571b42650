"""The bounds of prefill over a 4-bit cache reject results that are wrong: without one
128-token tile, without values, of operands rounded to bf16."""

import numpy as np
import pytest
import torch

from int4_cases import Case, assert_near, assert_within, prefill_bound
from oracle import int4

TYPES = [torch.bfloat16, torch.float16]
SHAPES = [([1], [5000], 4, 1), ([200], [3000], 4, 1), ([30], [2500], 4, 1)]


def _rejected(out, ref, bounds, dtype):
    """Whether both checks together see it."""
    for check in (lambda: assert_within(out, ref, prefill_bound(ref, bounds, dtype)),
                  lambda: assert_near(out, ref, dtype)):
        try:
            check()
        except AssertionError:
            return True
    return False


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("q,kv,hq,hkv", SHAPES)
def test_a_lost_tile_is_seen(dtype, q, kv, hq, hkv):
    c = Case(q, kv, hq, hkv, 16, dtype, seed=kv[0])
    ref, bounds = c.reference()
    assert not _rejected(torch.tensor(ref).to(dtype), ref, bounds, dtype)
    assert _rejected(torch.zeros(ref.shape), ref, bounds, dtype)
    tiles = range(0, kv[0] - q[0], 128)
    for first in list(tiles)[:: max(1, len(tiles) // 6)]:
        lost = Case(q, kv, hq, hkv, 16, dtype, seed=kv[0])
        pages = int4.Pages(lost.v.numpy())
        for token in range(first, min(first + 128, kv[0])):
            page, row = divmod(lost.slots[0][token], 16)
            pages.scales[page, :, row] = 0
        out, _ = lost.reference()
        assert _rejected(torch.tensor(out).to(dtype), ref, bounds, dtype), first


@pytest.mark.parametrize("q,kv,hq,hkv", SHAPES)
def test_operands_in_bf16_are_seen(q, kv, hq, hkv):
    # weights and values rounded to bf16: the bound of fp16 operands by norm is not met
    c = Case(q, kv, hq, hkv, 16, torch.bfloat16, seed=kv[0])
    ref, _ = c.reference()
    t = np.arange(kv[0])
    page = c.tables[0].numpy()[t // 16]
    k, v = (int4.Pages(x.numpy()).get(page, t % 16)[:, 0] for x in (c.k, c.v))
    rows = c.q[:, :1].double().numpy()[:, 0]
    s = rows @ k.T * c.scale
    s[t[None, :] > (kv[0] - q[0] + np.arange(q[0]))[:, None]] = -np.inf
    p = np.exp(s - s.max(1, keepdims=True))
    short = [torch.tensor(x).bfloat16().double().numpy() for x in (p, v)]
    out = torch.tensor(short[0] @ short[1] / p.sum(1, keepdims=True)).bfloat16()
    with pytest.raises(AssertionError, match="by norm"):
        assert_near(out, ref[:, 0], torch.bfloat16)
    assert_near(out, ref[:, 0], torch.bfloat16, wide=True)
