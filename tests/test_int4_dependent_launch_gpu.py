"""Decode over a 4-bit cache is launched before the kernel in front of it has ended: it
must not read what that kernel writes. The append in front lets it start early."""

import pytest
import torch

from int4_cases import Case
from my_vllm_b200 import ops

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("parts", [0, 1, 37])
def test_decode_right_behind_an_append_of_its_slots(cuda_device, parts):
    dev = cuda_device
    c = Case([1] * 48, [170] * 48, 8, 2, 16, torch.bfloat16, seed=31)
    q, tables, lens = (x.to(dev) for x in (c.q, c.tables, c.lens))
    key, value, slots = (x.to(dev) for x in (c.key, c.value, c.all_slots))
    # the same rows many times over in front of them: the append has blocks that start late
    many = [x.repeat(24, *[1] * (x.dim() - 1)) for x in (key, value)]
    skipped = torch.full((23 * slots.numel(),), -1, dtype=slots.dtype, device=dev)
    late = torch.cat([skipped, slots])
    plan = ops.plan_decode(48, 8, 2, 128, 16, 170, force_num_parts=parts, kv_int4=True)
    assert (plan.part_tokens == 0) == (parts == 0)
    ws = torch.empty(plan.workspace_bytes, dtype=torch.uint8, device=dev)
    other = [torch.randint(0, 256, c.k.shape, dtype=torch.uint8, device=dev) for _ in range(2)]
    k, v = (x.to(dev) for x in (c.k, c.v))
    want = ops.paged_decode(q, k, v, tables, lens, torch.empty_like(q), plan, c.scale, ws)
    for _ in range(10):
        k.copy_(other[0])
        v.copy_(other[1])
        out = torch.full_like(q, float("nan"))
        torch.cuda.synchronize()
        ops.store_kvcache(*many, k, v, late)
        ops.paged_decode(q, k, v, tables, lens, out, plan, c.scale, ws)
        assert torch.equal(out, want)
