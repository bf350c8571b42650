"""Inputs and tolerances shared by the 4-bit cache tests."""

from __future__ import annotations

import numpy as np
import torch

import oracle
from conftest import dtype_name, storage
from oracle import int4

# Largest relative error of one rounding to a type: half a step.
UNIT = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


class Case:
    """A 4-bit paged batch on the CPU: sequences of ``kv_lens`` tokens, the last
    ``q_lens`` of them queries, over a permuted pool of arbitrary bytes in which
    only the sequences' own slots hold rows."""

    def __init__(self, q_lens, kv_lens, hq, hkv, bs, dtype, seed=0, spread=1.0, v_spread=1.0):
        g = torch.Generator().manual_seed(seed)
        self.q_lens, self.kv_lens, self.hq, self.hkv, self.bs = q_lens, kv_lens, hq, hkv, bs
        self.dtype = dtype
        counts = [(n + bs - 1) // bs for n in kv_lens]
        pool = sum(counts) + 2
        perm = torch.randperm(pool, generator=g)[: sum(counts)].tolist()
        self.tables = torch.full((len(kv_lens), max(counts + [1])), -1, dtype=torch.int32)
        at, self.slots = 0, []
        for i, (n, c) in enumerate(zip(kv_lens, counts)):
            pages = perm[at: at + c]
            at += c
            self.tables[i, :c] = torch.tensor(pages, dtype=torch.int32)
            self.slots.append([pages[t // bs] * bs + t % bs for t in range(n)])
        shape = (pool, bs, hkv, int4.ROW_BYTES)
        self.k = torch.randint(0, 256, shape, generator=g, dtype=torch.uint8)
        self.v = torch.randint(0, 256, shape, generator=g, dtype=torch.uint8)
        n = sum(kv_lens)
        wide = torch.exp(0.5 * torch.randn(hkv, 128, generator=g))
        self.key = (spread * wide * torch.randn(n, hkv, 128, generator=g)).to(dtype)
        self.value = (v_spread * torch.randn(n, hkv, 128, generator=g)).to(dtype)
        self.all_slots = torch.tensor([s for row in self.slots for s in row], dtype=torch.int32)
        int4.kv_append_int4(storage(self.key), storage(self.value), self.k.numpy(),
                            self.v.numpy(), self.all_slots.numpy(), dtype_name(self.key))
        self.q = torch.randn(sum(q_lens), hq, 128, generator=g).to(dtype)
        self.starts = torch.tensor(np.cumsum([0] + list(q_lens)), dtype=torch.int32)
        self.lens = torch.tensor(kv_lens, dtype=torch.int32)
        self.scale = 128 ** -0.5

    def reference(self):
        return int4.attention(self.q.double().numpy(), self.k.numpy(), self.v.numpy(),
                              self.tables.numpy(), self.kv_lens, self.starts.numpy(), self.scale)


def decode_tolerance(ref, bounds, dtype):
    """Decode keeps scores in fp32 (up to 24 roundings of 2^-24 over a score's
    terms: below 2^-19 of them, and twice that on a weight, numerator and sum),
    rounds each weight times the value's scale to fp16 (2^-11) and the result to
    ``dtype``; 2^-19 covers the exponentials (2^-22) and the sums of weights."""
    weight = 2.0 ** -11 + 2.0 ** -19 + np.expm1(2 * 2.0 ** -19 * bounds["terms"])[..., None]
    return UNIT[dtype] * np.abs(ref) + weight * bounds["mass"] * (1 + UNIT[dtype]) + 1e-37


def prefill_tolerance(ref, bounds, dtype):
    """Prefill multiplies 16-bit operands: fp16 ones, exact but for the weights,
    or, for a bf16 call in which a scale leaves fp16's range, bf16 ones: keys and
    values round s (c - 8) then (2^-8 each) and weights to bf16. bf16 calls get the
    wider of the two bounds. Scores stay in fp32 as in decode."""
    u = UNIT[dtype]
    x = u if dtype == torch.bfloat16 else 0.0
    score = x * bounds["keys"] + 2.0 ** -19 * bounds["terms"]
    weight = u + x * (1 + u) + 2.0 ** -19 + np.expm1(2 * score)[..., None]
    return u * np.abs(ref) + weight * bounds["mass"] * (1 + u) + 1e-37


def assert_within(out, ref, tol):
    got = out.detach().double().cpu().numpy()
    assert np.isfinite(got).all()
    over = np.abs(got - ref) - tol
    assert over.max() <= 0, (
        f"{(over > 0).sum()} of {over.size} values off, worst "
        f"{np.abs(got - ref).flat[over.argmax()]:.3e} where {tol.flat[over.argmax()]:.3e} is "
        f"allowed, at {np.unravel_index(over.argmax(), over.shape)}")


def prefill_bound(ref, bounds, dtype, wide=False, bf16_keys=False):
    """The bound of prefill by the operands that a unit really runs with. fp16: keys and
    values are exact and weights round by 2^-11 (those below 2^-21 of a row's largest
    round to multiples of 2^-32 of it: that, for values whose scales lie up to 2^18
    apart, is within the 2^-19 that covers the exponentials). ``wide``: weights and
    values in bf16, keys still exact; ``bf16_keys``: keys, and the queries of fp16 calls, in
    bf16 too. Scores stay in fp32 as in decode. fp16 outputs below its normal range are off
    by half their step, 2^-25."""
    bf16 = UNIT[torch.bfloat16]
    rounded = 2 * bf16 + bf16 ** 2 if wide else UNIT[torch.float16]
    operands = (2 * bf16 + bf16 ** 2 if dtype == torch.float16 else bf16) if bf16_keys else 0.0
    score = operands * bounds["keys"] + 2.0 ** -19 * bounds["terms"]
    weight = rounded + 2.0 ** -19 + np.expm1(2 * score)[..., None]
    u = UNIT[dtype]
    least = 2.0 ** -25 if dtype == torch.float16 else 1e-37
    return u * np.abs(ref) + weight * bounds["mass"] * (1 + u) + least


def assert_near(out, ref, dtype, wide=False, carried=128):
    """By norm, over each output row [128]. A rounding to a unit of u is uniform within u of
    the value's power of two, whose square is 0.5435 of the value's in the mean at most
    (normal values of any deviation), so independent ones come to u sqrt(0.5435 / 3) of a
    row: the output's own, and, wide, the values'. Their squares, 3.5 / n of them in
    variance where n normal values carry the row, scatter by sqrt(3.5 / n), so the norm by
    half of that; four of these are left. A token's weight has one rounding for all its
    values: up to u by norm where one token carries the row, and 1.2 u where a few do that
    are not orthogonal."""
    own, operand = UNIT[dtype], UNIT[torch.bfloat16 if wide else torch.float16]
    spread = (1 + 2 * np.sqrt(3.5 / carried)) ** 2 * 0.5435 / 3
    limit = np.sqrt(spread * (own ** 2 + (operand ** 2 if wide else 0)) + (1.2 * operand) ** 2)
    err = np.linalg.norm(out.detach().double().cpu().numpy() - ref, axis=-1)
    ratio = err / np.maximum(np.linalg.norm(ref, axis=-1), 1e-37)
    assert ratio.max() <= limit, f"a row is {ratio.max():.2e} off by norm, {limit:.2e} is allowed"
