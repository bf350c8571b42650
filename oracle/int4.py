"""4-bit KV-cache format — TEST INFRASTRUCTURE ONLY (see ``oracle/__init__.py``).

No counterpart in the reference, whose attention contract accepts 16-bit caches
only (nanovllm/layers/attention_backend.py:516-519). A row is the 128 values of
one (slot, KV head) in four groups of 32; per group, with a = max |x|:

    s = bf16(a / 7), nearest even (float16 rows: at most 9344); 0 below 2^-126;
        NaN where a is not finite
    c = 8 + rint(fl32(x * fl32(1 / s)))   (8 where s is 0 or NaN)

stand for s * (c - 8). A page of ``bs`` slots holds codes [heads][bs][64] (even
elements in the low nibble), then scales [heads][bs][4] bf16. Everything is
computed in 64 bits and rounded to fp32 where the format says so.
"""

from __future__ import annotations

import numpy as np

from .paged_attention import to_f32

GROUP = 32
ROW_BYTES = 72
FP16_MAX_SCALE = 9344.0


def _round_bf16(x: np.ndarray) -> np.ndarray:
    """Nearest bf16, ties to even, of non-negative doubles (normal range)."""
    m, e = np.frexp(x)
    return np.ldexp(np.rint(np.ldexp(m, 8)), e - 8)


def quantize(x, dtype: str = "bfloat16"):
    """16-bit storage rows [..., 128] -> (codes uint8 [..., 128] of 0..15,
    scales float64 [..., 4])."""
    v = to_f32(x, dtype).astype(np.float64)
    g = v.reshape(v.shape[:-1] + (4, GROUP))
    a = np.max(np.abs(g), axis=-1)  # NaN propagates
    fine = np.isfinite(a)
    s = _round_bf16(np.where(fine, a, 0.0) / 7.0)
    if dtype == "float16":
        s = np.minimum(s, FP16_MAX_SCALE)
    s = np.where(s < 2.0 ** -126, 0.0, s)
    with np.errstate(divide="ignore"):
        r = np.where(s > 0, 1.0 / s, 0.0).astype(np.float32).astype(np.float64)
    product = np.where(fine[..., None], g, 0.0) * r[..., None]  # exact: 11 + 24 bits
    c = 8 + np.rint(product.astype(np.float32).astype(np.float64))
    return (c.reshape(v.shape).astype(np.uint8), np.where(fine, s, np.nan))


def dequantize(codes, scales) -> np.ndarray:
    """codes [..., 128], scales [..., 4] -> float64 values."""
    c = codes.astype(np.float64).reshape(codes.shape[:-1] + (4, GROUP)) - 8.0
    return (c * scales[..., None]).reshape(codes.shape)


def _scale_bits(s) -> np.ndarray:
    bits = np.asarray(s, dtype=np.float32).view(np.uint32)
    return np.where(np.isnan(s), 0x7FC0, bits >> 16).astype(np.uint16)


class Pages:
    """Views of a uint8 cache [blocks, bs, heads, 72] as its rows."""

    def __init__(self, cache: np.ndarray):
        assert cache.dtype == np.uint8 and cache.shape[3] == ROW_BYTES
        self.blocks, self.bs, self.heads, _ = cache.shape
        flat = cache.reshape(self.blocks, -1)
        n = self.heads * self.bs * 64
        self.codes = flat[:, :n].reshape(self.blocks, self.heads, self.bs, 64)
        self.scales = flat[:, n:].reshape(self.blocks, self.heads, self.bs, 8)

    def put(self, slot: int, codes: np.ndarray, scales: np.ndarray) -> None:
        """codes [heads, 128], scales [heads, 4]."""
        page, row = divmod(slot, self.bs)
        self.codes[page, :, row] = codes[:, 0::2] | (codes[:, 1::2] << 4)
        self.scales[page, :, row] = _scale_bits(scales).view(np.uint8).reshape(self.heads, 8)

    def get(self, page, row):
        """float64 [n, heads, 128] of the slots (page[i], row[i])."""
        raw = self.codes[page, :, row]
        codes = np.empty(raw.shape[:-1] + (128,), np.uint8)
        codes[..., 0::2] = raw & 15
        codes[..., 1::2] = raw >> 4
        bits = np.ascontiguousarray(self.scales[page, :, row]).view(np.uint16).astype(np.uint32)
        return dequantize(codes, (bits << 16).view(np.float32).astype(np.float64))


def kv_append_int4(key, value, k_cache, v_cache, slot_mapping, dtype="bfloat16") -> None:
    """In place: slot ``slot_mapping[i]`` of the uint8 caches <- row i quantised;
    -1 skipped. ``key``/``value``: 16-bit storage [tokens, heads, 128]."""
    kc, ks = quantize(key, dtype)
    vc, vs = quantize(value, dtype)
    kp, vp = Pages(k_cache), Pages(v_cache)
    for i, slot in enumerate(np.asarray(slot_mapping).tolist()):
        if slot != -1:
            kp.put(slot, kc[i], ks[i])
            vp.put(slot, vc[i], vs[i])


def kv_load_int4(cache, slots) -> np.ndarray:
    """float64 [n, heads, 128] of the slots."""
    pages = Pages(cache)
    slots = np.asarray(slots)
    return pages.get(slots // pages.bs, slots % pages.bs)


def attention(q, k_cache, v_cache, block_tables, seq_lens, query_start_loc, scale):
    """Causal attention in 64 bits over 4-bit caches. ``q`` float64 [T, Hq, 128].
    Returns (out, bounds). bounds["mass"] = sum_t p_t (|v_t| + s_t / 32) is what a
    relative error of the weights is multiplied with (s / 32: codes and their
    offset of 8 are summed apart, 16 s * 2^-20 being s / 32 * 2^-11);
    bounds["keys"] [T, Hq] the largest scale * sum_d |q_d k_d| and
    bounds["terms"] the largest scale * sum_d |q_d| (|k_d| + 16 s): what relative
    errors of the keys and of the score's terms are multiplied with. Rows
    without tokens give zeros."""
    kp, vp = Pages(k_cache), Pages(v_cache)
    T, hq, _ = q.shape
    out, mass = np.zeros(q.shape), np.zeros(q.shape)
    keys, terms = np.zeros((T, hq)), np.zeros((T, hq))
    group = hq // kp.heads
    for s, n in enumerate(np.asarray(seq_lens).tolist()):
        q0, q1 = int(query_start_loc[s]), int(query_start_loc[s + 1])
        if n <= 0 or q1 <= q0:
            continue
        t = np.arange(n)
        page = np.asarray(block_tables[s])[t // kp.bs]
        k, v = kp.get(page, t % kp.bs), vp.get(page, t % kp.bs)
        wide = np.abs(k) + 16 * _row_scales(kp, page, t % kp.bs)
        v_step = _row_scales(vp, page, t % kp.bs) / 32
        visible = t[None, :] <= (n - (q1 - q0) + np.arange(q1 - q0))[:, None]
        for h in range(hq):
            x = q[q0:q1, h]
            sc = (x @ k[:, h // group].T) * scale
            sc = np.where(visible, sc, -np.inf)
            km = np.where(visible, (np.abs(x) @ np.abs(k[:, h // group]).T) * scale, 0.0)
            tm = np.where(visible, (np.abs(x) @ wide[:, h // group].T) * scale, 0.0)
            top = sc.max(axis=1, keepdims=True)
            p = np.exp(sc - np.where(np.isneginf(top), 0.0, top))
            p /= np.maximum(p.sum(axis=1, keepdims=True), 1e-300)  # no token: a row of zeros
            vv = v[:, h // group]
            out[q0:q1, h] = p @ vv
            mass[q0:q1, h] = p @ (np.abs(vv) + v_step[:, h // group])
            keys[q0:q1, h] = km.max(axis=1)
            terms[q0:q1, h] = tm.max(axis=1)
    return out, {"mass": mass, "keys": keys, "terms": terms}


def _row_scales(pages: Pages, page, row) -> np.ndarray:
    """float64 [n, heads, 128]: the scale of each value."""
    bits = np.ascontiguousarray(pages.scales[page, :, row]).view(np.uint16).astype(np.uint32)
    return np.repeat((bits << 16).view(np.float32).astype(np.float64), GROUP, axis=-1)
