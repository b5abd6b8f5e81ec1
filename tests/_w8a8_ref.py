"""Plain forms of the W8A8 products and of the expert-sorted rows, in numpy.

The quantiser and the products are defined operation by operation in fp32
around a sum of whole numbers, so the references below give the calls' bits:
whole numbers are summed in float64 (exact up to 2^53), the fp32 operations are
numpy's own (IEEE).
"""
import numpy as np

TINY = np.float32(2.0**-126)


def bf16(v):
    """fp32 -> the nearest bf16 value (ties to even), as fp32."""
    v = np.ascontiguousarray(v, np.float32)
    u = v.view(np.uint32).astype(np.uint64)
    r = ((u + 0x7FFF + ((u >> 16) & 1)) & 0xFFFF0000).astype(np.uint32).view(np.float32)
    return np.where(np.isnan(v), v, r)


def f16(v):
    """fp32 -> the nearest fp16 value, finite values saturating, as fp32."""
    v = np.asarray(v, np.float32)
    return np.where(np.isfinite(v), np.clip(v, -65504, 65504), v).astype(np.float16).astype(np.float32)


ROUND = {"f32": lambda v: np.asarray(v, np.float32), "bf16": bf16, "f16": f16}


def quant(x):
    """(q as float64 whole numbers, scale fp32) of fp32 rows."""
    x = np.asarray(x, np.float32)
    with np.errstate(all="ignore"):
        a = np.abs(x).max(-1)
        bad = ~np.isfinite(a)
        s = np.where(a > 0, np.maximum(a / np.float32(127), TINY), np.float32(1)).astype(np.float32)
        q = np.rint(x * (np.float32(1) / s)[:, None])
    return np.where(bad[:, None], 0, q).astype(np.float64), np.where(bad, np.float32(np.nan), s).astype(np.float32)


def product(q, sx, W, sw):
    """fp32 values of the product before their rounding to the output's type."""
    sums = q @ np.asarray(W, np.float64).T
    with np.errstate(all="ignore"):
        return (sums.astype(np.float32) * sw[None, :].astype(np.float32)) * sx[:, None]


def sort(top_e, E):
    """(counts, offsets, tok_slot, pair_tok) of choices top_e [T][k]."""
    flat = top_e.reshape(-1).astype(np.int64)
    key = np.where((flat >= 0) & (flat < E), flat, E)
    order = np.argsort(key, kind="stable")
    counts = np.bincount(key, minlength=E + 1)[:E]
    offsets = np.concatenate([[0], np.cumsum(counts)])
    slot = np.empty(len(flat), np.int64)
    slot[order] = np.arange(len(flat))
    kept = offsets[-1]
    tok = np.where(np.arange(len(flat)) < kept, order // top_e.shape[1], -1)
    return counts, offsets, np.where(key < E, slot, -1).reshape(top_e.shape), tok


def tiles(counts, tile_m):
    """The (expert, first slot) list of a tile_m as qw_moe_route defines it."""
    out = []
    for e, c in enumerate(counts):
        m0 = 0
        while m0 < c:
            out.append((e, m0))
            rem, g = c - m0, -tile_m
            m0 += tile_m if tile_m > 0 else 4 * g if rem > 5 * g else (rem + g - 1) // g * g
    return out
