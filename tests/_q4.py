"""The 4-bit cache in numpy, in 64 bits, for the tests: packing, reading back, and attention over it."""

from __future__ import annotations

import numpy as np

GROUP, TILE, BLOCK = 64, 16, 1152


def _bf16(x: np.ndarray) -> np.ndarray:
    """Round to BF16, ties to even, as float64 (finite inputs that FP32 holds)."""
    bits = np.asarray(x, np.float32).view(np.uint32).astype(np.uint64)
    bits = (bits + 0x7FFF + ((bits >> 16) & 1)) & 0xFFFF0000
    return bits.astype(np.uint32).view(np.float32).astype(np.float64)


def quantise(rows: np.ndarray) -> tuple[np.ndarray, np.ndarray, np.ndarray]:
    """Codes, scale and low of rows [..., 64] of BF16 values; the quotients are exact to far below half a step away from
    a tie (a ratio of two BF16-grid numbers that is not a tie is at least 2^-17 from one)."""
    rows = np.asarray(rows, np.float64)
    low = rows.min(-1, keepdims=True)
    scale = _bf16((rows.max(-1, keepdims=True) - low) / 15)
    with np.errstate(divide="ignore", invalid="ignore"):
        codes = np.where(scale > 0, np.clip(np.rint((rows - low) / scale), 0, 15), 0)
    return codes, scale, low


def dequantise(rows: np.ndarray) -> np.ndarray:
    codes, scale, low = quantise(rows)
    return codes * scale + low


def attend(q: np.ndarray, cache: np.ndarray, lengths, heads: int) -> tuple[np.ndarray, np.ndarray]:
    """(out, bound) of queries [seqs, heads, head] over a packed uint8 cache [seqs, kv_heads, tiles, size]: the softmax
    average in 64 bits, and how far a BF16 result may be from it.

    The bound: the result's own rounding, half a BF16 step (2^-8 of it); each weight p_j scale_j in the products with
    the value codes rounded to FP16 (2^-11 of it), which moves the average by at most 2^-11 of the values' widest
    range R = 15 scale; a score computed from n products accumulated in FP32, the codes entering as 128 + code, off by
    at most n 2^-23 sum |q| (143 scale + |low|), twice that in the weights' ratio; the sums over the keys, n_keys 2^-23
    of R; and the exponentials, 2^-21 of R."""
    seqs, kv_heads, tiles, size = cache.shape
    groups = size // BLOCK
    head, share = groups * GROUP, heads // kv_heads
    out = np.zeros((seqs, heads, head))
    bound = np.zeros((seqs, heads, head))
    for s in range(seqs):
        n = int(np.clip(lengths[s], 0, tiles * TILE))
        if n == 0:
            continue
        for h in range(kv_heads):
            blocks = cache[s, h].reshape(tiles, groups, BLOCK)
            meta = np.ascontiguousarray(blocks[:, :, 1024:]).view(np.uint16).reshape(tiles, groups, TILE, 4)
            meta = (meta.astype(np.uint32) << 16).view(np.float32).astype(np.float64)
            kv, scales, lows = [], [], []
            for at in (0, 1):
                b = blocks[:, :, 512 * at:512 * at + 512].reshape(tiles, groups, TILE, 32)
                codes = np.stack([b & 15, b >> 4], -1).reshape(tiles, groups, TILE, GROUP).astype(np.float64)
                x = codes * meta[..., 2 * at, None] + meta[..., 2 * at + 1, None]
                kv.append(x.transpose(0, 2, 1, 3).reshape(tiles * TILE, head)[:n])
                scales.append(meta[..., 2 * at].transpose(0, 2, 1).reshape(-1, groups)[:n])
                lows.append(meta[..., 2 * at + 1].transpose(0, 2, 1).reshape(-1, groups)[:n])
            wide = np.repeat(15 * scales[1].max(0), GROUP)[None, :]
            for r in range(h * share, (h + 1) * share):
                score = kv[0] @ q[s, r]
                p = np.exp(score - score.max())
                p /= p.sum()
                out[s, r] = p @ kv[1]
                spread = np.abs(q[s, r]).sum() * (143 * scales[0].max() + np.abs(lows[0]).max())
                bound[s, r] = (2.0 ** -8 * np.abs(out[s, r]) +
                               wide * (2.0 ** -11 + 2 * head * 2.0 ** -23 * spread + n * 2.0 ** -23 + 2.0 ** -21) + 1e-30)
    return out, bound
