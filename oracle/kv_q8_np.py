"""The 8-bit K/V cache and the per-head norm with rotation, restated in numpy.

Everything is computed in fp64 from the formulas: codes are held as the values
they stand for before their scale, so a pool is an array of multiples of the
format's units and its rows are ``codes * scale``.
"""

from __future__ import annotations

import numpy as np

LARGEST = {"e4m3": 448.0, "int8": 127.0}


def scale_for(amax: float, fmt: str) -> float:
    """Smallest power of two s >= 2^-126 with amax <= largest * s."""
    s = 2.0 ** -126
    while amax > LARGEST[fmt] * s:
        s *= 2.0
    return s


def encode(x: np.ndarray, fmt: str) -> np.ndarray:
    """Nearest code values of x, ties to even; NaN stays NaN in e4m3, 0 in int8."""
    x = np.asarray(x, np.float64)
    if fmt == "int8":
        return np.clip(np.rint(np.where(np.isnan(x), 0.0, x)), -127, 127)
    # units of the last place: 2^(e - 3), e = floor(log2 |x|) but at least -6
    _, e = np.frexp(np.where(np.isfinite(x), x, 0.0))
    unit = np.ldexp(1.0, np.maximum(e - 1, -6) - 3)
    return np.clip(np.rint(x / unit) * unit, -448.0, 448.0)


def write(codes: np.ndarray, scale: np.ndarray, rows: np.ndarray, slots, bs: int,
          fmt: str) -> None:
    """Rows [N, Hkv, D] into codes [num_slots, Hkv, D] and scale [num_blocks, Hkv]
    in place; negative slots are skipped, the last row of a slot counts."""
    last = {int(s): i for i, s in enumerate(slots) if s >= 0}
    blocks: dict[int, dict[int, int]] = {}
    for s, i in last.items():
        blocks.setdefault(s // bs, {})[s % bs] = i
    for b, held in blocks.items():
        at = sorted(held)
        new = rows[[held[o] for o in at]].astype(np.float64)
        rest = [o for o in range(bs) if o not in held]
        for h in range(scale.shape[1]):
            x = new[:, h]
            fin = np.abs(x[np.isfinite(x)])
            need = scale_for(fin.max() if fin.size else 0.0, fmt)
            old = 0.0 if 0 in held else float(scale[b, h])
            now = max(old, need) if old == old else old
            if fmt == "int8" and not np.isfinite(x).all():
                now = np.nan
            if 0 not in held and now == now and now != old:
                base = [b * bs + o for o in rest]
                codes[base, h] = encode(codes[base, h] * (old / now), fmt)
            x = np.where(np.isfinite(x), x, np.nan)
            codes[[b * bs + o for o in at], h] = encode(x / now, fmt)
            scale[b, h] = now


def values(codes: np.ndarray, scale: np.ndarray, bs: int) -> np.ndarray:
    """fp64 rows of the whole pool."""
    return codes * np.repeat(scale.astype(np.float64), bs, axis=0)[:, :, None]


def attend(q: np.ndarray, k: np.ndarray, v: np.ndarray, scale: float):
    """One query row q [H, D] over k, v [T, Hkv, D] (fp64): ``(out [H, D],
    weighted magnitude [H, D], largest score sum [H])``. The second is
    sum_j p_j |v_j|, what a relative error of the weights is multiplied with;
    the third max_j sum_d |q_d k_jd| * scale, what rounding a score is relative
    to."""
    h, d = q.shape
    if k.shape[0] == 0:
        return np.zeros((h, d)), np.zeros((h, d)), np.zeros(h)
    rep = h // k.shape[1]
    kk, vv = np.repeat(k, rep, axis=1), np.repeat(v, rep, axis=1)
    q = q.astype(np.float64)
    s = np.einsum("hd,thd->ht", q, kk) * scale
    p = np.exp(s - s.max(axis=1, keepdims=True))
    p /= p.sum(axis=1, keepdims=True)
    size = np.einsum("hd,thd->ht", np.abs(q), np.abs(kk)).max(axis=1) * abs(scale)
    return np.einsum("ht,thd->hd", p, vv), np.einsum("ht,thd->hd", p, np.abs(vv)), size


def history(rows: np.ndarray, table: np.ndarray, n: int, bs: int) -> np.ndarray:
    """The first n rows of a sequence through its block table."""
    pos = np.arange(n)
    return rows[table[pos // bs].astype(np.int64) * bs + pos % bs]


def norm_rope(x: np.ndarray, w, cos: np.ndarray, sin: np.ndarray, eps: float) -> np.ndarray:
    """x [N, H, D], cos / sin [N, D] -> fp64 [N, H, D]."""
    x = x.astype(np.float64)
    y = x / np.sqrt(np.mean(x * x, axis=-1, keepdims=True) + eps)
    if w is not None:
        y = y * w.astype(np.float64)
    half = x.shape[-1] // 2
    turned = np.concatenate([-y[..., half:], y[..., :half]], axis=-1)
    return y * cos.astype(np.float64)[:, None] + turned * sin.astype(np.float64)[:, None]
