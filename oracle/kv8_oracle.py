"""64-bit restatement of the 8-bit slot cache (whisperdrz_amd.FlashKVCache8) and of the attention over it.

Blocks of 32 positions: scale 2^e, e the least whole number of [-100, 100] with max |x| <= 448 2^e over
the finite values; codes are e4m3 values, x 2^-e clamped to +-448 and rounded to nearest even; what is
not finite is NaN. Ring: position p in row p % 64. Written from the definition, apart from the kernels:
a cache here holds values, not bytes.
"""
from __future__ import annotations

import numpy as np

BLOCK, RING, D = 32, 64, 64


def e4m3(x: np.ndarray) -> np.ndarray:
    """Nearest e4m3 value (ties to even) of finite float64 values of at most 448 (464 would be the border)."""
    x = np.asarray(x, dtype=np.float64)
    _, e = np.frexp(x)  # x = m 2^e, m in [0.5, 1): four significant bits, the last worth 2^(e - 4)
    step = np.ldexp(1.0, np.maximum(e - 4, -9))
    return np.rint(x / step) * step


def quantize_block(x: np.ndarray) -> tuple[np.ndarray, float]:
    """(code values, scale) of one block's values ``[n, 64]``."""
    x = np.asarray(x, dtype=np.float64)
    fine = np.isfinite(x)
    top = float(np.max(np.abs(np.where(fine, x, 0.0)), initial=0.0))
    e = -100
    while e < 100 and np.ldexp(448.0, e) < top:
        e += 1
    c = e4m3(np.clip(np.where(fine, x, 0.0) * np.ldexp(1.0, -e), -448.0, 448.0))
    return np.where(fine, c, np.nan), float(np.ldexp(1.0, e))


class Cache:
    """The state of one cache in values: codes ``[S, H, blocks * 32, 64]``, scales, and rings or None."""

    def __init__(self, k_codes, v_codes, k_scales, v_scales, k_ring=None, v_ring=None, max_seq=None):
        self.codes = [np.array(k_codes, np.float64), np.array(v_codes, np.float64)]
        self.scales = [np.array(k_scales, np.float64), np.array(v_scales, np.float64)]
        self.ring = None if k_ring is None else [np.array(k_ring, np.float64), np.array(v_ring, np.float64)]
        self.max_seq = max_seq if max_seq is not None else self.codes[0].shape[2]

    def read(self, n: int, slot: int, length: int) -> np.ndarray:
        """``[H, length, 64]`` keys (n 0) or values (n 1) of the first ``length`` positions."""
        x = self.codes[n][slot] * np.repeat(self.scales[n][slot], BLOCK, axis=-1)[..., None]
        x = x[:, :length].copy()
        if self.ring is not None:
            for p in range(length // BLOCK * BLOCK, length):
                x[:, p] = self.ring[n][slot][:, p % RING]
        return x

    def append(self, slot: int, start: int, k: np.ndarray, v: np.ndarray) -> None:
        """Rows ``[T, H, 64]`` at positions ``start`` .. of a slot."""
        T, end = k.shape[0], start + k.shape[0]
        for n, new in enumerate((k, v)):
            seq = {p: self.ring[n][slot][:, p % RING].copy() for p in range(start // BLOCK * BLOCK, start)}
            seq.update({start + t: np.asarray(new[t], np.float64) for t in range(T)})
            for j in range(start // BLOCK, end // BLOCK):
                for h in range(new.shape[1]):
                    rows = np.stack([seq[p][h] for p in range(j * BLOCK, (j + 1) * BLOCK)])
                    self.codes[n][slot, h, j * BLOCK:(j + 1) * BLOCK], self.scales[n][slot, h, j] = quantize_block(rows)
            for p in range(max(start, (end // BLOCK - 1) * BLOCK), end):
                self.ring[n][slot][:, p % RING] = seq[p]

    def fill(self, slot: int, k: np.ndarray, v: np.ndarray) -> None:
        """Rows ``[T, H, 64]`` from position 0 on of a cache without a ring, the last block closed with zeros."""
        for n, new in enumerate((k, v)):
            for j in range(-(-new.shape[0] // BLOCK)):
                for h in range(new.shape[1]):
                    rows = np.zeros((BLOCK, D))
                    part = new[j * BLOCK:(j + 1) * BLOCK, h]
                    rows[:len(part)] = part
                    self.codes[n][slot, h, j * BLOCK:(j + 1) * BLOCK], self.scales[n][slot, h, j] = quantize_block(rows)


def attend(q: np.ndarray, k: np.ndarray, v: np.ndarray, limits, scale: float):
    """One row: ``q`` ``[T, H, 64]``, ``k`` / ``v`` ``[H, L, 64]``, query t sees the first ``limits[t]``
    positions. Returns the output ``[T, H, 64]`` and, for error bounds, sum_j p_j |v_j| and the largest
    scale * sum_d |q_d k_jd| of each (query, head)."""
    T, H, _ = q.shape
    out, mag, big = np.zeros((T, H, D)), np.zeros((T, H, D)), np.zeros((T, H, 1))
    with np.errstate(invalid="ignore", over="ignore"):
        for t in range(T):
            n = int(limits[t])
            if n == 0:
                continue
            for h in range(H):
                s = (k[h, :n] @ q[t, h]) * scale
                p = np.exp(s - s.max())
                p /= p.sum()
                out[t, h] = p @ v[h, :n]
                mag[t, h] = p @ np.abs(v[h, :n])
                big[t, h] = (np.abs(k[h, :n]) @ np.abs(q[t, h])).max() * scale
    return out, mag, big


def bound(out, mag, big, n_keys: int, half_step: float, one_part: bool = False) -> np.ndarray:
    """How far a kernel may be from ``attend``: the result's own rounding (half a step of its type), and in
    units of sum p |v|: twice the error of a score (64 products and a few factors in fp32; it counts in
    the probability and in the sum), the probability's two 16-bit parts (2^-16) with its exp2 (2^-22),
    and the fp32 sums over the keys. ``one_part``, for a form that holds less than the kernels do: the
    probabilities are one fp16 value each, p (1 + e) with
    |e| <= 2^-11, above and below the line alike: sum p e v - out sum p e over sum p, at most
    2^-11 (sum p |v| + |out|) <= 2^-10 sum p |v|; those under fp16's normal range, 2^-14 against a largest
    of at least 1, are off by 2^-25 instead, n_keys 2^-25 in all twice."""
    rel = 2 * 72 * 2.0 ** -24 * big + 2.0 ** -16 + 2.0 ** -20 + (n_keys + 64) * 2.0 ** -24
    if one_part:
        rel = rel + 2.0 ** -10 + n_keys * 2.0 ** -24
    return half_step * np.abs(out) + rel * mag + 2.0 ** -25
