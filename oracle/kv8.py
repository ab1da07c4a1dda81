"""The 8-bit block KV cache restated in numpy: e4m3 rounding, the quantising write, block tables, attention in 64 bits."""

from __future__ import annotations

import numpy as np

E4M3_MAX = 448.0


def _e4m3_values() -> np.ndarray:
    """The value of every code: sign, 4 exponent bits (bias 7), 3 significand bits; 0x7F and 0xFF are NaN."""
    out = np.empty(256)
    for c in range(256):
        e, m = (c >> 3) & 15, c & 7
        x = (m / 8) * 2.0 ** -6 if e == 0 else (1 + m / 8) * 2.0 ** (e - 7)
        out[c] = -x if c & 0x80 else x
    out[0x7F] = out[0xFF] = np.nan
    return out


E4M3 = _e4m3_values()


def to_e4m3(x: np.ndarray) -> np.ndarray:
    """Codes nearest to ``x`` (ties to the even code), saturated at +-448; NaN is 0x7F."""
    x = np.asarray(x, dtype=np.float64)
    pos = E4M3[:0x7F]
    a = np.minimum(np.abs(np.nan_to_num(x, nan=0.0, posinf=E4M3_MAX, neginf=E4M3_MAX)), E4M3_MAX)
    hi = np.searchsorted(pos, a)  # pos[hi - 1] < a <= pos[hi]
    lo = np.maximum(hi - 1, 0)
    d_hi, d_lo = pos[hi] - a, a - pos[lo]
    code = np.where((d_lo < d_hi) | ((d_lo == d_hi) & (lo % 2 == 0)), lo, hi)
    code = np.where(np.signbit(x), code | 0x80, code)
    return np.where(np.isnan(x), 0x7F, code).astype(np.uint8)


def scale_for(amax: np.ndarray) -> np.ndarray:
    """The smallest power of two s >= 2^-126 with amax <= 448 s."""
    amax = np.asarray(amax, dtype=np.float64)
    m, e = np.frexp(amax)
    k = np.where(amax > 0, np.where(m <= 0.875, e - 9, e - 8), -126)
    return np.ldexp(1.0, np.maximum(k, -126))


def append(codes: np.ndarray, scales: np.ndarray, x: np.ndarray, slots: np.ndarray) -> None:
    """Write rows ``x`` [tokens, kv, dim] into ``codes`` uint8 [blocks, kv, block, dim], in place."""
    block = codes.shape[2]
    t = 0
    while t < len(slots):
        if slots[t] < 0:
            t += 1
            continue
        b, off = divmod(int(slots[t]), block)
        n = 1
        while t + n < len(slots) and off + n < block and slots[t + n] == slots[t] + n:
            n += 1
        run = x[t:t + n].astype(np.float64)
        finite = np.where(np.isfinite(run), np.abs(run), 0.0)
        s = scale_for(finite.max(axis=(0, 2)))
        if off:
            old = scales[b].astype(np.float64)
            s = np.maximum(s, old)
            for h in range(len(s)):
                if s[h] != old[h]:
                    codes[b, h] = to_e4m3(E4M3[codes[b, h]] * (old[h] / s[h]))
        scales[b] = s
        codes[b, :, off:off + n] = to_e4m3(run / s[None, :, None]).transpose(1, 0, 2)
        t += n


def rows(codes: np.ndarray, scales: np.ndarray, slots: np.ndarray) -> np.ndarray:
    """The values of slots, float64 [n, kv, dim]; -1 gives zeros."""
    block = codes.shape[2]
    s = np.maximum(slots, 0)
    out = E4M3[codes[s // block, :, s % block]] * scales[s // block].astype(np.float64)[:, :, None]
    out[slots < 0] = 0.0
    return out


def attend(q: np.ndarray, k: np.ndarray, v: np.ndarray, scaling: float, v_scale: np.ndarray | None = None):
    """One query ``q`` [heads, dim] over ``k``, ``v`` [n, kv, dim]: ``(out, weight, spread, small)``, all float64.

    ``out`` [heads, dim]; ``weight`` [heads, dim] = sum_j w_j |v_j| (what relative errors of the weights are
    measured by); ``spread`` [heads] = max_j scaling * sum_d |q_d k_jd| (what errors of the scores are);
    ``small`` [heads, dim] = max_j (w_j s_j) sum_j |v_j| / s_j with the scales s_j = ``v_scale`` [n, kv] (what
    errors of the weights relative to the row's largest scaled weight are).
    """
    heads, dim = q.shape
    n, kv, _ = k.shape
    out, weight, spread = np.zeros((heads, dim)), np.zeros((heads, dim)), np.zeros(heads)
    small = np.zeros((heads, dim))
    if n == 0:
        return out, weight, spread, small
    for h in range(heads):
        kh, vh = k[:, h // (heads // kv)], v[:, h // (heads // kv)]
        s = kh @ q[h].astype(np.float64) * scaling
        p = np.exp(s - s.max())
        w = p / p.sum()
        out[h] = w @ vh
        weight[h] = w @ np.abs(vh)
        spread[h] = (np.abs(kh) @ np.abs(q[h].astype(np.float64))).max() * scaling
        if v_scale is not None:
            s_h = v_scale[:, h // (heads // kv)].astype(np.float64)
            small[h] = (w * s_h).max() * (np.abs(vh) / s_h[:, None]).sum(0)
    return out, weight, spread, small


class Tables:
    """Block tables with a ring of free blocks, one request at a time."""

    def __init__(self, num_blocks: int, max_reqs: int, max_blocks: int, block: int):
        self.block, self.max_blocks = block, max_blocks
        self.table = np.full((max_reqs, max_blocks), -1, dtype=np.int64)
        self.held = np.zeros(max_reqs, dtype=np.int64)
        self.free = list(range(num_blocks))

    def plan(self, reqs, seq, prefix, num_tokens):
        """``(slots, offsets, failed)``; ``failed``: the entries that got nothing."""
        slots = np.full(num_tokens, -1, dtype=np.int64)
        offsets = np.zeros(len(reqs) + 1, dtype=np.int64)
        failed, seen, wanted = [], set(), 0
        at, free_before, taken = 0, len(self.free), 0
        for i, (r, s, p) in enumerate(zip(reqs, seq, prefix)):
            offsets[i] = at
            if s == 0:
                continue
            n = s - p if p >= 0 and s >= p else 0
            good = p >= 0 and s >= p and 0 <= r < len(self.held) and s <= self.max_blocks * self.block and r not in seen
            if 0 <= r < len(self.held):
                seen.add(r)
            need = max(0, -(-s // self.block) - self.held[r]) if good else 0
            wanted += need
            if good and need and wanted > free_before:
                good = False
            if good:
                for _ in range(need):
                    self.table[r, self.held[r]] = self.free[taken]
                    taken += 1
                    self.held[r] += 1
                for t in range(n):
                    pos = p + t
                    if at + t < num_tokens:
                        slots[at + t] = self.table[r, pos // self.block] * self.block + pos % self.block
            else:
                failed.append(i)
            at += n
        offsets[len(reqs)] = at
        self.free = self.free[taken:]
        return slots, offsets, failed

    def trim(self, reqs, keep):
        for r, k in zip(reqs, keep):
            if r < 0:
                continue
            while self.held[r] > -(-k // self.block):
                pages = range(-(-k // self.block), self.held[r])
                self.free += [int(self.table[r, p]) for p in pages]
                self.table[r, list(pages)] = -1
                self.held[r] = -(-k // self.block)
