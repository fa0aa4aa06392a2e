"""The serving operators in 64 bits, from their definitions: the 8-bit paged cache and its attention,
the bookkeeping of pages, and token log probabilities.  Plain loops over tokens, heads and pages;
numpy only."""
from __future__ import annotations

import math
from typing import List, Optional, Tuple

import numpy as np

LARGEST = 448.0
SCALE_MIN, SCALE_MAX = 2.0 ** -40, 2.0 ** 80


def e4m3_table() -> np.ndarray:
    """The 256 values of e4m3 (no infinities; 0x7f and 0xff are NaN)."""
    out = np.empty(256)
    for b in range(256):
        e, m = b >> 3 & 15, b & 7
        v = math.nan if b & 0x7F == 0x7F else m * 2.0 ** -9 if e == 0 else (8 + m) * 2.0 ** (e - 10)
        out[b] = -v if b & 0x80 else v
    return out


E4M3 = e4m3_table()


def round_e4m3(x: np.ndarray) -> np.ndarray:
    """The nearest e4m3 value, ties to the even one, by search among the values themselves."""
    x = np.asarray(x, np.float64)
    pos = E4M3[:127]
    a = np.minimum(np.abs(np.nan_to_num(x, nan=0.0, posinf=LARGEST, neginf=-LARGEST)), LARGEST)
    hi = np.clip(np.searchsorted(pos, a), 1, 126)
    lo = hi - 1
    up, down = pos[hi] - a, a - pos[lo]
    pick = np.where(up < down, hi, np.where(down < up, lo, np.where(hi % 2 == 0, hi, lo)))
    y = np.copysign(pos[pick], x)
    return np.where(np.isnan(x), np.nan, y)


def scale_for(a: float) -> float:
    """The least power of two s with a <= 448 s, within the cache's limits."""
    if a <= 0:
        return SCALE_MIN
    m, e = math.frexp(a)  # a = m 2^e, 0.5 <= m < 1; 448 = 0.875 x 2^9
    return min(max(2.0 ** (e - 9 + (m > 0.875)), SCALE_MIN), SCALE_MAX)


def key_offset(t: int, x: int, d: int) -> int:
    return t // 16 * 16 * d + x // 64 * 1024 + x % 64 // 16 * 256 + t % 16 * 16 + x % 16


def value_offset(t: int, x: int, d: int) -> int:
    return t // 16 * 16 * d + x // 64 * 1024 + t % 16 // 4 * 256 + x % 16 * 16 + x % 64 // 16 * 4 + t % 4


def offsets(p: int, d: int) -> Tuple[np.ndarray, np.ndarray]:
    return tuple(np.array([[f(t, x, d) for x in range(d)] for t in range(p)]) for f in (key_offset, value_offset))


class Layer:
    """One layer of a cache in plain numbers: e4m3 values [pages, heads, 2, p, d] and scales."""

    def __init__(self, raw: np.ndarray, scales: np.ndarray):
        n, h, _, p, d = raw.shape
        at = offsets(p, d)
        flat = E4M3[raw.reshape(n, h, 2, p * d)]
        self.values = np.stack([flat[:, :, i][:, :, at[i]] for i in (0, 1)], 2)
        self.scales = scales.astype(np.float64).copy()
        self.p, self.d, self.heads = p, d, h

    def tiled(self) -> np.ndarray:
        """The values back in tile order."""
        n, h = self.values.shape[:2]
        out = np.empty((n, h, 2, self.p * self.d))
        for i, at in enumerate(offsets(self.p, self.d)):
            out[:, :, i, at.reshape(-1)] = self.values[:, :, i].reshape(n, h, -1)
        return out.reshape(self.values.shape)


def append(layer: Layer, k: np.ndarray, v: np.ndarray, table: np.ndarray, lengths: np.ndarray, cu: List[int],
           slots: Optional[List[int]] = None, max_new: Optional[int] = None) -> None:
    p, n = layer.p, layer.values.shape[0]
    for b in range(len(cu) - 1):
        slot = b if slots is None else slots[b]
        new = cu[b + 1] - cu[b]
        if not 0 <= slot < len(lengths) or new == 0:
            continue
        start = int(lengths[slot]) - new
        end = min(start + (new if max_new is None else min(new, max_new)), table.shape[1] * p)
        for j in range(max(start, 0) // p, -(-end // p)):
            page = int(table[slot, j])
            if not 0 <= page < n:
                continue
            lo, hi = max(start, j * p), min(end, (j + 1) * p)
            if lo >= hi:
                continue
            for i, x in enumerate((k, v)):
                for h in range(layer.heads):
                    fresh = x[cu[b] + lo - start:cu[b] + hi - start, h].astype(np.float64)
                    finite = np.abs(fresh[np.isfinite(fresh)])
                    s = scale_for(finite.max() if finite.size else 0.0)
                    if lo > j * p:
                        old = layer.scales[page, h, i]
                        s = max(s, old)
                        held = layer.values[page, h, i, : lo - j * p]
                        layer.values[page, h, i, : lo - j * p] = round_e4m3(held * (old / s))
                    layer.scales[page, h, i] = s
                    layer.values[page, h, i, lo - j * p:hi - j * p] = round_e4m3(fresh / s)


def attention(q: np.ndarray, layer: Layer, table: np.ndarray, lengths: np.ndarray, cu: List[int],
              slots: Optional[List[int]] = None, sm_scale: Optional[float] = None):
    """(out, lse, and per output the magnitudes that a bound on its error needs: sum p |v|, the
    largest sum |q k| sm_scale, the largest |v|, the number of tokens)."""
    t, hq, d = q.shape
    group = hq // layer.heads
    scale = d ** -0.5 if sm_scale is None else sm_scale
    out, lse = np.zeros((t, hq, d)), np.full((t, hq), -np.inf)
    mag, dots, vmax, count = np.zeros((t, hq, d)), np.zeros((t, hq)), np.zeros((t, hq)), np.zeros((t, hq))
    p, n = layer.p, layer.values.shape[0]
    for b in range(len(cu) - 1):
        slot = b if slots is None else slots[b]
        if not 0 <= slot < len(lengths):
            continue
        length = min(max(int(lengths[slot]), 0), table.shape[1] * p)
        pages = [int(table[slot, j]) for j in range(-(-length // p))]
        there = np.repeat([0 <= x < n for x in pages], p)[:length] if pages else np.zeros(0, bool)
        ids = [x if 0 <= x < n else 0 for x in pages]
        new = cu[b + 1] - cu[b]
        for h in range(layer.heads):
            k, v = ((layer.values[ids, h, i] * layer.scales[ids, h, i][:, None, None]).reshape(-1, d)[:length]
                    if ids else np.zeros((0, d)) for i in (0, 1))
            for i in range(new):
                seen = there & (np.arange(length) < length - new + i + 1)
                if not seen.any():
                    continue
                for g in range(group):
                    x = q[cu[b] + i, h * group + g].astype(np.float64)
                    at = (cu[b] + i, h * group + g)
                    s = k[seen] @ x * scale
                    w = np.exp(s - s.max())
                    total = w.sum()
                    out[at] = w @ v[seen] / total
                    lse[at] = s.max() + np.log(total)
                    mag[at] = w @ np.abs(v[seen]) / total
                    dots[at] = (np.abs(k[seen]) @ np.abs(x)).max() * abs(scale)
                    vmax[at] = np.abs(v[seen]).max()
                    count[at] = seen.sum()
    return out, lse, mag, dots, vmax, count


class Pool:
    """Page bookkeeping as a scheduler on the host would do it; `data` is any array by page id."""

    def __init__(self, table, lengths, refs, page_size: int, data=None):
        self.table = [list(map(int, r)) for r in table]
        self.lengths, self.refs = list(map(int, lengths)), list(map(int, refs))
        self.p = page_size
        self.data = None if data is None else list(data)

    def _drop(self, ids):
        for x in ids:
            if 0 <= x < len(self.refs):
                self.refs[x] -= 1

    def fork(self, parents, children):
        was, long = [list(r) for r in self.table], list(self.lengths)
        last = {c: i for i, (a, c) in enumerate(zip(parents, children))
                if 0 <= c < len(was) and 0 <= a < len(was)}
        for c, i in last.items():
            self._drop(was[c])
            for x in was[parents[i]]:
                if 0 <= x < len(self.refs):
                    self.refs[x] += 1
            self.table[c], self.lengths[c] = list(was[parents[i]]), long[parents[i]]

    def free(self, slots):
        for s in slots:
            if 0 <= s < len(self.table):
                self._drop(self.table[s])
                self.table[s], self.lengths[s] = [-1] * len(self.table[s]), 0

    def extend(self, new, slots=None):
        free = [i for i, r in enumerate(self.refs) if r == 0]
        had, asked, readers, served = len(free), 0, list(self.refs), []
        for b, add in enumerate(new):
            s = b if slots is None else slots[b]
            if not 0 <= s < len(self.table):
                served.append(0)
                continue
            length = self.lengths[s]
            have, want = -(-length // self.p), -(-(length + add) // self.p)
            if want > len(self.table[s]):
                served.append(0)
                continue
            inside = add > 0 and length % self.p != 0
            tail = self.table[s][have - 1] if inside else -1
            shared = inside and 0 <= tail < len(self.refs) and readers[tail] > 1
            split = inside and 0 <= tail < len(self.refs) and self.refs[tail] > 1
            need = want - have + split
            asked += need
            if asked > had and (need > 0 or shared):
                served.append(0)
                continue
            served.append(1)
            if split:
                x = free.pop(0)
                self.refs[tail] -= 1
                self.refs[x], self.table[s][have - 1] = 1, x
                if self.data is not None:
                    self.data[x] = self.data[tail]
            for j in range(have, want):
                self.table[s][j] = free.pop(0)
                self.refs[self.table[s][j]] = 1
            self.lengths[s] += add
        return served

    def compact(self):
        live = sum(r > 0 for r in self.refs)
        gaps = [i for i in range(live) if self.refs[i] <= 0]
        to = {}
        for x in range(live, len(self.refs)):
            if self.refs[x] > 0:
                y = to[x] = gaps.pop(0)
                self.refs[y], self.refs[x] = self.refs[x], 0
                if self.data is not None:
                    self.data[y] = self.data[x]
        self.table = [[to.get(x, x) for x in r] for r in self.table]
        return [live, len(to)]


def token_logprobs(x: np.ndarray, tokens: np.ndarray, k: int):
    """(logprob, entropy, top ids, top logprobs) of rows of logits."""
    x = np.asarray(x, np.float64)
    rows, vocab = x.shape
    lp, ent = np.full(rows, np.nan), np.zeros(rows)
    ids, top = np.zeros((rows, k), np.int64), np.zeros((rows, k))
    for r in range(rows):
        order = sorted(range(vocab), key=lambda i: (not math.isnan(x[r, i]), -x[r, i] if not math.isnan(x[r, i]) else 0.0, i))
        ids[r] = order[:k]
        if np.isnan(x[r]).any() or np.isposinf(x[r]).any():
            ent[r], top[r] = np.nan, np.nan
            continue
        if np.isneginf(x[r]).all():
            top[r] = -np.inf
            if 0 <= tokens[r] < vocab:
                lp[r] = -np.inf
            continue
        # relative to the largest: a logit near the end of its type's range would swallow the sum
        d = x[r] - x[r].max()
        total = np.log(np.exp(d).sum())
        p = np.exp(d - total)
        if 0 <= tokens[r] < vocab:
            lp[r] = d[tokens[r]] - total
        ent[r] = -(p[p > 0] * (d[p > 0] - total)).sum()
        top[r] = d[ids[r]] - total
    return lp, ent, ids, top
