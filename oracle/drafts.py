"""The operators of a step that drafts tokens in 64 bits, from their definitions: rotation on the way into the cache,
attention of a tree, verification of drafts, and what stays in the cache.  Plain loops; numpy only."""
from __future__ import annotations

from typing import List, Optional, Sequence

import numpy as np

from . import serving as orc


def tree_parent(parents: Sequence[int], i: int) -> int:
    """The parent of node i, or -1: only an earlier node is one."""
    return int(parents[i]) if 0 <= parents[i] < i else -1


def lineage(parents: Sequence[int], i: int) -> List[int]:
    """Node i and its ancestors."""
    out = []
    while i >= 0:
        out.append(i)
        i = tree_parent(parents, i)
    return out


def turn(x: np.ndarray, norm: Optional[np.ndarray], eps: float, cos: np.ndarray, sin: np.ndarray, pos: int, interleaved: bool):
    """(one token's heads [heads, d] normed and turned, for each channel the magnitudes that its rounding errors are
    relative to)."""
    x = np.asarray(x, np.float64).copy()
    if norm is not None:
        x = x / np.sqrt((x * x).mean(1, keepdims=True) + eps) * np.asarray(norm, np.float64)
    half = cos.shape[1]
    there = 0 <= pos < cos.shape[0]
    c = cos[pos].astype(np.float64) if there else np.full(half, np.nan)
    s = sin[pos].astype(np.float64) if there else np.full(half, np.nan)
    a, b = (slice(0, 2 * half, 2), slice(1, 2 * half, 2)) if interleaved else (slice(0, half), slice(half, 2 * half))
    y, mag = x.copy(), np.abs(x)
    y[:, a], y[:, b] = x[:, a] * c - x[:, b] * s, x[:, b] * c + x[:, a] * s
    mag[:, a], mag[:, b] = np.abs(x[:, a] * c) + np.abs(x[:, b] * s), np.abs(x[:, b] * c) + np.abs(x[:, a] * s)
    return y, mag


def turned(x, norm, eps, cos, sin, interleaved, lengths, cu, slots=None, positions=None, parents=None):
    """x [tokens, heads, d] of a batch, turned, and the magnitudes; tokens of no sequence stay NaN."""
    out, mags = np.full(x.shape, np.nan), np.full(x.shape, np.nan)
    for b in range(len(cu) - 1):
        slot, n = b if slots is None else slots[b], cu[b + 1] - cu[b]
        if not 0 <= slot < len(lengths):
            continue
        for i in range(n):
            pos = int(lengths[slot]) - n + i
            if positions is not None:
                pos = int(positions[cu[b] + i])
            elif parents is not None:
                pos = int(lengths[slot]) - n + len(lineage(parents[cu[b]:cu[b + 1]], i)) - 1
            out[cu[b] + i], mags[cu[b] + i] = turn(x[cu[b] + i], norm, eps, cos, sin, pos, interleaved)
    return out, mags


def tree_attention(q, parents, layer, table, lengths, cu, slots=None, sm_scale=None):
    """As oracle.serving.attention, of trees."""
    t, hq, d = q.shape
    group = hq // layer.heads
    scale = d ** -0.5 if sm_scale is None else sm_scale
    out, lse = np.zeros((t, hq, d)), np.full((t, hq), -np.inf)
    mag, dots, vmax, count = np.zeros((t, hq, d)), np.zeros((t, hq)), np.zeros((t, hq)), np.zeros((t, hq))
    p, pages = layer.p, layer.values.shape[0]
    for b in range(len(cu) - 1):
        slot = b if slots is None else slots[b]
        if not 0 <= slot < len(lengths):
            continue
        length = min(max(int(lengths[slot]), 0), table.shape[1] * p)
        ids = [int(table[slot, j]) for j in range(-(-length // p))]
        there = np.repeat([0 <= x < pages for x in ids], p)[:length] if ids else np.zeros(0, bool)
        ids = [x if 0 <= x < pages else 0 for x in ids]
        new = cu[b + 1] - cu[b]
        for h in range(layer.heads):
            k, v = ((layer.values[ids, h, i] * layer.scales[ids, h, i][:, None, None]).reshape(-1, d)[:length]
                    if ids else np.zeros((0, d)) for i in (0, 1))
            for i in range(new):
                seen = np.arange(length) < length - new
                for j in lineage(parents[cu[b]:cu[b + 1]], i):
                    if length - new + j >= 0:
                        seen[length - new + j] = True
                seen &= there
                if not seen.any():
                    continue
                for g in range(group):
                    at = (cu[b] + i, h * group + g)
                    x = q[at].astype(np.float64)
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


def _softmax(x: np.ndarray, temperature: float) -> Optional[np.ndarray]:
    x = np.asarray(x, np.float64)
    if np.isnan(x).any() or np.isposinf(x).any() or not np.isfinite(x).any():
        return None
    e = np.exp((x - x[np.isfinite(x)].max()) / temperature)
    return e / e.sum()


def _first_past(p: np.ndarray, u: float) -> int:
    sums = np.cumsum(p)
    return int(np.argmax(sums > u * sums[-1]))


def verify(logits, tokens, uniforms, parents=None, draft_logits=None, temperature=1.0, cu=None, max_new=None):
    """(accepted, path, tokens) of every sequence, as lists."""
    result = []
    for b in range(len(cu) - 1):
        first, n = cu[b], cu[b + 1] - cu[b]
        if max_new is not None:
            n = min(n, max_new)
        if n == 0:
            result.append((0, [], []))
            continue
        temp = float(temperature[b]) if np.ndim(temperature) else float(temperature)
        above = [i - 1 if parents is None else tree_parent(parents[first:first + n], i) for i in range(n)]
        path = [0]
        while True:
            at = path[-1]
            row = np.asarray(logits[first + at], np.float64)
            if not temp > 0:
                bad = np.isnan(row).any() or np.isposinf(row).any() or not np.isfinite(row).any()
                p = None if bad else np.eye(1, len(row), int(np.argmax(row)))[0]
            else:
                p = _softmax(row, temp)
            whole, refused, taken = p, set(), None
            for j in range(at + 1, n):
                if above[j] != at or p is None:
                    continue
                x, u = int(tokens[first + j]), float(uniforms[first + j])
                known = 0 <= x < len(row)
                if not temp > 0:
                    ok = known and p[x] == 1.0
                elif draft_logits is not None:
                    q = _softmax(draft_logits[first + at], temp)
                    ok = known and q is not None and u * q[x] < p[x]
                    if not ok:
                        left = np.zeros_like(p) if q is None else np.maximum(p - q, 0)
                        p = left if left.sum() > 0 else p
                        break
                else:
                    ok = known and x not in refused and u * (1 - sum(whole[y] for y in refused)) < whole[x]
                    if known:
                        refused.add(x)
                if ok:
                    taken = j
                    break
            if taken is None:
                break
            path.append(taken)
        if p is not None and temp > 0 and draft_logits is None:
            left = p.copy()
            left[list(refused)] = 0.0
            p = left if left.sum() > 0 else p
        new = -1 if p is None else _first_past(p, float(uniforms[first]))
        result.append((len(path), path, [int(tokens[first + j]) for j in path[1:]] + [new]))
    return result


def keep(layers: List[orc.Layer], pool: orc.Pool, path, accepted, news, slots=None) -> None:
    """pool.table, lengths and refs, and every layer's pages, after the accepted nodes have moved."""
    p = pool.p
    for b in range(len(accepted)):
        slot, n = b if slots is None else slots[b], news[b]
        if not 0 <= slot < len(pool.lengths) or n < 0 or pool.lengths[slot] < n or pool.lengths[slot] > len(pool.table[slot]) * p:
            continue
        start, kept = pool.lengths[slot] - n, []
        for x in list(path[b])[:max(0, accepted[b])]:
            if not 0 <= x < n or (kept and x <= kept[-1]):
                break
            kept.append(int(x))
        row = pool.table[slot]
        for layer in layers:
            count = layer.values.shape[0]
            moves = []
            for i, j in enumerate(kept):
                src, dst = row[(start + j) // p], row[(start + i) // p]
                if i != j and 0 <= src < count and 0 <= dst < count:
                    x = layer.values[src, :, :, (start + j) % p] * layer.scales[src][..., None]  # [heads, 2, d]
                    moves.append((dst, (start + i) % p, x))
            for page in sorted({m[0] for m in moves}):
                mine = [m for m in moves if m[0] == page]
                for h in range(layer.heads):
                    for kv in (0, 1):
                        all_x = np.concatenate([x[h, kv] for _, _, x in mine])
                        finite = np.abs(all_x[np.isfinite(all_x)])
                        old = layer.scales[page, h, kv]
                        s = max(old, orc.scale_for(finite.max() if finite.size else 0.0))
                        if s != old:
                            layer.values[page, h, kv] = orc.round_e4m3(layer.values[page, h, kv] * (old / s))
                            layer.scales[page, h, kv] = s
                        for _, t, x in mine:
                            layer.values[page, h, kv, t] = orc.round_e4m3(x[h, kv] / s)
        pool.lengths[slot] = start + len(kept)
        for j in range(-(-pool.lengths[slot] // p), -(-(start + n) // p)):
            if 0 <= row[j] < len(pool.refs):
                pool.refs[row[j]] -= 1
            row[j] = -1
