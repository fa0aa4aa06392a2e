"""Parity of the serving operators with oracle/serving.py (64 bits, from the definitions) on the GPU:
sizes and masks at which they can go wrong, refused calls, streams and graphs.

Tolerances, from the arithmetic:
- kv_append rounds by exact steps, so its bytes and scales are the oracle's.
- kv_attention: the output's own rounding u = 2^-11 (fp16) or 2^-8 (bf16) of |o|; each weight's
  rounding to fp16, 2^-11 relative or 2^-38 of the largest, times |v|; and the error of a score in 32
  bits, at most (D + 8) 2^-24 of sum |q k| sm_scale, which moves its weight by as much, in the
  sum above and in the one below.
- token_logprobs: 32-bit sums of weights whose exponents carry 2^-23 of up to 30 octaves, in
  chains of at most 128 terms: 2^-17 of 1 + |value|.
"""
from __future__ import annotations

import threading

import numpy as np
import pytest
import torch

import bsa_mi355x as bsa
from oracle import serving as orc

pytestmark = pytest.mark.gpu
F8 = torch.float8_e4m3fn
DT = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}


def _i32(v, dev):
    return torch.tensor(np.asarray(v), dtype=torch.int32, device=dev)


def _raw(pages):
    return pages.view(torch.uint8).cpu().numpy()


def _cache(rng, dev, lengths, heads, p, d, spare=3, each=None, poison=False):
    """Pages with random content for the given lengths: raw bytes, scales, table.  poison: every byte
    that no sequence's token owns is NaN."""
    per = [-(-n // p) for n in lengths]
    each = each or max(per + [1]) + 1
    count = sum(per) + spare
    raw = orc_bytes(rng, (count, heads, 2, p, d))
    scales = 2.0 ** rng.integers(-8, -3, (count, heads, 2)).astype(np.float32)
    ids = rng.permutation(count)
    table = np.full((len(lengths), each), -1, np.int64)
    at = 0
    for b, n in enumerate(per):
        table[b, :n] = ids[at:at + n]
        at += n
    if poison:
        owned = np.zeros((count, p), bool)
        for b, n in enumerate(lengths):
            for t in range(n):
                owned[table[b, t // p], t % p] = True
        for i, where in enumerate(orc.offsets(p, d)):
            flat = raw[:, :, i].reshape(count, heads, p * d)
            for page in range(count):
                flat[page][:, where[~owned[page]].reshape(-1)] = 0x7F
            raw[:, :, i] = flat.reshape(count, heads, p, d)
    pages = torch.from_numpy(raw).to(dev).view(F8)
    return raw, scales, table, pages, torch.from_numpy(scales).to(dev), _i32(table, dev)


def orc_bytes(rng, shape):
    """e4m3 bytes of normal numbers of spread 64."""
    x = torch.from_numpy(rng.standard_normal(shape).astype(np.float32) * 64).clamp(-448, 448)
    return x.to(F8).view(torch.uint8).numpy().copy()


def _same_pages(pages, scales, layer):
    got = orc.E4M3[_raw(pages)]
    np.testing.assert_array_equal(got, layer.tiled())
    np.testing.assert_array_equal(scales.cpu().numpy().astype(np.float64), layer.scales)


# ---------------------------------------------------------------------------------------- append


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("p,d", [(16, 64), (16, 128), (32, 128), (64, 64), (64, 128), (128, 128)])
@pytest.mark.parametrize("new", [[1, 1, 1], [3, 0, 1], [40, 129, 17], [16, 64, 128]])
def test_append(dev, dtype, p, d, new):
    rng = np.random.default_rng([p, d, *new, len(dtype)])
    heads = 3
    lengths = [n + o for n, o in zip(new, [5, 16, 131])]
    raw, sc, table, pages, scales, tab = _cache(rng, dev, lengths, heads, p, d)
    cu = np.concatenate([[0], np.cumsum(new)])
    k, v = (torch.from_numpy((rng.standard_normal((cu[-1], heads, d)) * np.exp(2 * rng.standard_normal((cu[-1], heads, 1))))
                             .astype(np.float32)).to(DT[dtype]).to(dev) for _ in range(2))
    layer = orc.Layer(raw, sc)
    orc.append(layer, k.float().cpu().numpy(), v.float().cpu().numpy(), table, np.array(lengths), list(cu))
    bsa.kv_append(k, v, pages, scales, tab, _i32(lengths, dev), cu_seqlens=_i32(cu, dev), max_new=max(new))
    _same_pages(pages, scales, layer)


def test_append_twice_is_the_same(dev):
    """The call writes where the lengths say, so a repeated one changes nothing."""
    rng = np.random.default_rng(5)
    _, _, _, pages, scales, tab = _cache(rng, dev, [21, 40], 2, 16, 64)
    k = torch.randn(4, 2, 64, device=dev, dtype=torch.float16) * 30
    args = (k, -k, pages, scales, tab, _i32([21, 40], dev))
    bsa.kv_append(*args)
    was = pages.view(torch.uint8).clone(), scales.clone()
    bsa.kv_append(*args)
    assert torch.equal(pages.view(torch.uint8), was[0]) and torch.equal(scales, was[1])


@pytest.mark.parametrize("case", ["nan_inf", "zeros", "tiny", "huge", "strided", "odd_stride", "slots", "bad_pages",
                                  "short_length", "table_full"])
def test_append_edges(dev, case):
    rng = np.random.default_rng(11)
    heads, p, d, dt = 2, 32, 64, torch.bfloat16
    lengths, new, slots, each = [35, 64, 9], [4, 40, 9], None, None
    if case == "short_length":
        new = [4, 70, 12]  # more tokens than the lengths hold: the first ones have no place
    if case == "table_full":
        each, new = 2, [4, 40, 9]
    raw, sc, table, pages, scales, tab = _cache(rng, dev, lengths, heads, p, d, each=each)
    if case == "table_full":
        lengths = [35, 80, 9]  # past the table's two pages
    cu = np.concatenate([[0], np.cumsum(new)])
    x = rng.standard_normal((2, cu[-1], heads, d)).astype(np.float32)
    if case == "nan_inf":
        x[0, 1, 0, 3], x[0, 2, 1, 5], x[1, 6, 0, 0], x[1, cu[-1] - 1, 1, 63] = np.nan, np.inf, -np.inf, np.nan
    elif case == "zeros":
        x[:, cu[1]:] = 0
    elif case == "tiny":
        x *= 1e-30
    elif case == "huge":
        x *= 1e37
    k, v = torch.from_numpy(x).to(dt).to(dev)
    kd, vd = k, v
    if case == "strided":  # as views of one projection's output
        fused = torch.randn(cu[-1], 4 * heads, d, device=dev).to(dt)
        fused[:, heads:2 * heads], fused[:, 2 * heads:3 * heads] = k, v
        kd, vd = fused[:, heads:2 * heads], fused[:, 2 * heads:3 * heads]
    elif case == "odd_stride":
        wide = torch.empty(cu[-1], heads, d + 1, device=dev, dtype=dt)
        wide[:, :, 1:] = k
        kd = wide[:, :, 1:]
    elif case == "slots":
        slots = [2, 7, 0]
        lengths = [lengths[2] + 3, lengths[1], lengths[0]]
        lengths[2] = 9
        lengths[0] = 35
    elif case == "bad_pages":
        table[0, 1], table[1, 1] = -1, 10 ** 6
        tab = _i32(table, dev)
    layer = orc.Layer(raw, sc)
    orc.append(layer, k.float().cpu().numpy(), v.float().cpu().numpy(), table, np.array(lengths), list(cu), slots)
    bsa.kv_append(kd, vd, pages, scales, tab, _i32(lengths, dev), cu_seqlens=_i32(cu, dev), max_new=max(new),
                  slots=None if slots is None else _i32(slots, dev))
    _same_pages(pages, scales, layer)


@pytest.mark.parametrize("p", [16, 128])
@pytest.mark.parametrize("max_new", [1, 3, 17, 40])
def test_append_writes_max_new_tokens(dev, p, max_new):
    """Tokens past max_new are not written, wherever a page ends, and do not weigh in a scale."""
    rng = np.random.default_rng([p, max_new])
    new, lengths = [5, 1, 0, 40, 12], [21, 1, 7, 150, 9]  # the last one's first three have no place
    raw, sc, table, pages, scales, tab = _cache(rng, dev, lengths, 2, p, 64)
    cu = np.concatenate([[0], np.cumsum(new)])
    k, v = (torch.from_numpy(rng.standard_normal((cu[-1], 2, 64)) * 2.0 ** np.arange(cu[-1])[:, None, None] ** 0.5).half().to(dev)
            for _ in range(2))
    layer = orc.Layer(raw, sc)
    orc.append(layer, k.float().cpu().numpy(), v.float().cpu().numpy(), table, np.array(lengths), list(cu), max_new=max_new)
    bsa.kv_append(k, v, pages, scales, tab, _i32(lengths, dev), cu_seqlens=_i32(cu, dev), max_new=max_new)
    _same_pages(pages, scales, layer)


def test_append_of_many_sequences_without_a_bound(dev):
    """300 sequences of 1 to 2000 new tokens with no max_new: a grid past what one launch takes."""
    rng = np.random.default_rng(19)
    heads, p, d, n = 24, 16, 64, 300
    new = rng.integers(1, 600, n)
    new[::60] = 2000
    lengths = new + rng.integers(0, 40, n)
    per = -(-lengths // p)
    table = np.full((n, per.max()), -1)
    ids = rng.permutation(int(per.sum()))
    for b, at in enumerate(np.cumsum(per) - per):
        table[b, : per[b]] = ids[at: at + per[b]]
    cu = np.concatenate([[0], np.cumsum(new)])
    g = torch.Generator(device=dev).manual_seed(1)
    k, v = (torch.randn(int(cu[-1]), heads, d, generator=g, device=dev, dtype=torch.float16) for _ in range(2))
    got = []
    for most in (2000, None):
        pages = torch.zeros(len(ids), heads, 2, p, d, dtype=torch.uint8, device=dev).view(F8)
        scales = torch.ones(len(ids), heads, 2, device=dev)
        bsa.kv_append(k, v, pages, scales, _i32(table, dev), _i32(lengths, dev), cu_seqlens=_i32(cu, dev), max_new=most)
        got.append((pages.view(torch.uint8), scales))
    assert torch.equal(got[0][0], got[1][0]) and torch.equal(got[0][1], got[1][1])
    some = [0, 1, 137, n - 1]  # the first call against the oracle
    part = np.concatenate([table[b, : per[b]] for b in some])
    raw = np.zeros((len(part), heads, 2, p, d), np.uint8)
    layer = orc.Layer(raw, np.ones((len(part), heads, 2), np.float32))
    own = np.full((len(some), per.max()), -1)
    own_cu = np.concatenate([[0], np.cumsum(new[some])])
    at = 0
    for i, b in enumerate(some):
        own[i, : per[b]] = np.arange(at, at + per[b])
        at += per[b]
    rows = np.concatenate([np.arange(cu[b], cu[b + 1]) for b in some])
    orc.append(layer, k[rows].float().cpu().numpy(), v[rows].float().cpu().numpy(), own, lengths[some], list(own_cu))
    index = torch.from_numpy(part).to(dev)
    _same_pages(got[0][0][index].view(F8), got[0][1][index], layer)


# ---------------------------------------------------------------------------------------- attention


def _check_attention(out, lse, ref, dtype, d, where=None):
    o, l, mag, dots, vmax, count = ref
    got, got_l = out.double().cpu().numpy(), lse.double().cpu().numpy()
    eps = (d + 8) * 2.0 ** -24 * dots + 2.0 ** -20
    u = 2.0 ** -11 if dtype == torch.float16 else 2.0 ** -8
    bound = u * np.abs(o) + (2.0 ** -11 + 2 * eps[..., None]) * mag + (count * vmax * 2.0 ** -38)[..., None] + 2.0 ** -24
    np.testing.assert_array_equal(np.isfinite(got), np.isfinite(o))
    fine = np.isfinite(o)
    worst = (np.abs(got - o) / bound)[fine]
    assert worst.size == 0 or worst.max() <= 1, f"error {worst.max():.3g} times its bound"
    empty = np.isneginf(l)
    np.testing.assert_array_equal(np.isneginf(got_l), empty)
    ok = np.isfinite(l)
    assert (np.abs(got_l[ok] - l[ok]) <= 2 * eps[ok] + 2.0 ** -20 * (1 + np.abs(l[ok]))).all()


def _attend(dev, rng, lengths, new, hq, heads, p, d, dtype, poison=True, **kw):
    raw, sc, table, pages, scales, tab = _cache(rng, dev, lengths, heads, p, d, poison=poison)
    cu = np.concatenate([[0], np.cumsum(new)])
    q = torch.from_numpy(rng.standard_normal((cu[-1], hq, d)).astype(np.float32)).to(dtype).to(dev)
    ref = orc.attention(q.double().cpu().numpy(), orc.Layer(raw, sc), table, np.array(lengths), list(cu))
    out, lse = bsa.kv_attention(q, pages, scales, tab, _i32(lengths, dev), cu_seqlens=_i32(cu, dev), max_new=max(new), **kw)
    _check_attention(out, lse, ref, dtype, d)


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("p,d", [(16, 64), (16, 128), (32, 64), (64, 128), (128, 128)])
@pytest.mark.parametrize("hq,heads", [(4, 4), (8, 2), (7, 1), (20, 1)])
def test_attention_decode(dev, dtype, p, d, hq, heads):
    rng = np.random.default_rng(p + d + hq)
    _attend(dev, rng, [1, 2, 15, 16, 17, 31, 32, 33, 127, 128, 129, 500], [1] * 12, hq, heads, p, d, DT[dtype])


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("new", [2, 5, 9, 33])
@pytest.mark.parametrize("hq,heads,p,d", [(2, 2, 16, 128), (6, 2, 32, 64), (8, 1, 64, 128)])
def test_attention_draft(dev, dtype, new, hq, heads, p, d):
    """Several new tokens, each seeing one token more than the one before."""
    rng = np.random.default_rng(new + hq)
    _attend(dev, rng, [new, new + 1, 64 + new, 200], [new] * 4, hq, heads, p, d, DT[dtype])


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("hq,heads,p,d", [(2, 1, 16, 64), (2, 2, 64, 128), (5, 1, 128, 64)])
@pytest.mark.parametrize("lengths,new", [([150, 257, 64], [150, 130, 1]), ([200, 70], [65, 70]), ([301], [300])])
def test_attention_prompt(dev, dtype, hq, heads, p, d, lengths, new):
    rng = np.random.default_rng(hq + p + len(new))
    _attend(dev, rng, lengths, new, hq, heads, p, d, DT[dtype])


@pytest.mark.parametrize("lengths,max_len", [([5000], None), ([5000, 3, 2049], 5000), ([5000, 1200], 700), ([4099], 1)])
def test_attention_split(dev, lengths, max_len):
    """Few sequences: the long axis is split, whatever max_len says of it."""
    rng = np.random.default_rng(3)
    _attend(dev, rng, lengths, [1] * len(lengths), 4, 2, 16, 128, torch.float16, max_len=max_len)
    _attend(dev, rng, lengths, [3] * len(lengths), 4, 2, 64, 64, torch.bfloat16, max_len=max_len)


# ---- prompts (more than 32 rows of a cached head) over more tokens than one turn of the kernel's page numbers
# (1024), in one part and in several, which take other paths at their ends


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("hq,heads,p,d", [(2, 2, 16, 64), (4, 2, 64, 128), (3, 1, 128, 64), (1, 1, 16, 128)])
@pytest.mark.parametrize("lengths,new,max_len", [([1100], [40], None), ([2049, 70, 1025], [130, 65, 33], None),
                                                 ([5000], [200], 700), ([5000, 1300], [35, 60], 1100), ([4099], [300], None)])
def test_prompt_over_long_caches(dev, dtype, hq, heads, p, d, lengths, new, max_len):
    rng = np.random.default_rng([hq, p, d, len(new), lengths[0]])
    _attend(dev, rng, lengths, new, hq, heads, p, d, DT[dtype], max_len=max_len)


@pytest.mark.parametrize("max_len", [None, 500])
@pytest.mark.parametrize("p", [16, 64, 128])
def test_prompt_pages_out_of_range(dev, p, max_len):
    """Pages that do not exist before and after token 1024, and a whole turn of them."""
    rng = np.random.default_rng(p)
    lengths, new = [3300, 2500], [70, 40]
    raw, sc, table, pages, scales, tab = _cache(rng, dev, lengths, 2, p, 64, poison=True)
    table[0, 300 // p], table[0, 1040 // p], table[0, 2064 // p], table[0, 3299 // p] = -1, 10 ** 7, -3, 2 ** 31 - 1
    table[1, 1024 // p: 2176 // p] = -1
    cu = np.concatenate([[0], np.cumsum(new)])
    q = torch.from_numpy(rng.standard_normal((cu[-1], 4, 64)).astype(np.float32)).half().to(dev)
    ref = orc.attention(q.double().cpu().numpy(), orc.Layer(raw, sc), table, np.array(lengths), list(cu))
    out, lse = bsa.kv_attention(q, pages, scales, _i32(table, dev), _i32(lengths, dev), cu_seqlens=_i32(cu, dev), max_new=70,
                                max_len=max_len)
    _check_attention(out, lse, ref, torch.float16, 64)


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("max_len", [None, 500])
@pytest.mark.parametrize("new", [3, 50])
@pytest.mark.parametrize("kind", ["keys_grow", "keys_shrink", "sink", "value_scales", "values_grow", "values_shrink"])
def test_attention_maximum_moves(dev, kind, new, max_len, dtype):
    """Scores and value scales that outgrow, late and by many octaves, what was the maximum at first, or
    never come near it again."""
    rng = np.random.default_rng(len(kind) + new)
    p, d, length, dt = 16, 64, 2200, DT[dtype]
    raw, sc, table, pages, scales, tab = _cache(rng, dev, [length, 700], 2, p, d)
    for row, n in ((0, length), (1, 700)):
        ids, at = table[row, : -(-n // p)], np.arange(-(-n // p))[:, None]
        if kind == "keys_grow":
            sc[ids, :, 0] = 2.0 ** (at * 8 // len(at) - 8)
        elif kind == "keys_shrink":
            sc[ids, :, 0] = 2.0 ** (-1 - at * 8 // len(at))
        elif kind == "sink":
            sc[ids[:1], :, 0] = 1.0
        elif kind == "value_scales":
            sc[ids, :, 1] = 2.0 ** rng.integers(-38, 20, (len(ids), 2))
        else:
            steps = at * 40 // len(at) - 20
            sc[ids, :, 1] = 2.0 ** (steps if kind == "values_grow" else -steps)
    q = torch.from_numpy(rng.standard_normal((2 * new, 4, d)).astype(np.float32)).to(dt).to(dev)
    ref = orc.attention(q.double().cpu().numpy(), orc.Layer(raw, sc), table, np.array([length, 700]), [0, new, 2 * new])
    out, lse = bsa.kv_attention(q, pages, torch.from_numpy(sc).to(dev), tab, _i32([length, 700], dev), max_len=max_len)
    if dt == torch.float16:  # outputs past its range are infinite (the ones about 65520 may be either)
        past = np.abs(ref[0]) >= 65520 * (1 - 2.0 ** -7)
        sure = np.abs(ref[0]) >= 65520 * (1 + 2.0 ** -7)
        assert (out.double().cpu().numpy()[sure] == np.copysign(np.inf, ref[0][sure])).all()
        out = torch.where(torch.from_numpy(past).to(dev), 0, out)
        ref = (np.where(past, 0.0, ref[0]), *ref[1:])
    _check_attention(out, lse, ref, dt, d)


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("new", [2, 60])
@pytest.mark.parametrize("sm_scale", [-0.125, -1.0, 0.0, -0.0, 1e-30, -1e-30, 2.0])
def test_attention_scales_of_any_sign(dev, sm_scale, new, dtype):
    rng = np.random.default_rng(new)
    lengths = [1500, 61]
    raw, sc, table, pages, scales, tab = _cache(rng, dev, lengths, 2, 32, 64, poison=True)
    q = torch.from_numpy(rng.standard_normal((2 * new, 4, 64)).astype(np.float32)).to(DT[dtype]).to(dev)
    ref = orc.attention(q.double().cpu().numpy(), orc.Layer(raw, sc), table, np.array(lengths), [0, new, 2 * new], sm_scale=sm_scale)
    for max_len in (None, 500):
        out, lse = bsa.kv_attention(q, pages, scales, tab, _i32(lengths, dev), sm_scale=sm_scale, max_len=max_len)
        _check_attention(out, lse, ref, DT[dtype], 64)


def test_prompt_split_graph_and_repeats(dev):
    """A prompt in several parts: the same numbers at every call, eager or replayed."""
    rng = np.random.default_rng(16)
    raw, sc, table, pages, scales, tab = _cache(rng, dev, [3000, 1900], 2, 16, 128)
    n = _i32([3000, 1900], dev)
    q = torch.randn(300, 4, 128, device=dev, dtype=torch.bfloat16)
    want, want_l = (x.clone() for x in bsa.kv_attention(q, pages, scales, tab, n))
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        out, lse = bsa.kv_attention(q, pages, scales, tab, n)
    for _ in range(4):
        out.fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(lse, want_l)
        eager = bsa.kv_attention(q, pages, scales, tab, n)
        assert torch.equal(eager[0], want) and torch.equal(eager[1], want_l)
    ref = orc.attention(q.double().cpu().numpy(), orc.Layer(raw, sc), table, np.array([3000, 1900]), [0, 150, 300])
    _check_attention(want, want_l, ref, torch.bfloat16, 128)


@pytest.mark.parametrize("octaves", [10, 20, 24, 26, 27, 28, 30, 40, 70])
@pytest.mark.parametrize("new,hq", [(1, 2), (3, 2), (30, 4)])
@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
def test_attention_far_scores(dev, dtype, new, hq, octaves):
    """Scores of up to 2^octaves that differ by as much: the values of the largest are averaged.  Queries and
    keys are small integers, so the products are exact; the outputs are rounded once (2^-11 or 2^-8) after weights
    that are equal or vanish, and the lse carries a few roundings of its own size."""
    rng = np.random.default_rng(octaves)
    p, d, lengths = 16, 64, [1300, 70]
    raw, sc, table, pages, scales, tab = _cache(rng, dev, lengths, 1, p, d)
    ints = torch.from_numpy(rng.integers(-1, 2, raw[:, :, 0].shape).astype(np.float32)).to(F8)
    raw[:, :, 0] = ints.view(torch.uint8).numpy()
    sc[..., 0], sc[..., 1] = 2.0 ** octaves, 0.125
    q = torch.from_numpy(rng.integers(-2, 3, (2 * new, hq, d)).astype(np.float32)).to(DT[dtype]).to(dev)
    o, l, *_ = orc.attention(q.double().cpu().numpy(), orc.Layer(raw, sc), table, np.array(lengths), [0, new, 2 * new], sm_scale=0.25)
    out, lse = bsa.kv_attention(q, torch.from_numpy(raw).to(dev).view(F8), torch.from_numpy(sc).to(dev), tab, _i32(lengths, dev),
                                sm_scale=0.25)
    u = 2.0 ** -10 if dtype == "fp16" else 2.0 ** -7
    assert (np.abs(out.double().cpu().numpy() - o) <= u * np.abs(o) + 2.0 ** -10).all()
    assert (np.abs(lse.double().cpu().numpy() - l) <= 2.0 ** -21 * np.abs(l)).all()


@pytest.mark.parametrize("octaves", [4, 8, 10, 12, 14, 16, 17, 18])
def test_prompt_equal_scores_weigh_the_same(dev, octaves):
    """Every token has the same key, so that a row's scores, however far from 0, are one number, and its output is the mean of what it
    sees: weights that are off by their rounding to fp16, 2^-11, and by at most 2^-13 of each other before."""
    rng = np.random.default_rng(octaves)
    p, d, lengths, new = 16, 64, [2200, 700], 50
    raw, sc, table, *_ = _cache(rng, dev, lengths, 2, p, d)
    key = torch.from_numpy(rng.integers(-2, 3, d).astype(np.float32)).to(F8).view(torch.uint8).numpy()
    one = np.zeros(p * d, np.uint8)
    for t in range(p):
        one[[orc.key_offset(t, x, d) for x in range(d)]] = key
    raw[:, :, 0] = one.reshape(p, d)
    sc[..., 0], sc[..., 1] = 2.0 ** octaves, 0.125
    args = (torch.from_numpy(raw).to(dev).view(F8), torch.from_numpy(sc).to(dev), _i32(table, dev), _i32(lengths, dev))
    for dtype, u in (("fp16", 2.0 ** -11), ("bf16", 2.0 ** -8)):
        q = torch.from_numpy(rng.integers(-2, 3, (2 * new, 4, d)).astype(np.float32)).to(DT[dtype]).to(dev)
        o, l, mag, *_ = orc.attention(q.double().cpu().numpy(), orc.Layer(raw, sc), table, np.array(lengths), [0, new, 2 * new], sm_scale=0.25)
        for max_len in (None, 500):
            out, lse = bsa.kv_attention(q, *args, sm_scale=0.25, max_len=max_len)
            assert (np.abs(out.double().cpu().numpy() - o) <= u * np.abs(o) + (2.0 ** -11 + 2.0 ** -13) * mag + 2.0 ** -20).all()
            assert (np.abs(lse.double().cpu().numpy() - l) <= 2.0 ** -21 * np.abs(l) + 2.0 ** -10).all()


def test_prompt_scores_of_minus_infinity_first(dev):
    """A prompt whose first tokens' scores pass the end of 32 bits: the later ones are seen as if alone."""
    rng = np.random.default_rng(17)
    p, d, length, new = 16, 64, 300, 40
    raw, sc, table, pages, scales, tab = _cache(rng, dev, [length], 1, p, d)
    sc[:] = 1.0
    minus = torch.tensor([-448.0, -8.0]).to(F8).view(torch.uint8).numpy()
    for t in range(length):
        tile = raw[table[0, t // p], 0, 0].reshape(-1)
        for x in range(d):
            tile[orc.key_offset(t % p, x, d)] = 0
        tile[orc.key_offset(t % p, 0, d)] = minus[0] if t < 128 else 0
        tile[orc.key_offset(t % p, 1, d)] = minus[1]
    q = torch.zeros(new, 1, d)
    q[..., 0], q[..., 1] = 1e38, 128
    q = q.bfloat16().to(dev)
    ref = orc.attention(q.double().cpu().numpy(), orc.Layer(raw, sc), table, np.array([length]), [0, new])
    out, lse = bsa.kv_attention(q, torch.from_numpy(raw).to(dev).view(F8), torch.from_numpy(sc).to(dev), tab, _i32([length], dev))
    assert np.allclose(ref[1][:, 0], np.log(length - 128 - new + 1 + np.arange(new)) - 128, atol=1e-9)
    _check_attention(out, lse, (*ref[:3], np.full_like(ref[3], 128.0), *ref[4:]), torch.bfloat16, d)


def test_attention_empty_rows(dev):
    """Sequences without tokens, new tokens that have no place, slots out of range: zeros and -inf."""
    rng = np.random.default_rng(2)
    lengths, new, slots = [0, 3, 40, 17], [2, 5, 1, 0, 1], [0, 1, 9, 3, 2]
    raw, sc, table, pages, scales, tab = _cache(rng, dev, lengths, 2, 16, 64, poison=True)
    cu = np.concatenate([[0], np.cumsum(new)])
    q = torch.randn(cu[-1], 2, 64, device=dev, dtype=torch.float16)
    ref = orc.attention(q.double().cpu().numpy(), orc.Layer(raw, sc), table, np.array(lengths), list(cu), slots)
    out, lse = bsa.kv_attention(q, pages, scales, tab, _i32(lengths, dev), cu_seqlens=_i32(cu, dev), max_new=5,
                                slots=_i32(slots, dev), out=torch.full_like(q, float("nan")))
    assert np.isneginf(ref[1][0]).all() and np.isneginf(ref[1][7]).all() and np.isfinite(ref[1][6]).all()
    _check_attention(out, lse, ref, torch.float16, 64)


def test_attention_pages_out_of_range(dev):
    """Tokens on a page that does not exist are not seen; nothing is read for them."""
    rng = np.random.default_rng(8)
    lengths = [70, 50, 16]
    raw, sc, table, pages, scales, tab = _cache(rng, dev, lengths, 2, 16, 128)
    table[0, 2], table[1, 0], table[2, 0] = -1, 10 ** 8, -7
    q = torch.randn(3, 4, 128, device=dev, dtype=torch.bfloat16)
    ref = orc.attention(q.double().cpu().numpy(), orc.Layer(raw, sc), table, np.array(lengths), [0, 1, 2, 3])
    out, lse = bsa.kv_attention(q, pages, scales, _i32(table, dev), _i32(lengths, dev))
    _check_attention(out, lse, ref, torch.bfloat16, 128)


@pytest.mark.parametrize("new,hq", [(4, 2), (40, 2), (70, 4)])
def test_attention_nan_in_unseen_tokens(dev, new, hq):
    """A NaN key or value of a later token does not reach the tokens before it, and does reach those
    that see it."""
    rng = np.random.default_rng(9)
    p, d, length = 16, 64, 90
    raw, sc, table, pages, scales, tab = _cache(rng, dev, [length], 1, p, d)
    bad_v, bad_k = length - new + new // 2, length - 1
    raw[table[0, bad_v // p], 0, 1].reshape(-1)[orc.value_offset(bad_v % p, 7, d)] = 0xFF
    raw[table[0, bad_k // p], 0, 0].reshape(-1)[orc.key_offset(bad_k % p, 3, d)] = 0x7F
    pages = torch.from_numpy(raw).to(dev).view(F8)
    q = torch.randn(new, hq, d, device=dev, dtype=torch.float16)
    with np.errstate(invalid="ignore"):
        ref = orc.attention(q.double().cpu().numpy(), orc.Layer(raw, sc), table, np.array([length]), [0, new])
    out, lse = bsa.kv_attention(q, pages, scales, tab, _i32([length], dev))
    assert np.isfinite(ref[0][: new // 2]).all() and np.isnan(ref[0][new // 2:-1, :, 7]).all() and np.isnan(ref[0][-1]).all()
    last = np.isnan(ref[1])
    assert last[-1].all() and np.isnan(lse.cpu().numpy()[last]).all()
    _check_attention(out, torch.where(torch.from_numpy(last).to(dev), 0.0, lse),
                     (ref[0], np.where(last, 0.0, ref[1]), *[np.nan_to_num(x) for x in ref[2:]]), torch.float16, d)


def test_attention_uneven_scales(dev):
    """Pages whose scales differ by many octaves, keys' and values' apart."""
    rng = np.random.default_rng(12)
    raw, sc, table, pages, scales, tab = _cache(rng, dev, [200, 33], 2, 16, 64)
    sc[..., 1] = 2.0 ** rng.integers(-38, 20, sc[..., 1].shape)
    sc[..., 0] = 2.0 ** rng.integers(-12, -4, sc[..., 0].shape)
    q = torch.randn(2, 4, 64, device=dev, dtype=torch.bfloat16)
    ref = orc.attention(q.double().cpu().numpy(), orc.Layer(raw, sc), table, np.array([200, 33]), [0, 1, 2])
    out, lse = bsa.kv_attention(q, pages, torch.from_numpy(sc).to(dev), tab, _i32([200, 33], dev))
    _check_attention(out, lse, ref, torch.bfloat16, 64)


def test_attention_strides_scale_and_prefix(dev):
    """q and out as views of wider tensors, a scale of the caller's, a named workspace."""
    rng = np.random.default_rng(4)
    lengths = [300, 20]
    raw, sc, table, pages, scales, tab = _cache(rng, dev, lengths, 2, 32, 128, poison=True)
    fused = torch.randn(2, 3 * 4, 128, device=dev, dtype=torch.float16)
    q = fused[:, 4:8]
    room = torch.full((2, 6, 132), 7.0, device=dev, dtype=torch.float16)
    out = room[:, 1:5, 4:]
    ref = orc.attention(q.double().cpu().numpy(), orc.Layer(raw, sc), table, np.array(lengths), [0, 1, 2], sm_scale=0.03)
    got, lse = bsa.kv_attention(q, pages, scales, tab, _i32(lengths, dev), sm_scale=0.03, out=out, workspace_prefix="test")
    assert got is out
    _check_attention(out, lse, ref, torch.float16, 128)
    assert (room[:, 0] == 7).all() and (room[:, 5] == 7).all() and (room[:, :, :4] == 7).all()


def test_attention_past_32_bit_offsets(dev):
    """Pages past 4 GiB of one layer: offsets in 64 bits, in append and in attention."""
    p, d, heads = 128, 128, 8
    count = (1 << 32) // (heads * 2 * p * d) + 40
    pages = torch.zeros(count, heads, 2, p, d, dtype=torch.uint8, device=dev).view(F8)
    scales = torch.ones(count, heads, 2, device=dev)
    tab = _i32([[count - 1, count - 7, 3]], dev)
    n = 300
    k, v = (torch.randn(n, heads, d, device=dev, dtype=torch.float16) for _ in range(2))
    bsa.kv_append(k, v, pages, scales, tab, _i32([n], dev))
    ids = tab[0].long()
    raw = pages.view(torch.uint8)[ids].cpu().numpy()
    layer = orc.Layer(raw, scales[ids].cpu().numpy())
    want = orc.Layer(np.zeros_like(raw), np.ones((3, heads, 2)))
    orc.append(want, k.float().cpu().numpy(), v.float().cpu().numpy(), np.array([[0, 1, 2]]), np.array([n]), [0, n])
    np.testing.assert_array_equal(layer.values, want.values)
    np.testing.assert_array_equal(layer.scales, want.scales)
    q = torch.randn(1, heads, d, device=dev, dtype=torch.float16)
    ref = orc.attention(q.double().cpu().numpy(), layer, np.array([[0, 1, 2]]), np.array([n]), [0, 1])
    out, lse = bsa.kv_attention(q, pages, scales, tab, _i32([n], dev))
    _check_attention(out, lse, ref, torch.float16, d)


def test_attention_graph_and_streams(dev):
    """Captured calls (split, so with counters) replayed beside eager ones, and two streams at once."""
    rng = np.random.default_rng(6)
    raw, sc, table, pages, scales, tab = _cache(rng, dev, [3000, 900], 4, 16, 128)
    n = _i32([3000, 900], dev)
    q = torch.randn(2, 4, 128, device=dev, dtype=torch.float16)
    want, want_l = (x.clone() for x in bsa.kv_attention(q, pages, scales, tab, n))
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=s):
        out, lse = bsa.kv_attention(q, pages, scales, tab, n)
    for _ in range(4):
        out.fill_(float("nan"))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(lse, want_l)
        eager = bsa.kv_attention(q, pages, scales, tab, n)
        assert torch.equal(eager[0], want)
    other = torch.cuda.Stream()
    other.wait_stream(torch.cuda.current_stream())
    results = []
    for _ in range(20):
        results.append(bsa.kv_attention(q, pages, scales, tab, n)[0])
        with torch.cuda.stream(other):
            results.append(bsa.kv_attention(q, pages, scales, tab, n)[0])
    torch.cuda.synchronize()
    assert all(torch.equal(r, want) for r in results)


# ---------------------------------------------------------------------------------------- pages


def _random_pool(rng, dev, slots, each, count, p, layers=2):
    """A pool in use, made by the oracle from nothing; data of a page is its id at first."""
    pool = orc.Pool([[-1] * each] * slots, [0] * slots, [0] * count, p, range(count))
    pool.extend(rng.integers(0, each * p // 2, slots).tolist())
    pool.fork(rng.integers(0, slots, slots // 2).tolist(), rng.permutation(slots)[: slots // 2].tolist())
    pool.free(rng.permutation(slots)[: slots // 5].tolist())
    heads, d = 2, 64
    pages = torch.from_numpy(orc_bytes(rng, (layers, count, heads, 2, p, d))).to(dev)
    scales = torch.rand(layers, count, heads, 2, device=dev)
    pool.data = list(range(count))
    return pool, pages, scales, _i32(pool.table, dev), _i32(pool.lengths, dev), _i32(pool.refs, dev)


def _same_pool(pool, tab, lengths, refs, pages=None, scales=None, was=None, live_only=True):
    assert tab.cpu().tolist() == pool.table
    assert lengths.cpu().tolist() == pool.lengths
    assert refs.cpu().tolist() == pool.refs
    if pages is not None:
        ids = [i for i, r in enumerate(pool.refs) if r > 0 or not live_only]
        src = [pool.data[i] for i in ids]
        assert torch.equal(pages[:, ids], was[0][:, src]) and torch.equal(scales[:, ids], was[1][:, src])


@pytest.mark.parametrize("slots,each,count,p", [(1, 3, 5, 16), (7, 5, 40, 16), (64, 9, 400, 32), (200, 40, 9001, 16),
                                                (1024, 4, 5000, 64)])
def test_pages_random_steps(dev, slots, each, count, p):
    """Forks, extensions (until the pool is full), releases and compactions against the oracle."""
    rng = np.random.default_rng(slots)
    pool, pages, scales, tab, lengths, refs = _random_pool(rng, dev, slots, each, count, p)
    was = pages.clone(), scales.clone()
    f8 = pages.view(F8)
    for step in range(4):
        n = int(rng.integers(1, slots + 1))
        parents, children = rng.integers(-1, slots + 1, n), rng.integers(-1, slots + 1, n)
        pool.fork(parents.tolist(), children.tolist())
        bsa.pages_fork(tab, lengths, refs, _i32(parents, dev), _i32(children, dev))
        _same_pool(pool, tab, lengths, refs)
        for long in (1, p + 3, each * p):
            at = rng.permutation(slots + 1)[:n]
            new = rng.integers(0, long + 1, n)
            served = bsa.pages_extend(f8, scales, tab, lengths, refs, _i32(new, dev), slots=_i32(at, dev))
            assert served.cpu().tolist() == pool.extend(new.tolist(), at.tolist())
            _same_pool(pool, tab, lengths, refs, pages, scales, was)
        gone = rng.integers(-1, slots + 1, max(1, n // 2))
        pool.free(gone.tolist())
        bsa.pages_free(tab, lengths, refs, _i32(gone, dev))
        _same_pool(pool, tab, lengths, refs)
        counts = bsa.pages_compact(f8, scales, tab, refs)
        assert counts.cpu().tolist() == pool.compact()
        _same_pool(pool, tab, lengths, refs, pages, scales, was)


def test_pages_of_a_large_pool(dev):
    """70001 pages (the plans walk them 4096 at a time), 4.6 GB of data: the free ids in the middle, then last."""
    slots, each, count, p = 300, 200, 70001, 32
    pool = orc.Pool([[-1] * each] * slots, [0] * slots, [0] * count, p, range(count))
    rng = np.random.default_rng(18)
    pool.extend(rng.integers(150 * p, each * p, slots).tolist())
    # the live pages lie in two blocks, the second one at the pool's end
    for s in range(slots):
        pool.table[s] = [x if x < 20000 or x < 0 else count - 1 - (x - 20000) for x in pool.table[s]]
    refs = [0] * count
    for row in pool.table:
        for x in row:
            if x >= 0:
                refs[x] = 1
    pool.refs = refs
    g = torch.Generator(device=dev).manual_seed(1)
    pages = torch.randint(0, 127, (2, count, 4, 2, p, 128), generator=g, device=dev, dtype=torch.uint8)
    scales = torch.rand(2, count, 4, 2, generator=g, device=dev)
    was = pages.clone(), scales.clone()
    tab, lengths, refs = _i32(pool.table, dev), _i32(pool.lengths, dev), _i32(pool.refs, dev)
    f8 = pages.view(F8)

    def check():
        assert torch.equal(tab, _i32(pool.table, dev)) and torch.equal(lengths, _i32(pool.lengths, dev))
        assert torch.equal(refs, _i32(pool.refs, dev))
        some = [i for i, r in enumerate(pool.refs) if r > 0]
        some = some[:500] + some[len(some) // 2 - 500: len(some) // 2 + 500] + some[-500:]
        src = [pool.data[i] for i in some]
        assert torch.equal(pages[:, some], was[0][:, src]) and torch.equal(scales[:, some], was[1][:, src])

    for step in range(3):
        parents, children = rng.integers(0, slots, 40), rng.permutation(slots)[:40]
        pool.fork(parents.tolist(), children.tolist())
        bsa.pages_fork(tab, lengths, refs, _i32(parents, dev), _i32(children, dev))
        new = rng.integers(0, 40, slots)
        served = bsa.pages_extend(f8, scales, tab, lengths, refs, _i32(new, dev))
        assert served.cpu().tolist() == pool.extend(new.tolist())
        check()
        counts = bsa.pages_compact(f8, scales, tab, refs)
        assert counts.cpu().tolist() == pool.compact()
        check()
        gone = rng.integers(0, slots, 30)
        pool.free(gone.tolist())
        bsa.pages_free(tab, lengths, refs, _i32(gone, dev))


def test_pages_extend_shared_tail_without_room(dev):
    """Readers of one partly filled page when the free pages do not reach: nobody writes to a page
    that another still reads."""
    p = 16
    for count in (2, 3, 4, 5):
        pool = orc.Pool([[0, -1]] * 4, [5] * 4, [4] + [0] * (count - 1), p, range(count))
        pages = torch.zeros(1, count, 1, 2, p, 64, dtype=torch.uint8, device=dev).view(F8)
        scales = torch.ones(1, count, 1, 2, device=dev)
        tab, lengths, refs = _i32(pool.table, dev), _i32(pool.lengths, dev), _i32(pool.refs, dev)
        served = bsa.pages_extend(pages, scales, tab, lengths, refs, _i32([1, 0, 1, 1], dev))
        assert served.cpu().tolist() == pool.extend([1, 0, 1, 1])
        _same_pool(pool, tab, lengths, refs)
        grown = [s for s in range(4) if pool.lengths[s] == 6]
        assert len({pool.table[s][0] for s in grown}) == len(grown)
        assert all(pool.refs[pool.table[s][0]] == 1 for s in grown)


def test_pages_copy(dev):
    rng = np.random.default_rng(1)
    pages = torch.from_numpy(orc_bytes(rng, (3, 50, 5, 2, 16, 64))).to(dev)
    scales = torch.rand(3, 50, 5, 2, device=dev)
    want = pages.clone(), scales.clone()
    src, dst = [3, 9, 3, -1, 7, 60, 5], [40, 41, 42, 43, -1, 44, 60]
    bsa.pages_copy(pages.view(F8), scales, _i32(src, dev), _i32(dst, dev))
    for a, b in zip(src[:3], dst[:3]):
        want[0][:, b], want[1][:, b] = want[0][:, a], want[1][:, a]
    assert torch.equal(pages, want[0]) and torch.equal(scales, want[1])


def test_threads_on_one_stream(dev):
    """Two threads, each with a cache of its own, on one stream: extensions, compactions and split attention
    give each what it asked for."""
    slots, count, p, rounds = 40, 900, 16, 60
    results = {}

    def work(seed):
        rng = np.random.default_rng(seed)
        pool, pages, scales, tab, lengths, refs = _random_pool(rng, dev, slots, 12, count, p)
        was = pages.clone(), scales.clone()
        f8 = pages.view(F8)
        raw, sc, table, kv, kv_scales, kv_tab = _cache(rng, dev, [3000], 2, 16, 64)
        q, n = torch.randn(1, 4, 64, device=dev, dtype=torch.float16), _i32([3000], dev)
        ok = []
        first = bsa.kv_attention(q, kv, kv_scales, kv_tab, n)[0]
        for _ in range(rounds):
            gone = rng.integers(0, slots, 8)
            pool.free(gone.tolist())
            bsa.pages_free(tab, lengths, refs, _i32(gone, dev))
            new = rng.integers(0, 20, slots)
            served = bsa.pages_extend(f8, scales, tab, lengths, refs, _i32(new, dev))
            out = bsa.kv_attention(q, kv, kv_scales, kv_tab, n)[0]
            counts = bsa.pages_compact(f8, scales, tab, refs)
            ok.append((served, pool.extend(new.tolist()), counts, pool.compact(), torch.equal(out, first)))
        for got, want, counts, moved, same in ok:
            assert got.tolist() == want and counts.tolist() == moved and same
        _same_pool(pool, tab, lengths, refs, pages, scales, was)
        results[seed] = True

    threads = [threading.Thread(target=work, args=(s,)) for s in (21, 22)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert results == {21: True, 22: True}


def test_cache_class_and_graph(dev):
    """A decode loop through KVCache: prompts, steps, a fork, a release and a compaction, the step as one
    replayed graph; attention against the oracle on the cache's own numbers at every stage."""
    torch.manual_seed(0)
    heads, hq, d, slots = 2, 4, 64, 6
    cache = bsa.KVCache(2, 64, heads, d, page_size=16, max_slots=slots, max_pages=8, device=dev)
    first = _i32([20, 0, 33, 0, 0, 0], dev)
    assert cache.extend(first).tolist() == [1] * slots
    cu = _i32([0, 20, 20, 53, 53, 53, 53], dev)
    for layer in range(2):
        k, v = (torch.randn(53, heads, d, device=dev, dtype=torch.float16) for _ in range(2))
        cache.append(layer, k, v, cu_seqlens=cu, max_new=33)
    cache.fork(_i32([0, 0, 2], dev), _i32([1, 3, 4], dev))
    live = _i32([0, 1, 2, 3, 4], dev)
    ones = torch.ones(5, dtype=torch.int32, device=dev)
    x = [[torch.randn(5, n, d, device=dev, dtype=torch.float16) for n in (heads, heads, hq)] for _ in range(2)]
    served = torch.zeros(5, dtype=torch.int32, device=dev)

    def step():
        cache.extend(ones, slots=live, served=served)
        outs = []
        for layer, (k, v, q) in enumerate(x):
            cache.append(layer, k, v, slots=live)
            outs.append(cache.attend(layer, q, slots=live))
        return outs

    def check(outs):
        assert served.tolist() == [1] * 5
        for layer, (out, lse) in enumerate(outs):
            ref = orc.attention(x[layer][2].double().cpu().numpy(),
                                orc.Layer(_raw(cache.pages[layer]), cache.scales[layer].cpu().numpy()),
                                cache.page_table.cpu().numpy(), cache.lengths.cpu().numpy(), [0, 1, 2, 3, 4, 5], [0, 1, 2, 3, 4])
            _check_attention(out, lse, ref, torch.float16, d)

    check(step())
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    for i in range(14):
        for group in x:
            for t in group:
                t.normal_()
        graph.replay()
        torch.cuda.synchronize()
        check(outs)
        if i == 6:
            cache.free(_i32([1, 1], dev))
            live.copy_(_i32([0, 5, 2, 3, 4], dev))  # slot 5 takes the row over
            live.copy_(_i32([0, 1, 2, 3, 4], dev))
            cache.fork(_i32([2], dev), _i32([1], dev))
            cache.compact()
    k, _ = cache.read(1, 2)
    assert k.shape == (heads, 33 + 15, d)
    assert int(cache.lengths[2]) == 48 and torch.isfinite(k).all()


def test_cache_grown_by_larger_tensors(dev):
    """All calls work on the tensors that the cache has now; layers are indexed as a list's entries are."""
    heads, d, layers = 2, 64, 3
    cache = bsa.KVCache(layers, 4, heads, d, page_size=16, max_slots=2, max_pages=8, device=dev)
    assert cache.extend(_i32([20, 9], dev)).tolist() == [1, 1]
    x = [torch.randn(29, heads, d, device=dev, dtype=torch.float16) for _ in range(layers)]
    cu = _i32([0, 20, 29], dev)
    for layer in range(layers):
        cache.append(layer, x[layer], -x[layer], cu_seqlens=cu)
    old = cache.pages
    cache.pages = torch.zeros(layers, 40, heads, 2, 16, d, dtype=torch.uint8, device=dev).view(F8)
    cache.pages.view(torch.uint8)[:, :4] = old.view(torch.uint8)
    cache.scales = torch.cat([cache.scales, torch.ones(layers, 36, heads, 2, device=dev)], 1)
    cache.refcounts = torch.cat([cache.refcounts, cache.refcounts.new_zeros(36)])
    old.view(torch.uint8).fill_(0x7F)
    assert cache.extend(_i32([60, 50], dev)).tolist() == [1, 1]
    new = [torch.randn(110, heads, d, device=dev, dtype=torch.float16) for _ in range(layers)]
    cu = _i32([0, 60, 110], dev)
    for layer in (0, 2, -2):
        cache.append(layer, new[layer], -new[layer], cu_seqlens=cu)
        q = torch.randn(2, heads, d, device=dev, dtype=torch.float16)
        out, lse = cache.attend(layer, q)
        ref = orc.attention(q.double().cpu().numpy(), orc.Layer(_raw(cache.pages[layer]), cache.scales[layer].cpu().numpy()),
                            cache.page_table.cpu().numpy(), cache.lengths.cpu().numpy(), [0, 1, 2])
        _check_attention(out, lse, ref, torch.float16, d)
        k, v = cache.read(layer, 0)
        want = torch.cat([x[layer][:20], new[layer][:60]]).transpose(0, 1).float()
        assert (k - want).abs().max() <= 0.3 and (v + want).abs().max() <= 0.3  # of at most 6: 2^-4 of a number
    for layer in (3, -4):
        with pytest.raises(IndexError):
            cache.append(layer, new[0], new[0], cu_seqlens=cu)
        with pytest.raises(IndexError):
            cache.attend(layer, q)
    with pytest.raises(TypeError):
        cache.attend(0.5, q)
    with pytest.raises(ValueError):
        bsa.kv_attention(q, cache.pages, cache.scales, cache.page_table, cache.lengths)
    with pytest.raises(ValueError):
        bsa.kv_attention(q, cache.pages[0], cache.scales[0], cache.page_table, cache.lengths, layer=0)


# ---------------------------------------------------------------------------------------- log probabilities


def _check_logprobs(got, ref):
    lp, ent, ids, top = ref
    assert got.top_ids.cpu().numpy().tolist() == ids.tolist()
    for a, b in ((got.logprob, lp), (got.entropy, ent), (got.top_logprobs, top)):
        a = a.double().cpu().numpy()
        np.testing.assert_array_equal(np.isnan(a), np.isnan(b))
        np.testing.assert_array_equal(np.isneginf(a), np.isneginf(b))
        fine = np.isfinite(b)
        assert (np.abs(a[fine] - b[fine]) <= 2.0 ** -17 * (1 + np.abs(b[fine]))).all()


@pytest.mark.parametrize("dtype", ["fp16", "bf16", "fp32"])
@pytest.mark.parametrize("rows,vocab,k", [(1, 1, 1), (3, 7, 7), (2, 63, 0), (5, 1000, 64), (3, 4099, 20), (2, 32000, 8),
                                          (1, 100003, 50), (700, 513, 3)])
def test_logprobs(dev, dtype, rows, vocab, k):
    rng = np.random.default_rng(vocab)
    x = torch.from_numpy(rng.standard_normal((rows, vocab)).astype(np.float32) * 3).to(DT[dtype])
    tokens = rng.integers(0, vocab, rows)
    got = bsa.token_logprobs(x.to(dev), _i32(tokens, dev), k)
    _check_logprobs(got, orc.token_logprobs(x.double().numpy(), tokens, k))


@pytest.mark.parametrize("dtype", ["fp16", "bf16", "fp32"])
@pytest.mark.parametrize("vocab", [40, 5000, 40000])
def test_logprobs_hard_rows(dev, dtype, vocab):
    """Equal, masked, ascending and non-finite rows, tokens out of range."""
    rng = np.random.default_rng(7)
    x = rng.standard_normal((12, vocab)).astype(np.float32)
    x[0] = 2.5
    x[1] = -np.inf
    x[2, 5:] = -np.inf
    x[3] = np.linspace(-8, 8, vocab)
    x[4] = np.linspace(8, -8, vocab)
    x[5, vocab // 2] = np.nan
    x[6, 3], x[6, vocab - 1] = np.inf, np.inf
    x[7] = np.where(rng.random(vocab) < 0.5, 0.0, -0.0)
    x[8] = np.finfo(np.float16).min if dtype != "bf16" else -3e38
    x[9, :-1] = -np.inf
    x[10] = np.round(x[10])
    x[11] = x[11] * 1e-3 + 1000
    tokens = rng.integers(0, vocab, 12)
    tokens[1], tokens[9], tokens[10], tokens[11] = 3, vocab - 1, -1, vocab
    t = torch.from_numpy(x).to(DT[dtype])
    got = bsa.token_logprobs(t.to(dev), _i32(tokens, dev), 20)
    with np.errstate(invalid="ignore"):
        _check_logprobs(got, orc.token_logprobs(t.double().numpy(), tokens, 20))


@pytest.mark.parametrize("vocab", [40, 5000, 40000])
@pytest.mark.parametrize("dtype,mask", [("fp16", -6e4), *[(t, m) for t in ("bf16", "fp32")
                                                          for m in (-1e6, -1e9, -1e10, -1e12, -1e20, -1e30, -3e38, -np.inf)]])
def test_logprobs_masks_of_any_size(dev, dtype, mask, vocab):
    """Rows of which a few logits, every other one, one or none is no mask, tokens under the mask and beside it."""
    rng = np.random.default_rng(vocab)
    x = rng.standard_normal((8, vocab)).astype(np.float32)
    lowest = max(mask, float(torch.finfo(DT[dtype]).min))
    x[0, 5:] = mask
    x[1, : vocab - 5] = mask
    x[2, ::2] = mask
    x[3] = mask
    x[4, np.arange(vocab) != vocab // 2] = mask
    x[5, : vocab // 2], x[5, vocab // 2:] = mask, lowest / 2
    x[6, 7:] = mask
    x[7, rng.random(vocab) < 0.9] = mask
    tokens = np.array([0, 3, 2, vocab - 1, vocab // 2, vocab - 1, vocab - 1, 5])
    t = torch.from_numpy(x).to(DT[dtype])
    for k in (0, 20):
        got = bsa.token_logprobs(t.to(dev), _i32(tokens, dev), k)
        _check_logprobs(got, orc.token_logprobs(t.double().numpy(), tokens, k))


@pytest.mark.parametrize("vocab", [40, 5000, 40000])
@pytest.mark.parametrize("middle", [2.0 ** 20, -(2.0 ** 20), 2.0 ** 21, 1e6, 1e8, -1e10, 1e30])
def test_logprobs_far_from_zero(dev, middle, vocab):
    """Logits that are far from zero, or on either side of where that begins, and close to each other."""
    rng = np.random.default_rng(3)
    x = (middle + 3 * rng.standard_normal((4, vocab))).astype(np.float32)
    x[1] = np.float32(middle) + np.spacing(np.float32(middle)) * rng.integers(-9, 9, vocab)
    x[2, rng.random(vocab) < 0.5] = 0
    x[3] = np.float32(middle) * rng.standard_normal(vocab)
    tokens = rng.integers(0, vocab, 4)
    got = bsa.token_logprobs(torch.from_numpy(x).to(dev), _i32(tokens, dev), 6)
    _check_logprobs(got, orc.token_logprobs(x.astype(np.float64), tokens, 6))


@pytest.mark.parametrize("rows,vocab", [(4200, 8192), (300, 32000), (3, 100003)])
@pytest.mark.parametrize("dtype", ["fp16", "fp32"])
def test_logprobs_confident_rows(dev, dtype, rows, vocab):
    """One logit 2 to 26 above the others, anywhere in its row, so that the entropy is small beside log2 l and
    t / l where the reference lies far below it.  Against 64 bits: weights of at most 3 octaves, so that
    the exponent, its logarithm and the quotient are each off by at most 2^-22, and sums whose
    roundings are independent, 2^-21: together below 2^-19 of 1 + |value|."""
    g = torch.Generator(device=dev).manual_seed(vocab)
    x = torch.randn(rows, vocab, generator=g, device=dev)
    at = torch.randint(0, vocab, (rows,), generator=g, device=dev)
    x[torch.arange(rows, device=dev), at] = x.amax(1) + torch.linspace(2, 26, rows, device=dev)
    x = x.to(DT[dtype])
    got = bsa.token_logprobs(x, at.int(), 1)
    assert torch.equal(got.top_ids[:, 0], at.int())
    for r in range(0, rows, 300):
        d = x[r:r + 300].double()
        d -= d.amax(1, keepdim=True)
        d -= d.exp().sum(1, keepdim=True).log()
        for a, b in ((got.logprob, d.amax(1)), (got.top_logprobs[:, 0], d.amax(1)), (got.entropy, -(d.exp() * d).sum(1))):
            assert ((a[r:r + 300].double() - b).abs() <= 2.0 ** -19 * (1 + b.abs())).all()


@pytest.mark.parametrize("dtype", ["fp16", "fp32"])
@pytest.mark.parametrize("offset,width", [(1, 1003), (3, 1009), (7, 1024)])
def test_logprobs_unaligned_rows(dev, dtype, offset, width):
    """Rows that begin anywhere and are followed by what is no logit of theirs."""
    rng = np.random.default_rng(offset)
    wide = torch.full((6, width), float("inf"), dtype=DT[dtype], device=dev)
    vocab = 990
    x = torch.from_numpy(rng.standard_normal((6, vocab)).astype(np.float32)).to(DT[dtype])
    view = wide[:, offset:offset + vocab]
    view.copy_(x)
    tokens = rng.integers(0, vocab, 6)
    got = bsa.token_logprobs(view, _i32(tokens, dev), 5)
    _check_logprobs(got, orc.token_logprobs(x.double().numpy(), tokens, 5))


def test_logprobs_graph(dev):
    x = torch.randn(3, 50000, device=dev)
    tokens = _i32([1, 2, 3], dev)
    graph = torch.cuda.CUDAGraph()
    bsa.token_logprobs(x, tokens, 10)
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        got = bsa.token_logprobs(x, tokens, 10)
    for _ in range(4):
        x.normal_()
        graph.replay()
        torch.cuda.synchronize()
        want = bsa.token_logprobs(x, tokens, 10)
        assert all(torch.equal(a, b) for a, b in zip(got, want))


# ---------------------------------------------------------------------------------------- refusals


def test_refusals(dev):
    pages = torch.zeros(4, 2, 2, 16, 64, dtype=torch.uint8, device=dev).view(F8)
    scales, tab, n = torch.ones(4, 2, 2, device=dev), _i32([[0, 1]], dev), _i32([3], dev)
    x = torch.zeros(1, 2, 64, device=dev, dtype=torch.float16)

    def attend(q=x, pages=pages, scales=scales, tab=tab, n=n, **kw):
        return bsa.kv_attention(q, pages, scales, tab, n, **kw)

    attend()
    for bad in (dict(q=x.float()), dict(pages=pages.view(torch.uint8)), dict(scales=scales.double()), dict(tab=tab.long()),
                dict(n=n.long()), dict(cu_seqlens=torch.zeros(2, device=dev))):
        with pytest.raises(TypeError):
            attend(**bad)
    for bad in (dict(q=x[:, :, :32]), dict(q=x[0]), dict(q=x[:, :1].expand(1, 3, 64).contiguous()), dict(q=x.cpu()),
                dict(scales=scales[:, :1]), dict(pages=pages[:, :1]), dict(tab=tab[0]), dict(n=_i32([3, 4], dev)),
                dict(q=torch.zeros(1, 64, 2, device=dev, dtype=torch.float16).transpose(1, 2)),
                dict(q=torch.zeros(1 * 2 * 64 + 1, device=dev, dtype=torch.float16)[1:].view(1, 2, 64)),
                dict(out=x[0]), dict(lse=scales), dict(max_new=2), dict(cu_seqlens=_i32([0, 1, 1], dev), slots=n)):
        with pytest.raises(ValueError):
            attend(**bad)
    for p, d in ((8, 64), (16, 32), (48, 64), (16, 256)):
        with pytest.raises((ValueError, NotImplementedError)):
            attend(q=torch.zeros(1, 2, d, device=dev, dtype=torch.float16),
                   pages=torch.zeros(4, 2, 2, p, d, dtype=torch.uint8, device=dev).view(F8))
    with pytest.raises(ValueError):
        bsa.kv_append(x, x.bfloat16(), pages, scales, tab, n)
    with pytest.raises(ValueError):
        bsa.kv_append(x, torch.zeros(2, 2, 64, device=dev, dtype=torch.float16), pages, scales, tab, n)
    refs = torch.zeros(4, dtype=torch.int32, device=dev)
    with pytest.raises(NotImplementedError):
        bsa.pages_free(tab, n, refs, torch.zeros(1025, dtype=torch.int32, device=dev))
    with pytest.raises(ValueError):
        bsa.pages_fork(tab, n, refs, _i32([0, 0], dev), _i32([0], dev))
    with pytest.raises(ValueError):
        bsa.pages_extend(pages, scales, tab, n, refs, _i32([1], dev))
    with pytest.raises(ValueError):
        bsa.pages_compact(pages[None], scales[None], tab, refs[:3])
    with pytest.raises(ValueError):
        bsa.KVCache(1, 4, 2, head_dim=96, device=dev)
    logits = torch.zeros(2, 30, device=dev)
    for k, t in ((31, [0, 0]), (-1, [0, 0]), (3, [0])):
        with pytest.raises(ValueError):
            bsa.token_logprobs(logits, _i32(t, dev), k)
    with pytest.raises(ValueError):
        bsa.token_logprobs(torch.zeros(2, 100, device=dev), _i32([0, 0], dev), 65)
    with pytest.raises(TypeError):
        bsa.token_logprobs(logits.double(), _i32([0, 0], dev))
    with pytest.raises(ValueError):
        bsa.token_logprobs(logits.t(), torch.zeros(30, dtype=torch.int32, device=dev))


def test_nothing_to_do(dev):
    pages = torch.zeros(1, 4, 2, 2, 16, 64, dtype=torch.uint8, device=dev).view(F8)
    scales, tab, n = torch.ones(1, 4, 2, 2, device=dev), _i32([[0, 1]], dev), _i32([0], dev)
    x = torch.zeros(0, 2, 64, device=dev, dtype=torch.float16)
    none = torch.zeros(0, dtype=torch.int32, device=dev)
    bsa.kv_append(x, x, pages[0], scales[0], tab, n, slots=none)
    out, lse = bsa.kv_attention(x, pages[0], scales[0], tab, n, slots=none)
    assert out.shape == (0, 2, 64) and lse.shape == (0, 2)
    refs = torch.zeros(4, dtype=torch.int32, device=dev)
    bsa.pages_fork(tab, n, refs, none, none)
    bsa.pages_free(tab, n, refs, none)
    assert bsa.pages_extend(pages, scales, tab, n, refs, none).numel() == 0
    bsa.pages_copy(pages, scales, none, none)
    assert bsa.token_logprobs(torch.zeros(0, 5, device=dev), none, 2).top_ids.shape == (0, 2)


def test_sizes_given_as_tensors_are_read_at_each_call(dev):
    """max_new, max_len and k as tensors that change between calls."""
    rng = np.random.default_rng(14)
    raw, sc, table, pages, scales, tab = _cache(rng, dev, [40], 2, 16, 64)
    n, cu = _i32([40], dev), _i32([0, 3], dev)
    q = torch.randn(3, 2, 64, device=dev, dtype=torch.float16)
    want = bsa.kv_attention(q, pages, scales, tab, n, cu_seqlens=cu, max_new=3)[0]
    most = torch.tensor(1)
    one = bsa.kv_attention(q, pages, scales, tab, n, cu_seqlens=cu, max_new=most, max_len=most, out=torch.zeros_like(q))[0]
    assert torch.equal(one[:1], want[:1]) and not one[1:].any()
    most.fill_(3)
    assert torch.equal(bsa.kv_attention(q, pages, scales, tab, n, cu_seqlens=cu, max_new=most, max_len=most, out=torch.zeros_like(q))[0], want)
    most.fill_(1)
    kept = pages.view(torch.uint8).clone()
    x = torch.ones(3, 2, 64, device=dev, dtype=torch.float16)
    bsa.kv_append(x, x, pages, scales, tab, n, cu_seqlens=cu, max_new=most)
    most.fill_(3)
    bsa.kv_append(x, x, pages, scales, tab, n, cu_seqlens=cu, max_new=most)
    again = kept.clone().view(F8)
    bsa.kv_append(x, x, again, scales, tab, n, cu_seqlens=cu, max_new=3)
    assert torch.equal(pages.view(torch.uint8), again.view(torch.uint8))
    k = torch.tensor(2)
    logits, tokens = torch.randn(2, 30, device=dev), _i32([0, 1], dev)
    assert bsa.token_logprobs(logits, tokens, k).top_ids.shape == (2, 2)
    k.fill_(5)
    assert bsa.token_logprobs(logits, tokens, k).top_ids.shape == (2, 5)
