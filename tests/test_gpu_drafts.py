"""Parity of the operators of drafted tokens with oracle/drafts.py (64 bits, from the definitions) on the GPU: sizes,
trees, masks and numbers at which they can go wrong, streams and graphs, and a step of all of them.

Tolerances, from the arithmetic:
- kv_append_rotated: a channel is two products and a sum, each off by half a step, 2^-24, of their magnitudes: 3 x 2^-24 of
  |a cos| + |b sin|, and 4 is allowed.  A norm adds a sum of 128 squares (chains of at most 40 terms, halved by the root),
  the root's own step, and two products: another 30 x 2^-24.  Then one rounding: half a step of the type, or of e4m3.
- kv_tree_attention: as kv_attention in test_gpu_serving.py.
- verify_drafts, pages_keep: none; both answers are exact.
"""
from __future__ import annotations

import threading

import numpy as np
import pytest
import torch

import bsa_mi355x as bsa
from oracle import drafts as dft
from oracle import serving as orc
from test_gpu_serving import DT, F8, _cache, _check_attention, _i32, _raw, _same_pages

pytestmark = pytest.mark.gpu


def _parents(rng, n, kind="any"):
    """A tree of n nodes: chain, star, or any; the first node a root, now and then another one."""
    if kind == "chain":
        return [i - 1 for i in range(n)]
    if kind == "star":
        return ([-1] + [0] * n)[:n]
    return [-1] + [int(rng.integers(-1, i)) if rng.random() < 0.1 else int(rng.integers(max(0, i - 6), i)) for i in range(1, n)]


def _cu(new):
    return [0, *np.cumsum(new).tolist()]


def _angles(positions, dims):
    a = np.arange(positions)[:, None] * 10000.0 ** (-np.arange(dims // 2) / (dims // 2))
    return np.cos(a).astype(np.float32), np.sin(a).astype(np.float32)


# ---------------------------------------------------------------------------------------- rotation into the cache


def _step8(x):
    """The step of e4m3 at x."""
    return 2.0 ** np.maximum(np.floor(np.log2(np.maximum(np.abs(x), 2.0 ** -9))) - 3, -9)


def _check_rotated(out, pages, scales, layer0, ref_q, mag_q, k, mag_k, v, table, lengths, cu, dtype, normed, slots=None, max_new=None):
    """out and the cache against the turned q and k (64 bits) and their magnitudes."""
    eps = (34 if normed else 4) * 2.0 ** -24
    u = 2.0 ** -11 if dtype == torch.float16 else 2.0 ** -8
    got = out.double().cpu().numpy()
    mine = np.zeros(len(got), bool)  # tokens whose queries the call writes
    for b in range(len(cu) - 1):
        if 0 <= (b if slots is None else slots[b]) < len(lengths):
            mine[cu[b]:min(cu[b + 1], cu[b] + (max_new or cu[b + 1]))] = True
    bound = eps * mag_q + u * (np.abs(ref_q) + eps * mag_q) + 2.0 ** -25
    np.testing.assert_array_equal(np.isnan(got[mine]), np.isnan(ref_q[mine]))
    fine = mine[:, None, None] & np.isfinite(ref_q)
    assert (np.abs(got - ref_q)[fine] <= bound[fine]).all(), np.max((np.abs(got - ref_q) / bound)[fine])
    want = layer0
    orc.append(want, k, v, table, np.asarray(lengths), cu, slots, max_new)
    np.testing.assert_array_equal(scales.cpu().numpy().astype(np.float64), want.scales)
    # the keys' bound, placed as the keys are
    err = orc.Layer(np.zeros_like(_raw(pages)), np.ones(scales.shape, np.float32))
    err.values[:] = 0.0
    for b in range(len(cu) - 1):
        slot, n = b if slots is None else slots[b], cu[b + 1] - cu[b]
        if not 0 <= slot < len(lengths):
            continue
        for i in range(n):
            pos = int(lengths[slot]) - n + i
            page = table[slot][pos // err.p] if 0 <= pos < len(table[slot]) * err.p else -1
            if 0 <= page < err.values.shape[0]:
                err.values[page, :, 0, pos % err.p] = np.nan_to_num(eps * mag_k[cu[b] + i])
    err.values /= want.scales[..., None, None]
    values = orc.E4M3[_raw(pages)]
    tiled = want.tiled()
    np.testing.assert_array_equal(np.isnan(values), np.isnan(tiled))
    off = np.abs(np.nan_to_num(values) - np.nan_to_num(tiled))
    # a number that its error carries over a border between two values is off by one step more than not at all
    slack = np.where(err.tiled() > 0, _step8(np.maximum(np.abs(np.nan_to_num(tiled)), np.abs(np.nan_to_num(values)))), 0.0)
    assert (off <= slack).all()
    # and few are: a border within the error is 2 err / step likely; ten times that, and ten
    assert np.count_nonzero(off) <= 10 + 10 * (2 * err.tiled() / _step8(np.nan_to_num(tiled))).sum()
    return mine


def _rotated(dev, rng, lengths, new, hq, heads, p, d, dims, dtype, interleaved=False, norm=False, mode="place", slots=None, **kw):
    raw, sc, table, pages, scales, tab = _cache(rng, dev, lengths, heads, p, d)
    cu = _cu(new)
    q, k, v = (torch.from_numpy((rng.standard_normal((cu[-1], h, d)) * np.exp(rng.standard_normal((cu[-1], h, 1)))).astype(np.float32)).to(dtype).to(dev)
               for h in (hq, heads, heads))
    cos, sin = _angles(max(lengths) + 3, dims)
    wq, wk = ((torch.from_numpy((1 + 0.3 * rng.standard_normal(d)).astype(np.float32)).to(dtype).to(dev) for _ in range(2)) if norm
              else (None, None))
    given, places = {}, {}
    if mode == "positions":
        places["positions"] = rng.integers(0, max(lengths) + 3, cu[-1])
    if mode == "tree":
        places["parents"] = [x for n in new for x in _parents(rng, n)]
    given = {name: _i32(x, dev) for name, x in places.items()}
    if slots is not None:
        given["slots"] = _i32(slots, dev)
    out = bsa.kv_append_rotated(q, k, v, torch.from_numpy(cos).to(dev), torch.from_numpy(sin).to(dev), pages, scales, tab, _i32(lengths, dev),
                                cu_seqlens=_i32(cu, dev), max_new=max(new), q_norm=wq, k_norm=wk, eps=1e-5, interleaved=interleaved,
                                **given, **kw)
    host = [None if x is None else x.double().cpu().numpy() for x in (q, wq, k, wk)]
    rq, mq = dft.turned(host[0], host[1], 1e-5, cos, sin, interleaved, lengths, cu, slots, **places)
    rk, mk = dft.turned(host[2], host[3], 1e-5, cos, sin, interleaved, lengths, cu, slots, **places)
    _check_rotated(out, pages, scales, orc.Layer(raw, sc), rq, mq, rk, mk, v.double().cpu().numpy(), table, lengths, cu, dtype, norm, slots)
    return out


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("p,d,dims", [(16, 64, 64), (16, 128, 128), (32, 128, 64), (64, 64, 32), (64, 128, 32), (128, 128, 16), (16, 64, 16)])
@pytest.mark.parametrize("interleaved,norm,mode", [(False, False, "place"), (True, True, "tree"), (False, True, "positions"), (True, False, "place")])
def test_rotated(dev, dtype, p, d, dims, interleaved, norm, mode):
    rng = np.random.default_rng([p, d, dims, interleaved, norm])
    _rotated(dev, rng, [1, 21, 38, 300], [1, 5, 33, 64], 6, 3, p, d, dims, DT[dtype], interleaved, norm, mode)


@pytest.mark.parametrize("hq,heads", [(1, 1), (7, 1), (32, 4), (40, 8)])
@pytest.mark.parametrize("new", [[1, 1, 1], [3, 0, 1], [40, 129, 17]])
def test_rotated_batches(dev, hq, heads, new):
    rng = np.random.default_rng([hq, *new])
    lengths = [n + o for n, o in zip(new, [5, 16, 131])]
    _rotated(dev, rng, lengths, new, hq, heads, 32, 128, 128, torch.bfloat16, norm=True)
    _rotated(dev, rng, lengths, new, hq, heads, 16, 64, 64, torch.float16)


def test_rotated_by_nothing_is_append(dev):
    """Angles of 0: the bytes that kv_append writes, and q as it is."""
    rng = np.random.default_rng(3)
    lengths, new = [40, 17, 200], [7, 17, 64]
    _, _, _, pages, scales, tab = _cache(rng, dev, lengths, 2, 16, 128)
    cu = _i32(_cu(new), dev)
    q, k, v = (torch.randn(88, h, 128, device=dev).half() for h in (4, 2, 2))
    k[3, 1, 5], k[9], v[20, 0, 7], v[21, 1] = float("inf"), 0.0, float("nan"), 60000.0
    pages2, scales2 = pages.view(torch.uint8).clone().view(F8), scales.clone()
    one, zero = torch.ones(210, 64, device=dev), torch.zeros(210, 64, device=dev)
    # an infinity times 0 is NaN, so the infinite pair does not turn but in the keys that have none
    k[3, 1, 5] = 3.0
    out = bsa.kv_append_rotated(q, k, v, one, zero, pages, scales, tab, _i32(lengths, dev), cu_seqlens=cu, max_new=64)
    bsa.kv_append(k, v, pages2, scales2, tab, _i32(lengths, dev), cu_seqlens=cu, max_new=64)
    assert torch.equal(pages.view(torch.uint8), pages2.view(torch.uint8)) and torch.equal(scales, scales2) and torch.equal(out, q)


@pytest.mark.parametrize("case", ["fused", "odd_stride", "in_place", "slots", "bad_pages", "short", "nan_inf", "rows_behind", "max_new",
                                  "layer", "position_out"])
def test_rotated_edges(dev, case):
    rng = np.random.default_rng(len(case))
    lengths, new, hq, heads, p, d = [37, 20, 16], [5, 20, 1], 4, 2, 16, 64
    raw, sc, table, pages, scales, tab = _cache(rng, dev, lengths, heads, p, d)
    cu, slots, max_new, dtype = _cu(new), None, 20, torch.float16
    total = cu[-1] + (4 if case == "rows_behind" else 0)
    qkv = torch.randn(total, hq + 2 * heads, d, device=dev).to(dtype)
    q, k, v = (x.contiguous() for x in qkv.split([hq, heads, heads], 1))
    cos, sin = _angles(40, d)
    kw, positions = {}, None
    if case == "fused":
        q, k, v = qkv.split([hq, heads, heads], 1)
    elif case == "odd_stride":
        k, v = (torch.randn(total, heads, d + 1, device=dev).to(dtype)[..., :d] for _ in range(2))
    elif case == "slots":
        slots = [2, 9, 0]
        lengths = [37, 20, 16]
        new = [5, 3, 1]
        cu, total = _cu(new), 9
        q, k, v = q[:9].contiguous(), k[:9].contiguous(), v[:9].contiguous()
    elif case == "bad_pages":
        table[1, 0], table[0, 2] = 10 ** 7, -1
        tab = _i32(table, dev)
    elif case == "short":
        lengths = [3, 20, 16]  # fewer tokens than the new ones: the first have no place
    elif case == "nan_inf":
        k[0, 0, 3], k[8, 1, 7], q[1, 2, 5], v[3, 0, 2], v[4, 1, 1] = float("nan"), float("inf"), float("inf"), float("inf"), float("nan")
    elif case == "max_new":
        max_new = 6
    elif case == "position_out":
        positions = np.arange(26) + 30
        positions[5] = -2
    if positions is not None:
        kw["positions"] = _i32(positions, dev)
    if slots is not None:
        kw["slots"] = _i32(slots, dev)
    host = [x.double().cpu().numpy() for x in (q, k, v)]
    out = torch.full(q.shape, 7.0, dtype=dtype, device=dev)
    if case == "in_place":
        out = q
    args = [pages, scales]
    if case == "layer":
        both = torch.stack([pages.view(torch.uint8)] * 3).view(F8), torch.stack([scales] * 3)
        args, kw["layer"] = list(both), -2
    got = bsa.kv_append_rotated(q, k, v, torch.from_numpy(cos).to(dev), torch.from_numpy(sin).to(dev), *args, tab, _i32(lengths, dev),
                                cu_seqlens=_i32(cu, dev), max_new=max_new, out=out, **kw)
    assert got is out
    if case == "layer":
        for i in (0, 2):
            assert torch.equal(both[0][i].view(torch.uint8), pages.view(torch.uint8)) and torch.equal(both[1][i], scales)
        pages, scales = both[0][1], both[1][1]
    with np.errstate(invalid="ignore"):
        (rq, mq), (rk, mk) = (dft.turned(x, None, 1e-6, cos, sin, False, lengths, cu, slots, positions) for x in host[:2])
        mine = _check_rotated(out, pages, scales, orc.Layer(raw, sc), rq, mq, rk, np.nan_to_num(mk, posinf=0.0), host[2], table, lengths, cu,
                              dtype, False, slots, max_new if case == "max_new" else None)
    assert mine.sum() == {"slots": 6, "max_new": 12}.get(case, 26)
    if case != "in_place":
        assert (out.cpu()[torch.from_numpy(~mine)] == 7.0).all()  # nobody's rows


@pytest.mark.parametrize("p,d", [(16, 64), (128, 128)])
def test_rotated_batches_of_many_sequences_without_a_bound(dev, p, d):
    """300 sequences of 1 to 2000 new tokens with no max_new: more tiles and more rows of queries than one launch takes.  The numbers of
    the call that is told of the longest, and some sequences' against the oracle."""
    rng = np.random.default_rng([19, p])
    hq, heads, n = 6, 24, 300
    new = rng.integers(1, 600, n)
    new[::60] = 2000
    lengths = new + rng.integers(0, 40, n)
    per = -(-lengths // p)
    table = np.full((n, per.max()), -1)
    ids = rng.permutation(int(per.sum()))
    for b, at in enumerate(np.cumsum(per) - per):
        table[b, : per[b]] = ids[at: at + per[b]]
    cu = np.asarray(_cu(new))
    g = torch.Generator(device=dev).manual_seed(1)
    q, k, v = (torch.randn(int(cu[-1]), h, d, generator=g, device=dev, dtype=torch.float16) for h in (hq, heads, heads))
    cos, sin = _angles(2100, d)
    got = []
    for most in (2000, None):
        pages = torch.zeros(len(ids), heads, 2, p, d, dtype=torch.uint8, device=dev).view(F8)
        scales = torch.ones(len(ids), heads, 2, device=dev)
        out = bsa.kv_append_rotated(q, k, v, torch.from_numpy(cos).to(dev), torch.from_numpy(sin).to(dev), pages, scales, _i32(table, dev),
                                    _i32(lengths, dev), cu_seqlens=_i32(cu, dev), max_new=most)
        got.append((pages.view(torch.uint8), scales, out))
    assert all(torch.equal(a, b) for a, b in zip(*got))
    some = [0, 1, 137, n - 1]
    index = torch.from_numpy(np.concatenate([table[b, : per[b]] for b in some])).to(dev)
    own, at = np.full((len(some), per.max()), -1), 0
    for i, b in enumerate(some):
        own[i, : per[b]] = np.arange(at, at + per[b])
        at += per[b]
    own_cu = _cu(new[some])
    rows = torch.cat([torch.arange(cu[b], cu[b + 1]) for b in some]).to(dev)
    host = [t[rows].double().cpu().numpy() for t in (q, k, v)]
    (rq, mq), (rk, mk) = (dft.turned(t, None, 1e-6, cos, sin, False, lengths[some], own_cu) for t in host[:2])
    layer = orc.Layer(np.zeros((at, heads, 2, p, d), np.uint8), np.ones((at, heads, 2), np.float32))
    _check_rotated(got[1][2][rows], got[1][0][index].view(F8), got[1][1][index], layer, rq, mq, rk, mk, host[2], own, lengths[some], own_cu,
                   torch.float16, False)


@pytest.mark.parametrize("dims,interleaved", [(16, False), (64, True), (128, False)])
def test_rotated_by_slices_of_a_table(dev, dims, interleaved):
    """cos and sin beside each other in one table, from a later position on, and a table of one position."""
    rng = np.random.default_rng(dims)
    lengths, new = [30, 17], [9, 17]
    _, _, _, pages, scales, tab = _cache(rng, dev, lengths, 2, 16, 128)
    n, cu = _i32(lengths, dev), _i32(_cu(new), dev)
    q, k, v = (torch.randn(26, h, 128, device=dev).half() for h in (4, 2, 2))
    cos, sin = (torch.from_numpy(x).to(dev) for x in _angles(50, dims))
    both = torch.cat([cos, sin], 1)
    was = pages.view(torch.uint8).clone(), scales.clone()

    def call(cos, sin, positions):
        pages.view(torch.uint8).copy_(was[0])
        scales.copy_(was[1])
        out = bsa.kv_append_rotated(q, k, v, cos, sin, pages, scales, tab, n, cu_seqlens=cu, max_new=17, interleaved=interleaved,
                                    positions=_i32(positions, dev))
        return out, pages.view(torch.uint8).clone(), scales.clone()

    at = rng.integers(7, 50, 26)
    want = call(cos, sin, at)
    for c, s, moved in ((both[:, :dims // 2], both[:, dims // 2:], 0), (both[7:, :dims // 2], both[7:, dims // 2:], 7), (cos[7:], sin[7:], 7)):
        assert all(torch.equal(x, y) for x, y in zip(call(c, s, at - moved), want))
    want = call(cos, sin, [11] * 26)
    assert all(torch.equal(x, y) for x, y in zip(call(both[11:12, :dims // 2], both[11:12, dims // 2:], [0] * 26), want))


@pytest.mark.parametrize("p,d", [(16, 64), (64, 128)])
def test_rotated_magnitudes_past_every_scale(dev, p, d):
    """bf16 numbers of 2^120 beside the largest scale, 2^80: the largest e4m3 number, with its sign, as kv_append."""
    rng = np.random.default_rng(7)
    lengths = [20, 5]
    _, _, _, pages, scales, tab = _cache(rng, dev, lengths, 2, p, d)
    pages2, scales2 = pages.view(torch.uint8).clone().view(F8), scales.clone()
    q, k, v = (torch.randn(10, 2, d, device=dev).bfloat16() for _ in range(3))
    k[2], v[3] = k[2] * 2.0 ** 120, v[3] * 2.0 ** 120
    one, zero = torch.ones(30, d // 2, device=dev), torch.zeros(30, d // 2, device=dev)
    bsa.kv_append_rotated(q, k, v, one, zero, pages, scales, tab, _i32(lengths, dev))
    bsa.kv_append(k, v, pages2, scales2, tab, _i32(lengths, dev))
    assert torch.equal(pages.view(torch.uint8), pages2.view(torch.uint8)) and torch.equal(scales, scales2)
    assert float(scales.max()) == 2.0 ** 80 and not torch.isnan(pages.float()).any()


def test_rotated_graph_and_streams(dev):
    """Captured and replayed with new inputs in the same tensors, and on another stream: the eager numbers."""
    rng = np.random.default_rng(5)
    lengths, new = [40, 9], [6, 3]
    _, _, _, pages, scales, tab = _cache(rng, dev, lengths, 2, 16, 128)
    n, cu, par = _i32(lengths, dev), _i32(_cu(new), dev), _i32([-1, 0, 0, 1, 2, 2, -1, 0, 0], dev)
    cos, sin = (torch.from_numpy(x).to(dev) for x in _angles(64, 128))
    q, k, v = (torch.randn(9, h, 128, device=dev).half() for h in (4, 2, 2))
    was, was_s = pages.view(torch.uint8).clone(), scales.clone()

    def reset():
        pages.view(torch.uint8).copy_(was)
        scales.copy_(was_s)

    def call():
        return bsa.kv_append_rotated(q, k, v, cos, sin, pages, scales, tab, n, cu_seqlens=cu, max_new=6, parents=par)

    call()
    reset()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    for i in range(3):
        for x in (q, k, v):
            x.copy_(torch.randn_like(x))
        reset()
        want = call()
        bytes_want, scales_want = pages.view(torch.uint8).clone(), scales.clone()
        reset()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(pages.view(torch.uint8), bytes_want) and torch.equal(scales, scales_want)
        reset()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            got = call()
        side.synchronize()
        assert torch.equal(got, want) and torch.equal(pages.view(torch.uint8), bytes_want)


# ---------------------------------------------------------------------------------------- attention of a tree


def _attend(dev, rng, lengths, new, hq, heads, p, d, dtype, kind="any", **kw):
    raw, sc, table, pages, scales, tab = _cache(rng, dev, lengths, heads, p, d, poison=True)
    cu = _cu(new)
    parents = [x for n in new for x in _parents(rng, n, kind)]
    q = torch.from_numpy(rng.standard_normal((cu[-1], hq, d)).astype(np.float32)).to(dtype).to(dev)
    ref = dft.tree_attention(q.double().cpu().numpy(), parents, orc.Layer(raw, sc), table, np.array(lengths), cu)
    out, lse = bsa.kv_tree_attention(q, _i32(parents, dev), pages, scales, tab, _i32(lengths, dev), cu_seqlens=_i32(cu, dev),
                                     max_new=max(new), **kw)
    _check_attention(out, lse, ref, dtype, d)


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("kind", ["any", "star", "chain"])
@pytest.mark.parametrize("new", [1, 2, 7, 16, 17, 33, 64])
@pytest.mark.parametrize("hq,heads,p,d", [(2, 2, 16, 128), (6, 2, 32, 64), (8, 1, 64, 128)])
def test_tree(dev, dtype, kind, new, hq, heads, p, d):
    rng = np.random.default_rng([new, hq, len(kind)])
    _attend(dev, rng, [new, new + 1, 64 + new, 200], [new] * 4, hq, heads, p, d, DT[dtype], kind)


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("hq,heads,p,d", [(3, 3, 16, 64), (4, 1, 128, 128), (12, 2, 64, 128), (20, 1, 16, 128)])
@pytest.mark.parametrize("lengths,new", [([150, 257, 64, 31], [64, 13, 1, 30]), ([1100, 2049], [40, 64]), ([33, 47, 48, 49, 63, 64, 65], [32, 32, 17, 18, 31, 64, 33])])
def test_tree_of_several_sizes(dev, dtype, hq, heads, p, d, lengths, new):
    rng = np.random.default_rng([hq, p, len(new)])
    _attend(dev, rng, lengths, new, hq, heads, p, d, DT[dtype])


@pytest.mark.parametrize("hq,heads,nodes", [(2, 2, 5), (4, 2, 16), (2, 1, 30), (4, 1, 64)])
@pytest.mark.parametrize("lengths,max_len", [([5000], None), ([5000, 90, 2049], 5000), ([5000, 1200], 700), ([4099], 1)])
def test_tree_split(dev, hq, heads, nodes, lengths, max_len):
    rng = np.random.default_rng(nodes)
    _attend(dev, rng, lengths, [nodes] * len(lengths), hq, heads, 16, 128, torch.float16, max_len=max_len)
    _attend(dev, rng, lengths, [nodes] * len(lengths), hq, heads, 64, 64, torch.bfloat16, max_len=max_len)


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("hq,heads,p,d", [(1, 1, 16, 128), (4, 2, 64, 64), (4, 1, 16, 128), (10, 2, 128, 64), (21, 7, 32, 128)])
@pytest.mark.parametrize("lengths,new", [([3000, 900, 70, 1500, 5000], [64, 33, 17, 48, 21]), ([64, 1025, 2112], [64, 1, 50]),
                                         ([40] * 40 + [2000], [34] * 40 + [43])])
def test_tree_uneven_batches(dev, dtype, hq, heads, p, d, lengths, new):
    """Work dealt out over sequences of very unequal lengths and tiles of unequal rows."""
    _attend(dev, np.random.default_rng([hq, len(new)]), lengths, new, hq, heads, p, d, DT[dtype])


@pytest.mark.parametrize("rows", [65, 130])
def test_tree_of_many_sequences(dev, rows):
    """More work-groups than begin at once: the longest sequences' first, of each 64; equal ones, empty ones, slots out of range."""
    rng = np.random.default_rng(rows)
    lengths = rng.choice([34, 40, 41, 90, 130], rows + 3).tolist()
    lengths[3] = lengths[70 % rows] = 0
    slots = rng.permutation(rows + 3)[:rows].tolist()
    slots[5], slots[rows - 1] = -1, rows + 3
    raw, sc, table, pages, scales, tab = _cache(rng, dev, lengths, 10, 16, 64, poison=True)
    new = rng.choice([33, 34], rows).tolist()
    cu = _cu(new)
    parents = [x for n in new for x in _parents(rng, n)]
    q = torch.randn(cu[-1], 10, 64, device=dev).half()
    with np.errstate(invalid="ignore"):
        ref = dft.tree_attention(q.double().cpu().numpy(), parents, orc.Layer(raw, sc), table, np.array(lengths), cu, slots)
    got, lse = bsa.kv_tree_attention(q, _i32(parents, dev), pages, scales, tab, _i32(lengths, dev), cu_seqlens=_i32(cu, dev),
                                     max_new=34, slots=_i32(slots, dev))
    _check_attention(got, lse, ref, torch.float16, 64)


@pytest.mark.parametrize("nodes,hq", [(9, 2), (30, 2), (40, 4)])
def test_tree_odd_parents_and_slots(dev, nodes, hq):
    """Parents that are no earlier node make roots; slots out of range and trees of more nodes than the sequence has
    tokens; sequences without tokens."""
    rng = np.random.default_rng(nodes)
    lengths, slots = [60, 0, nodes - 2, 200], [3, 17, 2, -1, 0, 1]
    raw, sc, table, pages, scales, tab = _cache(rng, dev, lengths, 2, 16, 64, poison=True)
    new = [nodes, 3, nodes, 2, 0, 4]
    cu = _cu(new)
    parents = rng.integers(-3, nodes + 3, cu[-1]).tolist()
    parents[1], parents[2] = 1, 2 ** 31 - 1
    q = torch.randn(cu[-1] + 2, 2 * hq, 64, device=dev).bfloat16()
    out = torch.full_like(q, 5.0)
    with np.errstate(invalid="ignore"):
        ref = dft.tree_attention(q[:cu[-1]].double().cpu().numpy(), parents, orc.Layer(raw, sc), table, np.array(lengths), cu, slots)
    got, lse = bsa.kv_tree_attention(q, _i32(parents + [0, 0], dev), pages, scales, tab, _i32(lengths, dev), cu_seqlens=_i32(cu, dev),
                                     max_new=nodes, slots=_i32(slots, dev), out=out)
    assert (got[cu[-1]:] == 5.0).all()
    _check_attention(got[:cu[-1]], lse[:cu[-1]], ref, torch.bfloat16, 64)


@pytest.mark.parametrize("nodes,hq", [(5, 2), (20, 4), (64, 2)])
def test_tree_nan_in_unseen_nodes(dev, nodes, hq):
    """A NaN of a node reaches its descendants and nobody else; pages out of range are not seen."""
    rng = np.random.default_rng(nodes)
    p, d, length = 16, 64, 150
    raw, sc, table, pages, scales, tab = _cache(rng, dev, [length], 1, p, d)
    parents = _parents(rng, nodes)
    at_v, at_k = length - nodes + nodes // 2, length - 1
    raw[table[0, at_v // p], 0, 1].reshape(-1)[orc.value_offset(at_v % p, 7, d)] = 0xFF
    raw[table[0, at_k // p], 0, 0].reshape(-1)[orc.key_offset(at_k % p, 3, d)] = 0x7F
    table[0, 1], table[0, 3] = -1, 10 ** 8
    q = torch.randn(nodes, hq, d, device=dev).half()
    with np.errstate(invalid="ignore"):
        ref = dft.tree_attention(q.double().cpu().numpy(), parents, orc.Layer(raw, sc), table, np.array([length]), [0, nodes])
    out, lse = bsa.kv_tree_attention(q, _i32(parents, dev), torch.from_numpy(raw).to(dev).view(F8), scales, _i32(table, dev), _i32([length], dev))
    bad = np.isnan(ref[1])
    assert bad[-1].all() and not bad.all() and np.isnan(ref[0][nodes // 2, :, 7]).all()
    assert np.isnan(lse.cpu().numpy()[bad]).all()
    _check_attention(out, torch.where(torch.from_numpy(bad).to(dev), 0.0, lse), (ref[0], np.where(bad, 0.0, ref[1]), *[np.nan_to_num(x) for x in ref[2:]]),
                     torch.float16, d)


def test_tree_graph_streams_and_threads(dev):
    """Split trees: the same numbers eager, replayed, on streams and from threads side by side."""
    rng = np.random.default_rng(2)
    raw, sc, table, pages, scales, tab = _cache(rng, dev, [3000, 1900], 2, 16, 128)
    n = _i32([3000, 1900], dev)
    for nodes in (8, 24, 60):
        q = torch.randn(2 * nodes, 4, 128, device=dev).bfloat16()
        parents = _i32(_parents(rng, nodes) + _parents(rng, nodes), dev)
        want, want_l = (x.clone() for x in bsa.kv_tree_attention(q, parents, pages, scales, tab, n))
        torch.cuda.synchronize()
        graphs = []
        for _ in range(2):
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                graphs.append((graph, *bsa.kv_tree_attention(q, parents, pages, scales, tab, n)))
        for _ in range(3):
            for g, out, lse in graphs:
                out.fill_(float("nan"))
                g.replay()
            eager = bsa.kv_tree_attention(q, parents, pages, scales, tab, n)
            torch.cuda.synchronize()
            for _, out, lse in [*graphs, (None, *eager)]:
                assert torch.equal(out, want) and torch.equal(lse, want_l)
        got = []

        def run():
            with torch.cuda.stream(torch.cuda.Stream()):
                got.append(bsa.kv_tree_attention(q, parents, pages, scales, tab, n))
                torch.cuda.current_stream().synchronize()

        threads = [threading.Thread(target=run) for _ in range(3)]
        [t.start() for t in threads]
        [t.join() for t in threads]
        assert len(got) == 3 and all(torch.equal(o, want) and torch.equal(l, want_l) for o, l in got)


# ---- hard scores, at 16 and 32 rows of a cached head (one kernel), and at 50 (small tiles), 120 (a large one) and 192 (a large
# and a small one) of the other: by max_len in parts, which are joined, and a work-group for each

HARD_TREES = [(8, 4), (16, 4), (50, 2), (60, 4), (64, 6)]  # nodes, query heads over two cached ones
CUTS = (None, 500)


def _hard(dev, rng, raw, sc, table, lengths, nodes, hq, dtype, d, q=None, **kw):
    """Both cuts against the oracle, whose answer for q is returned with theirs."""
    cu = [i * nodes for i in range(len(lengths) + 1)]
    parents = [x for _ in lengths for x in _parents(rng, nodes)]
    if q is None:
        q = torch.from_numpy(rng.standard_normal((cu[-1], hq, d)).astype(np.float32)).to(DT[dtype]).to(dev)
    with np.errstate(over="ignore"):
        ref = dft.tree_attention(q.double().cpu().numpy(), parents, orc.Layer(raw, sc), table, np.array(lengths), cu, **kw)
    for max_len in CUTS:
        yield ref, bsa.kv_tree_attention(q, _i32(parents, dev), torch.from_numpy(raw).to(dev).view(F8), torch.from_numpy(sc).to(dev),
                                         _i32(table, dev), _i32(lengths, dev), max_len=max_len, **kw)


@pytest.mark.parametrize("nodes,hq", HARD_TREES)
@pytest.mark.parametrize("kind", ["keys_grow", "keys_shrink", "sink", "value_scales", "values_grow", "values_shrink", "uneven"])
def test_tree_maximum_moves(dev, kind, nodes, hq):
    """Scores and value scales that outgrow, late and by many octaves, what was the maximum at first, or never come near it
    again: within a part, between the halves of a small tile's steps, and from part to part."""
    rng = np.random.default_rng([len(kind), nodes])
    p, d, lengths = 16, 64, [2200, 700]
    raw, sc, table, *_ = _cache(rng, dev, lengths, 2, p, d)
    for row, n in enumerate(lengths):
        ids, at = table[row, : -(-n // p)], np.arange(-(-n // p))[:, None]
        if kind == "keys_grow":
            sc[ids, :, 0] = 2.0 ** (at * 8 // len(at) - 8)
        elif kind == "keys_shrink":
            sc[ids, :, 0] = 2.0 ** (-1 - at * 8 // len(at))
        elif kind == "sink":
            sc[ids[:1], :, 0] = 1.0
        elif kind in ("value_scales", "uneven"):
            sc[ids, :, 1] = 2.0 ** rng.integers(-38, 20, (len(ids), 2))
            if kind == "uneven":
                sc[ids, :, 0] = 2.0 ** rng.integers(-12, -4, (len(ids), 2))
        else:
            steps = at * 40 // len(at) - 20
            sc[ids, :, 1] = 2.0 ** (steps if kind == "values_grow" else -steps)
    for dtype in ("fp16", "bf16"):
        for ref, (out, lse) in _hard(dev, rng, raw, sc, table, lengths, nodes, hq, dtype, d):
            if dtype == "fp16":
                # Outputs past its range are infinite, and what lies within its error of that, from either side, may be: an output's
                # is _check_attention's, the weights' 2^-11 of the magnitudes that it is the sum of, which are up to 2^8 times the
                # output's (1.7e7 for one of 64358: an error of up to 12336), and half a step of its own.
                o, _, mag, dots, vmax, count = ref
                eps = (d + 8) * 2.0 ** -24 * dots + 2.0 ** -20
                off = 2.0 ** -11 * np.abs(o) + (2.0 ** -11 + 2 * eps[..., None]) * mag + (count * vmax * 2.0 ** -38)[..., None] + 2.0 ** -24
                past, sure = np.abs(o) + off >= 65520, np.abs(o) - off >= 65520
                assert (out.double().cpu().numpy()[sure] == np.copysign(np.inf, ref[0][sure])).all()
                out = torch.where(torch.from_numpy(past).to(dev), 0, out)
                ref = (np.where(past, 0.0, ref[0]), *ref[1:])
            _check_attention(out, lse, ref, DT[dtype], d)


@pytest.mark.parametrize("nodes,hq", HARD_TREES)
@pytest.mark.parametrize("sm_scale", [-0.125, -1.0, 0.0, -0.0, 1e-30, -1e-30, 2.0])
def test_tree_scales_of_any_sign(dev, sm_scale, nodes, hq):
    rng = np.random.default_rng(nodes)
    lengths = [1500, 70]
    raw, sc, table, *_ = _cache(rng, dev, lengths, 2, 32, 64, poison=True)
    for dtype in ("fp16", "bf16"):
        for ref, (out, lse) in _hard(dev, rng, raw, sc, table, lengths, nodes, hq, dtype, 64, sm_scale=sm_scale):
            _check_attention(out, lse, ref, DT[dtype], 64)


@pytest.mark.parametrize("nodes,hq", HARD_TREES)
@pytest.mark.parametrize("octaves", [10, 20, 24, 26, 27, 28, 30, 40, 70])
def test_tree_far_scores(dev, octaves, nodes, hq):
    """Scores of up to 2^octaves that differ by as much, as test_attention_far_scores: the values of the largest are averaged, the
    products of small integers are exact, and outputs and lse carry a few roundings."""
    rng = np.random.default_rng([octaves, nodes])
    p, d, lengths = 16, 64, [1300, 70]
    raw, sc, table, *_ = _cache(rng, dev, lengths, 2, p, d)
    raw[:, :, 0] = torch.from_numpy(rng.integers(-1, 2, raw[:, :, 0].shape).astype(np.float32)).to(F8).view(torch.uint8).numpy()
    sc[..., 0], sc[..., 1] = 2.0 ** octaves, 0.125
    for dtype in ("fp16", "bf16"):
        q = torch.from_numpy(rng.integers(-2, 3, (2 * nodes, hq, d)).astype(np.float32)).to(DT[dtype]).to(dev)
        u = 2.0 ** -10 if dtype == "fp16" else 2.0 ** -7
        for (o, l, *_), (out, lse) in _hard(dev, rng, raw, sc, table, lengths, nodes, hq, dtype, d, q, sm_scale=0.25):
            assert (np.abs(out.double().cpu().numpy() - o) <= u * np.abs(o) + 2.0 ** -10).all()
            assert (np.abs(lse.double().cpu().numpy() - l) <= 2.0 ** -21 * np.abs(l)).all()


@pytest.mark.parametrize("nodes,hq", HARD_TREES)
@pytest.mark.parametrize("octaves", [4, 8, 10, 12, 14, 16, 17, 18])
def test_tree_equal_scores_weigh_the_same(dev, octaves, nodes, hq):
    """Every token has the same key, so that a row's scores, however far from 0, are one number, and its output is the mean of what it
    sees: weights that are off by their rounding to fp16, 2^-11, and by at most 2^-13 of each other before."""
    rng = np.random.default_rng([octaves, nodes])
    p, d, lengths = 16, 64, [2200, 700]
    raw, sc, table, *_ = _cache(rng, dev, lengths, 2, p, d)
    key = torch.from_numpy(rng.integers(-2, 3, d).astype(np.float32)).to(F8).view(torch.uint8).numpy()
    one = np.zeros(p * d, np.uint8)
    for t in range(p):
        one[[orc.key_offset(t, x, d) for x in range(d)]] = key
    raw[:, :, 0] = one.reshape(p, d)
    sc[..., 0], sc[..., 1] = 2.0 ** octaves, 0.125
    for dtype in ("fp16", "bf16"):
        q = torch.from_numpy(rng.integers(-2, 3, (2 * nodes, hq, d)).astype(np.float32)).to(DT[dtype]).to(dev)
        u = 2.0 ** -11 if dtype == "fp16" else 2.0 ** -8
        for (o, l, mag, *_), (out, lse) in _hard(dev, rng, raw, sc, table, lengths, nodes, hq, dtype, d, q, sm_scale=0.25):
            bound = u * np.abs(o) + (2.0 ** -11 + 2.0 ** -13) * mag + 2.0 ** -20
            assert (np.abs(out.double().cpu().numpy() - o) <= bound).all()
            assert (np.abs(lse.double().cpu().numpy() - l) <= 2.0 ** -21 * np.abs(l) + 2.0 ** -10).all()


@pytest.mark.parametrize("nodes,hq", HARD_TREES)
def test_tree_scores_of_minus_infinity_first(dev, nodes, hq):
    """The first 600 tokens' scores pass the end of 32 bits, whole parts of them: the later ones are seen as if alone."""
    rng = np.random.default_rng(nodes)
    p, d, length, first = 16, 64, 1100, 600
    raw, sc, table, *_ = _cache(rng, dev, [length], 2, p, d)
    sc[:] = 1.0
    minus = torch.tensor([-448.0, -8.0]).to(F8).view(torch.uint8).numpy()
    for t in range(length):
        for h in range(2):
            tile = raw[table[0, t // p], h, 0].reshape(-1)
            for x in range(d):
                tile[orc.key_offset(t % p, x, d)] = 0
            tile[orc.key_offset(t % p, 0, d)] = minus[0] if t < first else 0
            tile[orc.key_offset(t % p, 1, d)] = minus[1]
    q = torch.zeros(nodes, hq, d)
    q[..., 0], q[..., 1] = 1e38, 128
    for ref, (out, lse) in _hard(dev, rng, raw, sc, table, [length], nodes, hq, "bf16", d, q.bfloat16().to(dev)):
        assert (ref[1] >= np.log(length - first - nodes + 1) - 128 - 1e-9).all() and (ref[1] <= np.log(length - first) - 128 + 1e-9).all()
        _check_attention(out, lse, (*ref[:3], np.full_like(ref[3], 128.0), *ref[4:]), torch.bfloat16, d)


@pytest.mark.parametrize("hq,p,d", [(2, 16, 64), (8, 64, 128), (10, 16, 64)])
def test_tree_parts_of_sequences_that_take_no_part(dev, hq, p, d):
    """Work dealt out in parts over slots in any order, some of them out of range, sequences without tokens, shorter than their
    trees or empty, before, between and after long ones."""
    rng = np.random.default_rng(hq)
    lengths = [1500, 0, 2500, 30, 700, 64, 1100]
    slots, new = [9, 2, 1, -1, 6, 3, 0, 5, 4, 7], [50, 40, 33, 64, 0, 45, 37, 64, 0, 48]
    raw, sc, table, pages, scales, tab = _cache(rng, dev, lengths, 2, p, d, poison=True)
    cu, parents = _cu(new), [x for n in new if n for x in _parents(rng, n)]
    q = torch.from_numpy(rng.standard_normal((cu[-1], hq, d)).astype(np.float32)).bfloat16().to(dev)
    with np.errstate(invalid="ignore"):
        ref = dft.tree_attention(q.double().cpu().numpy(), parents, orc.Layer(raw, sc), table, np.array(lengths), cu, slots)
    for max_len in CUTS:
        out, lse = bsa.kv_tree_attention(q, _i32(parents, dev), pages, scales, tab, _i32(lengths, dev), cu_seqlens=_i32(cu, dev), max_new=64,
                                         slots=_i32(slots, dev), max_len=max_len)
        _check_attention(out, lse, ref, torch.bfloat16, d)


@pytest.mark.parametrize("nodes,hq", HARD_TREES)
def test_tree_queries_that_are_not_numbers(dev, nodes, hq):
    """A NaN or an infinity in a query makes its own row NaN and leaves the others what they are."""
    rng = np.random.default_rng(nodes)
    p, d, lengths = 16, 64, [1500, 90]
    raw, sc, table, *_ = _cache(rng, dev, lengths, 2, p, d, poison=True)
    q = torch.from_numpy(rng.standard_normal((2 * nodes, hq, d)).astype(np.float32)).half().to(dev)
    bad = torch.zeros(q.shape[:2], dtype=torch.bool, device=dev)
    for t, h, x in ((0, 0, float("nan")), (nodes // 2, hq - 1, float("inf")), (nodes, 1, float("-inf")), (2 * nodes - 1, hq // 2, float("nan"))):
        q[t, h, 7 + t % 5], bad[t, h] = x, True
    plain = torch.where(bad[..., None], torch.zeros_like(q), q)
    parents = [x for _ in lengths for x in _parents(rng, nodes)]
    ref = dft.tree_attention(plain.double().cpu().numpy(), parents, orc.Layer(raw, sc), table, np.array(lengths), [0, nodes, 2 * nodes])
    for max_len in CUTS:
        out, lse = bsa.kv_tree_attention(q, _i32(parents, dev), torch.from_numpy(raw).to(dev).view(F8), torch.from_numpy(sc).to(dev),
                                         _i32(table, dev), _i32(lengths, dev), max_len=max_len)
        assert torch.isnan(out[bad]).all() and torch.isnan(lse[bad]).all()
        zero = bad.cpu().numpy()  # whose reference is that of a row of zeros
        masked = [np.where(zero.reshape(zero.shape + (1,) * (x.ndim - 2)), 0.0, x) for x in ref]
        _check_attention(out.masked_fill(bad[..., None], 0.0), lse.masked_fill(bad, 0.0), masked, torch.float16, d)


@pytest.mark.parametrize("hq", [2, 4, 16])
def test_tree_max_new_bounds_the_rows(dev, hq):
    """The nodes past max_new are not computed; the others see what they do in the whole tree."""
    rng = np.random.default_rng(hq)
    new, lengths, most = [20, 9, 12], [150, 900, 12], 11
    raw, sc, table, pages, scales, tab = _cache(rng, dev, lengths, 2, 16, 64, poison=True)
    cu, parents = _cu(new), [x for n in new for x in _parents(rng, n)]
    q = torch.from_numpy(rng.standard_normal((cu[-1], hq, 64)).astype(np.float32)).half().to(dev)
    ref = dft.tree_attention(q.double().cpu().numpy(), parents, orc.Layer(raw, sc), table, np.array(lengths), cu)
    rows = np.concatenate([np.arange(a, min(b, a + most)) for a, b in zip(cu, cu[1:])])
    rest = np.setdiff1d(np.arange(cu[-1]), rows)
    for max_len in CUTS:
        out, lse = torch.full_like(q, 7.0), torch.full(q.shape[:2], 7.0, device=dev)
        bsa.kv_tree_attention(q, _i32(parents, dev), pages, scales, tab, _i32(lengths, dev), cu_seqlens=_i32(cu, dev), max_new=most,
                              max_len=max_len, out=out, lse=lse)
        assert (out[rest] == 7.0).all() and (lse[rest] == 7.0).all() and len(rest) == 10
        _check_attention(out[rows], lse[rows], [x[rows] for x in ref], torch.float16, 64)


# ---------------------------------------------------------------------------------------- verification


def _same_verdict(got, want, most):
    accepted, path, tokens = (x.cpu().tolist() for x in got)
    for b, (count, nodes, said) in enumerate(want):
        assert accepted[b] == count, (b, accepted[b], count)
        assert path[b] == nodes + [-1] * (most - len(nodes)), b
        assert tokens[b] == said + [-1] * (most - len(said)), (b, tokens[b], said)


def _drafts(rng, new, vocab, tree, spread=2.0):
    """Logits with a few likely tokens, trees of them, numbers."""
    total = sum(new)
    x = rng.standard_normal((total, vocab)) * spread
    for _ in range(2):
        x[np.arange(total), rng.integers(0, vocab, total)] += 8.0
    parents = [p for n in new for p in (_parents(rng, n) if tree else _parents(rng, n, "chain"))]
    tokens = rng.integers(0, vocab, total)
    at = 0
    for n in new:
        for i in range(1, n):
            p = dft.tree_parent(parents[at:at + n], i)
            if p >= 0 and rng.random() < 0.8:
                tokens[at + i] = np.argsort(-x[at + p])[min(rng.integers(0, 3), vocab - 1)]
        at += n
    return x, parents, tokens, rng.random(total).astype(np.float32)


@pytest.mark.parametrize("dtype", ["fp16", "bf16", "fp32"])
@pytest.mark.parametrize("vocab", [1, 2, 33, 500, 2048, 2049, 5003, 32000])
@pytest.mark.parametrize("temperature", [0.0, 0.3, 1.0])
def test_verify_trees(dev, dtype, vocab, temperature):
    rng = np.random.default_rng([vocab, int(10 * temperature)])
    new = [1, 2, 5, 16, 3, 9] + ([64] if vocab < 6000 else [])
    x, parents, tokens, u = _drafts(rng, new, vocab, True)
    logits = torch.from_numpy(x.astype(np.float32)).to(DT[dtype]).to(dev)
    want = dft.verify(logits.double().cpu().numpy(), tokens, u, parents, None, temperature, _cu(new))
    got = bsa.verify_drafts(logits, _i32(tokens, dev), torch.from_numpy(u).to(dev), parents=_i32(parents, dev), temperature=temperature,
                            cu_seqlens=_i32(_cu(new), dev), max_new=max(new))
    _same_verdict(got, want, max(new))


@pytest.mark.parametrize("dtype", ["fp16", "bf16", "fp32"])
@pytest.mark.parametrize("vocab", [2, 33, 2048, 5003, 32000])
@pytest.mark.parametrize("temperature", [0.0, 0.6, 1.0])
@pytest.mark.parametrize("noise", [0.0, 0.5, 3.0])
def test_verify_chains_of_drawn_drafts(dev, dtype, vocab, temperature, noise):
    rng = np.random.default_rng([vocab, int(10 * temperature), int(10 * noise)])
    new = [1, 2, 5, 8, 3, 12]
    x, _, tokens, u = _drafts(rng, new, vocab, False)
    logits = torch.from_numpy(x.astype(np.float32)).to(DT[dtype]).to(dev)
    draft = (logits.float() + noise * torch.from_numpy(rng.standard_normal(x.shape).astype(np.float32)).to(dev)).to(DT[dtype])
    want = dft.verify(logits.double().cpu().numpy(), tokens, u, None, draft.double().cpu().numpy(), temperature, _cu(new))
    got = bsa.verify_drafts(logits, _i32(tokens, dev), torch.from_numpy(u).to(dev), draft_logits=draft, temperature=temperature,
                            cu_seqlens=_i32(_cu(new), dev), max_new=12)
    _same_verdict(got, want, 12)
    if noise == 0 and temperature > 0:  # what the target would have drawn is accepted whatever the number
        assert [w[0] for w in want] == new


@pytest.mark.parametrize("draft", [False, True])
@pytest.mark.parametrize("vocab", [40, 5000])
def test_verify_hard_rows(dev, vocab, draft):
    """Masks, infinities and NaN in rows; tokens that do not exist, twice the same token among siblings, numbers at the
    ends of their range; a temperature for each sequence; sequences without nodes."""
    rng = np.random.default_rng([vocab, draft])
    new = [4, 4, 4, 4, 4, 4, 0, 4, 5, 5, 3]
    cu = _cu(new)
    x, _, tokens, u = _drafts(rng, new, vocab, False)
    parents = [p for n in new for p in ([i - 1 for i in range(n)] if draft else ([-1] + [0] * n)[:n])]
    x[cu[0]] = -np.inf                             # nothing
    x[cu[1], 3] = np.nan
    x[cu[2], 5] = np.inf
    x[cu[3]] = -np.inf
    x[cu[3], 7] = 2.0                              # one token only
    tokens[cu[3] + 1] = 7
    x[cu[4]] = np.where(np.arange(vocab) % 3 == 0, x[cu[4]], -np.inf)
    x[cu[5]] = np.where(np.arange(vocab) % 3 == 0, x[cu[5]], -6e4)
    tokens[cu[7] + 1], tokens[cu[7] + 2] = -1, vocab
    tokens[cu[8] + 1:cu[8] + 5] = int(np.argmax(x[cu[8]]))  # siblings of the same token
    u[cu[8] + 1], u[cu[8] + 2] = 1 - 2.0 ** -24, 0.0
    x[cu[9]] = 0.0                                 # every token alike; the last of them, or the first
    u[cu[9]] = 1 - 2.0 ** -24
    x[cu[10]], u[cu[10]] = 0.0, 0.0
    tokens[cu[10] + 1:] = vocab + 3
    temperature = np.array([1, 1, 1, 0.5, 1, 2, 1, 0.01, 1, 1, -1], np.float32)
    logits = torch.from_numpy(x.astype(np.float32)).to(dev)
    drafted = None
    if draft:
        d = x + 0.5 * rng.standard_normal(x.shape)
        d[cu[5]] = np.nan
        d[cu[9], : vocab // 2] = -np.inf
        drafted = torch.from_numpy(d.astype(np.float32)).to(dev)
    with np.errstate(invalid="ignore"):
        want = dft.verify(logits.double().cpu().numpy(), tokens, u, None if draft else parents,
                          None if drafted is None else drafted.double().cpu().numpy(), temperature, cu)
    got = bsa.verify_drafts(logits, _i32(tokens, dev), torch.from_numpy(u).to(dev), None if draft else _i32(parents, dev), drafted,
                            torch.from_numpy(temperature).to(dev), _i32(cu, dev), 5)
    _same_verdict(got, want, 5)
    assert [w[2][-1] for w in want[:3]] == [-1, -1, -1] and want[6] == (0, [], [])


@pytest.mark.parametrize("dtype", ["fp16", "bf16", "fp32"])
@pytest.mark.parametrize("draft", [False, True])
@pytest.mark.parametrize("each", [False, True])
def test_verify_temperatures_without_end(dev, dtype, draft, each):
    """From the least to infinity, where every token that has a finite logit is as likely; among them -inf."""
    rng = np.random.default_rng(12)
    temps = np.array([1e-45, 1e-38, 1e-30, 1e-3, 1e3, 1e30, 3.4e38, np.inf], np.float32)
    new = [4] * len(temps)
    x, _, tokens, u = _drafts(rng, new, 700, False)
    x[:, ::5] = -np.inf
    for i, t in enumerate(tokens):  # some of which are likely
        if i % 4:
            x[i - 1, t] = np.nanmax(x[i - 1]) + 0.25 * (i % 2)
    logits = torch.from_numpy(x).to(DT[dtype] if dtype != "fp32" else torch.float32).to(dev)
    drafted = logits.roll(1, 1).contiguous() if draft else None
    args = (logits.double().cpu().numpy(), tokens, u, None, None if drafted is None else drafted.double().cpu().numpy())
    exact = np.where(np.isinf(temps), 1e300, np.maximum(temps.astype(np.float64), 2.0 ** -126))
    with np.errstate(all="ignore"):
        want = dft.verify(*args, exact, _cu(new))
    ids, nums, cu = _i32(tokens, dev), torch.from_numpy(u).to(dev), _i32(_cu(new), dev)
    if each:
        _same_verdict(bsa.verify_drafts(logits, ids, nums, None, drafted, torch.from_numpy(temps).to(dev), cu, 4), want, 4)
    else:
        for b, t in enumerate(temps[:-1]):  # as a number infinity is refused
            got = bsa.verify_drafts(logits, ids, nums, None, drafted, float(t), cu, 4)
            _same_verdict([y[b:b + 1] for y in got], want[b:b + 1], 4)


@pytest.mark.parametrize("dtype", ["fp16", "bf16", "fp32"])
def test_verify_ties_take_the_first(dev, dtype):
    rng = np.random.default_rng(1)
    x = rng.integers(0, 4, (24, 9000)).astype(np.float32)  # thousands of equal maxima
    x[:, :2300] = np.minimum(x[:, :2300], 2)
    logits = torch.from_numpy(x).to(DT[dtype]).to(dev)
    tokens = np.concatenate([[0], np.argmax(x, 1)[:-1]])
    tokens[10] += 1
    want = dft.verify(x, tokens, np.zeros(24), None, None, 0.0, [0, 8, 16, 24])
    got = bsa.verify_drafts(logits, _i32(tokens, dev), torch.zeros(24, device=dev), temperature=0.0, max_new=8)
    _same_verdict(got, want, 8)
    assert want[0][0] == 8 and want[1][0] == 2


@pytest.mark.parametrize("dtype", ["fp16", "bf16", "fp32"])
@pytest.mark.parametrize("vocab", [3, 2050, 40000])
@pytest.mark.parametrize("each", [False, True])
def test_verify_greedy_rows_without_probabilities(dev, dtype, vocab, each):
    """By a number and by sequences: rows of nothing but -inf, with NaN, with +inf, at the root, within the path and at its end;
    children of the first token, which a row of -inf has first."""
    rng = np.random.default_rng(vocab)
    new = [6, 6, 6, 6, 6, 1, 0, 20]
    cu = _cu(new)
    x = rng.standard_normal((cu[-1], vocab))
    parents = [i - 1 for _ in range(5) for i in range(6)] + [-1] + _parents(rng, 20)
    tokens = rng.integers(0, vocab, cu[-1])
    for b in range(5):
        for i in range(5):
            tokens[cu[b] + i + 1] = int(np.argmax(x[cu[b] + i].astype(np.float16)))
    for i in range(1, 20):
        p = dft.tree_parent(parents[cu[7]:], i)
        if p >= 0 and i % 3:
            tokens[cu[7] + i] = int(np.argmax(x[cu[7] + p].astype(np.float16)))
    x = x.astype(np.float16).astype(np.float64)
    x[cu[0]], tokens[cu[0] + 1] = -np.inf, 0
    x[cu[1] + 2], tokens[cu[1] + 3] = -np.inf, 0
    x[cu[2] + 5] = -np.inf
    x[cu[3] + 1, vocab // 2] = np.nan
    x[cu[4] + 5, vocab - 1] = np.inf
    logits = torch.from_numpy(x).to(DT[dtype] if dtype != "fp32" else torch.float32).to(dev)
    u = rng.random(cu[-1]).astype(np.float32)
    want = dft.verify(logits.double().cpu().numpy(), tokens, u, parents, None, 0.0, cu)
    t = torch.zeros(len(new), device=dev) if each else 0.0
    got = bsa.verify_drafts(logits, _i32(tokens, dev), torch.from_numpy(u).to(dev), _i32(parents, dev), None, t, _i32(cu, dev), 20)
    _same_verdict(got, want, 20)
    assert want[0][2] == [-1] and max(w[0] for w in want) >= (1 if dtype == "bf16" else 5)


@pytest.mark.parametrize("offset,width,dtype", [(0, 5010, "fp16"), (3, 5007, "bf16"), (1, 2500, "fp32"), (5, 40, "fp16")])
def test_verify_strided_logits(dev, offset, width, dtype):
    rng = np.random.default_rng(width)
    new = [6, 3, 11]
    x, parents, tokens, u = _drafts(rng, new, width, True)
    wide = torch.full((20, width + 13), float("nan"), device=dev, dtype=DT[dtype])
    logits = wide[:, offset:offset + width]
    logits.copy_(torch.from_numpy(x.astype(np.float32)))
    want = dft.verify(logits.double().cpu().numpy(), tokens, u, parents, None, 0.9, _cu(new))
    got = bsa.verify_drafts(logits, _i32(tokens, dev), torch.from_numpy(u).to(dev), _i32(parents, dev), None, 0.9, _i32(_cu(new), dev), 11)
    _same_verdict(got, want, 11)


@pytest.mark.parametrize("dtype", ["fp16", "bf16", "fp32"])
@pytest.mark.parametrize("vocab", [300, 5003, 32000])
def test_verify_numbers_next_to_their_border(dev, dtype, vocab):
    """The 32-bit number below a child's border accepts it, the one above does not, after none, one and two rejected
    siblings: no nearer than 2^-25 of it, and 64-bit sums tell them apart.  The new token's number likewise."""
    rng = np.random.default_rng(vocab)
    new = [4] * 12
    x, _, _, u = _drafts(rng, new, vocab, False)
    logits = torch.from_numpy(x.astype(np.float32)).to(DT[dtype]).to(dev)
    host = logits.double().cpu().numpy()
    tokens, parents = np.zeros(48, np.int64), [-1, 0, 0, 0] * 12
    for b in range(12):
        best = np.argsort(-host[4 * b], kind="stable")
        tokens[4 * b + 1:4 * b + 4] = best[[5, 2, 3]]
        p = np.exp(host[4 * b] - host[4 * b].max())
        p /= p.sum()
        u[4 * b + 1:4 * b + 4] = 1 - 2.0 ** -24
        asked, up = b % 3, b // 3 % 2 == 0
        border = p[tokens[4 * b + 1 + asked]] / (1 - sum(p[tokens[4 * b + 1 + i]] for i in range(asked)))
        near = np.float32(border)
        near = near if (float(near) >= border) == up else np.nextafter(near, np.float32(2 if up else 0))
        u[4 * b + 1 + asked] = near
        assert (float(near) < border) != up and abs(float(near) / border - 1) < 2.0 ** -22
        # the new token's, between two tokens of the tail of what is left of its row
        at = 4 * b + (0 if up else 1 + asked)
        q = np.exp(host[at] - host[at].max())
        if up:
            q[tokens[4 * b + 1:4 * b + 4]] = 0
        sums = np.cumsum(q) / q.sum()
        u[4 * b] = np.float32(sums[(7919 * b) % vocab])
        assert u[4 * b] < 1
    want = dft.verify(host, tokens, u, parents, None, 1.0, _cu(new))
    got = bsa.verify_drafts(logits, _i32(tokens, dev), torch.from_numpy(u).to(dev), _i32(parents, dev), max_new=4)
    _same_verdict(got, want, 4)
    assert [w[0] for w in want] == [1, 1, 1, 2, 2, 2] * 2


@pytest.mark.parametrize("dtype", ["fp16", "bf16", "fp32"])
@pytest.mark.parametrize("vocab", [40, 5003, 65529])
@pytest.mark.parametrize("offset,constant", [(0, 0), (1, 0), (0, 8), (3, -16)])
def test_verify_drafts_as_likely_leave_nothing(dev, dtype, vocab, offset, constant):
    """A draft whose probabilities are the target's own, of the same logits or of ones that differ by a constant, cut at other addresses:
    what a rejected token (which does not exist) leaves is nothing, and the new one is drawn from the target's row."""
    rng = np.random.default_rng([vocab, offset])
    new = [2, 3, 2, 4, 2, 2]
    cu = _cu(new)
    x = rng.integers(-40, 41, (cu[-1], vocab)) / 4.0  # exact, and so with the constant, in each type
    x[np.arange(cu[-1]), rng.integers(0, vocab, cu[-1])] = 14.0
    tokens, u = rng.integers(0, vocab, cu[-1]), rng.random(cu[-1]).astype(np.float32)
    for b, bad in enumerate([-1, vocab, -7, vocab + 1, 2 ** 31 - 1, -1]):
        tokens[cu[b] + 1 + (b % 2) * (new[b] > 2)] = bad
    logits = torch.from_numpy(x.astype(np.float32)).to(DT[dtype]).to(dev)
    draft = torch.zeros(cu[-1], vocab + 5, dtype=DT[dtype], device=dev)[:, offset:offset + vocab]
    draft.copy_(logits + constant)
    assert torch.equal(draft.double() - constant, logits.double())
    args = (logits, _i32(tokens, dev), torch.from_numpy(u).to(dev))
    temps = np.array([1, 0.5, 2, 1, 0.25, 1], np.float32)
    want = dft.verify(logits.double().cpu().numpy(), tokens, u, None, logits.double().cpu().numpy(), temps, cu)
    got = bsa.verify_drafts(*args, draft_logits=draft, temperature=torch.from_numpy(temps).to(dev), cu_seqlens=_i32(cu, dev), max_new=4)
    _same_verdict(got, want, 4)
    assert [w[0] for w in want] == [1, 2, 1, 2, 1, 1]


# ---- rows of more pieces (1024 logits each) than a wave has lanes: 64 up to 65529 logits, 65 from there on

LARGE = [65529, 65530, 131073, 2 ** 20]


@pytest.mark.parametrize("dtype", ["fp16", "bf16", "fp32"])
@pytest.mark.parametrize("vocab", LARGE)
@pytest.mark.parametrize("kind", ["trees", "drawn", "same"])
def test_verify_large_vocabularies(dev, dtype, vocab, kind):
    """Trees, chains of drawn drafts, and chains whose drafts have the target's own logits, of which nothing is left where a token is
    rejected because it does not exist.  New tokens from all over the rows: of the first and the last piece, of rows whose
    only weights lie at one end, of rows of few weights far apart."""
    rng = np.random.default_rng([vocab, len(kind)])
    new = [1, 5, 4, 3, 2, 2, 3]
    cu = _cu(new)
    x, parents, tokens, u = _drafts(rng, new, vocab, kind == "trees")
    u[cu[1]], u[cu[2]] = 1 - 2.0 ** -24, 2.0 ** -24
    x[cu[3]:cu[4], : vocab - 70] = -np.inf
    x[cu[4]:cu[5], 70:] = -np.inf
    x[cu[5]:cu[6]] = np.where(np.arange(vocab) % (vocab // 7) == 3, x[cu[5]:cu[6]], -np.inf)
    tokens[cu[5] + 1] = 3 + 4 * (vocab // 7)
    if kind != "drawn":
        tokens[cu[2] + 2], tokens[cu[6] + 1] = vocab, -1
    logits = torch.from_numpy(x.astype(np.float32)).to(DT[dtype]).to(dev)
    draft = None
    if kind != "trees":
        noise = torch.from_numpy(rng.standard_normal(x.shape).astype(np.float32)).to(dev)
        draft = logits.clone() if kind == "same" else (logits.float() + noise).to(DT[dtype])
    temps = np.array([1, 0.7, 1, 0.8, 1, 2, 0.9], np.float32)
    host = (logits.double().cpu().numpy(), tokens, u, parents if kind == "trees" else None, None if draft is None else draft.double().cpu().numpy())
    with np.errstate(invalid="ignore"):
        want = dft.verify(*host, temps, cu)
    got = bsa.verify_drafts(logits, _i32(tokens, dev), torch.from_numpy(u).to(dev), _i32(parents, dev) if kind == "trees" else None, draft,
                            torch.from_numpy(temps).to(dev), _i32(cu, dev), 5)
    _same_verdict(got, want, 5)
    assert all(w[2][-1] >= vocab - 70 for w in want[3:4]) and 0 <= want[4][2][-1] < 70
    if kind == "same":  # accepted but for what does not exist, or has no weight in its row (the fourth and fifth)
        assert [w[0] for w in want[:3] + want[5:]] == [1, 5, 2, 2, 1]


@pytest.mark.parametrize("dtype", ["fp16", "bf16", "fp32"])
@pytest.mark.parametrize("vocab", [65529, 65530, 131073])
def test_verify_large_vocabularies_next_to_their_border(dev, dtype, vocab):
    """What 32-bit sums do not decide is added again over all of a row's pieces."""
    test_verify_numbers_next_to_their_border(dev, dtype, vocab)


@pytest.mark.parametrize("draft", [False, True])
def test_verify_rows_past_four_gigabytes(dev, draft):
    """The last rows of 4.6 GB of logits, and sequences that begin there: what the same rows give by themselves."""
    count, vocab, new = 1100, 2 ** 20, [3, 5]
    g = torch.Generator(device=dev).manual_seed(5)
    big = [torch.empty(count, vocab, device=dev) for _ in range(1 + draft)]
    last = [torch.randn(8, vocab, generator=g, device=dev) for _ in big]
    for x, rows in zip(big, last):
        rows[torch.arange(8), torch.arange(8) * 100000 + 77] += 14.0
        x[-8:] = rows
    tokens, u = torch.zeros(count, dtype=torch.int32, device=dev), torch.rand(count, generator=g, device=dev)
    tokens[-7:] = torch.arange(7, device=dev, dtype=torch.int32) * 100000 + 77
    first = count - 8
    want = bsa.verify_drafts(last[0], tokens[-8:].contiguous(), u[-8:].contiguous(), draft_logits=last[1] if draft else None, cu_seqlens=_i32([0, 3, 8], dev),
                             max_new=5)
    got = bsa.verify_drafts(big[0], tokens, u, draft_logits=big[1] if draft else None, cu_seqlens=_i32([first, first + 3, count], dev), max_new=5)
    assert all(torch.equal(a, b) for a, b in zip(got, want)) and int(want.accepted.max()) > 1 and (want.tokens.gather(1, want.accepted.long()[:, None] - 1) >= 0).all()
    if not draft:
        host = dft.verify(last[0].double().cpu().numpy(), tokens[-8:].cpu().numpy(), u[-8:].cpu().numpy(), None, None, 1.0, [0, 3, 8])
        _same_verdict(got, host, 5)


@pytest.mark.parametrize("dtype", ["fp16", "bf16", "fp32"])
@pytest.mark.parametrize("vocab", [300, 5003, 65530])
def test_verify_drawn_numbers_next_to_their_border(dev, dtype, vocab):
    """Against a draft: the 32-bit number below p(x) / q(x) accepts the token, the one above does not; and numbers of the new token next
    to a running sum of what p has over q."""
    rng = np.random.default_rng(vocab)
    x, _, _, u = _drafts(rng, [2] * 12, vocab, False)
    logits = torch.from_numpy(x.astype(np.float32)).to(DT[dtype]).to(dev)
    draft = (logits.float() + torch.from_numpy(rng.standard_normal(x.shape).astype(np.float32)).to(dev)).to(DT[dtype])
    hosts = [t.double().cpu().numpy() for t in (logits, draft)]
    tokens = np.zeros(24, np.int64)
    for b in range(12):
        p, q = (np.exp(h[2 * b] - h[2 * b].max()) for h in hosts)
        p, q = p / p.sum(), q / q.sum()
        shy = np.flatnonzero((p < 0.9 * q) & (p > 1e-3 * q))  # what the draft likes more
        tokens[2 * b + 1] = shy[np.argsort(-q[shy])[b % 3]]
        border, above = (p / q)[tokens[2 * b + 1]], b % 2 == 0
        near = np.float32(border)
        near = near if (float(near) >= border) == above else np.nextafter(near, np.float32(2 if above else 0))
        u[2 * b + 1] = near
        assert (float(near) >= border) == above and abs(float(near) / border - 1) < 2.0 ** -22
        left = np.maximum(p - q, 0) if above else np.exp(hosts[0][2 * b + 1] - hosts[0][2 * b + 1].max())
        u[2 * b] = np.float32((np.cumsum(left) / left.sum())[(7919 * b) % vocab])
        u[2 * b] = min(u[2 * b], np.float32(1 - 2.0 ** -24))
    want = dft.verify(hosts[0], tokens, u, None, hosts[1], 1.0, _cu([2] * 12))
    got = bsa.verify_drafts(logits, _i32(tokens, dev), torch.from_numpy(u).to(dev), draft_logits=draft, max_new=2)
    _same_verdict(got, want, 2)
    assert [w[0] for w in want] == [1, 2] * 6


@pytest.mark.parametrize("vocab,gap", [(50, 24.0), (50, 27.0), (50, 30.0), (3001, 12.0), (3001, 17.0), (3001, 20.0)])
def test_verify_drafts_almost_as_likely(dev, vocab, gap):
    """Two rows with all but e^-gap or so of their weight on the same token, and rejected drafts (which do not exist): little is
    left, 1e-5 to 1e-14 of the row, and the new token is drawn from just that.  A p or q near 1 is off by a sum's, an inverse's and a
    product's rounding, 3 x 2^-53 each, here and in the oracle: what is left, and each of its running sums, by 12 x 2^-53 of
    the row.  The others' polynomials are off by 2^-45.6 of what is not on that token, which is some three times what is left: 2^-43
    of that.  Numbers as near as twice that to a border are drawn again."""
    rng = np.random.default_rng([vocab, int(gap)])
    rows = 64
    x = (-gap - np.log(vocab) + rng.standard_normal((2, 2 * rows, vocab))).astype(np.float32)
    x[:, np.arange(2 * rows), rng.integers(0, vocab, rows).repeat(2)] = 0.0
    tokens, u = np.full(2 * rows, -1), rng.random(2 * rows).astype(np.float32)
    for b in range(rows):
        p, q = (np.exp(r.astype(np.float64)) / np.exp(r.astype(np.float64)).sum() for r in x[:, 2 * b])
        sums = np.cumsum(np.maximum(p - q, 0))
        assert 1e-14 < sums[-1] < 1e-5
        while np.abs(sums / sums[-1] - u[2 * b]).min() < 2 * (12 * 2.0 ** -53 / sums[-1] + 2.0 ** -43):
            u[2 * b] = rng.random(dtype=np.float32)
    logits, draft = (torch.from_numpy(r).to(dev) for r in x)
    want = dft.verify(x[0].astype(np.float64), tokens, u, None, x[1].astype(np.float64), 1.0, _cu([2] * rows))
    got = bsa.verify_drafts(logits, _i32(tokens, dev), torch.from_numpy(u).to(dev), draft_logits=draft, max_new=2)
    _same_verdict(got, want, 2)
    assert all(w[0] == 1 for w in want)


@pytest.mark.parametrize("vocab,places", [(40, (4, 5, 6)), (40, (36, 37, 2)), (5004, (8, 9, 4801)), (5004, (4104, 4105, 30)), (70000, (12, 13, 69999))])
def test_verify_where_nothing_is_left(dev, vocab, places):
    """A row of three tokens of weights 1, 2^-23 and 2^-46, all of them drafted and asked with 1 - 2^-24.  The last one's border is 1,
    from which its number is 2^-70 of the row away: it may be accepted.  Where it is refused nothing is left of the row, and
    the new token is drawn from all of it."""
    numbers = [0.0, 0.5, 1 - 2.0 ** -22, 1 - 2.0 ** -24]
    x = np.full((4 * len(numbers), vocab), -np.inf, np.float32)
    x[:, list(places)] = [0.0, -15.942384719848633, -31.8847713470459]
    u = np.full(len(x), 1 - 2.0 ** -24, np.float32)
    u[::4] = numbers
    got = bsa.verify_drafts(torch.from_numpy(x).to(dev), _i32([0, *places] * len(numbers), dev), torch.from_numpy(u).to(dev),
                            _i32([-1, 0, 0, 0] * len(numbers), dev), max_new=4)
    sums = np.cumsum(np.exp(x[0].astype(np.float64)))
    for b, number in enumerate(numbers):
        drawn = int(np.argmax(sums > number * sums[-1]))
        if got.accepted[b] == 1:
            assert got.path[b].tolist() == [0, -1, -1, -1] and got.tokens[b].tolist() == [drawn, -1, -1, -1], (b, got)
        else:
            assert got.path[b].tolist() == [0, 3, -1, -1] and got.tokens[b].tolist() == [places[2], drawn, -1, -1], (b, got)


def test_verify_max_new_bounds_the_nodes(dev):
    rng = np.random.default_rng(4)
    new = [9, 2, 7]
    x, parents, tokens, u = _drafts(rng, new, 300, True)
    logits = torch.from_numpy(x).float().to(dev)
    want = dft.verify(logits.double().cpu().numpy(), tokens, u, parents, None, 1.0, _cu(new), max_new=4)
    got = bsa.verify_drafts(logits, _i32(tokens, dev), torch.from_numpy(u).to(dev), _i32(parents, dev), cu_seqlens=_i32(_cu(new), dev), max_new=4)
    _same_verdict(got, want, 4)


@pytest.mark.parametrize("new", [[5], [2, 0, 4], [0, 0, 0]])
@pytest.mark.parametrize("max_new,width", [(16, 16), (64, 64), (1000, 64), (5, 5), (3, 3), (1, 1), (0, 0)])
def test_verify_answers_are_as_wide_as_max_new(dev, new, max_new, width):
    """[sequences, max_new], also where a batch has fewer tokens than that, and at most 64 columns; without max_new a column a token."""
    rng = np.random.default_rng(max_new)
    total, cu = sum(new), _cu(new)
    x, parents, tokens, u = _drafts(rng, [n for n in new if n], 300, True) if total else (np.zeros((0, 300)), [], [], np.zeros(0, np.float32))
    logits = torch.from_numpy(x).float().to(dev)
    args = (logits, _i32(tokens, dev), torch.from_numpy(u).to(dev), _i32(parents, dev))
    used = [torch.full((len(new) * 64,), 9, dtype=torch.int32, device=dev) for _ in range(3)]
    del used  # memory that the answers are given holds something
    host = (logits.double().cpu().numpy(), tokens, u, parents, None, 1.0, cu)
    got = bsa.verify_drafts(*args, cu_seqlens=_i32(cu, dev), max_new=max_new)
    assert got.accepted.shape == (len(new),) and got.path.shape == got.tokens.shape == (len(new), width)
    _same_verdict(got, dft.verify(*host, max_new=max_new), width)
    got = bsa.verify_drafts(*args, cu_seqlens=_i32(cu, dev))
    assert got.path.shape == got.tokens.shape == (len(new), total)
    _same_verdict(got, dft.verify(*host), total)


@pytest.mark.parametrize("kind", ["drawn", "likeliest"])
def test_verify_leaves_the_targets_distribution(dev, kind):
    """The first token that comes out is distributed as the target's first row says, whatever was drafted: of 16000
    sequences each token's share is within 5 standard deviations."""
    g = torch.Generator(device=dev).manual_seed(9)
    rows, vocab = 16000, 11
    p = torch.randn(3, vocab, generator=g, device=dev)
    q = p + torch.randn(3, vocab, generator=g, device=dev)
    logits = p.repeat(rows, 1).contiguous()
    u = torch.rand(3 * rows, generator=g, device=dev)
    if kind == "drawn":
        first = torch.multinomial(q[0].softmax(0), rows, replacement=True, generator=g)
        second = torch.multinomial(q[1].softmax(0), rows, replacement=True, generator=g)
        got = bsa.verify_drafts(logits, torch.stack([torch.zeros_like(first), first, second], 1).reshape(-1).int(), u,
                                draft_logits=q.repeat(rows, 1).contiguous(), max_new=3)
    else:
        best = q[0].topk(2)[1]
        tokens = torch.stack([torch.zeros_like(best[0]), best[0], best[1]]).repeat(rows).int()
        got = bsa.verify_drafts(logits, tokens, u, parents=_i32([-1, 0, 0] * rows, dev), max_new=3)
    share = torch.bincount(got.tokens[:, 0].long(), minlength=vocab).double() / rows
    want = p[0].double().softmax(0)
    assert (got.accepted > 1).float().mean() > 0.2
    assert ((share - want).abs() <= 5 * (want * (1 - want) / rows).sqrt()).all()


@pytest.mark.parametrize("kind", ["trees", "drawn", "greedy"])
@pytest.mark.parametrize("vocab", [300, 32000])
def test_verify_leaves_sequences_out(dev, kind, vocab):
    """A slot below 0: nothing accepted, no path, no tokens, whatever the sequence's rows hold; the others as without it.
    Eager, of equal sequences without offsets, all left out, and captured with other slots at each replay."""
    rng = np.random.default_rng([vocab, len(kind)])
    new = [5, 3, 1, 0, 8, 5]
    x, parents, tokens, u = _drafts(rng, [n for n in new if n], vocab, kind == "trees")
    temperature = 0.0 if kind == "greedy" else 0.8
    logits = torch.from_numpy(x).half().to(dev)
    draft = (logits.float() + 0.5 * torch.randn(logits.shape, device=dev)).half() if kind == "drawn" else None
    par = _i32(parents, dev) if kind == "trees" else None
    ids, nums, cu = _i32(tokens, dev), torch.from_numpy(u).to(dev), _i32(_cu(new), dev)
    host = (logits.double().cpu().numpy(), tokens, u, parents if par is not None else None, None if draft is None else draft.double().cpu().numpy(),
            temperature)
    want = dft.verify(*host, _cu(new))
    left_out = (0, [], [])

    def expected(slots):
        return [w if s >= 0 else left_out for w, s in zip(want, slots)]

    def call(slots):
        return bsa.verify_drafts(logits, ids, nums, par, draft, temperature, cu, 8, slots=slots)

    first, last = [4, -1, -9, 0, 70000, -(2 ** 31)], [-1, 3, 2, -1, -1, 2 ** 31 - 1]
    kept = logits.clone()
    logits[5:9], logits[17:] = float("nan"), float("inf")  # of the ones that are left out at first
    for _ in range(2):
        _same_verdict(call(_i32(first, dev)), expected(first), 8)
    logits.copy_(kept)
    for slots in (last, [-1] * 6, [0] * 6):
        _same_verdict(call(_i32(slots, dev)), expected(slots), 8)
    _same_verdict(call(None), want, 8)
    # sequences of equally many tokens, the last one and the first one of which are left out
    each = torch.cat([torch.arange(5), torch.arange(9, 14), torch.arange(17, 22)]).to(dev)
    even = (logits[each], ids[each], nums[each], None if par is None else par[each], None if draft is None else draft[each], temperature)
    verdict = [want[0], None, want[5]]
    for slots in ([3, -1, -1], [-1, -1, 5]):
        got = bsa.verify_drafts(*even, max_new=5, slots=_i32(slots, dev))
        _same_verdict(got, [w if s >= 0 else left_out for w, s in zip(verdict, slots)], 5)
    held = _i32(first, dev)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call(held)
    for slots in (first, last, [-1] * 6, [1] * 6, first):
        held.copy_(_i32(slots, dev))
        [t.fill_(99) for t in out]
        graph.replay()
        eager = call(held)
        torch.cuda.synchronize()
        _same_verdict(out, expected(slots), 8)
        _same_verdict(eager, expected(slots), 8)
    for bad, error in ((held.long(), TypeError), (held[:5], ValueError), (held.cpu(), ValueError), (_i32([0] * 12, dev)[::2], ValueError)):
        with pytest.raises(error):
            call(bad)


def test_verify_graph_threads_and_prefix(dev):
    rng = np.random.default_rng(8)
    new = [5, 3, 8, 1]
    x, _, tokens, u = _drafts(rng, new, 32000, False)
    logits = torch.from_numpy(x).half().to(dev)
    draft = (logits.float() + 0.5 * torch.randn(logits.shape, device=dev)).half()
    ids, nums, cu = _i32(tokens, dev), torch.from_numpy(u).to(dev), _i32(_cu(new), dev)

    def call(prefix=None):
        return bsa.verify_drafts(logits, ids, nums, draft_logits=draft, cu_seqlens=cu, max_new=8, workspace_prefix=prefix)

    call("verify test")
    torch.cuda.synchronize()
    graphs = []
    for prefix in (None, None, "verify test"):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            graphs.append((graph, call(prefix)))
    for i in range(4):
        nums.copy_(torch.rand_like(nums))
        want = dft.verify(logits.double().cpu().numpy(), tokens, nums.cpu().numpy(), None, draft.double().cpu().numpy(), 1.0, _cu(new))
        for graph, out in graphs:
            for t in out:
                t.fill_(99)
            graph.replay()
        eager = call()
        torch.cuda.synchronize()
        for out in [eager] + [o for _, o in graphs]:
            _same_verdict(out, want, 8)
    got = []

    def run():
        for _ in range(5):
            got.append(call())

    threads = [threading.Thread(target=run) for _ in range(3)]
    [t.start() for t in threads]
    [t.join() for t in threads]
    torch.cuda.synchronize()
    assert len(got) == 15
    for out in got:
        _same_verdict(out, want, 8)


# ---------------------------------------------------------------------------------------- what stays


def _kept(dev, rng, lengths, news, path, accepted, p, d, heads=2, layers=2, slots=None, spread=4, shared=()):
    most = len(path[0])
    made = [_cache(np.random.default_rng([rng.integers(1 << 30), 0]), dev, lengths, heads, p, d) for _ in range(layers)]
    table = made[0][2]
    refs = np.zeros(made[0][0].shape[0], np.int64)
    for b, n in enumerate(lengths):
        for j in range(-(-n // p)):
            refs[table[b, j]] += 1
    for page in shared:
        refs[table[page]] += 1
    scs = [2.0 ** rng.integers(-6 - spread, -6 + spread, m[1].shape).astype(np.float32) for m in made]
    pages = torch.stack([torch.from_numpy(m[0]) for m in made]).to(dev).view(F8)
    scales = torch.from_numpy(np.stack(scs)).to(dev)
    pool = orc.Pool(table, lengths, refs, p)
    ref = [orc.Layer(m[0], s) for m, s in zip(made, scs)]
    dft.keep(ref, pool, path, accepted, news, slots)
    tab, n, r = _i32(table, dev), _i32(lengths, dev), _i32(refs, dev)
    cu = _i32(_cu(news), dev)
    bsa.pages_keep(pages, scales, tab, n, r, _i32(path, dev), _i32(accepted, dev), cu_seqlens=cu, slots=None if slots is None else _i32(slots, dev))
    assert tab.cpu().tolist() == pool.table and n.cpu().tolist() == pool.lengths and r.cpu().tolist() == pool.refs
    for i in range(layers):
        _same_pages(pages[i], scales[i], ref[i])
    del most


@pytest.mark.parametrize("p,d", [(16, 64), (16, 128), (32, 128), (64, 64), (128, 128)])
@pytest.mark.parametrize("nodes", [1, 2, 7, 20, 64])
def test_keep(dev, p, d, nodes):
    """Paths of every kind over pages whose scales differ by octaves: moves within a page and from page to page."""
    rng = np.random.default_rng([p, d, nodes])
    lengths = [nodes, nodes + 1, nodes + 14, 2 * nodes + 33, 200 + nodes]
    news = [nodes] * 5
    path, accepted = [], []
    for b in range(5):
        count = int(rng.integers(0, nodes + 1)) if b else nodes
        accepted.append(count)
        path.append(sorted(rng.choice(nodes, count, replace=False).tolist()) + [-1] * (nodes - count))
    _kept(dev, rng, lengths, news, path, accepted, p, d)


@pytest.mark.parametrize("spread", [1, 12])
def test_keep_scales_grow(dev, spread):
    """A page takes tokens of later pages of much larger, or smaller, scales."""
    rng = np.random.default_rng(spread)
    path = [[5, 20, 33, 40, 47] + [-1] * 43, list(range(0, 48, 2)) + [-1] * 24, [47] + [-1] * 47]
    _kept(dev, rng, [61, 62, 50], [48, 48, 48], path, [5, 24, 1], 16, 64, heads=5, layers=3, spread=spread)


def test_keep_odd_paths_and_slots(dev):
    """What does not ascend or exist ends a path; slots out of range and sequences shorter than their new tokens are
    left as they are; counts of pages that others read."""
    rng = np.random.default_rng(3)
    lengths = [40, 5, 33, 64, 18, 30, 20]
    path = [[0, 2, 2, 3], [0, 1, 2, 3], [1, 3, 9, 2], [-1, 2, 3, 1], [0, 1, 2, 3], [2, 3, 1, 0], [3, 4, 5, 6]]
    accepted = [4, 3, 4, 2, 9, -3, 4]
    news = [7, 8, 4, 5, 4, 4, 4]
    slots = [0, 1, 2, 3, 9, 5, 6]
    _kept(dev, rng, lengths, news, path, accepted, 16, 64, slots=slots, shared=[(2, 2), (0, 0)])
    _kept(dev, rng, lengths, [4] * 7, path, accepted, 16, 128, slots=[3, 2, 6, 0, 1, -1, 4])


def test_keep_nan_and_bad_pages(dev):
    rng = np.random.default_rng(4)
    raw, sc, table, pages, scales, tab = _cache(rng, dev, [40, 40], 1, 16, 64)
    at = orc.key_offset(38 % 16, 5, 64)
    raw[table[0, 38 // 16], 0, 0].reshape(-1)[at] = 0xFF
    sc[table[0, 2], 0, 0], sc[table[0, 1], 0, 0] = 2.0, 0.25
    table[1, 1] = 10 ** 7
    layer, pool = orc.Layer(raw, sc), orc.Pool(table, [40, 40], [1] * raw.shape[0], 16)
    path = [[0, 8, -1, -1], [2, 7, 8, -1]]
    dft.keep([layer], pool, path, [2, 3], [10, 10])
    pages, scales = torch.from_numpy(raw)[None].to(dev).view(F8), torch.from_numpy(sc)[None].to(dev)
    tab, n, refs = _i32(table, dev), _i32([40, 40], dev), torch.ones(raw.shape[0], dtype=torch.int32, device=dev)
    bsa.pages_keep(pages, scales, tab, n, refs, _i32(path, dev), _i32([2, 3], dev), cu_seqlens=_i32([0, 10, 20], dev))
    assert tab.cpu().tolist() == pool.table and refs.cpu().tolist() == pool.refs
    _same_pages(pages[0], scales[0], layer)


def test_keep_graph(dev):
    rng = np.random.default_rng(6)
    _, _, table, pages, scales, tab = _cache(rng, dev, [50, 23], 2, 16, 64)
    pages, scales = torch.stack([pages.view(torch.uint8)] * 2).view(F8), torch.stack([scales] * 2)
    n, refs = _i32([50, 23], dev), torch.ones(pages.shape[1], dtype=torch.int32, device=dev)
    path, accepted = _i32([[0, 3, 9, -1], [1, -1, -1, -1]], dev), _i32([3, 1], dev)
    cu = _i32([0, 12, 16], dev)
    state = (pages.view(torch.uint8), scales, tab, n, refs)
    before = [x.clone() for x in state]

    def reset():
        for x, was in zip(state, before):
            x.copy_(was)

    def call():
        bsa.pages_keep(pages, scales, tab, n, refs, path, accepted, cu_seqlens=cu)

    call()
    want = [x.clone() for x in state]
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    reset()
    with torch.cuda.graph(graph):
        call()
    for _ in range(3):
        reset()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(x, w) for x, w in zip(state, want))
    assert n.tolist() == [41, 20]


# ---------------------------------------------------------------------------------------- a run of them together


class _Toy:
    """Two layers of the operators in turn, as a decoder that drafts calls them: a step takes a tree of each sequence's, whose first
    node is its last token, and leaves the accepted nodes in the cache and the next last token."""

    def __init__(self, dev, rng, prompts, dtype, slots, page=16, vocab=9, max_new=14):
        self.dev, self.vocab, self.max_new, self.hq, self.heads, self.d = dev, vocab, max_new, 6, 2, 64
        self.cache = bsa.KVCache(2, 64, self.heads, self.d, page, 6, 12, dev)
        self.slots = _i32(slots, dev)

        def weight(k, n):
            return torch.from_numpy(rng.standard_normal((k, n)).astype(np.float32) * k ** -0.5).to(dev).to(dtype)

        self.embed = weight(1, 64).expand(vocab, 64) * 0.3 + torch.from_numpy(rng.standard_normal((vocab, 64)).astype(np.float32)).to(dev).to(dtype)
        self.qkv = [weight(64, (self.hq + 2 * self.heads) * self.d) for _ in range(2)]
        self.o = [weight(self.hq * self.d, 64) for _ in range(2)]
        self.head = weight(64, vocab)
        self.norms = [torch.from_numpy((1 + 0.1 * rng.standard_normal(self.d)).astype(np.float32)).to(dev).to(dtype) for _ in range(2)]
        self.angles = _angles(400, self.d)
        self.cos, self.sin = (torch.from_numpy(x).to(dev) for x in self.angles)
        flat = _i32([t for p in prompts for t in p], dev)
        cu = _i32(_cu([len(p) for p in prompts]), dev)
        assert bool(self.cache.extend(cu.diff().to(torch.int32), slots=self.slots).all())
        self.forward(flat, cu, max(map(len, prompts)), None)
        self.last = _i32([1] * len(prompts), dev)  # the prompts' continuation, not yet in the cache
        self.seen = [list(p) + [1] for p in prompts]

    def forward(self, tokens, cu, max_new, parents):
        x = self.embed[tokens.long()]
        batch = dict(cu_seqlens=cu, max_new=max_new, slots=self.slots)
        for i in range(2):
            qkv = (x @ self.qkv[i]).view(len(x), -1, self.d)
            q, k, v = qkv.split([self.hq, self.heads, self.heads], 1)
            q = self.cache.append_rotated(i, q, k, v, self.cos, self.sin, parents=parents, q_norm=self.norms[0], k_norm=self.norms[1], **batch)
            out, _ = self.cache.attend(i, q, **batch) if parents is None else self.cache.attend_tree(i, q, parents, **batch)
            x = x + out.view(len(x), -1) @ self.o[i]
        return x @ self.head

    def step(self, drafts, parents, cu, uniforms):
        """drafts has the trees' tokens but for the first ones."""
        first = cu[:-1].long()
        tokens = drafts.index_copy(0, first, self.last)
        self.cache.extend(cu.diff().to(torch.int32), slots=self.slots)
        logits = self.forward(tokens, cu, self.max_new, parents)
        got = bsa.verify_drafts(logits, tokens, uniforms, parents, temperature=0.7, cu_seqlens=cu, max_new=self.max_new)
        self.cache.keep(got.path, got.accepted, cu_seqlens=cu, slots=self.slots)
        self.last.copy_(got.tokens.gather(1, got.accepted.long()[:, None] - 1)[:, 0])
        return tokens, logits, got


@pytest.mark.parametrize("dtype", ["fp16", "bf16"])
@pytest.mark.parametrize("captured", [False, True])
def test_a_run_of_steps(dev, dtype, captured):
    """Prompts, then steps of trees: each step's verdict is the oracle's of its logits, and at the end the first layer's cache
    holds the accepted tokens' keys at their own positions, in order, and pages for no more.

    Keys of the first layer depend on the token and its position alone: x W (computed here by the same call, one row's
    product in other company: 64 terms in 32 bits and a rounding, 2 u of the largest sum of magnitudes), normed and turned
    (34 x 2^-24), then e4m3 (2^-4 of it), then rounded again at most twice a step, which loses no more than half a step of
    what is subnormal, 2^-10 of the scale each."""
    rng = np.random.default_rng([5, captured])
    prompts = [rng.integers(0, 9, n).tolist() for n in (21, 5, 48)]
    toy = _Toy(dev, rng, prompts, DT[dtype], [4, 0, 2])
    sizes = [14, 9, 1]
    cu = _i32(_cu(sizes), dev)
    drafts, uniforms = torch.zeros(24, dtype=torch.int32, device=dev), torch.zeros(24, device=dev)
    parents = torch.zeros(24, dtype=torch.int32, device=dev)
    steps, graph, accepted = 8, None, 0

    def draw():
        drafts.copy_(_i32(rng.integers(0, 9, 24), dev))
        parents.copy_(_i32([x for n in sizes for x in _parents(rng, n)], dev))
        uniforms.copy_(torch.from_numpy(rng.random(24, dtype=np.float32)).to(dev))

    if captured:  # the capture itself runs nothing; allocations and first calls come before it, on a decoder of their own
        draw()
        _Toy(dev, np.random.default_rng(9), prompts, DT[dtype], [4, 0, 2]).step(drafts, parents, cu, uniforms)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = toy.step(drafts, parents, cu, uniforms)
    for _ in range(steps):
        draw()
        if graph is None:
            out = toy.step(drafts, parents, cu, uniforms)
        else:
            graph.replay()
        torch.cuda.synchronize()
        tokens, logits, got = out
        assert torch.isfinite(logits).all()
        _same_verdict(got, dft.verify(logits.double().cpu().numpy(), tokens.cpu().numpy(), uniforms.cpu().numpy(), parents.cpu().numpy(), None,
                                      0.7, _cu(sizes)), 14)
        for b, n in enumerate(got.accepted.tolist()):
            accepted += n - 1
            path = got.path[b, :n].tolist()
            assert [tokens[sizes[0] * (b > 0) + sizes[1] * (b > 1) + i].item() for i in path[1:]] == got.tokens[b, : n - 1].tolist()
            toy.seen[b] += got.tokens[b, :n].tolist()
    assert accepted  # or the run has moved nothing
    c = toy.cache
    lengths, table, refs = c.lengths.tolist(), c.page_table.tolist(), c.refcounts.tolist()
    assert [lengths[i] for i in (1, 3, 5)] == [0, 0, 0] and sum(refs) == sum(-(-n // 16) for n in lengths) and max(refs) == 1
    norm = toy.norms[1].double().cpu().numpy()
    for b, slot in enumerate((4, 0, 2)):
        seen = toy.seen[b][:-1]
        assert lengths[slot] == len(seen) and all(x < 0 for x in table[slot][-(-len(seen) // 16):])
        x = toy.embed[torch.tensor(seen, device=dev)]
        raw = (x @ toy.qkv[0]).view(len(seen), -1, 64)[:, 6:8]
        slack = (x.abs().float() @ toy.qkv[0].abs().float()).view(len(seen), -1, 64)[:, 6:8].double().cpu().numpy()
        cos, sin = toy.angles
        pairs = [dft.turn(r, norm, 1e-6, cos, sin, i, False) for i, r in enumerate(raw.double().cpu().numpy())]
        want = np.stack([w for w, _ in pairs]).transpose(1, 0, 2)
        mag = np.stack([m for _, m in pairs]).transpose(1, 0, 2)
        # an error e of each channel of x moves the normed x by at most 2 e |norm| / rms(x), and its turn by that of both channels
        u = 2.0 ** -11 if dtype == "fp16" else 2.0 ** -8
        rms = np.sqrt(np.square(raw.double().cpu().numpy()).mean(-1, keepdims=True))
        off = (2 * 2 * u * slack.max(-1, keepdims=True) * 2 * np.abs(norm).max() / rms).transpose(1, 0, 2)
        off = off + 34 * 2.0 ** -24 * mag
        largest = 2.0 ** np.ceil(np.log2(np.abs(want).max() * 1.1 / 448))
        got = c.read(0, slot)[0].double().cpu().numpy()
        assert (np.abs(got - want) <= off + 2.0 ** -4 * (np.abs(want) + off) + (1 + 2 * steps) * 2.0 ** -10 * largest).all()


class _GappyToy(_Toy):
    """Sequences that found no room, or have no nodes, take no part in a step; a sequence's last token is then what it was."""

    def step(self, drafts, parents, cu, uniforms):
        first = cu[:-1].long().clamp(max=len(drafts) - 1)
        tokens = drafts.scatter(0, torch.where(cu.diff() > 0, first, len(drafts) - 1), self.last)
        served = self.cache.extend(cu.diff().to(torch.int32), slots=self.slots)
        own = self.slots
        self.slots = torch.where(served > 0, own, -1)
        logits = self.forward(tokens, cu, self.max_new, parents)
        got = bsa.verify_drafts(logits, tokens, uniforms, parents, temperature=0.7, cu_seqlens=cu, max_new=self.max_new, slots=self.slots)
        self.cache.keep(got.path, got.accepted, cu_seqlens=cu, slots=self.slots)
        self.slots = own
        new = got.tokens.gather(1, (got.accepted.long() - 1).clamp(min=0)[:, None])[:, 0]
        self.last.copy_(torch.where(got.accepted > 0, new, self.last))
        return tokens, logits, got, served


@pytest.mark.parametrize("captured", [False, True])
def test_a_run_of_steps_some_take_no_part_in(dev, captured):
    """Every other step the pool is full, so that who needs a page is refused; one sequence has no nodes.  Who takes no part keeps
    its last token, its length and its bytes; the others' verdicts are the oracle's."""
    rng = np.random.default_rng(21)
    prompts = [rng.integers(0, 9, n).tolist() for n in (21, 5, 48, 30)]
    slots = [4, 0, 2, 5]
    toy = _GappyToy(dev, rng, prompts, torch.float16, slots)
    sizes = [14, 9, 0, 1]
    cu = _i32(_cu(sizes), dev)
    # one row more than the sequences have: where a sequence without nodes puts its last token
    drafts, uniforms, parents = _i32([0] * 25, dev), torch.zeros(25, device=dev), _i32([-1] * 25, dev)

    def draw():
        drafts.copy_(_i32(rng.integers(0, 9, 25), dev))
        parents.copy_(_i32([x for n in sizes if n for x in _parents(rng, n)] + [-1], dev))
        uniforms.copy_(torch.from_numpy(rng.random(25, dtype=np.float32)).to(dev))

    if captured:
        draw()
        _GappyToy(dev, np.random.default_rng(9), prompts, torch.float16, slots).step(drafts, parents, cu, uniforms)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = toy.step(drafts, parents, cu, uniforms)
    c, refused = toy.cache, 0
    for step in range(8):
        draw()
        held = (c.refcounts == 0).int() * (step % 2)  # a full pool
        c.refcounts.add_(held)
        before, last = [c.read(1, s) for s in slots], toy.last.tolist()
        if captured:
            graph.replay()
        else:
            out = toy.step(drafts, parents, cu, uniforms)
        torch.cuda.synchronize()
        c.refcounts.sub_(held)
        tokens, logits, got, served = out
        want = dft.verify(logits.double().cpu().numpy(), tokens.cpu().numpy(), uniforms.cpu().numpy(), parents.cpu().numpy(), None, 0.7, _cu(sizes))
        served = served.tolist()
        refused += served.count(0)
        _same_verdict(got, [w if ok else (0, [], []) for w, ok in zip(want, served)], 14)
        for b, (slot, n) in enumerate(zip(slots, got.accepted.tolist())):
            assert (n > 0) == (served[b] > 0 and sizes[b] > 0)
            toy.seen[b] += got.tokens[b, :n].tolist()
            assert toy.last[b].item() == (toy.seen[b][-1] if n else last[b]) and c.lengths[slot].item() == len(toy.seen[b]) - 1
            if n == 0:
                assert all(torch.equal(x, y) for x, y in zip(before[b], c.read(1, slot)))
    assert refused
    refs, table = c.refcounts.tolist(), c.page_table.tolist()
    assert sum(refs) == sum(-(-n // 16) for n in c.lengths.tolist()) and max(refs) == 1
    assert all(x < 0 for b, slot in enumerate(slots) for x in table[slot][-(-(len(toy.seen[b]) - 1) // 16):])


def test_calls_without_anything_to_do(dev):
    """No tokens, no sequences, no nodes: nothing is written, and what comes back has the shapes."""
    cache = bsa.KVCache(2, 8, 2, 64, 16, 3, 2, dev)
    before = [x.clone() for x in (cache.pages.view(torch.uint8), cache.scales, cache.page_table, cache.lengths, cache.refcounts)]
    cos, sin = (torch.from_numpy(x).to(dev) for x in _angles(8, 64))
    none = torch.zeros(0, dtype=torch.int32, device=dev)
    for rows in (0, 3):
        cu, slots = torch.zeros(rows + 1, dtype=torch.int32, device=dev), _i32(list(range(rows)), dev)
        q, k = (torch.zeros(0, h, 64, dtype=torch.float16, device=dev) for h in (4, 2))
        batch = dict(cu_seqlens=cu, max_new=5, slots=slots)
        assert cache.append_rotated(1, q, k, k, cos, sin, parents=none, **batch).shape == (0, 4, 64)
        out, lse = cache.attend_tree(1, q, none, **batch)
        assert out.shape == (0, 4, 64) and lse.shape == (0, 4)
        used = [torch.full((n,), 9, dtype=torch.int32, device=dev) for n in (3, 3, 3, 15, 15)]
        del used  # memory that the answers are given holds something
        got = bsa.verify_drafts(torch.zeros(0, 50, device=dev), none, torch.zeros(0, device=dev), none, cu_seqlens=cu, max_new=5)
        assert got.accepted.tolist() == [0] * rows and got.path.shape[0] == rows and (got.path == -1).all() and (got.tokens == -1).all()
        cache.keep(torch.zeros(rows, 5, dtype=torch.int32, device=dev), torch.ones(rows, dtype=torch.int32, device=dev), cu_seqlens=cu, slots=slots)
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(before, (cache.pages.view(torch.uint8), cache.scales, cache.page_table, cache.lengths, cache.refcounts)))


def test_batches_without_tokens_have_any_strides(dev):
    """An empty array's tensor has strides of 0, and is contiguous all the same."""
    cache = bsa.KVCache(1, 8, 2, 64, 16, 3, 2, dev)
    cos, sin = (torch.from_numpy(x).to(dev) for x in _angles(8, 64))
    none = torch.zeros(0, dtype=torch.int32, device=dev)
    q, k = (torch.from_numpy(np.zeros((0, h, 64), np.float16)).to(dev) for h in (4, 2))
    q, k, logits = (torch.as_strided(x, x.shape, (0,) * x.dim()) for x in (q, k, torch.zeros(0, 50, device=dev)))
    assert q.stride(2) == k.stride(2) == logits.stride(1) == 0 and q.is_contiguous()
    batch = dict(cu_seqlens=_i32([0, 0, 0], dev), max_new=5, slots=_i32([2, 0], dev))
    cache.append(0, k, k, **batch)
    assert cache.append_rotated(0, q, k, k, cos, sin, parents=none, **batch).shape == (0, 4, 64)
    for out, lse in (cache.attend(0, q, **batch), cache.attend_tree(0, q, none, **batch)):
        assert out.shape == (0, 4, 64) and lse.shape == (0, 4)
    for draft in (None, logits):
        got = bsa.verify_drafts(logits, none, torch.zeros(0, device=dev), None, draft, **batch)
        assert got.accepted.tolist() == [0, 0] and (got.path == -1).all() and (got.tokens == -1).all()


def test_refusals(dev):
    """Types, shapes, strides and devices that cannot be right, of each call; and the right ones, unharmed."""
    cache = bsa.KVCache(1, 8, 2, 64, 16, 3, 2, dev)
    q, k, n = torch.zeros(3, 4, 64, dtype=torch.float16, device=dev), torch.zeros(3, 2, 64, dtype=torch.float16, device=dev), _i32([-1, -1, -1], dev)
    cos, sin = (torch.from_numpy(x).to(dev) for x in _angles(8, 64))
    norm = torch.ones(64, dtype=torch.float16, device=dev)
    odd = torch.zeros(3 * 4 * 64 + 1, dtype=torch.float16, device=dev)[1:].view(3, 4, 64)
    turned = torch.zeros(3, 64, 4, dtype=torch.float16, device=dev).transpose(1, 2)

    def append(q=q, k=k, v=k, cos=cos, sin=sin, **kw):
        return cache.append_rotated(0, q, k, v, cos, sin, **kw)

    def attend(q=q, parents=n, **kw):
        return cache.attend_tree(0, q, parents, **kw)

    def verify(logits=torch.zeros(3, 30, device=dev), tokens=n, uniforms=torch.zeros(3, device=dev), max_new=3, **kw):
        return bsa.verify_drafts(logits, tokens, uniforms, max_new=max_new, **kw)

    def keep(path=_i32([[0], [0], [0]], dev), accepted=_i32([1, 1, 1], dev), **kw):
        return cache.keep(path, accepted, **kw)

    for call in (append, attend, verify, keep):
        call()
    many = torch.zeros(195, 4, 64, dtype=torch.float16, device=dev)
    for call, error, bads in (
            (append, TypeError, (dict(q=q.float(), k=k.float(), v=k.float()), dict(cos=cos.double()), dict(sin=sin.cpu()), dict(parents=n.long()),
                                 dict(positions=n.float()))),
            (append, ValueError, (dict(q=q[:2]), dict(q=q.bfloat16()), dict(v=k.bfloat16()), dict(k=k[:, :1], v=k[:, :1]), dict(q=q.cpu()), dict(q=turned),
                                  dict(sin=sin[:7]), dict(cos=cos.repeat(1, 2)[:, ::2]), dict(q_norm=norm[:32]), dict(k_norm=norm.float()),
                                  dict(q_norm=norm.cpu()), dict(parents=n[:2]), dict(positions=n.repeat(2)), dict(out=q[:2]), dict(out=q.float()),
                                  dict(out=turned), dict(max_new=2), dict(slots=n[:2]), dict(eps=-1.0), dict(positions=n, parents=n),
                                  dict(cos=cos[:0], sin=sin[:0]), dict(q=odd))),
            (append, NotImplementedError, (dict(cos=cos[:, :24].contiguous(), sin=sin[:, :24].contiguous()),)),
            (attend, TypeError, (dict(q=q.float()), dict(parents=n.long()))),
            (attend, ValueError, (dict(q=q[:, :3]), dict(q=q.cpu()), dict(q=turned), dict(q=odd), dict(parents=n[:2]), dict(parents=n.cpu()), dict(out=q[:2]),
                                  dict(out=turned), dict(lse=cos), dict(max_new=2), dict(sm_scale=float("inf")),
                                  dict(q=many, parents=n.repeat(65)))),
            (verify, TypeError, (dict(logits=torch.zeros(3, 30, device=dev).double()), dict(tokens=n.long()), dict(uniforms=torch.zeros(3, device=dev).half()),
                                 dict(parents=n.long()), dict(slots=torch.zeros(1, device=dev)))),
            (verify, ValueError, (dict(logits=torch.zeros(3, 30)), dict(logits=torch.zeros(30, device=dev)), dict(logits=torch.zeros(3, 0, device=dev)),
                                  dict(logits=torch.zeros(30, 3, device=dev).t()), dict(tokens=n[:2]), dict(uniforms=torch.zeros(2, device=dev)),
                                  dict(uniforms=torch.zeros(3)), dict(max_new=2), dict(max_new=None), dict(max_new=0),
                                  dict(draft_logits=torch.zeros(3, 30, device=dev), parents=n), dict(draft_logits=torch.zeros(3, 29, device=dev)),
                                  dict(draft_logits=torch.zeros(3, 30, device=dev).half()), dict(temperature=torch.ones(2, device=dev)),
                                  dict(temperature=torch.ones(1, device=dev).double()), dict(temperature=-1.0), dict(temperature=float("inf")),
                                  dict(temperature=float("nan")), dict(slots=n), dict(cu_seqlens=n[:0]),
                                  dict(logits=torch.zeros(65, 30, device=dev), tokens=n.new_zeros(65), uniforms=torch.zeros(65, device=dev), max_new=65))),
            (keep, TypeError, (dict(path=_i32([[0], [0], [0]], dev).long()), dict(accepted=torch.ones(3, device=dev)))),
            (keep, ValueError, (dict(path=n), dict(accepted=n[:2]), dict(slots=n[:2]), dict(cu_seqlens=n), dict(path=n.new_zeros(3, 65)),
                                dict(path=n.new_zeros(1025, 1), accepted=n.new_zeros(1025), slots=n.new_full((1025,), -1))))):
        for bad in bads:
            with pytest.raises(error):
                call(**bad)
    with pytest.raises((ValueError, NotImplementedError)):
        verify(logits=torch.zeros(3, 2 ** 20 + 1, device=dev))
    for call in (append, attend, verify, keep):
        call()
    torch.cuda.synchronize()


@pytest.mark.parametrize("nodes,hq", [(8, 2), (40, 4)])
def test_tree_strided_q_and_out(dev, nodes, hq):
    """q and out as slices of wider tensors; what lies between them is left as it is."""
    rng = np.random.default_rng(nodes)
    lengths, cu = [90, 300], [0, nodes, 2 * nodes]
    raw, sc, table, pages, scales, tab = _cache(rng, dev, lengths, 2, 32, 128, poison=True)
    parents = _parents(rng, nodes) + _parents(rng, nodes)
    wide = torch.randn(2 * nodes, 2 * hq + 3, 128, device=dev).half()
    out = torch.full((2 * nodes + 1, 4 * hq, 136), 7.0, dtype=torch.float16, device=dev)
    q, y = wide[:, 2:2 + 2 * hq], out[1:, ::2, :128]
    ref = dft.tree_attention(q.double().cpu().numpy(), parents, orc.Layer(raw, sc), table, np.array(lengths), cu)
    got, lse = bsa.kv_tree_attention(q, _i32(parents, dev), pages, scales, tab, _i32(lengths, dev), max_new=nodes, out=y)
    assert got is y
    _check_attention(y, lse, ref, torch.float16, 128)
    y.fill_(7.0)
    assert (out == 7.0).all()


@pytest.mark.parametrize("nodes,hq", [(12, 8), (50, 16)])
def test_pages_past_four_gigabytes(dev, nodes, hq):
    """The last pages of a pool of 4.4 GB give what its first ones do."""
    heads, p, d, count = 8, 128, 128, 17000
    rng = np.random.default_rng(nodes)
    pages = torch.empty(1, count, heads, 2, p, d, dtype=torch.uint8, device=dev)
    scales = torch.ones(1, count, heads, 2, device=dev)
    first = torch.from_numpy(rng.integers(0, 120, (3, heads, 2, p, d)).astype(np.uint8)).to(dev)
    length = 2 * p + 20
    q, k, v = (torch.from_numpy(rng.standard_normal((nodes, h, d)).astype(np.float32)).half().to(dev) for h in (hq, heads, heads))
    cos, sin = (torch.from_numpy(x).to(dev) for x in _angles(400, d))
    parents = _i32(_parents(rng, nodes), dev)
    path = _i32([sorted(rng.choice(nodes, 6, replace=False).tolist()) + [-1] * (nodes - 6)], dev)
    results = []
    for at in (0, count - 3):
        pages[0, at:at + 3], scales[0, at:at + 3] = first, 2.0 ** -8
        tab, n, refs = _i32([[at, at + 1, at + 2]], dev), _i32([length], dev), torch.ones(count, dtype=torch.int32, device=dev)
        args = (pages[0].view(F8), scales[0], tab, n)
        y = bsa.kv_append_rotated(q, k, v, cos, sin, *args, parents=parents)
        out, lse = bsa.kv_tree_attention(y, parents, *args)
        bsa.pages_keep(pages.view(F8), scales, tab, n, refs, path, _i32([6], dev))
        torch.cuda.synchronize()
        results.append([x.clone() for x in (y, out, lse, pages[0, at:at + 3], scales[0, at:at + 3], n)] + [refs[at:at + 3].tolist()])
    assert all(torch.equal(a, b) for a, b in zip(results[0][:-1], results[1][:-1])) and results[0][-1] == results[1][-1]
    assert results[0][5].tolist() == [length - nodes + 6] and not torch.equal(results[0][3], first)
