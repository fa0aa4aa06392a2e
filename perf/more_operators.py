"""The operators of a step that drafts tokens and verifies them over the 8-bit paged cache, whose speed this repository
answers for beside those of operators.py.

With `own` false, run() computes an operator in its plain form, from elementary torch operations in 32 bits (verification in
64: its answers are whole numbers next to borders); with `own` true it makes the calls that a user makes of bsa_mi355x.

op        what is called (own)
rotate    kv_append_rotated: queries and keys normed by head and rotated, keys and values quantised into the cache's pages
tree      kv_tree_attention: attention of a tree of drafted tokens over the cache
verify    verify_drafts: which drafted tokens the target's probabilities accept, and the token that follows them
keep      pages_keep: the accepted tokens' keys and values move together, the others leave the cache

The cache of one layer is pages [pages, heads, 2, P, D] in e4m3, keys then values, with scales [pages, heads, 2], powers
of two; page_table [sequences, pages each] names a sequence's pages.  Inside [P, D] lie tiles of 16 tokens x 64 channels:
keys as [tile, c, g, t, e] (token 16 tile + t, channel 64c + 16g + e), values as [tile, c, g, l, i, t] (token 16 tile + 4g
+ t, channel 64c + 16i + l).  The newest tokens of a sequence are the nodes of a tree: parents names each one's parent
among them, by its place, -1 for none.
"""
import os
import random
import sys

import torch

own = False

DEV = "cuda"
DTYPES = {"fp16": torch.float16, "bf16": torch.bfloat16, "fp32": torch.float32}
F8 = torch.float8_e4m3fn
SCALE_LOW, SCALE_HIGH = 2.0 ** -40, 2.0 ** 80
EPS = 1e-6


def _bsa():
    root = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "towards-batched-activation-sparsity_amd")
    if root not in sys.path:
        sys.path.insert(0, root)
    import bsa_mi355x

    return bsa_mi355x


def _rotate(name, bt, q, hq, hkv, d, page, length, dtype, rot, pairs, norm, tree):
    return {"name": name, "op": "rotate", "bt": bt, "q": q, "hq": hq, "hkv": hkv, "d": d, "page": page, "len": length,
            "dtype": dtype, "rot": rot, "pairs": pairs, "norm": norm, "tree": tree}


def _tree(name, bt, q, hq, hkv, d, page, length, dtype):
    return {"name": name, "op": "tree", "bt": bt, "q": q, "hq": hq, "hkv": hkv, "d": d, "page": page, "len": length,
            "dtype": dtype, "tree": True}


def _verify(name, bt, q, vocab, dtype, tree, draft, temperature):
    return {"name": name, "op": "verify", "bt": bt, "q": q, "vocab": vocab, "dtype": dtype, "tree": tree, "draft": draft,
            "temperature": temperature}


def _keep(name, bt, q, layers, hkv, d, page, length):
    return {"name": name, "op": "keep", "bt": bt, "q": q, "layers": layers, "hkv": hkv, "d": d, "page": page, "len": length}


def listed():
    return [
        # one sequence decoding one token: latency
        _rotate("rotate_b1", 1, 1, 32, 32, 128, 16, 300, "fp16", 128, False, False, False),
        # 64 sequences with trees of 16 drafted tokens, every layer of a step that verifies them
        _rotate("rotate_tree_b64", 64, 16, 32, 32, 128, 16, 500, "fp16", 128, False, False, True),
        # four prompts of up to 2000 tokens, a bf16 model with shared heads and norms of queries and keys
        _rotate("rotate_prompt", 4, 2000, 32, 8, 128, 64, 2500, "bf16", 128, False, True, False),
        # a batch of an odd size, small heads rotated in neighbouring pairs and only by half
        _rotate("rotate_odd", 37, 7, 28, 4, 64, 32, 333, "bf16", 32, True, True, True),
        # one sequence with a small tree: latency
        _tree("tree_b1", 1, 16, 32, 32, 128, 16, 777, "fp16"),
        # the batch of the decode step with trees of 16 tokens
        _tree("tree_b64", 64, 16, 32, 32, 128, 16, 1500, "fp16"),
        # large trees, four query heads to a cached head: 240 rows read the same cache
        _tree("tree_group", 16, 60, 32, 8, 128, 64, 6001, "bf16"),
        # 64 sequences with chains of 4 drafts, drawn from a draft model's probabilities
        _verify("verify_chain", 64, 5, 32000, "fp16", False, True, 1.0),
        # 64 sequences with trees of 16 of the likeliest tokens
        _verify("verify_tree", 64, 16, 32000, "bf16", True, False, 0.8),
        # one sequence, a large odd vocabulary in 32 bits, the likeliest token only
        _verify("verify_greedy", 1, 9, 100003, "fp32", True, False, 0.0),
        # after the trees of 64 sequences: what was accepted stays, in all of the step's 8 layers
        _keep("keep_b64", 64, 16, 8, 32, 128, 16, 500),
        # the same for few sequences with large trees and few heads
        _keep("keep_b5", 5, 60, 32, 4, 128, 64, 700),
    ]


def _log(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


def draw(rng):
    op = rng.choice(["rotate", "rotate", "tree", "tree", "tree", "verify", "verify", "keep"])
    dtype = rng.choice(["fp16", "bf16"])
    page, d = rng.choice([16, 16, 32, 64, 128]), rng.choice([64, 128, 128])
    hq, hkv = rng.choice([(32, 32), (32, 8), (16, 16), (40, 8), (28, 4), (8, 1)])
    if op == "rotate":
        kind = rng.choice(["decode", "tree", "prompt"])
        bt = _log(rng, 1, 4) if kind == "prompt" else _log(rng, 1, 64)
        q = {"decode": 1, "tree": rng.randint(2, 24), "prompt": _log(rng, 20, 2000)}[kind]
        return _rotate("", bt, q, hq, hkv, d, page, q + _log(rng, 10, 500), dtype, rng.choice([d, d, d // 2, d // 4]),
                       rng.random() < 0.3, rng.random() < 0.5, kind == "tree")
    if op == "tree":
        bt = _log(rng, 1, 64)
        q = rng.randint(2, 64)
        return _tree("", bt, q, hq, hkv, d, page, q + _log(rng, 8, max(16, min(20000, 60000 // bt))), dtype)
    if op == "verify":
        bt, tree = _log(rng, 1, 64), rng.random() < 0.5
        return _verify("", bt, rng.randint(2, 16 if tree else 8), _log(rng, 1000, 32000), rng.choice(["fp16", "bf16", "fp32"]),
                       tree, not tree and rng.random() < 0.7, rng.choice([0.0, 0.7, 1.0, 1.0]))
    return _keep("", _log(rng, 1, 64), rng.randint(8, 32), rng.randint(1, 8), rng.choice([4, 8, 16]), d, page, _log(rng, 40, 500))


# ------------------------------------------------------------------------------------------------ inputs


def _spread(lo, hi, n, salt):
    """n whole numbers between lo and hi, the last of them hi: lengths of a batch, the same for every seed."""
    r = random.Random(7919 * hi + 31 * n + salt)
    return [r.randint(lo, hi) for _ in range(n - 1)] + [hi]


def _new(c):
    """How many new tokens each sequence has: full trees and prompts of several lengths among them."""
    return [1] * c["bt"] if c["q"] == 1 else _spread(max(1, c["q"] // 2), c["q"], c["bt"], 1)


def _lengths(c):
    """Tokens of each sequence with its new ones, and how many are new."""
    new = _new(c)
    old = _spread((c["len"] - c["q"]) // 4, c["len"] - c["q"], c["bt"], 2)
    return [a + b for a, b in zip(old, new)], new


def _parents(c):
    """Trees level by level: a node's parent is never before the parent of the node before it."""
    if not c["tree"]:
        return [i - 1 for n in _new(c) for i in range(n)]
    r, out = random.Random(97 * c["q"] + c["bt"]), []
    for n in _new(c):
        wide = max(1, (n - 1) // 4)  # children of the first node
        for i in range(n):
            out.append(-1 if i == 0 else 0 if i <= wide else min(i - 1, max(out[-1], out[-1] + r.choice([0, 0, 0, 1, 1, 2]))))
    return out


def _paths(c):
    """The nodes that were accepted, of each sequence: the first one, then a few further ones.  None lies where another
    one goes to, so that the same pass can be made again."""
    r, out = random.Random(131 * c["q"] + c["bt"]), []
    for n in _new(c):
        most = min(n, r.choice([1, 2, 3, 3, 4, 4, 5, 6]))
        path = [0]
        while len(path) < most:
            lo = max(most, path[-1] + 1)
            if lo >= n:
                break
            path.append(1 if len(path) == 1 and r.random() < 0.4 else r.randint(lo, max(lo, min(n - 1, lo + n // 3))))
        out.append(path)
    return out


def _power(e):
    """2 to whole exponents, in 32 bits."""
    return ((e.to(torch.int32) + 127) << 23).view(torch.float32)


def _i32(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def _cu(new):
    cu = [0]
    for n in new:
        cu.append(cu[-1] + n)
    return cu


def _pages(g, layers, pages, heads, page, d):
    """Pages as a model's keys and values leave them: values of unit spread, stronger in some blocks than in others."""
    shape = (pages, heads, 2, page, d)
    data = torch.empty(layers, *shape, dtype=F8, device=DEV)
    for layer in data:
        layer.copy_(torch.randn(shape, generator=g, device=DEV).mul_(64.0).clamp_(-448.0, 448.0))
    e = torch.randint(-7, -4, (layers, pages, heads, 2), generator=g, device=DEV)
    return data, _power(e)


def _kv_state(c, g):
    total, new = _lengths(c)
    per = [-(-t // c["page"]) for t in total]
    most, layers = max(per) + 1, c.get("layers", 1)
    pages, scales = _pages(g, layers, sum(per) + 8, c["hkv"], c["page"], c["d"])
    ids = torch.randperm(sum(per) + 8, generator=g, device=DEV).to(torch.int32)
    table = torch.full((c["bt"], most), -1, dtype=torch.int32, device=DEV)
    refs = torch.zeros(len(ids), dtype=torch.int32, device=DEV)
    at = 0
    for b, n in enumerate(per):
        table[b, :n] = ids[at:at + n]
        at += n
    refs[ids[:at].long()] = 1
    cu = _cu(new)
    s = {"case": c, "table": table, "lengths": _i32(total), "cu": _i32(cu)}
    t = cu[-1]
    if c["op"] == "keep":
        paths = _paths(c)
        return {**s, "pages": pages, "scales": scales, "refs": refs, "before": [table.clone(), s["lengths"].clone(), refs.clone()],
                "accepted": _i32([len(p) for p in paths]), "path": _i32([p + [-1] * (c["q"] - len(p)) for p in paths])}
    s |= {"pages": pages[0], "scales": scales[0], "q": torch.randn(t, c["hq"], c["d"], generator=g, device=DEV).to(DTYPES[c["dtype"]])}
    if c["tree"]:
        s["parents"] = _i32(_parents(c))
    if c["op"] == "rotate":
        dt = DTYPES[c["dtype"]]
        # tokens of unequal strength: now and then a block's scale has to grow
        loud = torch.exp(0.5 * torch.randn(t, c["hkv"], 1, generator=g, device=DEV))
        s["k"] = (torch.randn(t, c["hkv"], c["d"], generator=g, device=DEV) * loud).to(dt)
        s["v"] = torch.randn(t, c["hkv"], c["d"], generator=g, device=DEV).to(dt)
        half = c["rot"] // 2
        angle = torch.arange(max(total) + 1, device=DEV)[:, None].double() * 10000.0 ** (-torch.arange(half, device=DEV).double() / half)
        s["cos"], s["sin"] = angle.cos().float(), angle.sin().float()
        for name in ("q_norm", "k_norm"):
            s[name] = (1.0 + 0.2 * torch.randn(c["d"], generator=g, device=DEV)).to(dt) if c["norm"] else None
    return s


def _verify_state(c, g):
    new = _new(c)
    cu, parents = _cu(new), _parents(c)
    t, vocab = cu[-1], c["vocab"]
    x = torch.randn(t, vocab, generator=g, device=DEV).mul_(2.0)
    for _ in range(3):  # a few likely tokens in each row, beside a tail that is not nothing
        at = torch.randint(0, vocab, (t, 1), generator=g, device=DEV)
        x.scatter_add_(1, at, 10.0 + 2.0 * torch.randn(t, 1, generator=g, device=DEV))
    x = x.to(DTYPES[c["dtype"]])
    s = {"case": c, "logits": x, "cu": _i32(cu), "parents": _i32(parents) if c["tree"] else None, "draft": None,
         "uniforms": torch.rand(t, generator=g, device=DEV)}
    # the draft model sees about what the target does
    guess = x.float() + 0.7 * torch.randn(t, vocab, generator=g, device=DEV)
    if c["draft"]:
        s["draft"] = guess.to(x.dtype)
        guess = s["draft"].float() / max(c["temperature"], 0.1) - torch.log(-torch.log(torch.rand(t, vocab, generator=g, device=DEV).clamp_(1e-9, 0.9999999)))
    # children of a node are its likeliest tokens, or in a chain one that was drawn
    rank, seen = [], {}
    first = [cu[b] for b, n in enumerate(new) for _ in range(n)]
    for i, p in enumerate(parents):
        at = first[i] + max(p, 0)
        rank.append(seen.get(at, 0) if p >= 0 else 0)
        seen[at] = seen.get(at, 0) + (p >= 0)
    best = guess.topk(max(rank) + 1, dim=1)[1]
    above = _i32([f + max(p, 0) for f, p in zip(first, parents)]).long()
    s["tokens"] = best[above].gather(1, _i32(rank).long()[:, None])[:, 0].to(torch.int32)
    return s


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    c = dict(case)
    return (_verify_state if c["op"] == "verify" else _kv_state)(c, g)


# ------------------------------------------------------------------------------------------------ one pass


def run(state):
    op = state["case"]["op"]
    if op == "keep":
        # the sequences as they were before the step, so that every pass has the same work
        for name, was in zip(("table", "lengths", "refs"), state["before"]):
            state[name].copy_(was)
    return (_RUN_OWN if own else _RUN_PLAIN)[op](state)


def _own_rotate(s):
    c = s["case"]
    q = _bsa().kv_append_rotated(s["q"], s["k"], s["v"], s["cos"], s["sin"], s["pages"], s["scales"], s["table"], s["lengths"],
                                 cu_seqlens=s["cu"], max_new=c["q"], parents=s.get("parents"), q_norm=s["q_norm"],
                                 k_norm=s["k_norm"], eps=EPS, interleaved=c["pairs"])
    return [q, s["pages"], s["scales"]]


def _own_tree(s):
    return list(_bsa().kv_tree_attention(s["q"], s["parents"], s["pages"], s["scales"], s["table"], s["lengths"],
                                         cu_seqlens=s["cu"], max_new=s["case"]["q"]))


def _own_verify(s):
    return list(_bsa().verify_drafts(s["logits"], s["tokens"], s["uniforms"], parents=s["parents"], draft_logits=s["draft"],
                                     temperature=s["case"]["temperature"], cu_seqlens=s["cu"], max_new=s["case"]["q"]))


def _own_keep(s):
    _bsa().pages_keep(s["pages"], s["scales"], s["table"], s["lengths"], s["refs"], s["path"], s["accepted"], cu_seqlens=s["cu"])
    return [s["table"], s["lengths"], s["refs"], s["pages"], s["scales"]]


_RUN_OWN = {"rotate": _own_rotate, "tree": _own_tree, "verify": _own_verify, "keep": _own_keep}


def _key_tiles(pages):
    """[..., heads, tile, c, g, t, e] of the keys; the values as [..., heads, tile, c, g, l, i, t] below."""
    *n, h, _, p, d = pages.shape
    return pages.view(*n, h, 2, p // 16, d // 64, 4, 16, 16).select(len(n) + 1, 0)


def _value_tiles(pages):
    *n, h, _, p, d = pages.shape
    return pages.view(*n, h, 2, p // 16, d // 64, 4, 16, 4, 4).select(len(n) + 1, 1)


def _e4m3(x):
    """To the nearest e4m3 value, as bytes; past the largest one to that."""
    return x.clamp(-448.0, 448.0).to(F8).view(torch.uint8)


def _token_rows(cu, total):
    """Which sequence each of the new tokens belongs to."""
    return torch.searchsorted(cu[1:].long(), torch.arange(total, device=DEV), right=True)


def _ancestors(s, row, i):
    """[sequences, q, q]: whether the second node is on the first one's way to the root, itself among it."""
    b, n = len(s["cu"]) - 1, s["case"]["q"]
    up = torch.eye(n, device=DEV).repeat(b, 1, 1)
    at = s["parents"].long()
    up[row, i, at.clamp(min=0)] += (at >= 0).float()
    return torch.matrix_power(up, 64) > 0


def _need(most):
    """The least power of two that brings a magnitude to 448 or below."""
    m, e = torch.frexp(most)
    return torch.where(most > 0, _power(e - 9 + (m > 0.875)).clamp(SCALE_LOW, SCALE_HIGH), SCALE_LOW)


def _turned(x, w, s, pos):
    """Normed by head where there is a weight, and rotated by position."""
    r, half = s["case"]["rot"], s["case"]["rot"] // 2
    x = x.float()
    if w is not None:
        x = x * torch.rsqrt(x.square().mean(2, keepdim=True) + EPS) * w.float()
    cos, sin = s["cos"][pos][:, None], s["sin"][pos][:, None]
    if s["case"]["pairs"]:
        a, b = x[..., 0:r:2], x[..., 1:r:2]
        y = torch.stack([a * cos - b * sin, a * sin + b * cos], -1).flatten(2)
    else:
        a, b = x[..., :half], x[..., half:r]
        y = torch.cat([a * cos - b * sin, a * sin + b * cos], -1)
    return torch.cat([y, x[..., r:]], -1)


def _plain_rotate(s):
    pages, scales, table, lengths, cu = s["pages"], s["scales"], s["table"], s["lengths"].long(), s["cu"].long()
    n, h, _, p, d = pages.shape
    t = s["k"].shape[0]
    row = _token_rows(s["cu"], t)
    i = torch.arange(t, device=DEV) - cu[row]
    start = lengths - (cu[1:] - cu[:-1])
    pos = start[row] + i
    turn = start[row] + _ancestors(s, row, i)[row, i].sum(1) - 1 if s["case"]["tree"] else pos
    q = _turned(s["q"], s["q_norm"], s, turn).to(s["q"].dtype)
    x = torch.stack([_turned(s["k"], s["k_norm"], s, turn), s["v"].float()], 2)  # [T, heads, 2, D]
    page = table[row, pos // p].long()
    # the largest magnitude of the new tokens of each page, and the power of two that holds it
    top = torch.where(torch.isfinite(x), x.abs(), 0.0).amax(3)
    need = _need(torch.zeros(n, h, 2, device=DEV).index_reduce_(0, page, top, "amax"))
    # only each sequence's first page can hold tokens already: those go over to the larger scale
    first = table.gather(1, (start // p)[:, None])[:, 0].long()
    held = start % p
    old = scales[first]
    keep = torch.where((held > 0)[:, None, None], torch.maximum(need[first], old), need[first])
    need[first] = keep
    shrink = (old / keep)[:, :, :, None, None, None, None, None]
    raw = pages.view(torch.uint8)
    tiles = pages[first].view(len(first), h, 2, p // 16, d // 64, 4, 16, 16)
    tile = torch.arange(p // 16, device=DEV)[:, None, None, None, None] * 16
    key_at = tile + torch.arange(16, device=DEV)[:, None]
    value_at = tile + torch.arange(4, device=DEV)[:, None, None] * 4 + torch.arange(16, device=DEV) % 4
    at = torch.stack([key_at.expand(p // 16, d // 64, 4, 16, 16), value_at.expand(p // 16, d // 64, 4, 16, 16)])
    before = at[None, None] < held.view(-1, 1, 1, 1, 1, 1, 1, 1)
    raw[first] = torch.where(before, _e4m3(tiles.float() * shrink), tiles.view(torch.uint8)).view(len(first), h, 2, p, d)
    touched = torch.zeros(n, dtype=torch.bool, device=DEV)
    touched[page] = True
    scales.copy_(torch.where(touched[:, None, None], need, scales))
    y = _e4m3(x / scales[page][..., None])
    t = pos % p
    _key_tiles(raw)[page, :, t // 16, :, :, t % 16] = y[:, :, 0].reshape(-1, h, d // 64, 4, 16)
    _value_tiles(raw)[page, :, t // 16, :, t % 16 // 4, :, :, t % 4] = y[:, :, 1].reshape(-1, h, d // 64, 4, 16).transpose(-1, -2)
    return [q, pages, scales]


def _plain_tree(s):
    q, pages, scales, lengths, cu = s["q"], s["pages"], s["scales"], s["lengths"].long(), s["cu"].long()
    _, h, _, p, d = pages.shape
    t, hq, _ = q.shape
    b, most = s["table"].shape
    n = s["case"]["q"]
    ids = s["table"].clamp(min=0).long()
    keys = _key_tiles(pages)[ids].float().permute(0, 2, 1, 3, 6, 4, 5, 7).reshape(b, h, most, p, d)
    values = _value_tiles(pages)[ids].float().permute(0, 2, 1, 3, 5, 8, 4, 7, 6).reshape(b, h, most, p, d)
    by = scales[ids].permute(0, 2, 1, 3)[..., None, None]
    keys, values = (keys * by[:, :, :, 0]).view(b, h, most * p, d), (values * by[:, :, :, 1]).view(b, h, most * p, d)
    at = torch.arange(most * p, device=DEV)
    values = torch.where((at < lengths[:, None])[:, None, :, None], values, 0.0)
    # the nodes of a sequence beside each other, the heads of a group under their cached head
    row = _token_rows(s["cu"], t)
    new, i = cu[1:] - cu[:-1], torch.arange(t, device=DEV) - cu[row]
    wide = torch.zeros(b, n, hq, d, device=DEV)
    wide[row, i] = q.float()
    wide = wide.view(b, n, h, hq // h, d).permute(0, 2, 1, 3, 4).reshape(b, h, -1, d)
    x = torch.matmul(wide, keys.transpose(2, 3)).mul_(d ** -0.5)
    # what a node sees: all that came before the tree, and its own ancestors in it
    node = (at - (lengths - new)[:, None])[:, None].expand(b, n, -1)
    sees = (node < 0) | ((node < n) & _ancestors(s, row, i).gather(2, node.clamp(0, n - 1)))
    x.masked_fill_(~sees.repeat_interleave(hq // h, 1)[:, None], float("-inf"))
    top = x.amax(3, keepdim=True)
    x.sub_(top).exp_()
    total = x.sum(3, keepdim=True)
    y = torch.matmul(x, values) / total
    y = y.view(b, h, n, hq // h, d).permute(0, 2, 1, 3, 4).reshape(b, n, hq, d)
    lse = (top + torch.log(total)).view(b, h, n, hq // h).permute(0, 2, 1, 3).reshape(b, n, hq)
    return [y[row, i].to(q.dtype), lse[row, i]]


def _plain_verify(s):
    c, cu = s["case"], s["cu"].long()
    b, n = len(cu) - 1, c["q"]
    t, vocab = s["logits"].shape
    row = _token_rows(s["cu"], t)
    i = torch.arange(t, device=DEV) - cu[row]
    parents = i - 1 if s["parents"] is None else s["parents"].long()
    up = cu[row] + parents.clamp(min=0)
    tokens = s["tokens"].long()
    if c["temperature"] > 0:
        z = s["logits"].double() / c["temperature"]
        w = torch.exp(z - z.amax(1, keepdim=True))
    else:  # all of the probability is the likeliest token's
        w = torch.zeros(t, vocab, dtype=torch.float64, device=DEV)
        w.scatter_(1, torch.argmax(s["logits"].float(), 1)[:, None], 1.0)
    total = w.sum(1)
    mine = w[up, tokens]
    if s["draft"] is not None and c["temperature"] > 0:
        z = s["draft"].double() / c["temperature"]
        e = torch.exp(z - z.amax(1, keepdim=True))
        w, e = w / total[:, None], e / e.sum(1, keepdim=True)
        total = torch.ones_like(total)
        mine, theirs = w[up, tokens], e[up, tokens]
    # the nodes in order, of all sequences at once: each is looked at where its parent is the last accepted one
    at, here = torch.zeros(b, dtype=torch.long, device=DEV), torch.arange(b, device=DEV)
    out, count = torch.zeros(b, dtype=torch.float64, device=DEV), torch.ones(b, dtype=torch.long, device=DEV)
    taken = torch.zeros(t, dtype=torch.bool, device=DEV)
    taken[cu[:-1]] = True
    refused = torch.zeros(t, dtype=torch.bool, device=DEV)
    for j in range(1, n):
        k = (cu[:-1] + j).clamp(max=t - 1)
        asked = (cu[:-1] + j < cu[1:]) & (parents[k] == at)
        if s["draft"] is not None and c["temperature"] > 0:
            ok = asked & (s["uniforms"][k].double() * theirs[k] < mine[k])
        else:
            ok = asked & (s["uniforms"][k].double() * (total[cu[:-1] + at] - out) < mine[k])
        out = torch.where(ok, 0.0, torch.where(asked, out + mine[k], out))
        at = torch.where(ok, j, at)
        count += ok
        taken[k] |= ok
        refused[k] |= asked & ~ok
    # what is left of the last row, and the token that the first number draws from it
    last = cu[:-1] + at
    refused &= parents == at[row]
    left = w[last]
    if s["draft"] is not None and c["temperature"] > 0:
        some = torch.zeros(b, dtype=torch.bool, device=DEV).index_fill_(0, row[refused], True)
        left = torch.where(some[:, None], (left - e[last]).clamp(min=0.0), left)
    else:
        left[row[refused], tokens[refused]] = 0.0
    sums = left.cumsum(1)
    more = sums > s["uniforms"][cu[:-1]].double()[:, None] * sums[:, -1:]
    drawn = torch.argmax(more.to(torch.uint8), 1)
    # nodes and tokens of the accepted ones beside each other, the new token behind them
    path = torch.full((b, n), -1, dtype=torch.int32, device=DEV)
    said = torch.full((b, n), -1, dtype=torch.int32, device=DEV)
    place = taken.long().cumsum(0) - 1
    place = place - place[cu[:-1]][row]
    path[row[taken], place[taken]] = i[taken].to(torch.int32)
    behind = taken & (i > 0)
    said[row[behind], place[behind] - 1] = s["tokens"][behind]
    said[here, count - 1] = drawn.to(torch.int32)
    return [count.to(torch.int32), path, said]


def _plain_keep(s):
    pages, scales, table, lengths, refs, cu = s["pages"], s["scales"], s["table"], s["lengths"], s["refs"], s["cu"].long()
    layers, _, h, _, p, d = pages.shape
    b, most = table.shape
    start = lengths.long() - (cu[1:] - cu[:-1])
    n = s["path"].shape[1]
    place = torch.arange(n, device=DEV)
    moves = (place < s["accepted"][:, None]) & (s["path"] != place)
    row, to = torch.nonzero(moves, as_tuple=True)
    src, dst = start[row] + s["path"][row, to].long(), start[row] + to
    sp, dp = table[row, src // p].long(), table[row, dst // p].long()
    raw = pages.view(torch.uint8)
    st, dt = src % p, dst % p
    k = _key_tiles(pages)[:, sp, :, st // 16, :, :, st % 16].float()  # [moved, layers, heads, c, g, e]
    v = _value_tiles(pages)[:, sp, :, st // 16, :, st % 16 // 4, :, :, st % 4].float()
    x = torch.stack([k.flatten(3), v.flatten(3)], 3) * scales[:, sp].transpose(0, 1)[..., None]  # [moved, layers, heads, 2, D]
    # a page whose scale is too small for what comes takes a larger one, and its tokens with it
    need = _need(torch.zeros(refs.shape[0], layers, h, 2, device=DEV).index_reduce_(0, dp, torch.where(torch.isfinite(x), x.abs(), 0.0).amax(4), "amax"))
    grown = torch.maximum(scales, need.transpose(0, 1))
    at = torch.unique(dp)
    raw[:, at] = _e4m3(pages[:, at].float() * (scales[:, at] / grown[:, at])[..., None, None])
    scales[:, at] = grown[:, at]
    y = _e4m3(x / scales[:, dp].transpose(0, 1)[..., None])
    _key_tiles(raw)[:, dp, :, dt // 16, :, :, dt % 16] = y[:, :, :, 0].reshape(k.shape)
    _value_tiles(raw)[:, dp, :, dt // 16, :, dt % 16 // 4, :, :, dt % 4] = y[:, :, :, 1].reshape(v.shape)
    # the pages past the new end go back
    left = start + s["accepted"]
    gone = (torch.arange(most, device=DEV) >= -(-left // p)[:, None]) & (table >= 0)
    refs.index_add_(0, table[gone].long(), torch.full_like(table[gone], -1))
    table[gone] = -1
    lengths.copy_(left)
    return [table, lengths, refs, pages, scales]


_RUN_PLAIN = {"rotate": _plain_rotate, "tree": _plain_tree, "verify": _plain_verify, "keep": _plain_keep}


# ------------------------------------------------------------------------------------------------ what a pass cannot do without


def work(case):
    c = case
    if c["op"] == "verify":
        size = 4 if c["dtype"] == "fp32" else 2
        # about six of ten drafts are accepted: the rows that are come to, as far as there are nodes behind each other
        parents, rows, at = _parents(c), 0.0, 0
        for n in _new(c):
            depth = []
            for i in range(n):
                depth.append(0 if i == 0 else depth[parents[at + i]] + 1)
            at += n
            rows += (1 - 0.6 ** (max(depth) + 1)) / 0.4
        return {"bytes": rows * c["vocab"] * size * (1.5 if c["draft"] else 1.0) + 12.0 * at, "flops": 4.0 * rows * c["vocab"]}
    total, new = _lengths(c)
    t = sum(new)
    if c["op"] == "keep":
        moved = sum(i != j for path in _paths(c) for i, j in enumerate(path))
        return {"bytes": moved * 4.0 * c["layers"] * c["hkv"] * c["d"] + 8.0 * c["bt"] * (max(total) // c["page"] + 2), "flops": 0.0}
    if c["op"] == "rotate":
        return {"bytes": float(t) * (c["hkv"] * 2 * c["d"] * 3 + c["hq"] * c["d"] * 4 + c["rot"] * 4),
                "flops": 4.0 * t * (c["hkv"] + c["hq"]) * c["d"]}
    held = sum(n * 2 * c["d"] + -(-n // c["page"]) * 8 for n in total) * float(c["hkv"])
    pairs = sum((n - m) * m + 3 * m for n, m in zip(total, new))
    return {"bytes": held + t * c["hq"] * (4.0 * c["d"] + 4), "flops": 4.0 * c["d"] * c["hq"] * pairs}


# ------------------------------------------------------------------------------------------------ the definition in 64 bits


def exact(case, seed):
    s = prepare(case, seed)
    return {"rotate": _exact_rotate, "tree": _exact_tree, "verify": _exact_verify, "keep": _exact_keep}[case["op"]](s)


def _offsets(p, d):
    """Where channel x of token t lies in a page's [P, D], for keys and for values."""
    t, x = torch.arange(p, device=DEV)[:, None], torch.arange(d, device=DEV)[None]
    tile, c, r = t // 16, x // 64, x % 64
    base = tile * 16 * d + c * 1024
    return base + r // 16 * 256 + t % 16 * 16 + r % 16, base + t % 16 // 4 * 256 + r % 16 * 16 + r // 16 * 4 + t % 4


def _round8(x):
    """The nearest e4m3 value of 64-bit numbers, ties to even: 4 significant bits down to a step of 2^-9."""
    x = x.clamp(-448.0, 448.0)
    _, e = torch.frexp(x)
    step = ((e - 4).clamp(min=-9).to(torch.int64) + 1023 << 52).view(torch.float64)
    return torch.round(x / step) * step


def _holding(top):
    """The least power of two that holds a magnitude within 448."""
    return torch.exp2(torch.ceil(torch.log2(top / 448.0))).clamp(SCALE_LOW, SCALE_HIGH)


def _depths(parents):
    depth = []
    for p in parents:
        depth.append(0 if p < 0 else depth[p] + 1)
    return depth


def _exact_rotate(s):
    c = s["case"]
    n, h, _, p, d = s["pages"].shape
    where = _offsets(p, d)
    pages, scales = s["pages"].double().view(n, h, 2, p * d), s["scales"].double()
    lengths, cu, table = s["lengths"].tolist(), s["cu"].tolist(), s["table"].tolist()
    parents = _parents(c)
    turned = []
    for x, w in ((s["q"], s["q_norm"]), (s["k"], s["k_norm"])):
        x = x.double()
        if w is not None:
            x = x / torch.sqrt((x * x).mean(2, keepdim=True) + EPS) * w.double()
        turn = [lengths[b] - (cu[b + 1] - cu[b]) + i for b in range(c["bt"]) for i in _depths(parents[cu[b]:cu[b + 1]])]
        turn = _i32(turn).long()
        cos, sin, y, half = s["cos"].double()[turn], s["sin"].double()[turn], x.clone(), c["rot"] // 2
        for j in range(half):
            a, b = (2 * j, 2 * j + 1) if c["pairs"] else (j, j + half)
            y[:, :, a] = x[:, :, a] * cos[:, None, j] - x[:, :, b] * sin[:, None, j]
            y[:, :, b] = x[:, :, b] * cos[:, None, j] + x[:, :, a] * sin[:, None, j]
        turned.append(y)
    q, k = turned
    for b, end in enumerate(lengths):
        pos = start = end - (cu[b + 1] - cu[b])
        while pos < end:
            j, stop = pos // p, min(end, (pos // p + 1) * p)
            at, first = table[b][j], cu[b] + pos - start
            for i, x in enumerate((k, s["v"].double())):
                x = x[first:first + stop - pos].transpose(0, 1)  # [heads, tokens, D]
                need = _holding(x.abs().amax((1, 2)))
                if pos % p:
                    old = scales[at, :, i].clone()
                    need = torch.maximum(need, old)
                    o = where[i][: pos % p].reshape(-1)
                    pages[at, :, i, o] = _round8(pages[at, :, i, o] * (old / need)[:, None])
                scales[at, :, i] = need
                pages[at, :, i, where[i][pos - j * p:stop - j * p].reshape(-1)] = _round8(x / need[:, None, None]).reshape(h, -1)
            pos = stop
    return [q, pages.view(n, h, 2, p, d), scales]


def _exact_tree(s):
    n, h, _, p, d = s["pages"].shape
    where = _offsets(p, d)
    group = s["q"].shape[1] // h
    raw = s["pages"].view(n, h, 2, p * d)
    lengths, cu, parents = s["lengths"].tolist(), s["cu"].tolist(), s["parents"].tolist()
    y, lse = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEV), torch.zeros(s["q"].shape[:2], dtype=torch.float64, device=DEV)
    for b, end in enumerate(lengths):
        ids = s["table"][b, : -(-end // p)].long()
        new, rows = cu[b + 1] - cu[b], slice(cu[b], cu[b + 1])
        sees = [[True] * (end - new) + [False] * new for _ in range(new)]
        for i in range(new):
            j = i
            while j >= 0:
                sees[i][end - new + j] = True
                j = parents[cu[b] + j]
        blind = ~torch.tensor(sees, device=DEV)
        for head in range(h):
            one = raw[ids, head].double() * s["scales"][ids, head].double()[..., None]
            k, v = (one[:, i, where[i].reshape(-1)].view(-1, d)[:end] for i in (0, 1))
            q = s["q"][rows, head * group:(head + 1) * group].double()
            x = (q.reshape(-1, d) @ k.t() / d ** 0.5).view(new, group, end)
            x.masked_fill_(blind[:, None], float("-inf"))
            total = torch.logsumexp(x, 2)
            y[rows, head * group:(head + 1) * group] = (torch.exp(x - total[..., None]).view(-1, end) @ v).view(q.shape)
            lse[rows, head * group:(head + 1) * group] = total
    return [y, lse]


def _exact_verify(s):
    """One sequence after the other, as the rule is told."""
    c, cu, parents = s["case"], s["cu"].tolist(), _parents(s["case"])
    tokens, numbers = s["tokens"].tolist(), s["uniforms"].double().tolist()
    counts, paths, said = [], [], []
    for b in range(c["bt"]):
        first, n = cu[b], cu[b + 1] - cu[b]

        def chances(x):
            if c["temperature"] == 0:
                p = torch.zeros(c["vocab"], dtype=torch.float64, device=DEV)
                p[int((x == x.max()).nonzero()[0, 0])] = 1.0
                return p
            return torch.softmax(x.double() / c["temperature"], 0)

        at, path = 0, [0]
        while True:
            p, none = chances(s["logits"][first + at]), True
            for j in range(at + 1, n):
                if parents[first + j] != at:
                    continue
                x, u = tokens[first + j], numbers[first + j]
                if s["draft"] is not None and c["temperature"] > 0:
                    e = chances(s["draft"][first + at])
                    if u * float(e[x]) < float(p[x]):
                        none = False
                        break
                    p = (p - e).clamp(min=0.0)
                else:
                    if u * float(p.sum()) < float(p[x]):
                        none = False
                        break
                    p[x] = 0.0
            if none:
                break
            at = j
            path.append(j)
        sums = p.cumsum(0)
        drawn = int((sums > numbers[first] * sums[-1]).nonzero()[0, 0])
        counts.append(len(path))
        paths.append(path + [-1] * (c["q"] - len(path)))
        said.append([tokens[first + j] for j in path[1:]] + [drawn] + [-1] * (c["q"] - len(path)))
    return [_i32(counts), _i32(paths), _i32(said)]


def _exact_keep(s):
    """Page by page: read what is accepted, write it where it goes."""
    layers, count, h, _, p, d = s["pages"].shape
    where = _offsets(p, d)
    pages, scales = s["pages"].double().view(layers, count, h, 2, p * d), s["scales"].double()
    table, lengths, refs, cu = s["table"].tolist(), s["lengths"].tolist(), s["refs"].tolist(), s["cu"].tolist()
    for b, path in enumerate(_paths(s["case"])):
        start = lengths[b] - (cu[b + 1] - cu[b])
        took = []
        for i, j in enumerate(path):
            if i != j:
                at, t = table[b][(start + j) // p], (start + j) % p
                x = torch.stack([pages[:, at, :, kv][:, :, where[kv][t]] * scales[:, at, :, kv, None] for kv in (0, 1)], 2)
                took.append((table[b][(start + i) // p], (start + i) % p, x))
        for page in sorted({t[0] for t in took}):
            mine = [t for t in took if t[0] == page]
            top = torch.stack([x.abs().amax(3) for _, _, x in mine]).amax(0)
            grown = torch.maximum(scales[:, page], _holding(top))
            pages[:, page] = _round8(pages[:, page] * (scales[:, page] / grown)[..., None])
            scales[:, page] = grown
            for _, t, x in mine:
                for kv in (0, 1):
                    pages[:, page, :, kv, where[kv][t]] = _round8(x[:, :, kv] / grown[:, :, kv, None])
        lengths[b] = start + len(path)
        for j in range(-(-lengths[b] // p), len(table[b])):
            if table[b][j] >= 0:
                refs[table[b][j]] -= 1
                table[b][j] = -1
    return [_i32(table), _i32(lengths), _i32(refs), pages.view(s["pages"].shape), scales]
