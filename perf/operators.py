"""The serving operators whose speed this repository answers for: the 8-bit paged cache of keys and values, the
attention that reads it, the bookkeeping of its pages, and the log probabilities that decide which sequences go on.

With `own` false, run() computes an operator in its plain form, from elementary torch operations in 32 bits; with
`own` true it makes the calls that a user makes of bsa_mi355x.

op        what is called (own)
append    kv_append: new keys and values quantised into the cache's pages
attend    kv_attention: attention of the newest `q` tokens of every sequence over its cached tokens
beam      pages_fork + pages_extend: sequences go on from chosen beams, each with room for one token more
retire    pages_free + pages_compact: finished sequences leave, the pool is made dense again
score     token_logprobs: log probabilities of given tokens, entropies and the k best alternatives

The cache of one layer is pages [pages, heads, 2, P, D] in e4m3, keys then values, with scales [pages, heads, 2], powers
of two; page_table [sequences, pages each] names a sequence's pages.  Inside [P, D] lie tiles of 16 tokens x 64 channels:
keys as [tile, c, g, t, e] (token 16 tile + t, channel 64c + 16g + e), values as [tile, c, g, l, i, t] (token 16 tile + 4g
+ t, channel 64c + 16i + l).
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


def _bsa():
    root = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "towards-batched-activation-sparsity_amd")
    if root not in sys.path:
        sys.path.insert(0, root)
    import bsa_mi355x

    return bsa_mi355x


def _kv(name, op, bt, q, hq, hkv, d, page, length, dtype):
    return {"name": name, "op": op, "bt": bt, "q": q, "hq": hq, "hkv": hkv, "d": d, "page": page, "len": length, "dtype": dtype}


def _pool(name, op, groups, width, layers, hkv, d, page, length):
    return {"name": name, "op": op, "groups": groups, "width": width, "layers": layers, "hkv": hkv, "d": d, "page": page,
            "len": length}


def _score(name, rows, vocab, k, dtype):
    return {"name": name, "op": "score", "rows": rows, "vocab": vocab, "k": k, "dtype": dtype}


def listed():
    return [
        # one token of each of 64 sequences into a layer's cache: every decode step, every layer
        _kv("append_b64", "append", 64, 1, 32, 32, 128, 16, 1000, "fp16"),
        # four prompts of up to 2000 tokens after what was cached of them, a bf16 model with shared heads
        _kv("append_prompt", "append", 4, 2000, 32, 8, 128, 64, 2500, "bf16"),
        # one sequence decoding: latency
        _kv("attend_b1", "attend", 1, 1, 32, 32, 128, 16, 777, "fp16"),
        # the decode batch of the step of linears, contexts of up to 4096 tokens
        _kv("attend_b64", "attend", 64, 1, 32, 32, 128, 16, 4096, "fp16"),
        # few long contexts, four query heads to a cached head
        _kv("attend_long", "attend", 5, 1, 32, 8, 128, 64, 60001, "bf16"),
        # 64 sequences checking 4 drafted tokens each
        _kv("attend_draft", "attend", 64, 4, 32, 32, 128, 32, 1500, "fp16"),
        # prompts, a part of each already cached
        _kv("attend_prompt", "attend", 3, 2000, 32, 8, 128, 64, 2800, "fp16"),
        # a step of beam search: 8 prompts x 8 beams
        _pool("beam_b64", "beam", 8, 8, 4, 32, 128, 16, 300),
        # half of 48 sequences are done: their pages are freed and the pool made dense
        _pool("retire_b48", "retire", 24, 2, 4, 32, 128, 16, 700),
        # the logits of a decode step at 64 sequences with 8 alternatives
        _score("score_b64", 64, 32000, 8, "fp16"),
        # every token of a prompt scored, one alternative
        _score("score_prompt", 4000, 32000, 1, "bf16"),
        # a large odd vocabulary, 32-bit logits, 20 alternatives
        _score("score_odd", 7, 100003, 20, "fp32"),
    ]


def _log(rng, lo, hi):
    return int(round(lo * (hi / lo) ** rng.random()))


def draw(rng):
    op = rng.choice(["append", "append", "attend", "attend", "attend", "attend", "beam", "retire", "score", "score"])
    dtype = rng.choice(["fp16", "bf16"])
    page, d = rng.choice([16, 16, 32, 64, 128]), rng.choice([64, 128, 128])
    hq, hkv = rng.choice([(32, 32), (32, 8), (16, 16), (40, 8), (28, 4), (8, 1)])
    if op == "append":
        bt, q = (_log(rng, 1, 64), rng.choice([1, 1, 4])) if rng.random() < 0.5 else (_log(rng, 1, 4), _log(rng, 20, 2000))
        return _kv("", op, bt, q, hq, hkv, d, page, q + _log(rng, 10, 1000), dtype)
    if op == "attend":
        kind = rng.choice(["decode", "decode", "draft", "prompt"])
        if kind == "prompt":
            q = _log(rng, 50, 2000)
            return _kv("", op, rng.randint(1, 3), q, hq, hkv, d, page, q + rng.choice([0, _log(rng, 1, 1000)]), dtype)
        bt = _log(rng, 1, 64)
        length = _log(rng, 8, max(16, min(60000, 200000 // bt)))
        return _kv("", op, bt, min(length, rng.randint(2, 8)) if kind == "draft" else 1, hq, hkv, d, page, length, dtype)
    if op in ("beam", "retire"):
        return _pool("", op, _log(rng, 2, 16), rng.randint(2, 4), rng.randint(1, 3), rng.choice([8, 16]), d, page,
                     _log(rng, 40, 600))
    return _score("", _log(rng, 1, 4000), _log(rng, 1000, 32000), rng.choice([0, 1, 5, 8, 20, 50]),
                  rng.choice(["fp16", "bf16", "fp32"]))


# ------------------------------------------------------------------------------------------------ inputs


def _spread(lo, hi, n, salt):
    """n whole numbers between lo and hi, the last of them hi: lengths of a batch, the same for every seed."""
    r = random.Random(7919 * hi + 31 * n + salt)
    return [r.randint(lo, hi) for _ in range(n - 1)] + [hi]


def _lengths(c):
    """Tokens of each sequence with its new ones, and how many are new."""
    new = [1] * c["bt"] if c["q"] == 1 else [c["q"]] * c["bt"] if c["q"] <= 8 else _spread(max(1, c["q"] // 2), c["q"], c["bt"], 1)
    old = _spread((c["len"] - c["q"]) // 4, c["len"] - c["q"], c["bt"], 2)
    return [a + b for a, b in zip(old, new)], new


def _power(e):
    """2 to whole exponents, in 32 bits."""
    return ((e.to(torch.int32) + 127) << 23).view(torch.float32)


def _i32(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def _cache(g, layers, pages, heads, page, d):
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
    most = max(per) + 1
    pages, scales = _cache(g, 1, sum(per) + 8, c["hkv"], c["page"], c["d"])
    ids = torch.randperm(sum(per) + 8, generator=g, device=DEV).to(torch.int32)
    table = torch.full((c["bt"], most), -1, dtype=torch.int32, device=DEV)
    at = 0
    for b, n in enumerate(per):
        table[b, :n] = ids[at:at + n]
        at += n
    cu = [0]
    for n in new:
        cu.append(cu[-1] + n)
    s = {"case": c, "pages": pages[0], "scales": scales[0], "table": table, "lengths": _i32(total), "cu": _i32(cu)}
    t, dt = cu[-1], DTYPES[c["dtype"]]
    if c["op"] == "append":
        # tokens of unequal strength: now and then a block's scale has to grow
        loud = torch.exp(0.5 * torch.randn(t, c["hkv"], 1, generator=g, device=DEV))
        s["k"] = (torch.randn(t, c["hkv"], c["d"], generator=g, device=DEV) * loud).to(dt)
        s["v"] = torch.randn(t, c["hkv"], c["d"], generator=g, device=DEV).to(dt)
    else:
        s["q"] = torch.randn(t, c["hq"], c["d"], generator=g, device=DEV).to(dt)
    return s


def _pool_state(c, g):
    """`groups` prompts, `width` sequences on each, which share the pages that the prompt fills."""
    n, p = c["groups"] * c["width"], c["page"]
    total = _spread(max(1, c["len"] // 3), c["len"], c["groups"], 3)
    shared = [t // 2 // p for t in total]
    private = [-(-t // p) - k for t, k in zip(total, shared)]
    used = sum(k + c["width"] * w for k, w in zip(shared, private))
    count = used + used // 4 + n
    pages, scales = _cache(g, c["layers"], count, c["hkv"], p, c["d"])
    ids = torch.randperm(count, generator=g, device=DEV).to(torch.int32)
    most = max(k + w for k, w in zip(shared, private)) + 2
    table = torch.full((n, most), -1, dtype=torch.int32, device=DEV)
    refs = torch.zeros(count, dtype=torch.int32, device=DEV)
    at = 0
    for i, (k, w) in enumerate(zip(shared, private)):
        rows = slice(i * c["width"], (i + 1) * c["width"])
        table[rows, :k] = ids[at:at + k]
        refs[ids[at:at + k].long()] = c["width"]
        at += k
        own_pages = ids[at:at + w * c["width"]]
        table[rows, k:k + w] = own_pages.view(c["width"], w)
        refs[own_pages.long()] = 1
        at += w * c["width"]
    lengths = _i32([t for t in total for _ in range(c["width"])])
    s = {"case": c, "pages": pages, "scales": scales, "table": table, "lengths": lengths, "refs": refs,
         "before": [table.clone(), lengths.clone(), refs.clone()]}
    if c["op"] == "beam":
        base = torch.arange(c["groups"], device=DEV).repeat_interleave(c["width"]) * c["width"]
        s["children"] = torch.arange(n, device=DEV).to(torch.int32)
        s["parents"] = (base + torch.randint(0, c["width"], (n,), generator=g, device=DEV)).to(torch.int32)
        s["new"] = torch.ones(n, dtype=torch.int32, device=DEV)
    else:
        s["done"] = torch.randperm(n, generator=g, device=DEV)[: n // 2].to(torch.int32)
    return s


def _score_state(c, g):
    x = torch.randn(c["rows"], c["vocab"], generator=g, device=DEV).mul_(2.0)
    for _ in range(3):  # a few likely tokens in each row
        at = torch.randint(0, c["vocab"], (c["rows"], 1), generator=g, device=DEV)
        x.scatter_add_(1, at, 6.0 + 2.0 * torch.randn(c["rows"], 1, generator=g, device=DEV))
    pick = torch.randint(0, c["vocab"], (c["rows"],), generator=g, device=DEV)
    likely = torch.rand(c["rows"], generator=g, device=DEV) < 0.7
    return {"case": c, "logits": x.to(DTYPES[c["dtype"]]), "tokens": torch.where(likely, at[:, 0], pick).to(torch.int32)}


def prepare(case, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    c = dict(case)
    return (_score_state if c["op"] == "score" else _pool_state if c["op"] in ("beam", "retire") else _kv_state)(c, g)


# ------------------------------------------------------------------------------------------------ one pass


def run(state):
    op = state["case"]["op"]
    if op in ("beam", "retire"):
        # the pool as it was before the step, so that every pass has the same work
        for name, was in zip(("table", "lengths", "refs"), state["before"]):
            state[name].copy_(was)
    return (_RUN_OWN if own else _RUN_PLAIN)[op](state)


def _own_append(s):
    _bsa().kv_append(s["k"], s["v"], s["pages"], s["scales"], s["table"], s["lengths"], cu_seqlens=s["cu"], max_new=s["case"]["q"])
    return [s["pages"], s["scales"]]


def _own_attend(s):
    return list(_bsa().kv_attention(s["q"], s["pages"], s["scales"], s["table"], s["lengths"], cu_seqlens=s["cu"],
                                    max_new=s["case"]["q"]))


def _own_beam(s):
    bsa = _bsa()
    bsa.pages_fork(s["table"], s["lengths"], s["refs"], s["parents"], s["children"])
    served = bsa.pages_extend(s["pages"], s["scales"], s["table"], s["lengths"], s["refs"], s["new"])
    return [s["table"], s["lengths"], s["refs"], served, s["pages"], s["scales"]]


def _own_retire(s):
    bsa = _bsa()
    bsa.pages_free(s["table"], s["lengths"], s["refs"], s["done"])
    counts = bsa.pages_compact(s["pages"], s["scales"], s["table"], s["refs"])
    return [s["table"], s["lengths"], s["refs"], counts, s["pages"], s["scales"]]


def _own_score(s):
    return list(_bsa().token_logprobs(s["logits"], s["tokens"], k=s["case"]["k"]))


_RUN_OWN = {"append": _own_append, "attend": _own_attend, "beam": _own_beam, "retire": _own_retire, "score": _own_score}


def _key_tiles(pages):
    """[pages, heads, tile, c, g, t, e] of the keys; the values as [pages, heads, tile, c, g, l, i, t] below."""
    n, h, _, p, d = pages.shape
    return pages.view(n, h, 2, p // 16, d // 64, 4, 16, 16)[:, :, 0]


def _value_tiles(pages):
    n, h, _, p, d = pages.shape
    return pages.view(n, h, 2, p // 16, d // 64, 4, 16, 4, 4)[:, :, 1]


def _e4m3(x):
    """To the nearest e4m3 value, as bytes; past the largest one to that."""
    return x.clamp(-448.0, 448.0).to(F8).view(torch.uint8)


def _token_rows(cu, total):
    """Which sequence each of the new tokens belongs to."""
    return torch.searchsorted(cu[1:].long(), torch.arange(total, device=DEV), right=True)


def _plain_append(s):
    pages, scales, table, lengths, cu = s["pages"], s["scales"], s["table"], s["lengths"].long(), s["cu"].long()
    n, h, _, p, d = pages.shape
    x = torch.stack([s["k"], s["v"]], 2).float()  # [T, heads, 2, D]
    row = _token_rows(s["cu"], x.shape[0])
    start = lengths - (cu[1:] - cu[:-1])
    pos = start[row] + torch.arange(x.shape[0], device=DEV) - cu[row]
    page = table[row, pos // p].long()
    # the largest magnitude of the new tokens of each page, and the power of two that holds it
    top = torch.where(torch.isfinite(x), x.abs(), 0.0).amax(3)
    most = torch.zeros(n, h, 2, device=DEV).index_reduce_(0, page, top, "amax")
    m, e = torch.frexp(most)
    need = torch.where(most > 0, _power(e - 9 + (m > 0.875)).clamp(SCALE_LOW, SCALE_HIGH), SCALE_LOW)
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
    return [pages, scales]


def _plain_attend(s):
    q, pages, scales, lengths, cu = s["q"], s["pages"], s["scales"], s["lengths"].long(), s["cu"].long()
    _, h, _, p, d = pages.shape
    t, hq, _ = q.shape
    b, most = s["table"].shape
    ids = s["table"].clamp(min=0).long()
    keys = _key_tiles(pages)[ids].float().permute(0, 2, 1, 3, 6, 4, 5, 7).reshape(b, h, most, p, d)
    values = _value_tiles(pages)[ids].float().permute(0, 2, 1, 3, 5, 8, 4, 7, 6).reshape(b, h, most, p, d)
    by = scales[ids].permute(0, 2, 1, 3)[..., None, None]
    keys, values = (keys * by[:, :, :, 0]).view(b, h, most * p, d), (values * by[:, :, :, 1]).view(b, h, most * p, d)
    seen = torch.arange(most * p, device=DEV)
    values = torch.where((seen < lengths[:, None])[:, None, :, None], values, 0.0)
    # the new tokens of a sequence beside each other, the heads of a group under their cached head
    row = _token_rows(s["cu"], t)
    new, i = cu[1:] - cu[:-1], torch.arange(t, device=DEV) - cu[row]
    wide = torch.zeros(b, s["case"]["q"], hq, d, device=DEV)
    wide[row, i] = q.float()
    wide = wide.view(b, -1, h, hq // h, d).permute(0, 2, 1, 3, 4).reshape(b, h, -1, d)
    x = torch.matmul(wide, keys.transpose(2, 3)).mul_(d ** -0.5)
    last = (lengths - new)[:, None] + torch.arange(s["case"]["q"], device=DEV).repeat_interleave(hq // h)
    x.masked_fill_((seen[None, None] > last[:, :, None])[:, None], float("-inf"))
    top = x.amax(3, keepdim=True)
    top = torch.where(torch.isfinite(top), top, 0.0)
    x.sub_(top).exp_()
    total = x.sum(3, keepdim=True)
    y = torch.matmul(x, values) / torch.where(total > 0, total, 1.0)
    y = y.view(b, h, -1, hq // h, d).permute(0, 2, 1, 3, 4).reshape(b, -1, hq, d)
    lse = (top + torch.log(total)).view(b, h, -1, hq // h).permute(0, 2, 1, 3).reshape(b, -1, hq)
    return [y[row, i].to(q.dtype), lse[row, i]]


def _count(refs, ids, by):
    """Adds `by` to the counts of the pages that `ids` names (-1 names none)."""
    ids = ids.reshape(-1).long()
    refs.index_add_(0, ids.clamp(min=0), torch.where(ids >= 0, by, 0).to(refs.dtype))


def _plain_beam(s):
    pages, scales, table, lengths, refs = s["pages"], s["scales"], s["table"], s["lengths"], s["refs"]
    p = pages.shape[4]
    children, parents = s["children"].long(), s["parents"].long()
    _count(refs, table[children], -1)
    _count(refs, table[parents], 1)
    table[children], lengths[children] = table[parents], lengths[parents]
    # room for the new tokens: fresh pages, and a copy of a last page that others go on reading
    n, most = table.shape
    have, want = -(-lengths // p), -(-(lengths + s["new"]) // p)
    tail = table.gather(1, (have - 1).clamp(min=0).long()[:, None])[:, 0]
    inside = (lengths % p != 0) & (s["new"] > 0)
    row = torch.arange(n, device=DEV)
    fits = want <= most
    earlier = ((tail[:, None] == tail[None]) & (inside & fits)[None] & (row[None] < row[:, None])).sum(1)
    readers = torch.where(inside, refs[tail.clamp(min=0).long()], 1)
    split = fits & inside & (readers - earlier > 1)
    need = torch.where(fits, want - have + split, 0)
    until = need.cumsum(0)
    served = fits & ((until <= (refs == 0).sum()) | ((need == 0) & (readers == 1)))
    free = torch.argsort((refs > 0).to(torch.int8), stable=True)
    first = until - need
    moves = split & served
    src, dst = tail[moves].long(), free[first[moves]]
    pages.view(torch.uint8)[:, dst] = pages.view(torch.uint8)[:, src]
    scales[:, dst] = scales[:, src]
    refs.index_add_(0, src, torch.full_like(src, -1, dtype=refs.dtype))
    refs[dst] = 1
    table[moves, have[moves].long() - 1] = dst.to(torch.int32)
    slot = torch.arange(most, device=DEV)
    fresh = served[:, None] & (slot >= have[:, None]) & (slot < want[:, None])
    at = ((first + split)[:, None] + slot - have[:, None])[fresh]
    table[fresh] = free[at].to(torch.int32)
    refs[free[at]] = 1
    lengths.add_(torch.where(served, s["new"], 0))
    return [table, lengths, refs, served.to(torch.int32), pages, scales]


def _plain_retire(s):
    pages, scales, table, lengths, refs = s["pages"], s["scales"], s["table"], s["lengths"], s["refs"]
    done = s["done"].long()
    _count(refs, table[done], -1)
    table[done] = -1
    lengths[done] = 0
    # the highest live pages into the lowest free ones, until the live ones are the first of the pool
    live = refs > 0
    count = live.sum()
    ids = torch.arange(len(refs), device=DEV)
    src, dst = ids[live & (ids >= count)], ids[~live & (ids < count)]
    to = ids.clone()
    to[src] = dst
    pages.view(torch.uint8)[:, dst] = pages.view(torch.uint8)[:, src]
    scales[:, dst] = scales[:, src]
    refs[dst] = refs[src]
    refs[src] = 0
    table.copy_(torch.where(table >= 0, to[table.clamp(min=0).long()], -1))
    moved = torch.full_like(count, len(src))
    return [table, lengths, refs, torch.stack([count, moved]).to(torch.int32), pages, scales]


def _plain_score(s):
    x, k = s["logits"].float(), s["case"]["k"]
    top = x.amax(1, keepdim=True)
    e = torch.exp(x - top)
    total = e.sum(1, keepdim=True)
    lse = top + torch.log(total)
    logprob = (x.gather(1, s["tokens"].long()[:, None]) - lse)[:, 0]
    entropy = (torch.log(total) - (e * (x - top)).sum(1, keepdim=True) / total)[:, 0]
    best = torch.argsort(x, dim=1, descending=True, stable=True)[:, :k]
    return [logprob, entropy, best.to(torch.int32), x.gather(1, best) - lse]


_RUN_PLAIN = {"append": _plain_append, "attend": _plain_attend, "beam": _plain_beam, "retire": _plain_retire,
              "score": _plain_score}


# ------------------------------------------------------------------------------------------------ what a pass cannot do without


def work(case):
    c = case
    if c["op"] == "score":
        size = 4 if c["dtype"] == "fp32" else 2
        return {"bytes": float(c["rows"]) * (c["vocab"] * size + 4 + 8 + 8 * c["k"]), "flops": 4.0 * c["rows"] * c["vocab"]}
    if c["op"] in ("beam", "retire"):
        n, p = c["groups"] * c["width"], c["page"]
        page = 2.0 * c["layers"] * c["hkv"] * (2 * p * c["d"] + 8)  # read and written
        total = _spread(max(1, c["len"] // 3), c["len"], c["groups"], 3)
        own_pages, shared = [-(-t // p) - t // 2 // p for t in total], [t // 2 // p for t in total]
        used = sum(k + c["width"] * w for k, w in zip(shared, own_pages))
        count = used + used // 4 + n
        if c["op"] == "beam":
            twice = c["width"] - c["width"] * (1 - (1 - 1.0 / c["width"]) ** c["width"])  # beams whose parent has another child
            copied = twice * sum(t % p != 0 for t in total)
        else:
            left = sum(0.75 * k + c["width"] * 0.5 * w for k, w in zip(shared, own_pages)) if c["width"] == 2 else 0.5 * used
            copied = left * (count - left) / count
        return {"bytes": copied * page + 8.0 * n * (max(own_pages) + max(shared)) + 8.0 * count, "flops": 0.0}
    total, new = _lengths(c)
    t = sum(new)
    if c["op"] == "append":
        return {"bytes": float(t) * c["hkv"] * 2 * c["d"] * 3, "flops": 4.0 * t * c["hkv"] * c["d"]}
    held = sum(n * 2 * c["d"] + -(-n // c["page"]) * 8 for n in total) * float(c["hkv"])
    pairs = sum(n * m - m * (m - 1) / 2 for n, m in zip(total, new))
    return {"bytes": held + t * c["hq"] * (4.0 * c["d"] + 4), "flops": 4.0 * c["d"] * c["hq"] * pairs}


# ------------------------------------------------------------------------------------------------ the definition in 64 bits


def exact(case, seed):
    s = prepare(case, seed)
    return {"append": _exact_append, "attend": _exact_attend, "beam": _exact_beam, "retire": _exact_retire,
            "score": _exact_score}[case["op"]](s)


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


def _exact_append(s):
    n, h, _, p, d = s["pages"].shape
    where = _offsets(p, d)
    pages, scales = s["pages"].double().view(n, h, 2, p * d), s["scales"].double()
    lengths, cu, table = s["lengths"].tolist(), s["cu"].tolist(), s["table"].tolist()
    for b, end in enumerate(lengths):
        pos = start = end - (cu[b + 1] - cu[b])
        while pos < end:
            j, stop = pos // p, min(end, (pos // p + 1) * p)
            at, k = table[b][j], cu[b] + pos - start
            for i, x in enumerate((s["k"], s["v"])):
                x = x[k:k + stop - pos].double().transpose(0, 1)  # [heads, tokens, D]
                need = torch.exp2(torch.ceil(torch.log2(x.abs().amax((1, 2)) / 448.0))).clamp(SCALE_LOW, SCALE_HIGH)
                if pos % p:
                    old = scales[at, :, i].clone()
                    need = torch.maximum(need, old)
                    o = where[i][: pos % p].reshape(-1)
                    pages[at, :, i, o] = _round8(pages[at, :, i, o] * (old / need)[:, None])
                scales[at, :, i] = need
                pages[at, :, i, where[i][pos - j * p:stop - j * p].reshape(-1)] = _round8(x / need[:, None, None]).reshape(h, -1)
            pos = stop
    return [pages.view(n, h, 2, p, d), scales]


def _exact_attend(s):
    n, h, _, p, d = s["pages"].shape
    where = _offsets(p, d)
    group = s["q"].shape[1] // h
    raw = s["pages"].view(n, h, 2, p * d)
    lengths, cu = s["lengths"].tolist(), s["cu"].tolist()
    y, lse = torch.zeros(s["q"].shape, dtype=torch.float64, device=DEV), torch.zeros(s["q"].shape[:2], dtype=torch.float64, device=DEV)
    for b, end in enumerate(lengths):
        ids = s["table"][b, : -(-end // p)].long()
        new = cu[b + 1] - cu[b]
        for head in range(h):
            one = raw[ids, head].double() * s["scales"][ids, head].double()[..., None]
            k, v = (one[:, i, where[i].reshape(-1)].view(-1, d)[:end] for i in (0, 1))
            for first in range(0, new, 512):
                rows = slice(cu[b] + first, min(cu[b] + first + 512, cu[b + 1]))
                q = s["q"][rows, head * group:(head + 1) * group].double()
                x = (q.reshape(-1, d) @ k.t() / d ** 0.5).view(q.shape[0], group, end)
                last = end - new + first + torch.arange(q.shape[0], device=DEV)
                x.masked_fill_((torch.arange(end, device=DEV)[None] > last[:, None])[:, None], float("-inf"))
                total = torch.logsumexp(x, 2)
                y[rows, head * group:(head + 1) * group] = (torch.exp(x - total[..., None]).view(-1, end) @ v).view(q.shape)
                lse[rows, head * group:(head + 1) * group] = total
    return [y, lse]


def _exact_beam(s):
    """The step as a scheduler on the host would take it, one sequence after the other."""
    p = s["pages"].shape[4]
    table, lengths, refs = s["table"].tolist(), s["lengths"].tolist(), s["refs"].tolist()
    was, long = [list(r) for r in table], list(lengths)
    for child, parent in zip(s["children"].tolist(), s["parents"].tolist()):
        for at in was[child]:
            refs[at] -= at >= 0
        for at in was[parent]:
            refs[at] += at >= 0
        table[child], lengths[child] = list(was[parent]), long[parent]
    pages, scales = s["pages"].double(), s["scales"].double()
    free = [i for i, r in enumerate(refs) if r == 0]
    asked, served, was_free, readers = 0, [], len(free), list(refs)
    for b, new in enumerate(s["new"].tolist()):
        have, want = -(-lengths[b] // p), -(-(lengths[b] + new) // p)
        tail, fits = table[b][have - 1], want <= len(table[b])
        inside = new > 0 and lengths[b] % p != 0
        split = inside and refs[tail] > 1
        need = (want - have + split) * fits
        asked += need
        ok = fits and (asked <= was_free or need == 0 and not (inside and readers[tail] > 1))
        served.append(int(ok))
        if not ok:
            continue
        if split:
            at = free.pop(0)
            pages[:, at], scales[:, at] = pages[:, tail], scales[:, tail]
            refs[tail] -= 1
            refs[at], table[b][have - 1] = 1, at
        for j in range(have, want):
            table[b][j] = free.pop(0)
            refs[table[b][j]] = 1
        lengths[b] += new
    return [_i32(table), _i32(lengths), _i32(refs), _i32(served), pages, scales]


def _exact_retire(s):
    table, lengths, refs = s["table"].tolist(), s["lengths"].tolist(), s["refs"].tolist()
    for b in s["done"].tolist():
        for at in table[b]:
            refs[at] -= at >= 0
        table[b], lengths[b] = [-1] * len(table[b]), 0
    live = sum(r > 0 for r in refs)
    pages, scales = s["pages"].double(), s["scales"].double()
    to = {}
    gaps = [i for i in range(live) if refs[i] == 0]
    for at in range(live, len(refs)):
        if refs[at] > 0:
            to[at] = gaps.pop(0)
            pages[:, to[at]], scales[:, to[at]] = pages[:, at], scales[:, at]
            refs[to[at]], refs[at] = refs[at], 0
    table = [[to.get(at, at) for at in r] for r in table]
    return [_i32(table), _i32(lengths), _i32(refs), _i32([live, len(to)]), pages, scales]


def _exact_score(s):
    k, out = s["case"]["k"], []
    for first in range(0, s["logits"].shape[0], 512):
        x = s["logits"][first:first + 512].double()
        logp = torch.log_softmax(x, 1)
        best = x.sort(dim=1, descending=True, stable=True)[1][:, :k]
        out.append([logp.gather(1, s["tokens"][first:first + 512].long()[:, None])[:, 0], -(logp.exp() * logp).sum(1),
                    best.to(torch.int32), logp.gather(1, best)])
    return [torch.cat(v) for v in zip(*out)]
