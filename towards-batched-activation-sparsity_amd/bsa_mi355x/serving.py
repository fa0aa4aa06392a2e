"""What a decode loop needs beside its linears: a paged cache of keys and values held in 8 bits, the
attention that reads it, the bookkeeping of its pages, and the log probabilities of tokens.

    kv_append       new keys and values into the cache, a scale for each page, head and K/V
    kv_attention    attention of each sequence's newest tokens over its cached ones
    pages_fork      sequences go on from others and share their pages
    pages_extend    room for new tokens; a shared last page is copied before it is written to
    pages_free      finished sequences release their pages
    pages_compact   the live pages become the first of the pool
    pages_copy      whole pages copied
    token_logprobs  log probabilities of given tokens, entropies and the likeliest alternatives
    KVCache         the tensors of a cache of several layers, and these calls as its methods

All of it runs on the device with no host round trip (csrc/kv_append.hip, kv_attention.hip, pages.hip,
logprobs.hip through include/bsgserve.h), on torch's current stream, and can be captured.  The
reference leaves attention and cache to the model's own library, so these have no counterpart there.

Layout.  pages is [layers, pages, heads, 2, page_size, head_dim] in torch.float8_e4m3fn, keys then
values, in tile order inside [page_size, head_dim] (include/bsgserve.h; `read_pages` gives plain
numbers); scales is fp32 [layers, pages, heads, 2], powers of two.  page_table int32 [slots, pages
each] names the pages of a sequence in order (-1 none), lengths int32 [slots] its tokens, refcounts
int32 [pages] how many table entries name a page.
"""
from __future__ import annotations

import threading
from operator import index as _index
from typing import Dict, NamedTuple, Optional, Tuple

import torch

from . import _lib
from ._lib import check, load
from .runtime import _cu_count, _dtype_code, _require_cuda

PAGE_SIZES = (16, 32, 64, 128)
HEAD_DIMS = (64, 128)
COUNTER_BYTES = 65536  # BSG_KV_COUNTER_BYTES
MAX_ROWS = 1024  # BSG_PAGES_MAX_ROWS
MAX_ALTERNATIVES = 64  # BSG_LOGPROBS_MAX_K

_F8 = torch.float8_e4m3fn
_WORKSPACES: Dict[tuple, list] = {}  # by (device, prefix)
_OF_THREAD = threading.local()  # its attributes by (device, stream)


# What a call's shapes, strides, types and devices decide (the checks, the sizes, the library's
# fixed arguments) is worked out once for each such signature; addresses and values come with each call.
_CALLS: Dict[tuple, tuple] = {}
_CALLS_MAX = 4096


def _sigs(*tensors: Optional[torch.Tensor]) -> tuple:
    return tuple([t if t is None else (t.shape, t.stride(), t.dtype, t.get_device()) for t in tensors])


def _remember(key: tuple, call: tuple) -> tuple:
    if len(_CALLS) >= _CALLS_MAX:
        _CALLS.clear()
    _CALLS[key] = call
    return call


def _ptr(t: Optional[torch.Tensor]) -> int:
    return 0 if t is None else t.data_ptr()


_MOLDS: Dict[tuple, torch.Tensor] = {}


def _mold(shape, dtype: torch.dtype, dev: torch.device) -> torch.Tensor:
    """A tensor of this shape over one element, for torch.empty_like: a contiguous tensor of the shape
    at half of what torch.empty costs from Python."""
    one = _MOLDS.get((dtype, dev))
    if one is None:
        one = _MOLDS[dtype, dev] = torch.empty(1, dtype=dtype, device=dev)
    return one.expand(shape)


def _launch(index: int, fn, *args) -> None:
    """fn(*args, the current stream of device `index`), with that device current."""
    if torch._C._cuda_getDevice() == index:
        status = fn(*args, torch._C._cuda_getCurrentRawStream(index))
    else:
        with torch.cuda.device(index):
            status = fn(*args, torch._C._cuda_getCurrentRawStream(index))
    if status != _lib.BSG_OK:
        check(status)


def _workspace(index: int, nbytes: int, prefix: Optional[str], cleared: bool = True) -> torch.Tensor:
    """At least `nbytes`, the first COUNTER_BYTES of them zero (the kernels leave them zero).

    Without a prefix an eager call takes the buffer that its thread has for its stream, which the
    thread's calls on that stream use in turn (another thread's could come between the two launches of
    a page plan), and a captured one a buffer of its own in the graph's memory, its counters cleared by
    the graph (where `cleared`): graphs may then replay beside each other.  With a prefix both take the
    prefix's buffer, and calls of several threads, or that may overlap, must not share one.  A buffer is
    never given back while a graph may hold it: a larger one is made beside it."""
    if torch._C._cuda_getDevice() != index:  # the capture asked for below is the current device's
        with torch.cuda.device(index):
            return _workspace(index, nbytes, prefix, cleared)
    if prefix is None:
        key, all_held = (index, torch._C._cuda_getCurrentRawStream(index)), _OF_THREAD.__dict__
    else:
        key, all_held = (index, prefix), _WORKSPACES
    if torch._C._cuda_isCurrentStreamCapturing():
        if prefix is None:
            ws = torch.empty(nbytes, dtype=torch.uint8, device=torch.device("cuda", index))
            if cleared:
                ws[:COUNTER_BYTES].zero_()
            return ws
        held = all_held.get(key)
        if not held or held[-1].numel() < nbytes:
            raise RuntimeError(f"workspace {prefix!r} is too small for this call: run it once before capturing it")
        return held[-1]
    held = all_held.setdefault(key, [])
    if not held or held[-1].numel() < nbytes:
        held.append(torch.zeros(1 << max(20, (nbytes - 1).bit_length()), dtype=torch.uint8, device=torch.device("cuda", index)))
    return held[-1]


def _i32(t: Optional[torch.Tensor], dev: torch.device, what: str, n: Optional[int] = None) -> int:
    """Address of a contiguous int32 tensor on `dev` (of n entries), or None's."""
    if t is None:
        return 0
    if t.dtype is not torch.int32:
        raise TypeError(f"{what} must be int32, got {t.dtype}")
    if t.device != dev:
        raise ValueError(f"{what} must be on {dev}, got {t.device}")
    if not t.is_contiguous():
        raise ValueError(f"{what} must be contiguous")
    if n is not None and t.numel() != n:
        raise ValueError(f"{what} has {t.numel()} entries, needs {n}")
    return t.data_ptr()


def _table(page_table: torch.Tensor, dev: torch.device) -> None:
    if page_table.dtype is not torch.int32:
        raise TypeError(f"page_table must be int32, got {page_table.dtype}")
    if page_table.dim() != 2 or page_table.device != dev:
        raise ValueError(f"page_table must be [slots, pages each] on {dev}, got {tuple(page_table.shape)} on {page_table.device}")
    if page_table.stride(1) != 1 or (page_table.shape[0] > 1 and page_table.stride(0) < page_table.shape[1]):
        raise ValueError(f"page_table rows must be contiguous, strides {page_table.stride()}")


def _storage(pages: torch.Tensor, scales: torch.Tensor, dims: int) -> torch.device:
    dev = _require_cuda(pages, scales)
    if pages.dtype is not _F8:
        raise TypeError(f"pages must be {_F8}, got {pages.dtype}")
    if scales.dtype is not torch.float32:
        raise TypeError(f"scales must be float32, got {scales.dtype}")
    if pages.dim() != dims or pages.shape[-3] != 2 or scales.shape != pages.shape[:-2]:
        lead = "layers, " if dims == 6 else ""
        raise ValueError(f"pages must be [{lead}pages, heads, 2, page_size, head_dim] with scales [{lead}pages, heads, 2], "
                         f"got {tuple(pages.shape)} and {tuple(scales.shape)}")
    if not pages.is_contiguous() or not scales.is_contiguous():
        raise ValueError("pages and scales must be contiguous")
    return dev


def _layer(pages: torch.Tensor, scales: torch.Tensor, page_table: torch.Tensor, lengths: torch.Tensor, layer: Optional[int]):
    """The device of one layer's tensors, the sizes of its bsg_kv_cache, and of pages and scales of
    several layers their number and the bytes from one to the next."""
    dev = _storage(pages, scales, 5 if layer is None else 6)
    _table(page_table, dev)
    n, h, _, p, d = pages.shape[-5:]
    slots, each = page_table.shape
    _i32(lengths, dev, "lengths", slots)
    steps = (1, 0, 0) if layer is None else (pages.shape[0], n * h * 2 * p * d, n * h * 2 * 4)
    return dev, (n, h, p, d, slots, each, page_table.stride(0) if slots > 1 else each), steps


def _from_end(i: int, layers: int) -> int:
    if not -layers <= i < layers:
        raise IndexError(f"layer {i} of {layers}")
    return i % layers


def _batch(x: torch.Tensor, what: str, heads: int, d: int, dev: torch.device, rows: int, cu, max_new) -> int:
    """Checks a [tokens, heads, head_dim] tensor of a batch; returns max_new."""
    if x.dim() != 3 or x.shape[2] != d or (heads and x.shape[1] != heads):
        raise ValueError(f"{what} must be [tokens, {heads or 'heads'}, {d}], got {tuple(x.shape)}")
    if x.device != dev:
        raise ValueError(f"{what} must be on {dev}, got {x.device}")
    if x.stride(2) != 1:
        raise ValueError(f"{what} must have contiguous channels, strides {x.stride()}")
    if cu is None:
        if rows and x.shape[0] % rows:
            raise ValueError(f"without cu_seqlens {what}'s {x.shape[0]} tokens must divide over {rows} sequences")
        per = x.shape[0] // rows if rows else 0
        if max_new is not None and max_new != per:
            raise ValueError(f"max_new={max_new}, but each of {rows} sequences has {per} tokens")
        return per
    return x.shape[0] if max_new is None else min(max_new, x.shape[0])


def _rows(slots: Optional[torch.Tensor], cu: Optional[torch.Tensor], lengths: torch.Tensor) -> int:
    if slots is not None:
        return slots.numel()
    return cu.numel() - 1 if cu is not None else lengths.numel()


def kv_append(k: torch.Tensor, v: torch.Tensor, pages: torch.Tensor, scales: torch.Tensor, page_table: torch.Tensor,
              lengths: torch.Tensor, cu_seqlens: Optional[torch.Tensor] = None, max_new: Optional[int] = None,
              slots: Optional[torch.Tensor] = None, layer: Optional[int] = None) -> None:
    """Write the new keys and values of a batch, [tokens, heads, head_dim] fp16/bf16, into one
    layer's pages.  Row b (slot slots[b], or b) has the tokens cu_seqlens[b] .. cu_seqlens[b+1], or an
    equal share of them; they are the last of its lengths, which already count them.

    Each page, head and K/V has one scale: the least power of two that brings its largest finite
    magnitude to 448 or below, and no less than the scale of tokens that the page held before (which
    are rounded again where it grows).  Infinities become +-448 x scale, NaN stays NaN.  max_new bounds
    the tokens of one sequence (default: all of them; a tight one makes a smaller launch); the ones past
    it are not written.  With
    `layer`, pages and scales are those of all layers, of which it names one."""
    if max_new is not None:
        max_new = int(max_new)  # a number, not a tensor that may change, in the signature
    key = ("append", _sigs(k, v, pages, scales, page_table, lengths, cu_seqlens, slots), max_new, layer is None)
    call = _CALLS.get(key)
    if call is None:
        dev, sizes, steps = _layer(pages, scales, page_table, lengths, layer)
        rows = _rows(slots, cu_seqlens, lengths)
        most = _batch(k, "k", sizes[1], sizes[3], dev, rows, cu_seqlens, max_new)
        _batch(v, "v", sizes[1], sizes[3], dev, rows, cu_seqlens, None if cu_seqlens is None else most)
        if v.dtype is not k.dtype or v.shape[0] != k.shape[0]:
            raise ValueError(f"k and v must match, got {tuple(k.shape)} {k.dtype} and {tuple(v.shape)} {v.dtype}")
        _i32(cu_seqlens, dev, "cu_seqlens", rows + 1)
        _i32(slots, dev, "slots")
        call = _remember(key, (dev.index, load().bsg_kv_append, sizes, rows, most, _dtype_code(k), k.stride(0), k.stride(1),
                               v.stride(0), v.stride(1), k.shape[0], *steps))
    index, fn, sizes, rows, most, code, kt, kh, vt, vh, tokens, layers, page_step, scale_step = call
    at, scales_at = pages.data_ptr(), scales.data_ptr()
    if layer is not None:
        i = _index(layer)
        if not 0 <= i < layers:
            i = _from_end(i, layers)
        at, scales_at = at + i * page_step, scales_at + i * scale_step
    cache = _lib.KvCache(at, scales_at, *sizes, page_table.data_ptr(), lengths.data_ptr())
    _launch(index, fn, k.data_ptr(), kt, kh, v.data_ptr(), vt, vh, tokens, cache, _ptr(slots), rows, _ptr(cu_seqlens), most, code)


def kv_attention(q: torch.Tensor, pages: torch.Tensor, scales: torch.Tensor, page_table: torch.Tensor,
                 lengths: torch.Tensor, cu_seqlens: Optional[torch.Tensor] = None, max_new: Optional[int] = None,
                 slots: Optional[torch.Tensor] = None, sm_scale: Optional[float] = None, max_len: Optional[int] = None,
                 out: Optional[torch.Tensor] = None, lse: Optional[torch.Tensor] = None,
                 workspace_prefix: Optional[str] = None,
                 layer: Optional[int] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """Attention of a batch's new tokens q, [tokens, query heads, head_dim] fp16/bf16, over one
    layer's cached tokens, their own (appended before) among them: token i of a sequence's n new ones sees the
    first length - n + i + 1 tokens.  Query head h reads cached head h // (query heads / heads).
    Returns (out like q, lse fp32 [tokens, query heads]); a token that sees nothing gets zeros and -inf.

    Rows, cu_seqlens, max_new and layer as kv_append (tokens past max_new are not computed); sm_scale is
    1 / sqrt(head_dim) by default.  max_len, the longest sequence (default: what a table row holds),
    decides how the long axis is split and bounds nothing.  q rows must be 16-byte aligned, out rows
    8-byte aligned."""
    if max_new is not None:
        max_new = int(max_new)
    if max_len is not None:
        max_len = int(max_len)
    key = ("attend", _sigs(q, pages, scales, page_table, lengths, cu_seqlens, slots, out, lse), max_new, max_len, layer is None)
    call = _CALLS.get(key)
    if call is None:
        call = _remember(key, _attention_call(q, pages, scales, page_table, lengths, cu_seqlens, max_new, slots, max_len, out, lse, layer))
    index, fn, sizes, rows, most, code, qt, qh, tokens, heads, out_mold, lse_mold, longest, need, cus, scale, layers, page_step, scale_step = call
    if out is None:
        out = torch.empty_like(out_mold)
    if lse is None:
        lse = torch.empty_like(lse_mold)
    at, scales_at = pages.data_ptr(), scales.data_ptr()
    if layer is not None:
        i = _index(layer)
        if not 0 <= i < layers:
            i = _from_end(i, layers)
        at, scales_at = at + i * page_step, scales_at + i * scale_step
    cache = _lib.KvCache(at, scales_at, *sizes, page_table.data_ptr(), lengths.data_ptr())
    ws, room = 0, 0
    if need > 0:
        held = _workspace(index, need, workspace_prefix)
        ws, room = held.data_ptr(), held.numel()
    _launch(index, fn, q.data_ptr(), qt, qh, tokens, heads, cache, _ptr(slots), rows, _ptr(cu_seqlens), most, longest,
            scale if sm_scale is None else sm_scale, out.data_ptr(), out.stride(0), out.stride(1), lse.data_ptr(), code, ws, room, cus)
    return out, lse


def _attention_call(q, pages, scales, page_table, lengths, cu_seqlens, max_new, slots, max_len, out, lse, layer) -> tuple:
    """The checks of kv_attention and what follows from its arguments' shapes."""
    dev, sizes, steps = _layer(pages, scales, page_table, lengths, layer)
    rows = _rows(slots, cu_seqlens, lengths)
    most = _batch(q, "q", 0, sizes[3], dev, rows, cu_seqlens, max_new)
    code = _dtype_code(q)
    tokens, heads, d = q.shape
    if out is not None and (out.shape != q.shape or out.dtype is not q.dtype or out.device != dev or out.stride(2) != 1):
        raise ValueError(f"out must match q {tuple(q.shape)} {q.dtype} with contiguous channels, got {tuple(out.shape)} {out.dtype}")
    if lse is not None and (lse.shape != q.shape[:2] or lse.dtype is not torch.float32 or lse.device != dev
                            or not lse.is_contiguous()):
        raise ValueError(f"lse must be contiguous float32 [{tokens}, {heads}] on {dev}")
    _i32(cu_seqlens, dev, "cu_seqlens", rows + 1)
    _i32(slots, dev, "slots")
    lib, cus = load(), _cu_count(dev)
    longest = 0 if max_len is None else max(1, max_len)
    cache = _lib.KvCache(pages.data_ptr(), scales.data_ptr(), *sizes, page_table.data_ptr(), lengths.data_ptr())
    need = int(lib.bsg_kv_attention_workspace_bytes(cache, rows, heads, most, longest, cus))
    return (dev.index, lib.bsg_kv_attention, sizes, rows, most, code, q.stride(0), q.stride(1), tokens, heads,
            _mold(q.shape, q.dtype, dev), _mold(q.shape[:2], torch.float32, dev), longest, need, cus, d ** -0.5, *steps)


# The int32 tensors of each page call beside the cache's own.
_PAGE_CALLS = {"copy": ("src", "dst"), "fork": ("parents", "children"), "extend": ("new_tokens", "slots", "served"),
               "free": ("slots",), "compact": ("counts",)}


def _pool(kind: str, page_table, lengths, refcounts, pages, scales, *others) -> tuple:
    """What a page call needs beside `others`, its own int32 tensors: the device index, the library's
    function, the bsg_page_pool and the bytes of a plan's lists."""
    key = (kind, _sigs(page_table, lengths, refcounts, pages, scales, *others))
    call = _CALLS.get(key)
    if call is None:
        dev = (page_table if page_table is not None else pages).device
        if dev.type != "cuda":
            raise ValueError("a cache's tensors must live on a ROCm (cuda) device")
        layers = page_bytes = page_scales = slots = each = stride = 0
        page_size = 1
        if pages is not None:
            _storage(pages, scales, 6)
            if pages.device != dev:
                raise ValueError(f"pages must be on {dev}, got {pages.device}")
            layers, count, h, _, page_size, d = pages.shape
            page_bytes, page_scales = h * 2 * page_size * d, h * 2
        if page_table is not None:
            _table(page_table, dev)
            slots, each = page_table.shape
            stride = page_table.stride(0) if slots > 1 else each
            _i32(lengths, dev, "lengths", slots)
            _i32(refcounts, dev, "refcounts", None if pages is None else pages.shape[1])
            count = refcounts.numel()
        n = 2 if kind == "compact" else others[0].numel()
        for what, t in zip(_PAGE_CALLS[kind], others):
            _i32(t, dev, what, n)
        need = int(load().bsg_pages_workspace_bytes(count)) if kind in ("extend", "compact") else 0
        call = _remember(key, (dev.index, getattr(load(), "bsg_pages_" + kind),
                               (layers, count, page_bytes, page_scales, page_size, slots, each, stride), need))
    index, fn, sizes, need = call
    return index, fn, _lib.PagePool(_ptr(pages), _ptr(scales), *sizes, _ptr(page_table), _ptr(lengths), _ptr(refcounts)), need


def pages_copy(pages: torch.Tensor, scales: torch.Tensor, src: torch.Tensor, dst: torch.Tensor) -> None:
    """Copy pages src[i] -> dst[i] (int32) with their scales in every layer of pages [layers, pages,
    heads, 2, page_size, head_dim].  Pairs with an id out of range are skipped.  No page may be
    written twice, or both read and written, in one call."""
    index, fn, pool, _ = _pool("copy", None, None, None, pages, scales, src, dst)
    _launch(index, fn, pool, src.data_ptr(), dst.data_ptr(), src.numel())


def pages_fork(page_table: torch.Tensor, lengths: torch.Tensor, refcounts: torch.Tensor, parents: torch.Tensor,
               children: torch.Tensor) -> None:
    """Slot children[i] goes on from slot parents[i] (int32): it takes its pages, which both then
    share, and its length, and releases what it held.  All pairs at once, so that a reordering of
    beams is one call.  Pairs with a slot out of range are skipped; of pairs with the same child the
    last one counts.  At most 1024 pairs."""
    index, fn, pool, _ = _pool("fork", page_table, lengths, refcounts, None, None, parents, children)
    _launch(index, fn, pool, parents.data_ptr(), children.data_ptr(), parents.numel())


def pages_extend(pages: torch.Tensor, scales: torch.Tensor, page_table: torch.Tensor, lengths: torch.Tensor,
                 refcounts: torch.Tensor, new_tokens: torch.Tensor, slots: Optional[torch.Tensor] = None,
                 served: Optional[torch.Tensor] = None, workspace_prefix: Optional[str] = None) -> torch.Tensor:
    """Room for new_tokens[i] (int32) more tokens of slot slots[i] (or i): lengths grow, pages come
    from the free ones, lowest id first, in the order of the rows, and a partly filled last page that
    other slots read as well is copied first (the last of its readers in the call keeps it).

    Returns served, int32: 1, or 0 where nothing was changed because the slot is out of range, its
    table row is too short, or the free pages do not reach.  Rows are served in order until the first
    that they do not reach; of the later ones only those that need no page and write to no shared
    one.  Slots must be distinct; at most 1024 rows."""
    n = new_tokens.numel()
    if served is None:
        served = torch.empty(n, dtype=torch.int32, device=new_tokens.device)
    index, fn, pool, need = _pool("extend", page_table, lengths, refcounts, pages, scales, new_tokens, slots, served)
    held, ws, room = _plan_workspace(index, need, workspace_prefix)
    _launch(index, fn, pool, _ptr(slots), new_tokens.data_ptr(), n, served.data_ptr(), ws, room)
    return served


def _plan_workspace(index: int, need: int, prefix: Optional[str]) -> Tuple[torch.Tensor, int, int]:
    """A workspace, with the address and bytes of its room for a plan's lists, past the counters that
    other calls need zero."""
    held = _workspace(index, COUNTER_BYTES + need, prefix, cleared=False)
    return held, held.data_ptr() + COUNTER_BYTES, held.numel() - COUNTER_BYTES


def pages_free(page_table: torch.Tensor, lengths: torch.Tensor, refcounts: torch.Tensor, slots: torch.Tensor) -> None:
    """Release every page of the given slots (int32): their table rows become -1, their lengths 0.
    Slots out of range are skipped, one named twice is released once.  At most 1024 slots."""
    index, fn, pool, _ = _pool("free", page_table, lengths, refcounts, None, None, slots)
    _launch(index, fn, pool, slots.data_ptr(), slots.numel())


def pages_compact(pages: torch.Tensor, scales: torch.Tensor, page_table: torch.Tensor, refcounts: torch.Tensor,
                  counts: Optional[torch.Tensor] = None, workspace_prefix: Optional[str] = None) -> torch.Tensor:
    """Make the pool dense: the live pages past the first `live` ids move, in order, to the free
    ids before, and every entry of page_table (all slots) follows.  Returns counts, int32 [live, moved]."""
    if counts is None:
        counts = torch.empty(2, dtype=torch.int32, device=page_table.device)
    index, fn, pool, need = _pool("compact", page_table, None, refcounts, pages, scales, counts)
    held, ws, room = _plan_workspace(index, need, workspace_prefix)
    _launch(index, fn, pool, counts.data_ptr(), ws, room)
    return counts


class TokenLogprobs(NamedTuple):
    logprob: torch.Tensor       # fp32 [rows]
    entropy: torch.Tensor       # fp32 [rows], nats
    top_ids: torch.Tensor       # int32 [rows, k]
    top_logprobs: torch.Tensor  # fp32 [rows, k]


_LOGIT_DTYPES = {torch.float16: _lib.BSG_F16, torch.bfloat16: _lib.BSG_BF16, torch.float32: _lib.BSG_F32}


def token_logprobs(logits: torch.Tensor, tokens: torch.Tensor, k: int = 0,
                   workspace_prefix: Optional[str] = None) -> TokenLogprobs:
    """Log probabilities of tokens (int32 [rows]) under logits [rows, vocab] (fp16, bf16 or fp32, any
    row stride), the entropy of each row and its k <= 64 likeliest tokens, by (logit desc, id asc).

    A token outside the vocabulary gives NaN.  A row of nothing but -inf gives -inf, entropy 0 and the
    lowest ids; a NaN or +inf in a row makes its numbers NaN (NaN ranks first among the ids, -0 equals
    +0)."""
    k = int(k)
    key = ("logprobs", _sigs(logits, tokens), k)
    call = _CALLS.get(key)
    if call is None:
        call = _remember(key, _logprobs_call(logits, tokens, k))
    index, fn, rows, vocab, stride, k, code, need, cus, molds = call
    out = TokenLogprobs(*map(torch.empty_like, molds))
    ws, room = 0, 0
    if need > 0:
        held = _workspace(index, need, workspace_prefix)
        ws, room = held.data_ptr(), held.numel()
    _launch(index, fn, logits.data_ptr(), stride, rows, vocab, tokens.data_ptr(), k, out[0].data_ptr(), out[1].data_ptr(),
            out[2].data_ptr(), out[3].data_ptr(), code, ws, room, cus)
    return out


def _logprobs_call(logits: torch.Tensor, tokens: torch.Tensor, k: int) -> tuple:
    """The checks of token_logprobs and what follows from its arguments' shapes."""
    dev = _require_cuda(logits)
    if logits.dtype not in _LOGIT_DTYPES:
        raise TypeError(f"logits must be float16, bfloat16 or float32, got {logits.dtype}")
    if logits.dim() != 2 or logits.shape[1] < 1:
        raise ValueError(f"logits must be [rows, vocab], got {tuple(logits.shape)}")
    rows, vocab = logits.shape
    if logits.stride(1) != 1 and vocab > 1:
        raise ValueError(f"logits rows must be contiguous, strides {logits.stride()}")
    if not 0 <= k <= min(MAX_ALTERNATIVES, vocab):
        raise ValueError(f"k={k} (0 to {min(MAX_ALTERNATIVES, vocab)})")
    _i32(tokens, dev, "tokens", rows)
    code = _LOGIT_DTYPES[logits.dtype]
    lib, cus = load(), _cu_count(dev)
    need = int(lib.bsg_token_logprobs_workspace_bytes(rows, vocab, k, code, cus))
    molds = [_mold(s, t, dev) for s, t in (((rows,), torch.float32), ((rows,), torch.float32), ((rows, k), torch.int32),
                                           ((rows, k), torch.float32))]
    return dev.index, lib.bsg_token_logprobs, rows, vocab, logits.stride(0), k, code, need, cus, molds


def read_pages(pages: torch.Tensor, scales: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """Keys and values of pages [..., heads, 2, page_size, head_dim] as fp32 [..., heads, page_size,
    head_dim] each: tile order undone, scales applied (for inspection, any device)."""
    p, d = pages.shape[-2:]
    lead = pages.shape[:-3]
    x = pages.float() * scales[..., None, None]
    k = x[..., 0, :, :].reshape(*lead, p // 16, d // 64, 4, 16, 16)  # tile, c, g, t, e
    v = x[..., 1, :, :].reshape(*lead, p // 16, d // 64, 4, 16, 4, 4)  # tile, c, g, l, i, t
    n = len(lead)
    k = k.permute(*range(n), n, n + 3, n + 1, n + 2, n + 4).reshape(*lead, p, d)
    v = v.permute(*range(n), n, n + 2, n + 5, n + 1, n + 4, n + 3).reshape(*lead, p, d)
    return k, v


class KVCache:
    """The tensors of a paged 8-bit cache of `layers` layers, and the calls on them as methods.

    A slot is a sequence: `extend` gives it pages for new tokens (once for all layers), `append`
    writes a layer's keys and values, `attend` reads them, `fork` lets slots go on from others, `free`
    releases them, `compact` makes the pool dense."""

    def __init__(self, layers: int, num_pages: int, heads: int, head_dim: int = 128, page_size: int = 16,
                 max_slots: int = 64, max_pages: int = 256, device: Optional[torch.device] = None):
        if page_size not in PAGE_SIZES or head_dim not in HEAD_DIMS:
            raise ValueError(f"page_size must be one of {PAGE_SIZES} and head_dim one of {HEAD_DIMS}, got {page_size}, {head_dim}")
        if min(layers, num_pages, heads, max_slots, max_pages) < 1:
            raise ValueError("layers, num_pages, heads, max_slots and max_pages must be at least 1")
        dev = torch.device(device) if device is not None else torch.device("cuda", torch.cuda.current_device())
        self.pages = torch.empty((layers, num_pages, heads, 2, page_size, head_dim), dtype=_F8, device=dev)
        self.scales = torch.ones((layers, num_pages, heads, 2), dtype=torch.float32, device=dev)
        self.page_table = torch.full((max_slots, max_pages), -1, dtype=torch.int32, device=dev)
        self.lengths = torch.zeros(max_slots, dtype=torch.int32, device=dev)
        self.refcounts = torch.zeros(num_pages, dtype=torch.int32, device=dev)
        self.page_size, self.head_dim, self.heads = page_size, head_dim, heads

    def extend(self, new_tokens: torch.Tensor, slots: Optional[torch.Tensor] = None, **kw) -> torch.Tensor:
        return pages_extend(self.pages, self.scales, self.page_table, self.lengths, self.refcounts, new_tokens, slots, **kw)

    def append(self, layer: int, k: torch.Tensor, v: torch.Tensor, **kw) -> None:
        kv_append(k, v, self.pages, self.scales, self.page_table, self.lengths, layer=layer, **kw)

    def attend(self, layer: int, q: torch.Tensor, **kw) -> Tuple[torch.Tensor, torch.Tensor]:
        return kv_attention(q, self.pages, self.scales, self.page_table, self.lengths, layer=layer, **kw)

    def fork(self, parents: torch.Tensor, children: torch.Tensor) -> None:
        pages_fork(self.page_table, self.lengths, self.refcounts, parents, children)

    def free(self, slots: torch.Tensor) -> None:
        pages_free(self.page_table, self.lengths, self.refcounts, slots)

    def compact(self, **kw) -> torch.Tensor:
        return pages_compact(self.pages, self.scales, self.page_table, self.refcounts, **kw)

    def copy(self, src: torch.Tensor, dst: torch.Tensor) -> None:
        pages_copy(self.pages, self.scales, src, dst)

    def read(self, layer: int, slot: int) -> Tuple[torch.Tensor, torch.Tensor]:
        """The cached keys and values of a slot, fp32 [heads, tokens, head_dim] (synchronises)."""
        n = int(self.lengths[slot])
        ids = self.page_table[slot, : -(-n // self.page_size)].long()
        k, v = read_pages(self.pages[layer].view(torch.uint8)[ids].view(_F8), self.scales[layer][ids])
        return tuple(x.transpose(0, 1).reshape(self.heads, -1, self.head_dim)[:, :n] for x in (k, v))
