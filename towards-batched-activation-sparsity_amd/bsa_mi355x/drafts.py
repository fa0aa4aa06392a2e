"""A step that drafts tokens and verifies them, over the 8-bit paged cache of serving.py.

    kv_append_rotated  queries and keys normed by head and rotated by position, keys and values into the cache
    kv_tree_attention  attention of a tree of drafted tokens over the cache
    verify_drafts      which drafted tokens the target's probabilities accept, and the token that follows them
    pages_keep         the accepted tokens stay in the cache, the others leave it

All of it runs on the device with no host round trip (csrc/kv_rotate.hip, kv_tree.hip, verify.hip, pages_keep.hip
through include/bsgdraft.h and bsgdraft_slots.h), on torch's current stream, and can be captured.  The reference decodes one token at a
time, so these have no counterpart there.

A tree is the newest tokens of a sequence, its nodes, at most 64 of them.  parents int32 [tokens] holds for each
token its parent's place among its sequence's new tokens; what names no earlier node (-1) makes it a root.  One
step: pages_extend gives every node a place, kv_append_rotated and kv_tree_attention run in each layer, verify_drafts
reads the logits, and pages_keep leaves the accepted nodes behind the tokens that were there before.  Batches
(cu_seqlens, max_new, slots) are described as in serving.py.  A sequence that pages_extend had no room for takes no
part: its slot is -1 in the calls that follow, verify_drafts among them.
"""
from __future__ import annotations

from operator import index as _index
from typing import NamedTuple, Optional, Tuple, Union

import torch

from . import _lib
from ._lib import load
from .runtime import _cu_count, _dtype_code, _require_cuda
from .serving import (MAX_ROWS, _CALLS, _LOGIT_DTYPES, _batch, _from_end, _i32, _launch, _layer, _mold, _plan_workspace, _ptr, _remember,
                      _rows, _sigs, _storage, _table, _workspace)

MAX_NODES = 64  # BSG_TREE_NODES


def _nodes(max_new: int) -> None:
    if max_new > MAX_NODES:
        raise ValueError(f"a tree has at most {MAX_NODES} nodes: give max_new, a bound on the new tokens of a sequence (here {max_new})")


def kv_append_rotated(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor,
                      pages: torch.Tensor, scales: torch.Tensor, page_table: torch.Tensor, lengths: torch.Tensor,
                      cu_seqlens: Optional[torch.Tensor] = None, max_new: Optional[int] = None,
                      slots: Optional[torch.Tensor] = None, positions: Optional[torch.Tensor] = None,
                      parents: Optional[torch.Tensor] = None, q_norm: Optional[torch.Tensor] = None,
                      k_norm: Optional[torch.Tensor] = None, eps: float = 1e-6, interleaved: bool = False,
                      out: Optional[torch.Tensor] = None, layer: Optional[int] = None) -> torch.Tensor:
    """kv_append of keys that are normed and rotated on the way; returns the queries, treated alike, in `out` (by
    default a new tensor; q itself is fine).

    q [tokens, query heads, head_dim], k and v [tokens, heads, head_dim] fp16/bf16.  With q_norm and k_norm
    [head_dim], of the same type, each head's x becomes x * rsqrt(mean(x^2) + eps) * norm.  cos and sin are fp32
    [positions, dims / 2]; of a head's channels the first `dims` (16, 32, 64 or 128) are rotated in pairs (i, i +
    dims / 2), or (2 i, 2 i + 1) where `interleaved`: (a, b) -> (a cos - b sin, a sin + b cos).  A token's position is
    its place in its sequence, or positions[token] (int32), or with `parents` the place of its tree's first node
    plus its depth in the tree.  All of it is in 32 bits; q is rounded once, k and v once, as kv_append rounds.

    A position that the tables do not have makes the rotated channels NaN.  Rows of q that belong to no sequence
    (or one whose slot is out of range, or past max_new) are left as they are in `out`.  Batches and layer as
    kv_append.  Rows of q and out must be 16-byte aligned."""
    if max_new is not None:
        max_new = int(max_new)
    key = ("append_rotated", _sigs(q, k, v, cos, sin, pages, scales, page_table, lengths, cu_seqlens, slots, positions, parents,
                                   q_norm, k_norm, out), max_new, layer is None, interleaved)
    call = _CALLS.get(key)
    if call is None:
        call = _remember(key, _rotated_call(q, k, v, cos, sin, pages, scales, page_table, lengths, cu_seqlens, max_new, slots,
                                            positions, parents, q_norm, k_norm, interleaved, out, layer))
    index, fn, sizes, rows, most, code, strides, tokens, heads, mold, turn, layers, page_step, scale_step = call
    if out is None:
        out = torch.empty_like(mold)
    at, scales_at = pages.data_ptr(), scales.data_ptr()
    if layer is not None:
        i = _index(layer)
        if not 0 <= i < layers:
            i = _from_end(i, layers)
        at, scales_at = at + i * page_step, scales_at + i * scale_step
    cache = _lib.KvCache(at, scales_at, *sizes, page_table.data_ptr(), lengths.data_ptr())
    rotary = _lib.Rotary(cos.data_ptr(), sin.data_ptr(), *turn, eps, _ptr(q_norm), _ptr(k_norm), _ptr(positions), _ptr(parents))
    qt, qh, kt, kh, vt, vh = strides
    _launch(index, fn, q.data_ptr(), qt, qh, heads, out.data_ptr(), out.stride(0), out.stride(1), k.data_ptr(), kt, kh, v.data_ptr(),
            vt, vh, tokens, rotary, cache, _ptr(slots), rows, _ptr(cu_seqlens), most, code)
    return out


def _rotated_call(q, k, v, cos, sin, pages, scales, page_table, lengths, cu_seqlens, max_new, slots, positions, parents, q_norm,
                  k_norm, interleaved, out, layer) -> tuple:
    """The checks of kv_append_rotated and what follows from its arguments' shapes."""
    dev, sizes, steps = _layer(pages, scales, page_table, lengths, layer)
    d = sizes[3]
    rows = _rows(slots, cu_seqlens, lengths)
    most = _batch(k, "k", sizes[1], d, dev, rows, cu_seqlens, max_new)
    given = None if cu_seqlens is None else most
    _batch(v, "v", sizes[1], d, dev, rows, cu_seqlens, given)
    _batch(q, "q", 0, d, dev, rows, cu_seqlens, given)
    code = _dtype_code(k)
    for what, t in (("q", q), ("v", v)):
        if t.dtype is not k.dtype or t.shape[0] != k.shape[0]:
            raise ValueError(f"{what} and k must match, got {tuple(t.shape)} {t.dtype} and {tuple(k.shape)} {k.dtype}")
    if out is not None and (out.shape != q.shape or out.dtype is not q.dtype or out.device != dev or out.stride(2) != 1):
        raise ValueError(f"out must match q {tuple(q.shape)} {q.dtype} with contiguous channels, got {tuple(out.shape)} {out.dtype}")
    for what, t in (("cos", cos), ("sin", sin)):
        if t.dtype is not torch.float32 or t.device != dev:
            raise TypeError(f"{what} must be float32 on {dev}, got {t.dtype} on {t.device}")
        if t.dim() != 2 or t.shape != cos.shape or t.stride(1) != 1 or t.stride(0) != cos.stride(0):
            raise ValueError(f"cos and sin must be [positions, dims / 2] alike with contiguous rows, got {tuple(cos.shape)} and {tuple(t.shape)}")
    for what, t in (("q_norm", q_norm), ("k_norm", k_norm)):
        if t is not None and (t.shape != (d,) or t.dtype is not k.dtype or t.device != dev or not t.is_contiguous()):
            raise ValueError(f"{what} must be contiguous [{d}] {k.dtype} on {dev}, got {tuple(t.shape)} {t.dtype} on {t.device}")
    _i32(cu_seqlens, dev, "cu_seqlens", rows + 1)
    _i32(slots, dev, "slots")
    _i32(positions, dev, "positions", k.shape[0])
    _i32(parents, dev, "parents", k.shape[0])
    if parents is not None:
        _nodes(most)
    turn = (cos.stride(0) if cos.shape[0] > 1 else 0, cos.shape[0], 2 * cos.shape[1], int(bool(interleaved)))
    strides = (q.stride(0), q.stride(1), k.stride(0), k.stride(1), v.stride(0), v.stride(1))
    return (dev.index, load().bsg_kv_append_rotated, sizes, rows, most, code, strides, k.shape[0], q.shape[1],
            _mold(q.shape, q.dtype, dev), turn, *steps)


def kv_tree_attention(q: torch.Tensor, parents: torch.Tensor, pages: torch.Tensor, scales: torch.Tensor,
                      page_table: torch.Tensor, lengths: torch.Tensor, cu_seqlens: Optional[torch.Tensor] = None,
                      max_new: Optional[int] = None, slots: Optional[torch.Tensor] = None,
                      sm_scale: Optional[float] = None, max_len: Optional[int] = None, out: Optional[torch.Tensor] = None,
                      lse: Optional[torch.Tensor] = None, workspace_prefix: Optional[str] = None,
                      layer: Optional[int] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """kv_attention of a tree: node i of a sequence's n new tokens (appended before) sees the first length - n
    tokens, its own ancestors by `parents` (int32 [tokens]) and itself.  At most 64 nodes a sequence (max_new bounds
    them); everything else as kv_attention."""
    if max_new is not None:
        max_new = int(max_new)
    if max_len is not None:
        max_len = int(max_len)
    key = ("tree", _sigs(q, parents, pages, scales, page_table, lengths, cu_seqlens, slots, out, lse), max_new, max_len, layer is None)
    call = _CALLS.get(key)
    if call is None:
        call = _remember(key, _tree_call(q, parents, pages, scales, page_table, lengths, cu_seqlens, max_new, slots, max_len, out, lse,
                                         layer))
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
    _launch(index, fn, q.data_ptr(), qt, qh, tokens, heads, parents.data_ptr(), cache, _ptr(slots), rows, _ptr(cu_seqlens), most,
            longest, scale if sm_scale is None else sm_scale, out.data_ptr(), out.stride(0), out.stride(1), lse.data_ptr(), code, ws,
            room, cus)
    return out, lse


def _tree_call(q, parents, pages, scales, page_table, lengths, cu_seqlens, max_new, slots, max_len, out, lse, layer) -> tuple:
    """The checks of kv_tree_attention and what follows from its arguments' shapes."""
    dev, sizes, steps = _layer(pages, scales, page_table, lengths, layer)
    rows = _rows(slots, cu_seqlens, lengths)
    most = _batch(q, "q", 0, sizes[3], dev, rows, cu_seqlens, max_new)
    _nodes(most)
    code = _dtype_code(q)
    tokens, heads, d = q.shape
    if out is not None and (out.shape != q.shape or out.dtype is not q.dtype or out.device != dev or out.stride(2) != 1):
        raise ValueError(f"out must match q {tuple(q.shape)} {q.dtype} with contiguous channels, got {tuple(out.shape)} {out.dtype}")
    if lse is not None and (lse.shape != q.shape[:2] or lse.dtype is not torch.float32 or lse.device != dev
                            or not lse.is_contiguous()):
        raise ValueError(f"lse must be contiguous float32 [{tokens}, {heads}] on {dev}")
    _i32(parents, dev, "parents", tokens)
    _i32(cu_seqlens, dev, "cu_seqlens", rows + 1)
    _i32(slots, dev, "slots")
    lib, cus = load(), _cu_count(dev)
    longest = 0 if max_len is None else max(1, max_len)
    cache = _lib.KvCache(pages.data_ptr(), scales.data_ptr(), *sizes, page_table.data_ptr(), lengths.data_ptr())
    need = int(lib.bsg_kv_tree_attention_workspace_bytes(cache, rows, heads, most, longest, cus))
    return (dev.index, lib.bsg_kv_tree_attention, sizes, rows, most, code, q.stride(0), q.stride(1), tokens, heads,
            _mold(q.shape, q.dtype, dev), _mold(q.shape[:2], torch.float32, dev), longest, need, cus, d ** -0.5, *steps)


class Verified(NamedTuple):
    accepted: torch.Tensor  # int32 [sequences]: accepted nodes, the first one among them
    path: torch.Tensor      # int32 [sequences, max_new]: the accepted nodes, then -1 (max_new: at most 64; where not given, the tokens)
    tokens: torch.Tensor    # int32 [sequences, max_new]: the accepted drafts and the new token, then -1


def verify_drafts(logits: torch.Tensor, tokens: torch.Tensor, uniforms: torch.Tensor, parents: Optional[torch.Tensor] = None,
                  draft_logits: Optional[torch.Tensor] = None, temperature: Union[float, torch.Tensor] = 1.0,
                  cu_seqlens: Optional[torch.Tensor] = None, max_new: Optional[int] = None,
                  workspace_prefix: Optional[str] = None, slots: Optional[torch.Tensor] = None) -> Verified:
    """Which drafted tokens the target model accepts, and the token that follows them, from given random numbers.

    Row t of logits [tokens, vocab] (fp16, bf16 or fp32, any row stride) is the target's after token t; tokens int32,
    parents int32 (None: each token's parent is the one before it) and uniforms fp32 in [0, 1) have an entry for each.  A
    sequence has the tokens cu_seqlens[b] .. cu_seqlens[b + 1], or max_new each; its first one, which it began with, is
    accepted.  Then the children of the last accepted one are asked in order, until one is accepted, and so on.  With p =
    softmax(logits / temperature) of the last accepted row, x a child's token and u its number, it is accepted

        without draft_logits   if u (1 - r) < p(x), r the sum of p over its rejected siblings' tokens; the new token is drawn
                               from p without these tokens (for drafts that are chosen, not drawn: the likeliest ones)
        with draft_logits      like logits, for chains only (row t is what token t + 1 was drawn from), q their softmax at
                               the same temperature: if u q(x) < p(x); after a rejection the new token is drawn from max(p - q, 0)
        temperature 0          if x is the likeliest token (of equal ones the first), which is also the new one

    and drawn by the first token's number: the first token whose running sum exceeds it times the whole.  The tokens that
    come out are then distributed as the target's own.  temperature is a finite number from 0 on, or fp32 [sequences], by which
    0 or less (or NaN) is greedy and infinity makes all tokens of finite logits alike.  Decisions are those of 64-bit
    weights and sums.  A row of logits with NaN, +inf, or nothing but -inf ends its path with a new token of -1, which is no
    token for a next step: the sequence has failed; a token
    outside the vocabulary is rejected.  slots (int32 [sequences]) are the batch's: one below 0 leaves its sequence out, which
    then has nothing accepted, no path and no tokens, whatever its logits hold.  At most 64 tokens a sequence, 2^20 in the vocabulary, 16384 sequences."""
    if max_new is not None:
        max_new = int(max_new)
    each = temperature if isinstance(temperature, torch.Tensor) else None
    key = ("verify", _sigs(logits, tokens, uniforms, parents, draft_logits, each, cu_seqlens, slots), max_new)
    call = _CALLS.get(key)
    if call is None:
        call = _remember(key, _verify_call(logits, tokens, uniforms, parents, draft_logits, each, cu_seqlens, max_new, slots))
    index, fn, rows, most, vocab, count, stride, draft_stride, code, need, molds = call
    out = Verified(*map(torch.empty_like, molds))
    held = _workspace(index, need, workspace_prefix)
    _launch(index, fn, logits.data_ptr(), stride, _ptr(draft_logits), draft_stride, count, vocab, tokens.data_ptr(),
            uniforms.data_ptr(), _ptr(parents), _ptr(cu_seqlens), _ptr(slots), rows, most, 0.0 if each is not None else temperature, _ptr(each),
            out[0].data_ptr(), out[1].data_ptr(), out[2].data_ptr(), code, held.data_ptr(), held.numel())
    return out


def _verify_call(logits, tokens, uniforms, parents, draft_logits, temperatures, cu_seqlens, max_new, slots) -> tuple:
    """The checks of verify_drafts and what follows from its arguments' shapes."""
    dev = _require_cuda(logits)
    if logits.dtype not in _LOGIT_DTYPES:
        raise TypeError(f"logits must be float16, bfloat16 or float32, got {logits.dtype}")
    if logits.dim() != 2 or logits.shape[1] < 1:
        raise ValueError(f"logits must be [tokens, vocab], got {tuple(logits.shape)}")
    count, vocab = logits.shape
    if draft_logits is not None:
        if draft_logits.shape != logits.shape or draft_logits.dtype is not logits.dtype or draft_logits.device != dev:
            raise ValueError(f"draft_logits must match logits {tuple(logits.shape)} {logits.dtype} on {dev}, got "
                             f"{tuple(draft_logits.shape)} {draft_logits.dtype} on {draft_logits.device}")
        if parents is not None:
            raise ValueError("draft_logits go with chains: parents must be None")
    for what, t in (("logits", logits), ("draft_logits", draft_logits)):
        if t is not None and t.stride(1) != 1 and vocab > 1 and count > 0:
            raise ValueError(f"{what} rows must be contiguous, strides {t.stride()}")
    _i32(tokens, dev, "tokens", count)
    _i32(parents, dev, "parents", count)
    if uniforms.dtype is not torch.float32:
        raise TypeError(f"uniforms must be float32, got {uniforms.dtype}")
    if uniforms.device != dev or uniforms.numel() != count or not uniforms.is_contiguous():
        raise ValueError(f"uniforms must be contiguous [{count}] on {dev}, got {tuple(uniforms.shape)} on {uniforms.device}")
    if cu_seqlens is None:
        if max_new is None or max_new < 1 or count % max_new:
            raise ValueError(f"without cu_seqlens max_new must divide the {count} tokens, got {max_new}")
        rows, most = count // max_new, max_new
    else:
        _i32(cu_seqlens, dev, "cu_seqlens")
        # the answers' width is max_new whatever the batch's tokens are; only these are a tree's nodes
        rows, most = cu_seqlens.numel() - 1, count if max_new is None else max(0, max_new)
        if rows < 0:
            raise ValueError("cu_seqlens has no entries")
    _nodes(min(most, count))
    most = min(most, MAX_NODES)
    _i32(slots, dev, "slots", rows)
    if temperatures is not None and (temperatures.dtype is not torch.float32 or temperatures.device != dev
                                     or temperatures.shape != (rows,) or not temperatures.is_contiguous()):
        raise ValueError(f"temperature must be a number or contiguous float32 [{rows}] on {dev}, got {tuple(temperatures.shape)} "
                         f"{temperatures.dtype} on {temperatures.device}")
    code = _LOGIT_DTYPES[logits.dtype]
    lib = load()
    need = int(lib.bsg_verify_drafts_workspace_bytes(count, rows, vocab, most, code, int(draft_logits is not None)))
    if need < 0:
        raise _lib.BsgUnsupported(_lib.BSG_ERR_UNSUPPORTED, _lib.last_error())
    molds = [_mold(s, torch.int32, dev) for s in ((rows,), (rows, most), (rows, most))]
    return (dev.index, lib.bsg_verify_drafts_slots, rows, most, vocab, count, logits.stride(0),
            0 if draft_logits is None else draft_logits.stride(0), code, need, molds)


def pages_keep(pages: torch.Tensor, scales: torch.Tensor, page_table: torch.Tensor, lengths: torch.Tensor,
               refcounts: torch.Tensor, path: torch.Tensor, accepted: torch.Tensor, cu_seqlens: Optional[torch.Tensor] = None,
               slots: Optional[torch.Tensor] = None, workspace_prefix: Optional[str] = None) -> None:
    """What was accepted of a tree stays in the cache, in all layers of pages [layers, pages, heads, 2, page_size,
    head_dim]: of the newest tokens of row b (slot slots[b], or b), cu_seqlens[b + 1] - cu_seqlens[b] of them or as many
    as path has columns, those at the places path[b][:accepted[b]] (int32 [rows, places] and [rows], of verify_drafts) move
    together, in order, behind the tokens that were there before; the length shrinks to hold them and the pages past
    it are released.

    A token that changes its page is rounded again under that page's scale, which grows as kv_append's does.  No scale
    shrinks: what a louder token that is rejected now cost its page's other tokens when it was appended stays lost.  Of a
    path only what ascends and exists counts.  A slot out of range, or of fewer tokens than its new ones, is left as it
    is.  Slots must be distinct, and the new tokens' pages a sequence's own (pages_extend sees to that); at most 64
    places and 1024 rows."""
    key = ("keep", _sigs(pages, scales, page_table, lengths, refcounts, path, accepted, cu_seqlens, slots))
    call = _CALLS.get(key)
    if call is None:
        dev = _storage(pages, scales, 6)
        layers, count, h, _, p, d = pages.shape
        _table(page_table, dev)
        n, each = page_table.shape
        _i32(lengths, dev, "lengths", n)
        _i32(refcounts, dev, "refcounts", count)
        _i32(path, dev, "path")
        if path.dim() != 2:
            raise ValueError(f"path must be [rows, places], got {tuple(path.shape)}")
        rows, most = path.shape
        _nodes(most)
        _i32(accepted, dev, "accepted", rows)
        _i32(cu_seqlens, dev, "cu_seqlens", rows + 1)
        _i32(slots, dev, "slots", rows)
        sizes = (layers, count, h * 2 * p * d, h * 2, p, n, each, page_table.stride(0) if n > 1 else each)
        need = int(load().bsg_pages_keep_workspace_bytes(rows))
        if need < 0:
            raise ValueError(f"at most {MAX_ROWS} rows, got {rows}")
        call = _remember(key, (dev.index, load().bsg_pages_keep, sizes, h, d, rows, most, need))
    index, fn, sizes, h, d, rows, most, need = call
    held, ws, room = _plan_workspace(index, need, workspace_prefix)  # held: till the launch
    pool = _lib.PagePool(pages.data_ptr(), scales.data_ptr(), *sizes, page_table.data_ptr(), lengths.data_ptr(), refcounts.data_ptr())
    _launch(index, fn, pool, h, d, path.data_ptr(), accepted.data_ptr(), _ptr(cu_seqlens), _ptr(slots), rows, most, ws, room)
