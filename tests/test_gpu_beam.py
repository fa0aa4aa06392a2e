"""The beam decoder as a whole: its best beams against the same tokens fed one by one through a cache
that never forks, the cache's counts, and a step as a replayed graph."""
from __future__ import annotations

import pytest
import torch

from bsa_mi355x import token_logprobs
from bsa_mi355x.beam import BeamDecoder

pytestmark = pytest.mark.gpu

SMALL = dict(hidden=256, intermediate=704, heads=4, kv_heads=2, layers=2, vocab=500, prompts=3, width=4, max_len=64,
             density=1.0, seed=1)


def test_best_beams_score_what_their_tokens_do(dev):
    """With every block active the same tokens give the same numbers whoever else is in the batch, so the
    scores agree to the sums' own rounding: steps x 2^-20 of their size."""
    dec = BeamDecoder(device=dev, **SMALL)
    prompts = torch.randint(0, 500, (3, 21), device=dev, dtype=torch.int32, generator=torch.Generator(device=dev).manual_seed(2))
    steps = 17
    out = dec.generate(prompts, steps)
    best = dec.scores.max(1).values
    lengths = dec.cache.lengths.clone()
    assert (lengths == 21 + steps).all()
    named = dec.cache.page_table[dec.cache.page_table >= 0]
    assert torch.equal(torch.bincount(named.long(), minlength=dec.cache.refcounts.numel()).int(), dec.cache.refcounts)

    dec.prefill(prompts)
    first = token_logprobs(dec.forward(prompts.reshape(-1), torch.arange(21, device=dev).repeat(3), False,
                                       torch.arange(1, 4, device=dev) * 21 - 1, slots=dec.slots[::4].contiguous()),
                           out[:, 0].int().contiguous())
    total = first.logprob.clone()
    # every beam of a prompt takes the winner's tokens; slots' tails are shared, so each writes a copy of its own
    for i in range(steps):
        tokens = out[:, i].int().repeat_interleave(4).contiguous()
        assert bool(dec.cache.extend(dec.ones).all())
        logits = dec.forward(tokens, dec.cache.lengths - 1, True)
        total += token_logprobs(logits, out[:, i + 1].int().repeat_interleave(4).contiguous()).logprob[::4]
    assert (total - best).abs().max() <= steps * 2.0 ** -20 * best.abs().max(), (total, best)


def test_step_as_a_graph(dev):
    """A captured step replayed gives the beams that eager steps give."""
    prompts = torch.randint(0, 500, (3, 10), device=dev, dtype=torch.int32, generator=torch.Generator(device=dev).manual_seed(3))
    eager = BeamDecoder(device=dev, **SMALL)
    eager.prefill(prompts)
    want = []
    for _ in range(6):
        tokens, parents, _ = eager.step()
        want.append((tokens.clone(), parents.clone(), eager.scores.clone()))
    dec = BeamDecoder(device=dev, **SMALL)
    dec.prefill(prompts)
    dec.step()  # settles plans and workspaces
    dec.prefill(prompts)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        tokens, parents, served = dec.step()
    dec.prefill(prompts)
    for t, p, s in want:
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(tokens, t) and torch.equal(parents, p) and torch.equal(dec.scores, s)
        assert bool(served.all())


@pytest.mark.parametrize("left", [0, 2, 5, 9])
def test_a_beam_without_room_writes_nothing(dev, left):
    """With `left` pages left, the beams that got none leave every page that they read as it was, and
    others go on in their places."""
    dec = BeamDecoder(device=dev, **SMALL)
    prompts = torch.randint(0, 500, (3, 21), device=dev, dtype=torch.int32, generator=torch.Generator(device=dev).manual_seed(5))
    dec.prefill(prompts)
    cache = dec.cache
    free = (cache.refcounts == 0).nonzero()[:, 0]
    cache.refcounts[free[left:]] = 1  # taken by someone else
    table, lengths = cache.page_table.clone(), cache.lengths.clone()
    pages, scales = cache.pages.view(torch.uint8).clone(), cache.scales.clone()
    tokens, parents, served = dec.step()
    got = served.tolist()
    # of four readers of a prompt's last page three need a copy, and the last one keeps it
    assert sum(got) == (12 if left >= 9 else left // 3 * 4 + left % 3)
    for beam, ok in enumerate(got):
        if not ok:
            ids = table[beam, : -(-int(lengths[beam]) // cache.page_size)].long()
            assert torch.equal(cache.pages.view(torch.uint8)[:, ids], pages[:, ids]) and torch.equal(cache.scales[:, ids], scales[:, ids])
    for prompt in range(3):
        some = [b for b in range(4 * prompt, 4 * prompt + 4) if got[b]]
        if some:
            assert set(parents[4 * prompt:4 * prompt + 4].tolist()) <= set(some)
            assert (cache.lengths[4 * prompt:4 * prompt + 4] == 22).all() and dec.scores[prompt].isfinite().all()
        else:
            assert (cache.lengths[4 * prompt:4 * prompt + 4] == 21).all() and dec.scores[prompt].isneginf().all()


def test_decoders_beside_each_other(dev):
    """Two decoders of one shape on two streams, one as a replayed graph: each has workspaces of its own, gives
    what it gives alone, and leaves nothing behind."""
    from bsa_mi355x import runtime

    small = dict(SMALL, density=0.5)
    prompts = [torch.randint(0, 500, (3, 21), device=dev, dtype=torch.int32, generator=torch.Generator(device=dev).manual_seed(i))
               for i in (6, 7)]
    decs = [BeamDecoder(device=dev, **small) for _ in prompts]

    def buffers(dec):
        return {b.data_ptr() for k, b in runtime._WORKSPACE_CACHE["bufs"].items() if k[0] == dec._prefix}

    want = []
    for dec, p in zip(decs, prompts):
        dec.prefill(p)
        want.append([])
        for _ in range(8):
            dec.step()
            want[-1].append((dec.tokens.clone(), dec.scores.clone()))
        dec.prefill(p)
    assert buffers(decs[0]) and buffers(decs[1]) and not buffers(decs[0]) & buffers(decs[1])
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        decs[0].step()
    decs[0].prefill(prompts[0])
    streams = [torch.cuda.Stream() for _ in decs]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(8):
        for i, dec in enumerate(decs):
            with torch.cuda.stream(streams[i]):
                graph.replay() if i == 0 else dec.step()
                got[i].append((dec.tokens.clone(), dec.scores.clone()))
    torch.cuda.synchronize()
    for a, b in zip(want, got):
        for (t, s), (u, v) in zip(a, b):
            assert torch.equal(t, u) and torch.equal(s, v)
    names = [d._prefix for d in decs]
    del dec, decs, graph
    import gc
    gc.collect()
    assert not [k for k in runtime._WORKSPACE_CACHE["bufs"] if k[0] in names]


def test_refuses_what_it_has_no_room_for(dev):
    dec = BeamDecoder(device=dev, **dict(SMALL, max_len=32))
    with pytest.raises(ValueError):
        dec.prefill(torch.zeros(2, 5, dtype=torch.int32, device=dev))
    with pytest.raises(RuntimeError):
        dec.prefill(torch.zeros(3, 33, dtype=torch.int32, device=dev))
    with pytest.raises(RuntimeError):
        dec.generate(torch.zeros(3, 20, dtype=torch.int32, device=dev), 20)
