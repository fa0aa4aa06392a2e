"""Beam search over a Llama-shaped decoder with batch-shared activation sparsity and an 8-bit paged
cache: the package's operators as a decode loop runs them together.

    python -m bsa_mi355x.beam --hidden 4096 --layers 8 --prompts 8 --width 8 --steps 32

Every beam is a slot of one KVCache.  A step takes one token of every beam: each layer selects blocks
and runs its linears on them (select_gemm_packed), writes its keys and values (append) and attends
over the cache (attend); the head's logits go through token_logprobs, whose alternatives, with the
beams' scores, decide which beams go on; fork makes them share their parents' pages and extend
gives each room for its next token, copying the page it is about to write where others read it.
Nothing but the finished tokens comes to the host, so a step can be captured.

Weights are random (N(0, 0.02), the architecture's shapes); norms, rotation of q and k, the gate and
the choice among width^2 candidates are plain torch.
"""
from __future__ import annotations

import argparse
import itertools
import time
import weakref
from typing import List, Optional, Tuple

import torch

from .runtime import _release_workspaces, gemm_packed, n_keep_for_density, nblk_of, pack_weight
from .select import select_gemm_packed
from .serving import KVCache, token_logprobs


_NUMBER = itertools.count()


def _rms(x: torch.Tensor) -> torch.Tensor:
    f = x.float()
    return (f * torch.rsqrt(f.square().mean(-1, keepdim=True) + 1e-5)).to(x.dtype)


def _rotate(x: torch.Tensor, pos: torch.Tensor) -> torch.Tensor:
    """Rotary embedding of x [tokens, heads, head_dim] at integer positions [tokens]."""
    half = x.shape[-1] // 2
    angle = pos[:, None].float() * 10000.0 ** (-torch.arange(half, device=x.device) / half)
    cos, sin = angle.cos()[:, None], angle.sin()[:, None]
    a, b = x[..., :half].float(), x[..., half:].float()
    return torch.cat([a * cos - b * sin, a * sin + b * cos], -1).to(x.dtype)


class BeamDecoder:
    """A decoder of `layers` layers for `prompts` x `width` beams of up to max_len tokens each.

    Its linears' workspaces are its own, so decoders may run beside each other on several streams; one
    decoder's eager steps and replayed graphs come one after the other."""

    def __init__(self, hidden: int = 4096, intermediate: int = 11008, heads: int = 32, kv_heads: int = 32, layers: int = 8,
                 vocab: int = 32000, prompts: int = 8, width: int = 8, max_len: int = 1024, page_size: int = 16,
                 density: float = 0.5, device: Optional[torch.device] = None, seed: int = 0, dtype=torch.float16):
        self.device = device or torch.device("cuda", torch.cuda.current_device())
        self.hidden, self.heads, self.kv_heads, self.vocab = hidden, heads, kv_heads, vocab
        self.prompts, self.width, self.density = prompts, width, density
        self.head_dim = hidden // heads
        self._prefix = f"beam {next(_NUMBER)}"
        weakref.finalize(self, _release_workspaces, self._prefix)
        g = torch.Generator(device=self.device).manual_seed(seed)

        def weight(k: int, n: int, spread: float = 0.02) -> Tuple[torch.Tensor, int, int]:
            w = (torch.randn(k, n, generator=g, device=self.device) * spread).to(dtype)
            return pack_weight(w, layout="kn"), k, n

        qkv = (heads + 2 * kv_heads) * self.head_dim
        self.embed = torch.randn(vocab, hidden, generator=g, device=self.device).to(dtype)
        self.layers: List[dict] = [{"qkv": weight(hidden, qkv), "o": weight(heads * self.head_dim, hidden),
                                    "gate_up": weight(hidden, 2 * intermediate), "down": weight(intermediate, hidden)}
                                   for _ in range(layers)]
        self.head = weight(hidden, vocab, 0.05)
        beams = prompts * width
        each = -(-max_len // page_size)
        # a prompt's full pages are shared by its beams, so twice a beam's share of one prompt is ample
        self.cache = KVCache(layers, beams * each + beams, kv_heads, self.head_dim, page_size, beams, each, self.device)
        self.slots = torch.arange(beams, dtype=torch.int32, device=self.device)
        self.ones = torch.ones(beams, dtype=torch.int32, device=self.device)
        self.base = (torch.arange(prompts, device=self.device) * width)[:, None]
        self.scores = torch.zeros(prompts, width, device=self.device)
        self.tokens = torch.zeros(beams, dtype=torch.int32, device=self.device)
        self.history: List[Tuple[torch.Tensor, torch.Tensor]] = []

    def _linear(self, x: torch.Tensor, w, sparse: bool) -> torch.Tensor:
        packed, k, n = w
        y = torch.empty(x.shape[0], n, dtype=x.dtype, device=x.device)
        if sparse:
            select_gemm_packed(x, packed, n, n_keep_for_density(self.density, nblk_of(k)), y, workspace_prefix=self._prefix)
        else:
            gemm_packed(x, packed, n, None, y, workspace_prefix=self._prefix)
        return y

    def forward(self, tokens: torch.Tensor, pos: torch.Tensor, sparse: bool, last: Optional[torch.Tensor] = None, **batch) -> torch.Tensor:
        """Logits after `tokens` [T] at positions pos [T], whose pages the cache has already given;
        batch: cu_seqlens, max_new, slots of append and attend; last: the rows to take logits of."""
        x = self.embed[tokens.long()]
        h, kv, d = self.heads, self.kv_heads, self.head_dim
        for i, w in enumerate(self.layers):
            qkv = self._linear(_rms(x), w["qkv"], sparse).view(-1, h + 2 * kv, d)
            q, k = _rotate(qkv[:, :h], pos), _rotate(qkv[:, h:h + kv], pos)
            self.cache.append(i, k, qkv[:, h + kv:], **batch)
            out, _ = self.cache.attend(i, q, **batch)
            x = x + self._linear(out.view(-1, h * d), w["o"], sparse)
            gate, up = self._linear(_rms(x), w["gate_up"], sparse).chunk(2, -1)
            x = x + self._linear(torch.nn.functional.silu(gate) * up, w["down"], sparse)
        if last is not None:
            x = x[last]
        return self._linear(_rms(x), self.head, sparse=False)

    def prefill(self, prompts: torch.Tensor) -> None:
        """Start every prompt [prompts, n] on its first beam and fork the others from it."""
        p, n = prompts.shape
        if p != self.prompts or n < 1:
            raise ValueError(f"prompts must be [{self.prompts}, tokens], got {tuple(prompts.shape)}")
        self.cache.free(self.slots)
        first = self.slots[:: self.width].contiguous()
        served = self.cache.extend(torch.full((p,), n, dtype=torch.int32, device=self.device), slots=first)
        if not bool(served.all()):
            raise RuntimeError(f"the cache has no room for prompts of {n} tokens")
        last = torch.arange(1, p + 1, device=self.device) * n - 1
        logits = self.forward(prompts.reshape(-1), torch.arange(n, device=self.device).repeat(p), False, last, slots=first)
        # the beams begin with the prompt's likeliest continuations
        got = token_logprobs(logits, self.tokens[:p], k=self.width)
        self.scores.copy_(got.top_logprobs)
        self.tokens.copy_(got.top_ids.reshape(-1))
        self.cache.fork((self.base.expand(-1, self.width)).reshape(-1).to(torch.int32).contiguous(), self.slots)
        self.history = [(self.tokens.clone(), self.slots.clone())]

    def step(self) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
        """One token of every beam; returns (tokens, parents, served) of the beams that go on.  A beam
        that found no room (served 0) has its token written nowhere and does not go on."""
        served = self.cache.extend(self.ones)
        pos = self.cache.lengths - 1
        room = served > 0
        # without room the newest place is an older token's, on a page that other beams may read
        logits = self.forward(self.tokens, pos, True, slots=torch.where(room, self.slots, -1))
        got = token_logprobs(logits, self.tokens, k=self.width)
        total = self.scores[:, :, None] + got.top_logprobs.view(self.prompts, self.width, self.width)
        total = torch.where(room.view(self.prompts, self.width, 1), total, -torch.inf)
        best, at = total.view(self.prompts, -1).topk(self.width, dim=1)
        parents = (self.base + at // self.width).reshape(-1)
        self.scores.copy_(best)
        self.tokens.copy_(got.top_ids.reshape(-1)[(parents * self.width).view_as(at).add(at % self.width).reshape(-1)])
        parents = parents.to(torch.int32)
        self.cache.fork(parents, self.slots)
        return self.tokens, parents, served

    def generate(self, prompts: torch.Tensor, steps: int) -> torch.Tensor:
        """The best beam's continuation of each prompt, [prompts, steps + 1] tokens; scores in self.scores."""
        self.prefill(prompts)
        ok = []
        for _ in range(steps):
            tokens, parents, served = self.step()
            self.history.append((tokens.clone(), parents.clone()))
            ok.append(served)
        if ok and not bool(torch.stack(ok).all()):
            raise RuntimeError("a beam found no free page or its table is full: raise max_len")
        beam = (self.base[:, 0] + self.scores.argmax(1)).long()
        out = []
        for tokens, parents in reversed(self.history):
            out.append(tokens[beam])
            beam = parents[beam].long()
        return torch.stack(out[::-1], 1)


def main() -> None:
    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    for name, value in (("hidden", 4096), ("intermediate", 11008), ("heads", 32), ("kv-heads", 32), ("layers", 8), ("vocab", 32000),
                        ("prompts", 8), ("width", 8), ("prompt-len", 200), ("steps", 32), ("page-size", 16)):
        ap.add_argument("--" + name, type=int, default=value)
    ap.add_argument("--density", type=float, default=0.5)
    a = ap.parse_args()
    dec = BeamDecoder(a.hidden, a.intermediate, a.heads, a.kv_heads, a.layers, a.vocab, a.prompts, a.width,
                      a.prompt_len + a.steps + 1, a.page_size, a.density)
    prompts = torch.randint(0, a.vocab, (a.prompts, a.prompt_len), device=dec.device, dtype=torch.int32)
    dec.generate(prompts, 2)
    torch.cuda.synchronize()
    start = time.perf_counter()
    out = dec.generate(prompts, a.steps)
    torch.cuda.synchronize()
    seconds = time.perf_counter() - start
    live = int((dec.cache.refcounts > 0).sum())
    flat = int(-(-dec.cache.lengths // a.page_size).sum())
    print(f"{a.prompts} prompts x {a.width} beams, {a.steps} steps: {seconds / a.steps * 1e3:.2f} ms a step with the prompts' share, "
          f"{a.prompts * a.width * a.steps / seconds:.0f} tokens/s; {live} pages hold what {flat} would without sharing; "
          f"best scores {[round(s, 2) for s in dec.scores.max(1).values.tolist()]}; first tokens {out[0, :8].tolist()}")


if __name__ == "__main__":
    main()
