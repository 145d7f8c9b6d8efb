"""Serving a layer after its sparse prefill: a paged K/V cache, appended to and attended over.

The reference stops at prefill: its callback sends decode to SDPA over the model's dense cache
(kernels/sparse_prefill.py:63-65).  Here a prompt runs the selector and the block-sparse attention and leaves its keys
and values in pages; every later chunk or token is appended with its head norms and rotation in one launch and attends
over the pages.

``PagedKVCache`` owns the pages of every layer and the sequences' page tables (host), ``PagedStep`` is one forward's
batch (device), ``PagedSparseLayer`` runs one layer of it.  A cache that keeps the attention weight of its keys
(``track_mass``) can be cut to a budget: ``PagedKVCache.evict`` keeps each head's heaviest.

    python -m spruce_research_b200.paged          # a small layer: prompts, then decode steps, with their times
    python -m spruce_research_b200.paged 2048     # the same, then cut to 2048 tokens a sequence and decoded further
"""
from __future__ import annotations

import sys
from dataclasses import dataclass

import torch

from . import native
from .pipeline import SparsePrefillLayer


@dataclass
class PagedStep:
    """The new tokens of one forward: packed sequence by sequence, in the order given to :meth:`PagedKVCache.step`."""

    seq_ids: list
    block_table: torch.Tensor   # int32 [S, pages of the longest sequence]
    cu_q: torch.Tensor          # int32 [S + 1]
    kv_lens: torch.Tensor       # int32 [S], the new tokens included
    max_q_len: int
    max_kv_len: int
    tokens: int
    positions: torch.Tensor | None = None   # int64 [tokens] in their sequences, where an eviction left these ahead of the slots
    max_position: int = 0                    # positions end before this
    counts: list | None = None               # each sequence's new tokens, and its length with them
    lengths: list | None = None
    serial: int = 0                          # of the cache's steps


class PagedKVCache:
    """Pages of ``page_size`` tokens for ``num_layers`` layers: ``k`` and ``v`` [layers, pages, Hkv, page_size, D].

    A page id names the same page of every layer.  Heads lie outside the tokens of a page, so that one head's page
    is one contiguous block.  With ``track_mass``, ``mass`` float32 [layers, pages, Hkv, page_size] holds the attention weight
    that each key has received, which layers add to and :meth:`evict` goes by.
    """

    def __init__(self, num_layers: int, num_pages: int, page_size: int, kv_heads: int, head_dim: int,
                 dtype: torch.dtype = torch.bfloat16, device="cuda", track_mass: bool = False):
        if page_size < 16 or page_size % 16:
            raise ValueError(f"page_size must be a multiple of 16, got {page_size}")
        if min(num_layers, num_pages, kv_heads, head_dim) < 1:
            raise ValueError("layers, pages, KV heads and head_dim must be positive")
        shape = (num_layers, num_pages, kv_heads, page_size, head_dim)
        self.k = torch.empty(shape, dtype=dtype, device=device)
        self.v = torch.empty(shape, dtype=dtype, device=device)
        self.mass = torch.zeros(shape[:4], dtype=torch.float32, device=device) if track_mass else None
        self.page_size = page_size
        self._free = list(range(num_pages - 1, -1, -1))
        self._pages: dict = {}
        self._length: dict = {}
        self._evicted: dict = {}   # tokens that evictions took, and the slots that the last one left
        self._last: dict = {}      # each sequence's last step, while no eviction has moved its tokens
        self._steps = 0

    @property
    def free_pages(self) -> int:
        return len(self._free)

    def length(self, seq_id) -> int:
        """Tokens the sequence holds (0 for one the cache does not know)."""
        return self._length.get(seq_id, 0)

    def position(self, seq_id) -> int:
        """Position of the sequence's next token: its length and what evictions took from it."""
        return self.length(seq_id) + self._evicted.get(seq_id, (0, 0))[0]

    def drop(self, seq_id) -> None:
        """Return a sequence's pages.  Kernels of its last step may still run: the next step's follow them."""
        self._free.extend(reversed(self._pages.pop(seq_id, [])))
        self._length.pop(seq_id, None)
        self._evicted.pop(seq_id, None)
        self._last.pop(seq_id, None)

    def truncate(self, seq_id, length: int) -> None:
        """Keep a sequence's first ``length`` tokens: drafts that were rejected, or a step whose forward did not run.

        The weight that the other tokens gave to keys before them stays in ``mass``, and the old ones have faded once for their step:
        drafts go through :meth:`PagedSparseLayer.draft`, which gives none until they are accepted.
        """
        held = self.length(seq_id)
        if not 0 <= length <= held:
            raise ValueError(f"a sequence of {held} tokens cannot be cut to {length}")
        if length < self._evicted.get(seq_id, (0, 0))[1]:
            raise ValueError(f"the first {self._evicted[seq_id][1]} slots are an eviction's: each head holds other tokens there")
        if seq_id in self._pages:
            pages, keep = self._pages[seq_id], -(-length // self.page_size)
            self._free.extend(reversed(pages[keep:]))
            del pages[keep:]
            self._length[seq_id] = length

    def step(self, new_tokens) -> PagedStep:
        """Make room for ``new_tokens``, pairs (seq_id, count), and describe the batch on the device.

        Unknown sequences start empty.  Nothing changes when the pages do not suffice (RuntimeError).
        The lengths count the new tokens from here on: :meth:`truncate` takes them back if they are not written.
        """
        new_tokens = [(s, int(n)) for s, n in new_tokens]
        if len({s for s, _ in new_tokens}) < len(new_tokens):
            raise ValueError("a sequence appears twice in one step")
        if any(n < 0 for _, n in new_tokens):
            raise ValueError("token counts must not be negative")
        lengths = [self.length(s) + n for s, n in new_tokens]
        need = [-(-m // self.page_size) - len(self._pages.get(s, [])) for (s, _), m in zip(new_tokens, lengths)]
        if sum(need) > len(self._free):
            raise RuntimeError(f"the cache needs {sum(need)} more pages and has {len(self._free)}")
        for (s, _), m, count in zip(new_tokens, lengths, need):
            self._pages.setdefault(s, []).extend(self._free.pop() for _ in range(count))
            self._length[s] = m
        self._steps += 1
        self._last.update((s, self._steps) for s, _ in new_tokens)
        dev = self._describe([s for s, _ in new_tokens], [n for _, n in new_tokens], lengths)
        ends = [self.position(s) for s, _ in new_tokens]
        positions = None
        if any(self._evicted.get(s, (0, 0))[0] for s, _ in new_tokens):
            positions = torch.cat([torch.arange(end - n, end) for end, (_, n) in zip(ends, new_tokens)]).to(self.k.device)
        return PagedStep([s for s, _ in new_tokens], *dev, max((n for _, n in new_tokens), default=0), max(lengths, default=0),
                         sum(n for _, n in new_tokens), positions, max(ends, default=0), [n for _, n in new_tokens], lengths,
                         self._steps)

    def accepted(self, step: PagedStep) -> list:
        """How many of a step's new tokens each of its sequences still holds, before anything but :meth:`truncate` and :meth:`drop`."""
        if step.counts is None:
            raise ValueError("this step was not described by a cache")
        kept = []
        for s, n, length in zip(step.seq_ids, step.counts, step.lengths):
            if s in self._length and self._last.get(s) != step.serial:
                raise ValueError(f"sequence {s!r} has gone on or lost tokens to an eviction since this step")
            kept.append(max(0, n - length + self.length(s)))
        return kept

    def _describe(self, seq_ids, counts, lengths):
        """Page table, offsets of ``counts`` and lengths of sequences, on the device."""
        width = max([len(self._pages[s]) for s in seq_ids], default=0)
        S = len(seq_ids)
        # One host tensor and one copy: table, offsets, lengths.
        host = torch.zeros(S * width + 2 * S + 1, dtype=torch.int32)
        table, cu, kv = host[:S * width].view(S, width), host[S * width:S * width + S + 1], host[S * width + S + 1:]
        for i, (s, n) in enumerate(zip(seq_ids, counts)):
            pages = self._pages[s]
            table[i, :len(pages)] = torch.tensor(pages, dtype=torch.int32)
            cu[i + 1] = cu[i] + n
            kv[i] = lengths[i]
        dev = host.to(self.k.device)
        return dev[:S * width].view(S, width), dev[S * width:S * width + S + 1], dev[S * width + S + 1:]

    def evict(self, seq_ids, keep: int, *, sinks: int = 0, recent: int = 0) -> list:
        """Cut sequences to ``keep`` tokens in every layer and return the pages that this empties.

        Each KV head keeps its first ``sinks`` slots, its last ``recent`` ones and of those between the keys of the largest mass;
        they move, in their order, to the first slots.  Sequences of at most ``keep`` tokens stay as they are.  New tokens go on at
        :meth:`position`.  Steps described before do not hold any more.  Returns the sequences that were cut.
        """
        if self.mass is None:
            raise ValueError("this cache was made without track_mass")
        keep, sinks, recent = int(keep), int(sinks), int(recent)
        if keep < 1 or sinks < 0 or recent < 0 or sinks + recent > keep:
            raise ValueError(f"cannot keep {sinks} first and {recent} last of {keep} tokens")
        seq_ids = list(seq_ids)
        if len(set(seq_ids)) < len(seq_ids):
            raise ValueError("a sequence appears twice in one eviction")
        cut = [s for s in seq_ids if self.length(s) > keep]
        if not cut:
            return cut
        lengths = [self.length(s) for s in cut]
        table, _, lens = self._describe(cut, [0] * len(cut), lengths)
        for k, v, mass in zip(self.k, self.v, self.mass):
            native.paged_evict(k, v, mass, table, lens, keep, sinks=sinks, recent=recent, max_kv_len=max(lengths))
        left = -(-keep // self.page_size)
        for s, n in zip(cut, lengths):
            pages = self._pages[s]
            self._free.extend(reversed(pages[left:]))
            del pages[left:]
            self._length[s] = keep
            self._evicted[s] = (self._evicted.get(s, (0, 0))[0] + n - keep, keep)
            self._last.pop(s, None)
        return cut


class PagedSparseLayer:
    """One attention layer over a :class:`PagedKVCache`: sparse prefill of prompts, then chunks and single tokens.

    Takes the projections before norms and rotation, packed ``q [N, Hq, D]``, ``k`` / ``v`` [N, Hkv, D].  ``rope`` is a
    :func:`rope.rope_table` of the longest sequence (None: no rotation); ``q_weight`` / ``k_weight`` are head norms (None: no norm).

    Where the cache keeps its keys' weights, each step multiplies the old ones of its sequences by ``decay`` and adds
    what its queries give; a sparse prefill sets them by its last ``observe`` queries, which attend to the whole prompt for it.
    Tokens that may be taken back go through :meth:`draft` and :meth:`accept`.
    """

    def __init__(self, cache: PagedKVCache, layer_idx: int, rope: torch.Tensor | None, *,
                 prefill: SparsePrefillLayer | None = None, q_weight: torch.Tensor | None = None,
                 k_weight: torch.Tensor | None = None, eps: float = 1e-6, interleaved: bool = False,
                 decay: float = 1.0, observe: int = 64):
        if not 0 <= layer_idx < cache.k.shape[0]:
            raise ValueError(f"layer_idx {layer_idx} is outside the cache's {cache.k.shape[0]} layers")
        if not 0 <= decay <= 1:
            raise ValueError(f"decay must be in [0, 1], got {decay}")
        if observe < 1:
            raise ValueError(f"observe must be positive, got {observe}")
        self.cache = cache
        self.k_cache, self.v_cache = cache.k[layer_idx], cache.v[layer_idx]
        self.mass = None if cache.mass is None else cache.mass[layer_idx]
        self.decay, self.observe = decay, observe
        self.rope, self.sparse = rope, prefill
        self.rotation = dict(q_weight=q_weight, k_weight=k_weight, eps=eps, interleaved=interleaved)

    def _check(self, tensors, step: PagedStep, spare: bool) -> None:
        """What the host knows: the kernels would leave rows out, take the nearest angles and only report it in a status."""
        rows = [x.shape[0] for x in tensors]
        if min(rows) < step.tokens or not spare and max(rows) > step.tokens:
            raise ValueError(f"the step has {step.tokens} tokens, q, k and v have {rows}")
        most = max(step.max_kv_len, step.max_position)
        if self.rope is not None and most > self.rope.shape[0]:
            raise ValueError(f"sequences of {most} tokens need a rotation table of as many positions, got "
                             f"{self.rope.shape[0]}")

    def _attend(self, q, step: PagedStep, cu_q, max_q_len: int, out=None):
        """Attention of ``q`` over the cache and, where the cache keeps weights, the rows' log-sums: ``(out, lse)``."""
        lse = None if self.mass is None else torch.empty(q.shape[:2], dtype=torch.float32, device=q.device)
        out = native.paged_attention(q, self.k_cache, self.v_cache, step.block_table, cu_q, step.kv_lens, out=out,
                                     max_q_len=max_q_len, max_kv_len=step.max_kv_len, lse=lse)
        return out, lse

    def _weigh(self, q, lse, step: PagedStep, cu_q, kv_lens, max_q_len: int, decay: float) -> None:
        """Add the weight that ``q`` gives, if the cache keeps any."""
        if self.mass is not None:
            native.paged_key_mass(q, self.k_cache, self.mass, step.block_table, cu_q, kv_lens, lse, decay=decay,
                                  max_q_len=max_q_len, max_kv_len=step.max_kv_len)

    def _extend(self, q, k, v, step: PagedStep, out):
        """Append and attend: ``(out, rotated q, lse)``."""
        self._check((q, k, v), step, spare=True)
        positions = step.positions
        if positions is not None and positions.shape[0] < k.shape[0]:  # rows past the step's tokens are left out
            positions = torch.nn.functional.pad(positions, (0, k.shape[0] - positions.shape[0]))
        q = native.paged_append(k, v, self.k_cache, self.v_cache, step.block_table, step.cu_q, step.kv_lens, q=q,
                                rope=self.rope, positions=positions, **self.rotation)
        out, lse = self._attend(q, step, step.cu_q, step.max_q_len, out)
        return out, q, lse

    def extend(self, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, step: PagedStep,
               out: torch.Tensor | None = None) -> torch.Tensor:
        """Append the step's tokens and attend over all each sequence holds: [N, Hq, D].

        N may exceed the step's tokens; the rows past them are not written.
        """
        out, q, lse = self._extend(q, k, v, step, out)
        self._weigh(q, lse, step, step.cu_q, step.kv_lens, step.max_q_len, self.decay)
        return out

    def draft(self, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, step: PagedStep,
              out: torch.Tensor | None = None):
        """:meth:`extend` by tokens that may be taken back: ``(out, seen)``.

        The cache's weights stay as they are until :meth:`accept` gets ``seen``.
        """
        out, q, lse = self._extend(q, k, v, step, out)
        return out, (q, lse)

    def accept(self, seen, step: PagedStep) -> None:
        """Add the weight of those of a drafted step's tokens that the cache still holds, as a step of these alone does.

        Once a step and layer, after :meth:`PagedKVCache.truncate` and before the sequences' next step or eviction.  A sequence that
        keeps none of the step's tokens keeps its weights.
        """
        counts = self.cache.accepted(step)
        most = max(counts, default=0)
        if self.mass is None or most == 0:
            return
        (q, lse), cu_q, kv_lens = seen, step.cu_q, step.kv_lens
        if counts != step.counts:
            n, S = sum(counts), len(counts)
            # One host tensor and one copy: the tokens kept, their offsets, what the lengths lose.
            host, at = torch.zeros(n + 2 * S + 1, dtype=torch.int32), 0
            rows, cu, less = host[:n], host[n:n + S + 1], host[n + S + 1:]
            for i, (kept, count) in enumerate(zip(counts, step.counts)):
                first = int(cu[i])
                rows[first:first + kept] = torch.arange(at, at + kept)
                cu[i + 1], less[i] = first + kept, count - kept
                at += count
            dev = host.to(q.device)
            q, lse = q.index_select(0, dev[:n]), lse.index_select(0, dev[:n])
            cu_q, kv_lens = dev[n:n + S + 1], kv_lens - dev[n + S + 1:]
        self._weigh(q, lse, step, cu_q, kv_lens, most, self.decay)

    def prefill(self, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, step: PagedStep):
        """Block-sparse prefill of one whole prompt; its keys and values go to the cache.

        Returns ``(out [N, Hq, D], selected [1, Hkv, blocks, K])``.
        """
        if self.sparse is None:
            raise ValueError("this layer was made without a SparsePrefillLayer")
        if len(step.seq_ids) != 1 or step.max_q_len != step.max_kv_len:
            raise ValueError("the sparse prefill takes one whole prompt: one sequence that held nothing before")
        self._check((q, k, v), step, spare=False)
        qs, ks, vs = (x.transpose(0, 1).unsqueeze(0) for x in (q, k, v))       # [1, H, T, D] views
        rope = self.rope if self.rope is not None else q.new_empty((step.tokens, 0), dtype=torch.float32)  # norms alone
        qr, kr = native.qk_norm_rope(qs, ks, rope, **self.rotation)
        native.paged_append(kr[0].transpose(0, 1), v, self.k_cache, self.v_cache, step.block_table, step.cu_q,
                            step.kv_lens)
        out, selected = self.sparse(qr, kr, vs)
        if self.mass is not None and step.tokens:
            last = min(self.observe, step.tokens)
            cu_q = torch.arange(0, 2 * last, last, device=q.device, dtype=torch.int32)
            rows = qr[0, :, -last:].transpose(0, 1)
            _, lse = self._attend(rows, step, cu_q, last)
            self._weigh(rows, lse, step, cu_q, step.kv_lens, last, 0.0)
        return out[0], selected


def main(prompt_tokens: int = 8192, sequences: int = 4, decode_steps: int = 32, budget: int = 0) -> None:
    """Prompts through the sparse prefill, then decode steps of all of them, on one 28-query / 4-KV-head layer; with a
    ``budget``, the cache keeps its keys' weights, is cut to so many tokens a sequence and decodes on."""
    from .rope import rope_table
    from .synthetic import k_for_density, make_gate_weights

    Hq, Hkv, D, page = 28, 4, 128, 64
    total = prompt_tokens + (2 if budget else 1) * decode_steps
    cache = PagedKVCache(1, sequences * -(-total // page), page, Hkv, D, track_mass=budget > 0)
    wq, wk = make_gate_weights(1, D, D, seed=2, device="cuda")
    sparse = SparsePrefillLayer(wq[0], wk[0], max(2, k_for_density(-(-prompt_tokens // 64), 0.10)))
    layer = PagedSparseLayer(cache, 0, rope_table(D, total, 1e6), prefill=sparse)
    g = torch.Generator(device="cuda").manual_seed(1)

    def project(n):
        x = torch.randn(n, Hq + 2 * Hkv, D, generator=g, device="cuda", dtype=torch.bfloat16)
        return x[:, :Hq], x[:, Hq:Hq + Hkv], x[:, Hq + Hkv:]

    def timed(f):
        a, b = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        a.record()
        f()
        b.record()
        b.synchronize()
        return a.elapsed_time(b)

    def decode():
        for _ in range(decode_steps):
            qkv, step = project(sequences), cache.step([(s, 1) for s in range(sequences)])
            ms = timed(lambda: layer.extend(*qkv, step))
        print(f"decode: {sequences} sequences at {step.max_kv_len} tokens, {1e3 * ms:.1f} us for the last step")

    for s in range(sequences):
        qkv, step = project(prompt_tokens), cache.step([(s, prompt_tokens)])
        ms = timed(lambda: layer.prefill(*qkv, step))
        print(f"prompt {s}: {prompt_tokens} tokens, {sparse.k_selected} blocks a row, {ms:.3f} ms")
    decode()
    if budget > 0:
        before = cache.free_pages
        ms = timed(lambda: cache.evict(range(sequences), budget, sinks=min(64, budget // 8), recent=budget // 4))
        print(f"eviction: {sequences} sequences cut to {budget} tokens, {cache.free_pages - before} pages returned, "
              f"{1e3 * ms:.1f} us")
        decode()


if __name__ == "__main__":
    main(budget=int(sys.argv[1]) if len(sys.argv) > 1 else 0)
