"""Serving a layer after its sparse prefill: a paged K/V cache, appended to and attended over.

The reference stops at prefill: its callback sends decode to SDPA over the model's dense cache
(kernels/sparse_prefill.py:63-65).  Here a prompt runs the selector and the block-sparse attention and leaves its keys
and values in pages; every later chunk or token is appended with its head norms and rotation in one launch and attends
over the pages.

``PagedKVCache`` owns the pages of every layer and the sequences' page tables (host), ``PagedStep`` is one forward's
batch (device), ``PagedSparseLayer`` runs one layer of it.

    python -m spruce_research_b200.paged          # a small layer: prompts, then decode steps, with their times
"""
from __future__ import annotations

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


class PagedKVCache:
    """Pages of ``page_size`` tokens for ``num_layers`` layers: ``k`` and ``v`` [layers, pages, Hkv, page_size, D].

    A page id names the same page of every layer.  Heads lie outside the tokens of a page, so that one head's page
    is one contiguous block.
    """

    def __init__(self, num_layers: int, num_pages: int, page_size: int, kv_heads: int, head_dim: int,
                 dtype: torch.dtype = torch.bfloat16, device="cuda"):
        if page_size < 16 or page_size % 16:
            raise ValueError(f"page_size must be a multiple of 16, got {page_size}")
        if min(num_layers, num_pages, kv_heads, head_dim) < 1:
            raise ValueError("layers, pages, KV heads and head_dim must be positive")
        shape = (num_layers, num_pages, kv_heads, page_size, head_dim)
        self.k = torch.empty(shape, dtype=dtype, device=device)
        self.v = torch.empty(shape, dtype=dtype, device=device)
        self.page_size = page_size
        self._free = list(range(num_pages - 1, -1, -1))
        self._pages: dict = {}
        self._length: dict = {}

    @property
    def free_pages(self) -> int:
        return len(self._free)

    def length(self, seq_id) -> int:
        """Tokens the sequence holds (0 for one the cache does not know)."""
        return self._length.get(seq_id, 0)

    def drop(self, seq_id) -> None:
        """Return a sequence's pages.  Kernels of its last step may still run: the next step's follow them."""
        self._free.extend(reversed(self._pages.pop(seq_id, [])))
        self._length.pop(seq_id, None)

    def truncate(self, seq_id, length: int) -> None:
        """Keep a sequence's first ``length`` tokens: drafts that were rejected, or a step whose forward did not run."""
        held = self.length(seq_id)
        if not 0 <= length <= held:
            raise ValueError(f"a sequence of {held} tokens cannot be cut to {length}")
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
        width = max([len(self._pages[s]) for s, _ in new_tokens], default=0)
        S = len(new_tokens)
        # One host tensor and one copy: table, offsets, lengths.
        host = torch.zeros(S * width + 2 * S + 1, dtype=torch.int32)
        table, cu, kv = host[:S * width].view(S, width), host[S * width:S * width + S + 1], host[S * width + S + 1:]
        for i, (s, n) in enumerate(new_tokens):
            pages = self._pages[s]
            table[i, :len(pages)] = torch.tensor(pages, dtype=torch.int32)
            cu[i + 1] = cu[i] + n
            kv[i] = lengths[i]
        dev = host.to(self.k.device)
        return PagedStep([s for s, _ in new_tokens], dev[:S * width].view(S, width), dev[S * width:S * width + S + 1],
                         dev[S * width + S + 1:], max((n for _, n in new_tokens), default=0), max(lengths, default=0),
                         int(cu[-1]))


class PagedSparseLayer:
    """One attention layer over a :class:`PagedKVCache`: sparse prefill of prompts, then chunks and single tokens.

    Takes the projections before norms and rotation, packed ``q [N, Hq, D]``, ``k`` / ``v`` [N, Hkv, D].  ``rope`` is a
    :func:`rope.rope_table` of the longest sequence (None: no rotation); ``q_weight`` / ``k_weight`` are head norms (None: no norm).
    """

    def __init__(self, cache: PagedKVCache, layer_idx: int, rope: torch.Tensor | None, *,
                 prefill: SparsePrefillLayer | None = None, q_weight: torch.Tensor | None = None,
                 k_weight: torch.Tensor | None = None, eps: float = 1e-6, interleaved: bool = False):
        if not 0 <= layer_idx < cache.k.shape[0]:
            raise ValueError(f"layer_idx {layer_idx} is outside the cache's {cache.k.shape[0]} layers")
        self.k_cache, self.v_cache = cache.k[layer_idx], cache.v[layer_idx]
        self.rope, self.sparse = rope, prefill
        self.rotation = dict(q_weight=q_weight, k_weight=k_weight, eps=eps, interleaved=interleaved)

    def _check(self, tensors, step: PagedStep, spare: bool) -> None:
        """What the host knows: the kernels would leave rows out, take the nearest angles and only report it in a status."""
        rows = [x.shape[0] for x in tensors]
        if min(rows) < step.tokens or not spare and max(rows) > step.tokens:
            raise ValueError(f"the step has {step.tokens} tokens, q, k and v have {rows}")
        if self.rope is not None and step.max_kv_len > self.rope.shape[0]:
            raise ValueError(f"sequences of {step.max_kv_len} tokens need a rotation table of as many positions, got "
                             f"{self.rope.shape[0]}")

    def extend(self, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, step: PagedStep,
               out: torch.Tensor | None = None) -> torch.Tensor:
        """Append the step's tokens and attend over all each sequence holds: [N, Hq, D].

        N may exceed the step's tokens; the rows past them are not written.
        """
        self._check((q, k, v), step, spare=True)
        q = native.paged_append(k, v, self.k_cache, self.v_cache, step.block_table, step.cu_q, step.kv_lens, q=q,
                                rope=self.rope, **self.rotation)
        return native.paged_attention(q, self.k_cache, self.v_cache, step.block_table, step.cu_q, step.kv_lens,
                                      max_q_len=step.max_q_len, max_kv_len=step.max_kv_len, out=out)

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
        return out[0], selected


def main(prompt_tokens: int = 8192, sequences: int = 4, decode_steps: int = 32) -> None:
    """Prompts through the sparse prefill, then decode steps of all of them, on one 28-query / 4-KV-head layer."""
    from .rope import rope_table
    from .synthetic import k_for_density, make_gate_weights

    Hq, Hkv, D, page = 28, 4, 128, 64
    total = prompt_tokens + decode_steps
    cache = PagedKVCache(1, sequences * -(-total // page), page, Hkv, D)
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

    for s in range(sequences):
        qkv, step = project(prompt_tokens), cache.step([(s, prompt_tokens)])
        ms = timed(lambda: layer.prefill(*qkv, step))
        print(f"prompt {s}: {prompt_tokens} tokens, {sparse.k_selected} blocks a row, {ms:.3f} ms")
    for i in range(decode_steps):
        qkv, step = project(sequences), cache.step([(s, 1) for s in range(sequences)])
        ms = timed(lambda: layer.extend(*qkv, step))
    print(f"decode: {sequences} sequences at {step.max_kv_len} tokens, {1e3 * ms:.1f} us for the last step")


if __name__ == "__main__":
    main()
