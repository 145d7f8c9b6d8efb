"""The serving path as a user runs it: sparse prefill into the pages, then chunks and single tokens over them.

At 100% density the block-sparse prefill is dense causal attention, so every row of prompt, chunk and decode must
match one dense attention over the whole sequence (64 bits, rotations and norms included).  The packed K in the cache
and Q are rounded to bf16 (u = 2^-8) before the attention: a score moves by at most 2 u S, S = scale sum |q_d k_d|, which at
these inputs stays under 0.2, and the tolerance of the framework's bf16 attention tests (2e-2 max, 2e-3 mean) covers
the outputs.
"""
import pytest
import torch

from spruce_research_b200.paged import PagedKVCache, PagedSparseLayer
from spruce_research_b200.pipeline import SparsePrefillLayer
from spruce_research_b200.rope import rope_table
from spruce_research_b200.synthetic import make_gate_weights

pytestmark = pytest.mark.gpu


def reference(q, k, v, wq, wk, table, eps=1e-6):
    """Dense causal attention [T, Hq, D] of one sequence from its projections; rotated Q / K rounded to bf16."""
    T, Hq, D = q.shape

    def turn(x, w):
        x = x.double()
        x = x / (x.square().mean(-1, keepdim=True) + eps).sqrt() * w.double()
        cos, sin = (t[:T, None].double() for t in table.chunk(2, dim=1))
        a, b = x.chunk(2, dim=-1)
        return torch.cat([a * cos - b * sin, b * cos + a * sin], dim=-1).to(torch.bfloat16).double()

    q, k, v = turn(q, wq), turn(k, wk), v.double()
    k, v = (x.repeat_interleave(Hq // x.shape[1], dim=1) for x in (k, v))
    s = torch.einsum("thd,shd->hts", q, k) * D ** -0.5
    s.masked_fill_(torch.ones(T, T, dtype=torch.bool, device=q.device).triu(1), float("-inf"))
    return torch.einsum("hts,shd->thd", s.softmax(-1), v)


@pytest.mark.parametrize("Hq,Hkv,D,page", [(28, 4, 128, 64), (4, 2, 64, 16)])
def test_prefill_chunks_and_decode_match_one_dense_attention(Hq, Hkv, D, page):
    g = torch.Generator(device="cuda").manual_seed(11)
    lengths = {"a": 700, "b": 333}
    prompt, chunk = {"a": 600, "b": 200}, {"a": 90, "b": 128}
    wq, wk = (1 + 0.1 * torch.randn(D, generator=g, device="cuda") for _ in range(2))
    table = rope_table(D, 1024, 1e6)
    gq, gk = make_gate_weights(1, D, D, seed=3, device="cuda")
    cache = PagedKVCache(2, 80, page, Hkv, D)
    cache.k.fill_(float("nan"))
    cache.v.fill_(float("nan"))
    layer = PagedSparseLayer(cache, 1, table, q_weight=wq, k_weight=wk)
    x = {s: torch.randn(n, Hq + 2 * Hkv, D, generator=g, device="cuda", dtype=torch.bfloat16) for s, n in lengths.items()}
    split = lambda y: (y[:, :Hq], y[:, Hq:Hq + Hkv], y[:, Hq + Hkv:])  # noqa: E731
    got = {s: [] for s in lengths}
    for s, n in prompt.items():
        layer.sparse = SparsePrefillLayer(gq[0], gk[0], max(2, -(-n // 64)))         # every block
        out, selected = layer.prefill(*split(x[s][:n]), cache.step([(s, n)]))
        assert selected.shape[1] == Hkv
        got[s].append(out)
    step = cache.step(list(chunk.items()))
    out = layer.extend(*split(torch.cat([x[s][prompt[s]:prompt[s] + n] for s, n in chunk.items()])), step)
    for s, part in zip(chunk, out.split(list(chunk.values()))):
        got[s].append(part)
    at = {s: prompt[s] + chunk[s] for s in lengths}
    while any(at[s] < lengths[s] for s in lengths):
        live = [s for s in lengths if at[s] < lengths[s]]
        out = layer.extend(*split(torch.cat([x[s][at[s]:at[s] + 1] for s in live])), cache.step([(s, 1) for s in live]))
        for i, s in enumerate(live):
            got[s].append(out[i:i + 1])
            at[s] += 1
    for s in lengths:
        want = reference(*split(x[s]), wq, wk, table)
        err = (torch.cat(got[s]).double() - want).abs()
        assert err.max().item() < 2e-2 and err.mean().item() < 2e-3, (s, err.max().item(), err.mean().item())
    assert cache.k[0].isnan().all() and cache.v[0].isnan().all()      # the other layer's pages


def test_the_module_runs_as_a_command(capsys):
    from spruce_research_b200 import paged

    paged.main(prompt_tokens=700, sequences=2, decode_steps=3)
    lines = capsys.readouterr().out.splitlines()
    assert len(lines) == 3 and lines[-1].startswith("decode: 2 sequences at 703 tokens")
