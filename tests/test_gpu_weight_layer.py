"""Attention weight as a user runs it: a layer that serves, is cut to a budget and goes on, and a gate that is taught.

After an eviction each head attends to tokens of its own; the cache then says which keys it holds, so the next step is checked
against 64-bit attention over those, its new tokens rotated to their true positions.  Tolerances of outputs are the framework's for
bf16 attention (2e-2 max, 2e-3 mean); weights of bf16 scores that a rounding of Q and K moved are compared loosely, as their
kernel has tests of its own.
"""
import math

import pytest
import torch

from spruce_research_b200 import native
from spruce_research_b200.paged import PagedKVCache, PagedSparseLayer
from spruce_research_b200.pipeline import SparsePrefillLayer
from spruce_research_b200.rope import rope_table
from spruce_research_b200.selector import train
from spruce_research_b200.selector.gate import FlatGate
from spruce_research_b200.synthetic import make_gate_weights

pytestmark = pytest.mark.gpu


def rows(cache, x, layer, seq, n):
    """Rows [n, Hkv, ...] of a sequence's slots."""
    j = torch.arange(n, device="cuda")
    pages = torch.tensor(cache._pages[seq], device="cuda")
    return x[layer][pages[j // cache.page_size], :, j % cache.page_size]


def turned(x, table, first):
    """Rotation of x [n, H, D] from position `first` on, in 64 bits, rounded to bf16."""
    n = x.shape[0]
    cos, sin = (t[first:first + n, None].double() for t in table.chunk(2, dim=1))
    a, b = x.double().chunk(2, dim=-1)
    return torch.cat([a * cos - b * sin, b * cos + a * sin], dim=-1).to(torch.bfloat16)


def attend(q, k, v):
    """64-bit causal attention and weights of the last rows: q [a, Hq, D], k / v [n, Hkv, D] -> [a, Hq, D], [n, Hkv]."""
    a, Hq, D = q.shape
    n, Hkv, _ = k.shape
    kk, vv = (x.double().repeat_interleave(Hq // Hkv, dim=1) for x in (k, v))
    s = torch.einsum("thd,shd->hts", q.double(), kk) * D ** -0.5
    s.masked_fill_(torch.arange(n, device="cuda") > torch.arange(n - a, n, device="cuda")[:, None], -math.inf)
    p = s.softmax(-1)
    return torch.einsum("hts,shd->thd", p, vv), p.sum(1).view(Hkv, Hq // Hkv, n).sum(1).T


@pytest.mark.parametrize("Hq,Hkv,D,page", [(28, 4, 128, 64), (4, 2, 64, 16)])
@pytest.mark.parametrize("rope", [True, False])
def test_a_layer_serves_is_cut_and_goes_on(Hq, Hkv, D, page, rope):
    g = torch.Generator(device="cuda").manual_seed(5)
    table = rope_table(D, 2048, 1e6) if rope else None
    plain = rope_table(D, 2048, 1e6) if rope else torch.cat([torch.ones(2048, D // 2), torch.zeros(2048, D // 2)], 1).cuda()
    gq, gk = make_gate_weights(1, D, D, seed=3, device="cuda")
    cache = PagedKVCache(2, 200, page, Hkv, D, track_mass=True)
    cache.mass.fill_(float("nan"))                       # new tokens start from zero, whatever a page held
    layer = PagedSparseLayer(cache, 1, table, decay=0.5, observe=32)
    split = lambda y: (y[:, :Hq], y[:, Hq:Hq + Hkv], y[:, Hq + Hkv:])  # noqa: E731

    def tokens(n):
        return torch.randn(n, Hq + 2 * Hkv, D, generator=g, device="cuda", dtype=torch.bfloat16)

    prompt, keep = {"a": 700, "b": 150}, 200
    mass = {}
    for s, n in prompt.items():
        x = tokens(n)
        layer.sparse = SparsePrefillLayer(gq[0], gk[0], max(2, -(-n // 64)))
        layer.prefill(*split(x), cache.step([(s, n)]))
        q, k, v = split(x)
        _, mass[s] = attend(turned(q, plain, 0)[-32:], turned(k, plain, 0), v)
        got = rows(cache, cache.mass, 1, s, n)
        assert torch.allclose(got.double(), mass[s], rtol=0.1, atol=1e-4) and abs(got.sum() / (32 * Hq) - 1) < 1e-2

    for round in range(3):
        n = {"a": 5, "b": 1}
        x = tokens(6)
        held = {s: (rows(cache, cache.k, 1, s, cache.length(s)), rows(cache, cache.v, 1, s, cache.length(s)),
                    rows(cache, cache.mass, 1, s, cache.length(s))) for s in n}
        at = {s: cache.position(s) for s in n}
        step = cache.step(list(n.items()))
        out = layer.extend(*split(x), step)
        for s, part, y in zip(n, out.split([5, 1]), x.split([5, 1])):
            q, k, v = split(y)
            k = torch.cat([held[s][0], turned(k, plain, at[s])])
            want, weight = attend(turned(q, plain, at[s]), k, torch.cat([held[s][1], v]))
            err = (part.double() - want).abs()
            assert err.max() <= 2e-2 and err.mean() <= 2e-3
            got = rows(cache, cache.mass, 1, s, cache.length(s)).double()
            old = torch.cat([0.5 * held[s][2].double(), torch.zeros(n[s], Hkv, device="cuda")])
            assert torch.allclose(got, old + weight, rtol=0.1, atol=1e-4)
            assert (rows(cache, cache.k, 1, s, cache.length(s)) - k).abs().max() <= 2.0 ** -5   # the new keys' rounding
        before = {s: [rows(cache, y, 1, s, cache.length(s)) for y in (cache.k, cache.v, cache.mass)] for s in n}
        lengths = {s: cache.length(s) for s in n}
        free = cache.free_pages
        assert cache.evict(["a", "b"], keep, sinks=4, recent=50) == [s for s in n if lengths[s] > keep]
        for s in n:
            assert cache.length(s) == min(lengths[s], keep) and cache.position(s) == at[s] + n[s]
            after = [rows(cache, y, 1, s, cache.length(s)) for y in (cache.k, cache.v, cache.mass)]
            for h in range(Hkv):
                kept = torch.arange(lengths[s], device="cuda")
                if lengths[s] > keep:
                    w = before[s][2][4:lengths[s] - 50, h]
                    best = torch.sort(w, dim=0, descending=True, stable=True).indices[:keep - 54].sort().values + 4
                    kept = torch.cat([kept[:4], best, kept[-50:]])
                for x0, x1 in zip(before[s], after):
                    assert torch.equal(x0[kept, h], x1[:, h])
        assert cache.free_pages == free + sum(-(-lengths[s] // page) - -(-cache.length(s) // page) for s in n)


def test_the_paged_command_evicts(capsys):
    from spruce_research_b200 import paged

    paged.main(prompt_tokens=512, sequences=2, decode_steps=3, budget=128)
    said = capsys.readouterr().out
    assert "2 sequences at 515 tokens" in said and "cut to 128 tokens" in said and "2 sequences at 131 tokens" in said


@pytest.mark.parametrize("P, tau", [(1, 1.0), (1, 2.0), (4, 1.0)])
def test_the_gates_gradient_is_the_formulas(P, tau):
    """Wq and Wk by the loss against 64-bit autograd of the formula.  fp32 projections, scores and their gradients are each sums of at
    most 64 products of values under 10: relative to the largest gradient they are good to 1e-4."""
    g = torch.Generator(device="cuda").manual_seed(2)
    L, G, qb, d, K = 2, 3, 20, 64, 5
    gate = FlatGate(L, d, 32).cuda()
    q, k = (torch.randn(L, G, qb, P, d, generator=g, device="cuda", dtype=torch.bfloat16) for _ in range(2))
    mass = torch.rand(L, G, qb, qb, generator=g, device="cuda").tril()
    ids, teacher = train.teacher_top_blocks(mass / mass.sum(-1, keepdim=True), K)
    loss = train.gate_loss(gate, q, k, ids, teacher, temperature=tau)
    loss.backward()
    W = [w.detach().double().requires_grad_() for w in (gate.Wq, gate.Wk)]
    qp, kp = (torch.einsum("lgqpd,lde->lgqpe", x.double(), w) for x, w in zip((q, k), W))
    s = torch.einsum("lgqpe,lgkre->lgqkpr", qp, kp).amax((-1, -2)) / 32 ** 0.5 / tau
    s = s.masked_fill(torch.ones(qb, qb, device="cuda", dtype=torch.bool).triu(1), -math.inf)
    p = torch.softmax((teacher.double() / tau).masked_fill(ids < 0, -math.inf), -1)
    log_q = torch.log_softmax(s, -1).gather(-1, ids.long().clamp(min=0))
    want = torch.where(ids >= 0, p * (p.clamp(min=1e-300).log() - log_q), 0.0).sum(-1).mean()
    want.backward()
    assert abs(loss.item() - want.item()) <= 1e-5 * max(1.0, want.item())
    for w, x in zip((gate.Wq, gate.Wk), W):
        assert (w.grad - x.grad).abs().max() <= 1e-4 * x.grad.abs().max()


def test_a_layers_teacher_and_the_training_command():
    g = torch.Generator(device="cuda").manual_seed(2)
    q, k = (torch.randn(1, h, 400, 64, generator=g, device="cuda", dtype=torch.bfloat16) for h in (4, 2))
    ids, teacher = train.layer_teacher(q, k, 3)
    mass = native.block_mass(q, k)
    assert ids.shape == teacher.shape == (1, 2, 7, 3) and (ids[:, :, 0] == torch.tensor([0, -1, -1], device="cuda")).all()
    assert torch.equal(teacher[:, :, 6].exp().round(decimals=5), mass[:, :, 6].topk(3, -1).values.round(decimals=5))
    losses = train.main(tokens=512, steps=2, top=4)
    assert len(losses) == 2 and all(math.isfinite(x) for x in losses)


@pytest.mark.parametrize("Hq,Hkv,D,page", [(28, 4, 128, 64), (4, 2, 64, 16)])
def test_rejected_drafts_leave_no_weight(Hq, Hkv, D, page):
    """Draft, truncate, accept, twice, against the same tokens without the rejected ones.  The keys are the same; the log-sums may come
    from kernels of other row counts, each good to 1e-4, twice that for every weight, which fading does not enlarge."""
    g = torch.Generator(device="cuda").manual_seed(8)
    table = rope_table(D, 1024, 1e6)
    caches = [PagedKVCache(1, 120, page, Hkv, D, track_mass=True) for _ in range(2)]
    layers = [PagedSparseLayer(c, 0, table, decay=0.75) for c in caches]
    split = lambda y: (y[:, :Hq], y[:, Hq:Hq + Hkv], y[:, Hq + Hkv:])  # noqa: E731

    def tokens(n):
        return torch.randn(n, Hq + 2 * Hkv, D, generator=g, device="cuda", dtype=torch.bfloat16)

    held = {"a": 300, "b": 77, "c": 40}
    x = tokens(sum(held.values()))
    for c, layer in zip(caches, layers):
        layer.extend(*split(x), c.step(list(held.items())))
    before = rows(caches[0], caches[0].mass, 0, "c", 40).clone()
    for drafts, good in (((5, 9, 3), (2, 9, 0)), ((12, 1, 4), (7, 0, 0))):
        parts = [tokens(n) for n in drafts]
        step = caches[0].step(list(zip("abc", drafts)))
        out, seen = layers[0].draft(*split(torch.cat(parts)), step)
        for s, n, kept in zip("abc", drafts, good):
            caches[0].truncate(s, caches[0].length(s) - n + kept)
        layers[0].accept(seen, step)
        kept = [(s, n) for s, n in zip("abc", good) if n]
        want = layers[1].extend(*split(torch.cat([p[:n] for p, n in zip(parts, good)])), caches[1].step(kept))
        got = torch.cat([o[:n] for o, n in zip(out.split(drafts), good)])
        assert (got.double() - want.double()).abs().max() <= 2e-2
    assert torch.equal(rows(caches[0], caches[0].mass, 0, "c", 40), before)
    x = tokens(3)
    for c, layer in zip(caches, layers):
        layer.extend(*split(x), c.step([("a", 1), ("b", 1), ("c", 1)]))
    for s, n in {"a": 310, "b": 87, "c": 41}.items():
        assert caches[0].length(s) == caches[1].length(s) == n
        a, b = (rows(c, c.mass, 0, s, n) for c in caches)
        assert torch.allclose(a, b, rtol=2e-4, atol=1e-6) and a.sum() > Hq
