"""Operators on accumulated attention weight, measured: the weight each cached key has received, eviction from the
paged cache by it, the weight of whole key blocks (the gate's teacher), and the distillation of a teacher's top entries.

Where ``own`` is false ``run`` computes the plain form (elementary torch operations in fp32, rounded once); where
it is true it makes the calls of ``spruce_research_b200.native`` and ``spruce_research_b200.selector.loss``.
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
BLOCK = 64


# ------------------------------------------------------------------ cases
def listed():
    return [
        # One decode step of a serving batch: 64 sequences of unequal lengths up to 8192 tokens.
        dict(name="mass_decode_64_at_8k", op="mass", dtype="bf16", seqs=64, q_lo=1, q_hi=1, c_lo=300, c_hi=8191, hq=28,
             hkv=4, d=128, page=64, decay=1.0),
        # The last 64 queries of a whole prompt vote on its keys, before the cache is cut to a budget.
        dict(name="mass_window_64_at_128k", op="mass", dtype="bf16", seqs=1, q_lo=64, q_hi=64, c_lo=131008, c_hi=131008,
             hq=28, hkv=4, d=128, page=64, decay=0.0),
        # A mixed step of idle, decoding and prefilling sequences with odd lengths and small pages; old weight fades.
        dict(name="mass_mixed_f16_page16", op="mass", dtype="f16", seqs=9, q_lo=0, q_hi=300, c_lo=1, c_hi=3001, hq=4,
             hkv=2, d=64, page=16, decay=0.875),
        # A whole prompt cut to an eighth.
        dict(name="evict_one_128k", op="evict", dtype="bf16", seqs=1, c_lo=131072, c_hi=131072, keep=16384, sinks=64,
             recent=1024, hkv=4, d=128, page=64),
        # A serving batch cut to a budget that some of its sequences have not reached.
        dict(name="evict_64_at_8k", op="evict", dtype="bf16", seqs=64, c_lo=300, c_hi=8191, keep=2048, sinks=4,
             recent=256, hkv=4, d=128, page=64),
        # Latency: a few short sequences, an odd budget, small pages.
        dict(name="evict_small_f16", op="evict", dtype="f16", seqs=5, c_lo=40, c_hi=700, keep=333, sinks=1, recent=17,
             hkv=2, d=64, page=16),
        # The teacher of one layer's gate on a 32K prompt.
        dict(name="blocks_32k", op="blocks", dtype="bf16", batch=1, tokens=32768, hq=28, hkv=4, d=128),
        # The same on a shorter prompt of a length that ends inside a block.
        dict(name="blocks_8k_odd", op="blocks", dtype="bf16", batch=1, tokens=8100, hq=28, hkv=4, d=128),
        # A small batch.
        dict(name="blocks_small_f16", op="blocks", dtype="f16", batch=2, tokens=1000, hq=4, hkv=2, d=64),
        # The gate's rows of one layer at 8192 tokens: latency. Loss, then its backward pass.
        dict(name="distill_gate_8k", op="distill", dtype="f32", rows=512, n=128, k=16, causal=True, tau=1.0, fused=False),
        # The gate's rows of 28 layers at 32K tokens, loss and gradient in one call.
        dict(name="distill_gate_28x32k", op="distill", dtype="f32", rows=57344, n=512, k=27, causal=True, tau=2.0,
             fused=True),
        # Rows of a vocabulary from a teacher's 64 best tokens. Loss, then its backward pass.
        dict(name="distill_vocab_131k", op="distill", dtype="bf16", rows=4096, n=131072, k=64, causal=False, tau=1.0,
             fused=False),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["mass", "mass", "evict", "evict", "blocks", "distill", "distill"])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    hq, hkv, d = rng.choice([(28, 4, 128), (4, 2, 64), (16, 16, 64), (32, 8, 128), (14, 2, 64), (8, 1, 128)])
    if op == "distill":
        causal = rng.random() < 0.5
        n = _log(rng, 16, 2048) if causal else _log(rng, 1000, 131072)
        most = 4096 * 131072 // (2 if dtype == "f32" else 1)
        rows = _log(rng, 16, max(17, min(57344, most // n)))
        return dict(op=op, dtype=dtype, rows=rows, n=n, k=min(n, _log(rng, 1, 256)), causal=causal,
                    tau=rng.choice([1.0, 1.0, 2.0, 0.5]), fused=rng.random() < 0.5)
    if op == "blocks":
        batch = rng.choice([1, 1, 2, 3])
        most = 32768 * math.sqrt(28 * 128 / (batch * hq * d)) / (5 if dtype == "f32" else 1)
        return dict(op=op, dtype=dtype, batch=batch, tokens=min(32768, _log(rng, 30, most)), hq=hq, hkv=hkv, d=d)
    seqs = _log(rng, 1, 64)
    page = rng.choice([16, 32, 64, 64, 128])
    if op == "evict":
        c_hi = min(131072, _log(rng, 64, 64 * 8192 * 512 // (seqs * hkv * d) // (2 if dtype == "f32" else 1)))
        c_lo = rng.randint(c_hi // 4, c_hi)
        keep = _log(rng, 16, c_hi)
        recent = rng.randint(0, keep // 2)
        return dict(op=op, dtype=dtype, seqs=seqs, c_lo=c_lo, c_hi=c_hi, keep=keep,
                    sinks=rng.randint(0, min(64, keep - recent)), recent=recent, hkv=hkv, d=d, page=page)
    q_hi = rng.choice([1, 1, _log(rng, 2, 9), _log(rng, 10, 512)])
    budget = 28 * 64 * 131072 // (8 if dtype == "f32" else 1)
    c_most = min(131072 - q_hi, budget // (seqs * hq * q_hi), 64 * 8192 * 512 // (seqs * hkv * d))
    if c_most < 64:
        seqs, c_most = 1, max(64, min(131072 - q_hi, budget // (hq * q_hi)))
    c_hi = _log(rng, 16, c_most)
    return dict(op=op, dtype=dtype, seqs=seqs, q_lo=rng.randint(0, q_hi) if seqs > 1 else q_hi, q_hi=q_hi,
                c_lo=rng.randint(0, c_hi), c_hi=c_hi, hq=hq, hkv=hkv, d=d, page=page,
                decay=rng.choice([1.0, 0.0, 0.5]))


def _spread(lo, hi, n, step):
    """n whole numbers spread over lo .. hi, the last one at the end."""
    return [lo + int(((i + 1) * step) % 1.0 * (hi - lo)) for i in range(n - 1)] + [hi]


def _lengths(case):
    """New tokens and cached tokens of each sequence."""
    n = case["seqs"]
    return (_spread(case["q_lo"], case["q_hi"], n, 0.6180339887498949),
            _spread(case["c_lo"], case["c_hi"], n, 0.7548776662466927))


def work(case):
    es = 4 if case["dtype"] == "f32" else 2
    if case["op"] == "distill":
        rows, n, k = case["rows"], case["n"], case["k"]
        seen = sum(min(n, r % n + 1) for r in range(rows)) if case["causal"] else rows * n
        return {"bytes": seen * es + rows * n * es + rows * k * 8 + rows * 12, "flops": 6 * seen}
    if case["op"] == "blocks":
        b, t, hq, hkv, d = (case[x] for x in ("batch", "tokens", "hq", "hkv", "d"))
        blocks = -(-t // BLOCK)
        return {"bytes": b * t * (hq + hkv) * d * es + 4 * b * hkv * blocks * blocks,
                "flops": 2 * d * b * hq * (t * (t + 1) // 2)}
    hkv, d = case["hkv"], case["d"]
    if case["op"] == "evict":
        held = _spread(case["c_lo"], case["c_hi"], case["seqs"], 0.7548776662466927)
        kept = sum(min(x, case["keep"]) for x in held)
        return {"bytes": hkv * (4 * sum(held) + kept * (4 * d * es + 8)), "flops": hkv * sum(held)}
    hq = case["hq"]
    q, c = _lengths(case)
    seen = sum(a * b + a * (a + 1) // 2 for a, b in zip(q, c))
    keys = sum(a + b for a, b in zip(q, c) if a)
    old = sum(b for a, b in zip(q, c) if a) if case["decay"] else 0
    return {"bytes": keys * hkv * (d * es + 4) + 4 * hkv * old + sum(q) * hq * (d * es + 4), "flops": 2 * d * hq * seen}


# ------------------------------------------------------------------ inputs
def _pages(held, page, seed):
    """A page table of sequences that hold so many tokens, over pages in no order, as after some time of serving."""
    need = [-(-x // page) for x in held]
    order = torch.randperm(sum(need) + 3, generator=torch.Generator().manual_seed(seed))
    table = torch.full((len(held), max(1, max(need))), -1, dtype=torch.int32)
    at = 0
    for s, m in enumerate(need):
        table[s, :m] = order[at:at + m].int()
        at += m
    return table.to("cuda"), sum(need) + 3


def _row_lse(st, seq, a, b, dtype):
    """Natural log of each new token's softmax sum over what it sees: [a, Hq] of a sequence that held b tokens before."""
    c = st["case"]
    rep, page = c["hq"] // c["hkv"], c["page"]
    n = a + b
    pages = st["table"][seq, :-(-n // page)].long()
    q = st["q"][st["at"][seq]:st["at"][seq] + a]
    out = torch.empty(a, c["hq"], device="cuda", dtype=dtype)
    step = max(1, 64 * 1024 * 1024 // (n * rep))
    for g in range(c["hkv"]):
        k = st["k_cache"][pages, g].flatten(0, 1)[:n].to(dtype)
        for t in range(0, a, step):
            e = min(a, t + step)
            z = torch.einsum("thd,kd->htk", q[t:e, g * rep:(g + 1) * rep].to(dtype), k) * c["d"] ** -0.5
            late = torch.arange(n, device="cuda") > torch.arange(b + t, b + e, device="cuda")[:, None]
            out[t:e, g * rep:(g + 1) * rep] = torch.logsumexp(z.masked_fill_(late, -math.inf), -1).T
    return out


def prepare(case, seed):
    dev = "cuda"
    g = torch.Generator(device=dev).manual_seed(seed)
    dt = DTYPES[case["dtype"]]

    def rand(*shape, scale=1.0):
        return torch.randn(*shape, generator=g, device=dev, dtype=dt) * scale

    st = dict(case=case)
    if case["op"] == "distill":
        rows, n, k = case["rows"], case["n"], case["k"]
        # A student that follows its teacher loosely; both peaked, as logits are.
        st["scores"] = rand(rows, n, scale=2.0)
        st["visible"] = None
        if case["causal"]:  # row r scores the key blocks up to its own
            st["visible"] = (torch.arange(rows, device=dev) % n + 1).int()
        ids = torch.empty(rows, k, device=dev, dtype=torch.int64)
        best = torch.empty(rows, k, device=dev)
        for r in range(0, rows, 1024):
            t = st["scores"][r:r + 1024].float() * 0.7 + torch.randn(len(st["scores"][r:r + 1024]), n, generator=g,
                                                                      device=dev)
            if case["causal"]:
                t.masked_fill_(torch.arange(n, device=dev) >= st["visible"][r:r + 1024, None], -math.inf)
            best[r:r + 1024], ids[r:r + 1024] = t.topk(k, -1)
        gone = best == -math.inf
        st["ids"], st["teacher"] = ids.masked_fill(gone, -1).int(), best.masked_fill(gone, 0.0)
        st["weight"] = 0.5 + torch.rand(rows, generator=g, device=dev)
        return st
    hkv, d = case["hkv"], case["d"]
    if case["op"] == "blocks":
        b, t, hq = case["batch"], case["tokens"], case["hq"]
        # [B, H, T, D] views of the fused projection [B, T, (Hq + Hkv) * D]
        qk = rand(b, t, hq + hkv, d)
        st["q"], st["k"] = qk[:, :, :hq].transpose(1, 2), qk[:, :, hq:].transpose(1, 2)
        return st
    page = case["page"]
    if case["op"] == "evict":
        held = _spread(case["c_lo"], case["c_hi"], case["seqs"], 0.7548776662466927)
        st["table"], n = _pages(held, page, seed)
        st["held"] = torch.tensor(held, device=dev, dtype=torch.int32)
        st["k_cache"], st["v_cache"] = rand(n, hkv, page, d), rand(n, hkv, page, d)
        # Few keys carry most of the weight; some have none that fp32 can hold.
        mass = torch.exp(2.5 * torch.randn(n, hkv, page, generator=g, device=dev))
        st["mass"] = torch.where(torch.rand(n, hkv, page, generator=g, device=dev) < 0.05, 0.0, mass)
        # Where the kept rows go: other pages.
        st["to_table"], m = _pages([min(x, case["keep"]) for x in held], page, seed + 1)
        st["to"] = rand(m, hkv, page, d), rand(m, hkv, page, d), torch.zeros(m, hkv, page, device=dev)
        st["most"] = max(held)
        return st
    qlen, clen = _lengths(case)
    kv = [a + b for a, b in zip(qlen, clen)]
    st["table"], n = _pages(kv, page, seed)
    st["cu_q"] = torch.tensor([0] + qlen, device=dev, dtype=torch.int32).cumsum(0, dtype=torch.int32)
    st["kv_lens"] = torch.tensor(kv, device=dev, dtype=torch.int32)
    st["max_q"], st["max_kv"] = max(qlen), max(kv)
    st["k_cache"] = rand(n, hkv, page, d)
    st["mass"] = torch.rand(n, hkv, page, generator=g, device=dev)
    st["to"] = torch.zeros(n, hkv, page, device=dev)
    # Twice the unit scale: about one key in fifty carries a query's weight.
    st["q"] = rand(sum(qlen), case["hq"], d, scale=2.0)
    st["at"] = [sum(qlen[:s]) for s in range(len(qlen))]
    # What the attention of these tokens leaves behind.
    st["lse"] = torch.cat([_row_lse(st, s, a, b, torch.float32) for s, (a, b) in enumerate(zip(qlen, clen))])
    return st


# ------------------------------------------------------------------ plain forms
def _plain_mass(st):
    c = st["case"]
    q, n = st["q"], st["q"].shape[0]
    hq, hkv, d, rep, page = c["hq"], c["hkv"], c["d"], c["hq"] // c["hkv"], c["page"]
    most_q, most_kv = st["max_q"], st["max_kv"]
    cu, table = st["cu_q"].long(), st["table"].long().clamp(min=0)
    i, j = torch.arange(most_q, device=q.device), torch.arange(most_kv, device=q.device)
    out = st["to"]
    step = max(1, (1 << 28) // (most_kv * most_q * hq))  # sequences at a time
    for s0 in range(0, c["seqs"], step):
        kv = st["kv_lens"][s0:s0 + step].long()
        first = cu[s0:s0 + len(kv)]
        qlen = cu[s0 + 1:s0 + 1 + len(kv)] - first
        pages = table[s0:s0 + len(kv)]
        k = st["k_cache"][pages].transpose(1, 2).reshape(len(kv), hkv, -1, d)[:, :, :most_kv].float()
        at = (first[:, None] + i).clamp(max=max(n - 1, 0))
        rows = q[at].float().reshape(len(kv), most_q, hkv, rep, d).permute(0, 2, 3, 1, 4)
        lse = st["lse"][at].reshape(len(kv), most_q, hkv, rep).permute(0, 2, 3, 1)
        p = (rows.reshape(len(kv), hkv, rep * most_q, d) * d ** -0.5) @ k.transpose(-1, -2)
        p = p.view(len(kv), hkv, rep, most_q, most_kv).sub_(lse[..., None]).exp_()
        seen = (j <= (kv - qlen)[:, None, None] + i[:, None]) & (i < qlen[:, None])[..., None]
        p.masked_fill_(~seen[:, None, None], 0.0)
        total = p.sum((2, 3))                                                     # [S, Hkv, K]
        s, x = torch.nonzero((j < kv[:, None]) & (qlen > 0)[:, None], as_tuple=True)
        at_page, row = pages[s, x // page], x % page
        old = torch.where((x < (kv - qlen)[s])[:, None], st["mass"][at_page, :, row] * c["decay"], 0.0)
        out[at_page, :, row] = total[s, :, x] + old
    return {"mass": out}


def _plain_evict(st):
    c = st["case"]
    hkv, page, keep = c["hkv"], c["page"], c["keep"]
    held, table, to_table = st["held"].long(), st["table"].long().clamp(min=0), st["to_table"].long()
    most = table.shape[1] * page
    j = torch.arange(most, device=held.device)
    rank = st["mass"][table].transpose(1, 2).reshape(c["seqs"], hkv, most).clone()
    always = (j < c["sinks"]) | (j >= held[:, None] - c["recent"])
    rank.masked_fill_(always[:, None], math.inf)
    rank.masked_fill_((j >= held[:, None])[:, None], -math.inf)
    width = min(keep, st["most"])
    kept = torch.sort(rank, dim=-1, descending=True, stable=True).indices[..., :width]
    new = held.clamp(max=keep)
    there = (torch.arange(width, device=held.device) < new[:, None])[:, None].expand(-1, hkv, -1)
    kept = kept.masked_fill(~there, most).sort(-1).values
    s, h, x = torch.nonzero(there, as_tuple=True)
    src = kept[s, h, x]
    for a, b in zip((st["k_cache"], st["v_cache"], st["mass"]), st["to"]):
        b[to_table[s, x // page], h, x % page] = a[table[s, src // page], h, src % page]
    k, v, m = st["to"]
    return {"kept": kept.masked_fill(~there, -1).int(), "lens": new.int(), "k": k, "v": v, "mass": m}


def _plain_blocks(st):
    c = st["case"]
    b, t, hq, hkv, d = (c[x] for x in ("batch", "tokens", "hq", "hkv", "d"))
    rep, blocks = hq // hkv, -(-t // BLOCK)
    out = torch.zeros(b, hkv, blocks, blocks, device="cuda")
    step = max(BLOCK, (1 << 28) // (rep * t) // BLOCK * BLOCK)  # queries at a time
    u = torch.arange(t, device="cuda")
    for x in range(b):
        for g in range(hkv):
            k = st["k"][x, g].float()
            for t0 in range(0, t, step):
                t1 = min(t, t0 + step)
                s = (st["q"][x, g * rep:(g + 1) * rep, t0:t1].float() * d ** -0.5) @ k[:t1].T
                s.masked_fill_(u[:t1] > u[t0:t1, None], -math.inf)
                s.sub_(s.amax(-1, keepdim=True)).exp_()
                s.div_(s.sum(-1, keepdim=True))
                p = torch.zeros(-(-(t1 - t0) // BLOCK) * BLOCK, -(-t1 // BLOCK) * BLOCK, device="cuda")
                p[:t1 - t0, :t1] = s.sum(0)
                p = p.view(p.shape[0] // BLOCK, BLOCK, p.shape[1] // BLOCK, BLOCK).sum((1, 3))
                first = torch.arange(t0, t1, BLOCK, device="cuda")
                n = (t1 - first).clamp(max=BLOCK)
                out[x, g, t0 // BLOCK:t0 // BLOCK + len(first), :p.shape[1]] = p / (n * rep)[:, None]
    return {"mass": out}


def _plain_distill(st):
    c = st["case"]
    s, ids, tau = st["scores"], st["ids"].long(), c["tau"]
    z = s.float() / tau
    if st["visible"] is not None:
        z = z.masked_fill(torch.arange(c["n"], device=s.device) >= st["visible"][:, None], -math.inf)
    z = z - z.amax(-1, keepdim=True)
    lsum = z.exp().sum(-1, keepdim=True).log()
    there = ids >= 0
    t = (st["teacher"].float() / tau).masked_fill(~there, -math.inf)
    t = t - t.amax(-1, keepdim=True)
    log_p = t - t.exp().sum(-1, keepdim=True).log()
    p = log_p.exp()
    log_q = z.gather(-1, ids.clamp(min=0)) - lsum
    loss = torch.where(there, p * (log_p - log_q), 0.0).sum(-1)
    grad = (z - lsum).exp_()
    grad.scatter_add_(-1, ids.clamp(min=0), -p)
    grad *= (st["weight"] / tau)[:, None]
    return {"loss": loss, "grad": grad.to(s.dtype)}


def run(st):
    c = st["case"]
    op = c["op"]
    if not own:
        return {"mass": _plain_mass, "evict": _plain_evict, "blocks": _plain_blocks, "distill": _plain_distill}[op](st)
    from spruce_research_b200 import native
    from spruce_research_b200.selector.loss import topk_distill_loss

    if op == "mass":
        return {"mass": native.paged_key_mass(st["q"], st["k_cache"], st["mass"], st["table"], st["cu_q"],
                                              st["kv_lens"], st["lse"], max_q_len=st["max_q"],
                                              max_kv_len=st["max_kv"], decay=c["decay"], out=st["to"])}
    if op == "evict":
        k, v, m = st["to"]
        kept, lens = native.paged_evict(st["k_cache"], st["v_cache"], st["mass"], st["table"], st["held"], c["keep"],
                                        sinks=c["sinks"], recent=c["recent"], max_kv_len=st["most"],
                                        into=(k, v, m, st["to_table"]))
        return {"kept": kept, "lens": lens, "k": k, "v": v, "mass": m}
    if op == "blocks":
        return {"mass": native.block_mass(st["q"], st["k"])}
    if c["fused"]:
        loss, grad = native.topk_distill(st["scores"], st["ids"], st["teacher"], visible=st["visible"],
                                         temperature=c["tau"], grad_weight=st["weight"])
        return {"loss": loss, "grad": grad}
    scores = st["scores"].detach().requires_grad_()
    loss = topk_distill_loss(scores, st["ids"], st["teacher"], visible=st["visible"], temperature=c["tau"])
    grad, = torch.autograd.grad(loss, scores, st["weight"])
    return {"loss": loss.detach(), "grad": grad}


# ------------------------------------------------------------------ the definition in 64 bits
def _exact_mass(st, case):
    qlen, clen = _lengths(case)
    page, rep, d = case["page"], case["hq"] // case["hkv"], case["d"]
    out = st["to"].double()
    at = 0
    for s, (a, b) in enumerate(zip(qlen, clen)):
        if not a:
            continue
        n = a + b
        pages = st["table"][s, :-(-n // page)].long()
        x = torch.arange(n, device="cuda")
        old = torch.where(x < b, case["decay"], 0.0).double()
        for g in range(case["hkv"]):
            k = st["k_cache"][pages, g].double().flatten(0, 1)[:n]
            total = old * st["mass"][pages, g].double().flatten()[:n]
            for t in range(0, a, 32):
                e = min(a, t + 32)
                z = torch.einsum("thd,kd->thk", st["q"][at + t:at + e, g * rep:(g + 1) * rep].double(), k) / math.sqrt(d)
                z = z - st["lse"][at + t:at + e, g * rep:(g + 1) * rep].double()[..., None]
                seen = x <= torch.arange(b + t, b + e, device="cuda")[:, None, None]
                total += torch.where(seen, torch.exp(z), 0.0).sum((0, 1))
            out[pages[x // page], g, x % page] = total
        at += a
    return {"mass": out}


def _exact_evict(st, case):
    held = _spread(case["c_lo"], case["c_hi"], case["seqs"], 0.7548776662466927)
    page, hkv = case["page"], case["hkv"]
    k, v, m = (x.double() for x in st["to"])
    width = min(case["keep"], max(held))
    kept = torch.full((len(held), hkv, width), -1, device="cuda", dtype=torch.int32)
    table, to_table = st["table"].long(), st["to_table"].long()
    for s, n in enumerate(held):
        slot = torch.arange(n, device="cuda")
        for h in range(hkv):
            weight = st["mass"][table[s, slot // page], h, slot % page]
            if n <= case["keep"]:
                chosen = slot
            else:
                lo, hi = case["sinks"], n - case["recent"]
                order = torch.argsort(weight[lo:hi], descending=True, stable=True)[:case["keep"] - lo - case["recent"]]
                chosen = torch.cat([slot[:lo], lo + order.sort().values, slot[hi:]])
            kept[s, h, :len(chosen)] = chosen.int()
            to = slot[:len(chosen)]
            for a, b in zip((st["k_cache"], st["v_cache"], st["mass"]), (k, v, m)):
                b[to_table[s, to // page], h, to % page] = a[table[s, chosen // page], h, chosen % page].double()
    return {"kept": kept, "lens": torch.tensor([min(n, case["keep"]) for n in held], device="cuda", dtype=torch.int32),
            "k": k, "v": v, "mass": m}


def _exact_blocks(st, case):
    b, t, hq, hkv, d = (case[x] for x in ("batch", "tokens", "hq", "hkv", "d"))
    rep, blocks = hq // hkv, -(-t // BLOCK)
    out = torch.zeros(b, hkv, blocks, blocks, device="cuda", dtype=torch.float64)
    member = (torch.arange(t, device="cuda")[:, None] // BLOCK == torch.arange(blocks, device="cuda")).double()
    for x in range(b):
        for h in range(hq):
            k = st["k"][x, h // rep].double()
            for t0 in range(0, t, 2048):
                t1 = min(t, t0 + 2048)
                z = st["q"][x, h, t0:t1].double() @ k[:t1].T / math.sqrt(d)
                late = torch.arange(t1, device="cuda") > torch.arange(t0, t1, device="cuda")[:, None]
                p = torch.softmax(z.masked_fill(late, -math.inf), -1)
                mine = member[t0:t1]
                out[x, h // rep] += mine.T @ (p @ member[:t1])
    return {"mass": out / (member.sum(0) * rep)[:, None]}


def _exact_distill(st, case):
    rows, n, tau = case["rows"], case["n"], case["tau"]
    loss = torch.empty(rows, device="cuda", dtype=torch.float64)
    grad = torch.empty(rows, n, device="cuda", dtype=torch.float64)
    step = max(1, (1 << 25) // n)
    for r in range(0, rows, step):
        z = st["scores"][r:r + step].double() / tau
        if st["visible"] is not None:
            z = z.masked_fill(torch.arange(n, device="cuda") >= st["visible"][r:r + step, None], -math.inf)
        ids = st["ids"][r:r + step].long()
        p = torch.softmax((st["teacher"][r:r + step].double() / tau).masked_fill(ids < 0, -math.inf), -1)
        target = torch.zeros_like(z).scatter_add_(-1, ids.clamp(min=0), p)
        log_q = torch.log_softmax(z, -1)
        # Entropy and cross entropy; what the teacher gives no weight counts as nothing.
        loss[r:r + step] = torch.special.xlogy(p, p).sum(-1) - torch.where(target > 0, target * log_q, 0.0).sum(-1)
        grad[r:r + step] = (log_q.exp() - target) * (st["weight"][r:r + step].double() / tau)[:, None]
    return {"loss": loss, "grad": grad}


def exact(case, seed):
    st = prepare(case, seed)
    return {"mass": _exact_mass, "evict": _exact_evict, "blocks": _exact_blocks,
            "distill": _exact_distill}[case["op"]](st, case)
