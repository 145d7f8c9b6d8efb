"""The serving operators around a sparse-prefill layer, measured: the rotation with its head norms, the append
to a paged K/V cache, and the attention of new tokens over that cache.

Where ``own`` is false ``run`` computes the plain form (elementary torch operations in fp32, rounded once); where
it is true it makes the calls of ``spruce_research_b200.native``.
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
EPS = 1e-6


# ------------------------------------------------------------------ cases
def listed():
    return [
        # A whole prompt of the 128K-token layer (28 query / 4 KV heads, d = 128): rotation only.
        dict(name="rope_prompt_128k", op="rope", dtype="bf16", batch=1, tokens=131072, hq=28, hkv=4, d=128, rd=128,
             interleaved=False, norm=False),
        # A chunk of an odd length with head norms; half of each head is rotated.
        dict(name="norm_rope_chunk_f16", op="rope", dtype="f16", batch=1, tokens=4097, hq=28, hkv=4, d=128, rd=64,
             interleaved=False, norm=True),
        # A small batch in fp32, interleaved pairs.
        dict(name="norm_rope_small_f32", op="rope", dtype="f32", batch=3, tokens=333, hq=4, hkv=2, d=64, rd=32,
             interleaved=True, norm=True),
        # One decode step of 64 sequences: a token each.
        dict(name="append_decode_64", op="append", dtype="bf16", seqs=64, q_lo=1, q_hi=1, c_lo=100, c_hi=2000, hq=28,
             hkv=4, d=128, page=64, rd=128, interleaved=False, norm=True),
        # Prefill chunks of four prompts.
        dict(name="append_chunks_8k", op="append", dtype="bf16", seqs=4, q_lo=1800, q_hi=2300, c_lo=0, c_hi=6000,
             hq=28, hkv=4, d=128, page=64, rd=128, interleaved=False, norm=False),
        # A mixed step: idle sequences, single tokens and short chunks; small pages, interleaved pairs, partial rotation.
        dict(name="append_mixed_f16", op="append", dtype="f16", seqs=17, q_lo=0, q_hi=65, c_lo=0, c_hi=700, hq=4,
             hkv=2, d=64, page=16, rd=32, interleaved=True, norm=True),
        # Decode of one short sequence: latency.
        dict(name="decode_one_1k", op="attention", dtype="bf16", seqs=1, q_lo=1, q_hi=1, c_lo=1000, c_hi=1000, hq=28,
             hkv=4, d=128, page=64),
        # A serving batch: 64 sequences of unequal lengths up to 8192 tokens.
        dict(name="decode_64_at_8k", op="attention", dtype="bf16", seqs=64, q_lo=1, q_hi=1, c_lo=300, c_hi=8191, hq=28,
             hkv=4, d=128, page=64),
        # One sequence at the full context.
        dict(name="decode_one_128k", op="attention", dtype="bf16", seqs=1, q_lo=1, q_hi=1, c_lo=131071, c_hi=131071,
             hq=28, hkv=4, d=128, page=64),
        # A short turn of a conversation over its cached history.
        dict(name="chunk_512_at_32k", op="attention", dtype="bf16", seqs=1, q_lo=512, q_hi=512, c_lo=32256, c_hi=32256,
             hq=28, hkv=4, d=128, page=64),
        # A prefill chunk deep in a long prompt.
        dict(name="chunk_2048_at_64k", op="attention", dtype="bf16", seqs=1, q_lo=2048, q_hi=2048, c_lo=63488,
             c_hi=63488, hq=28, hkv=4, d=128, page=64),
        # A mixed step of idle, decoding and prefilling sequences with odd lengths and small pages.
        dict(name="mixed_f16_page16", op="attention", dtype="f16", seqs=9, q_lo=0, q_hi=300, c_lo=1, c_hi=3001, hq=4,
             hkv=2, d=64, page=16),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["rope", "append", "attention", "attention"])
    dtype = rng.choice(["bf16", "bf16", "f16", "f32"])
    hq, hkv, d = rng.choice([(28, 4, 128), (4, 2, 64), (16, 16, 64), (32, 8, 128), (14, 2, 64), (8, 1, 128)])
    if op == "rope":
        batch = rng.choice([1, 1, 2, 5])
        tokens = _log(rng, 1, 131072 * 32 * 128 // (batch * (hq + hkv) * d) // (2 if dtype == "f32" else 1))
        return dict(op=op, dtype=dtype, batch=batch, tokens=min(tokens, 131072), hq=hq, hkv=hkv, d=d,
                    rd=rng.choice([d, d // 2, d // 4]), interleaved=rng.random() < 0.4, norm=rng.random() < 0.6)
    seqs = _log(rng, 1, 64)
    page = rng.choice([16, 32, 64, 64, 128])
    if op == "append":
        q_hi = _log(rng, 1, max(1, 8192 // seqs))
        q_lo = rng.randint(0, q_hi) if seqs > 1 else q_hi
        c_hi = _log(rng, 1, 16384 // seqs)
        return dict(op=op, dtype=dtype, seqs=seqs, q_lo=q_lo, q_hi=q_hi, c_lo=rng.randint(0, c_hi), c_hi=c_hi, hq=hq,
                    hkv=hkv, d=d, page=page, rd=rng.choice([d, d // 2, d // 4]), interleaved=rng.random() < 0.4,
                    norm=rng.random() < 0.6)
    # Attention: single tokens, a few tokens (drafts), or chunks; scores and cache within the largest listed cases.
    q_hi = rng.choice([1, 1, _log(rng, 2, 9), _log(rng, 10, 2048)])
    budget = 28 * 2048 * 65536 // (16 if dtype == "f32" else 1)
    c_most = min(131071, budget // (seqs * hq * q_hi), 64 * 8192 * 512 // (seqs * hkv * d))
    if c_most < 64:
        seqs, c_most = 1, min(131071, budget // (hq * q_hi))
    c_hi = _log(rng, 16, c_most)
    return dict(op=op, dtype=dtype, seqs=seqs, q_lo=rng.randint(0, q_hi) if seqs > 1 else q_hi, q_hi=q_hi,
                c_lo=rng.randint(0, c_hi), c_hi=c_hi, hq=hq, hkv=hkv, d=d, page=page)


def _lengths(case):
    """New tokens and cached tokens of each sequence: spread over the case's ranges, the last one at their ends."""
    n = case["seqs"]
    at = [((i + 1) * 0.6180339887498949) % 1.0 for i in range(n - 1)] + [1.0]
    of = [((i + 1) * 0.7548776662466927) % 1.0 for i in range(n - 1)] + [1.0]
    q = [case["q_lo"] + int(a * (case["q_hi"] - case["q_lo"])) for a in at]
    c = [case["c_lo"] + int(a * (case["c_hi"] - case["c_lo"])) for a in of]
    return q, c


def work(case):
    es = 4 if case["dtype"] == "f32" else 2
    hq, hkv, d = case["hq"], case["hkv"], case["d"]
    if case["op"] == "rope":
        rows = case["batch"] * case["tokens"] * (hq + hkv)
        return {"bytes": 2 * rows * d * es + 4 * case["tokens"] * case["rd"], "flops": rows * (3 * case["rd"] + (4 * d if case["norm"] else 0))}
    q, c = _lengths(case)
    if case["op"] == "append":
        rows = sum(q) * (hq + 2 * hkv)
        return {"bytes": 2 * rows * d * es + 4 * sum(q) * case["rd"],
                "flops": sum(q) * (hq + hkv) * (3 * case["rd"] + (4 * d if case["norm"] else 0))}
    seen = sum(a * b + a * (a + 1) // 2 for a, b in zip(q, c))
    read = sum(a + b for a, b in zip(q, c) if a)
    return {"bytes": 2 * sum(q) * hq * d * es + 2 * read * hkv * d * es, "flops": 4 * d * hq * seen}


# ------------------------------------------------------------------ inputs
def _table(positions, rd, device):
    """cos | sin of position * base^(-2i/rd), formed in 64 bits."""
    freq = 1000000.0 ** (-torch.arange(0, rd, 2, device=device, dtype=torch.float64) / rd)
    ang = torch.arange(positions, device=device, dtype=torch.float64)[:, None] * freq
    return torch.cat([ang.cos(), ang.sin()], dim=-1).float()


def prepare(case, seed):
    dev = "cuda"
    g = torch.Generator(device=dev).manual_seed(seed)
    dt = DTYPES[case["dtype"]]
    hq, hkv, d = case["hq"], case["hkv"], case["d"]

    def rand(*shape, scale=1.0):
        return torch.randn(*shape, generator=g, device=dev, dtype=dt) * scale

    st = dict(case=case)
    if case["op"] in ("rope", "append") and case["norm"]:
        st["q_weight"] = 1 + 0.1 * torch.randn(d, generator=g, device=dev)
        st["k_weight"] = 1 + 0.1 * torch.randn(d, generator=g, device=dev)
    if case["op"] == "rope":
        b, t = case["batch"], case["tokens"]
        # [B, H, T, D] views of the fused projection [B, T, (Hq + Hkv) * D]
        qk = rand(b, t, hq + hkv, d)
        st["q"], st["k"] = qk[:, :, :hq].transpose(1, 2), qk[:, :, hq:].transpose(1, 2)
        st["rope"] = _table(t, case["rd"], dev)
        return st
    qlen, clen = _lengths(case)
    page, n = case["page"], sum(qlen)
    kv = [a + b for a, b in zip(qlen, clen)]
    need = [-(-x // page) for x in kv]
    # Pages lie in no order in the pool, as after some time of serving.
    order = torch.randperm(sum(need) + 3, generator=torch.Generator().manual_seed(seed))
    table = torch.full((len(kv), max(1, max(need))), -1, dtype=torch.int32)
    at = 0
    for s, m in enumerate(need):
        table[s, :m] = order[at:at + m].int()
        at += m
    st["table"] = table.to(dev)
    st["cu_q"] = torch.tensor([0] + qlen, device=dev, dtype=torch.int32).cumsum(0, dtype=torch.int32)
    st["kv_lens"] = torch.tensor(kv, device=dev, dtype=torch.int32)
    st["max_q"], st["max_kv"] = max(qlen), max(kv)
    st["k_cache"], st["v_cache"] = rand(sum(need) + 3, hkv, page, d), rand(sum(need) + 3, hkv, page, d)
    if case["op"] == "append":
        qkv = rand(n, hq + 2 * hkv, d)
        st["q"], st["k"], st["v"] = qkv[:, :hq], qkv[:, hq:hq + hkv], qkv[:, hq + hkv:]
        st["rope"] = _table(max(kv) + 1, case["rd"], dev)
    else:
        # Twice the unit scale: about one key in fifty carries a query's weight.
        st["q"] = rand(n, hq, d, scale=2.0)
    return st


# ------------------------------------------------------------------ plain forms
def _turned(x, weight, cos, sin, rd, interleaved):
    """Head norm (where a weight is given) and rotation in fp32; cos / sin broadcast over x[..., :rd // 2]."""
    x = x.float()
    if weight is not None:
        x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + EPS) * weight
    if interleaved:
        a, b = x[..., 0:rd:2], x[..., 1:rd:2]
        turned = torch.stack([a * cos - b * sin, b * cos + a * sin], dim=-1).flatten(-2)
    else:
        a, b = x[..., :rd // 2], x[..., rd // 2:rd]
        turned = torch.cat([a * cos - b * sin, b * cos + a * sin], dim=-1)
    return torch.cat([turned, x[..., rd:]], dim=-1)


def _plain_rope(st):
    c = st["case"]
    rd = c["rd"]
    cos, sin = st["rope"][:, :rd // 2], st["rope"][:, rd // 2:]
    q, k = (_turned(st[x].transpose(1, 2), st.get(x + "_weight"), cos[:, None], sin[:, None], rd,
                    c["interleaved"]).to(st[x].dtype).transpose(1, 2) for x in ("q", "k"))
    return {"q": q, "k": k}


def _where(st, n):
    """Sequence and position in it of each packed token."""
    token = torch.arange(n, device=st["cu_q"].device)
    seq = torch.searchsorted(st["cu_q"].long(), token, right=True) - 1
    first = st["kv_lens"].long() - (st["cu_q"][1:] - st["cu_q"][:-1]).long()
    return seq, first[seq] + token - st["cu_q"].long()[seq]


def _plain_append(st):
    c, rd = st["case"], st["case"]["rd"]
    seq, pos = _where(st, st["k"].shape[0])
    row = st["rope"][pos][:, None]
    q, k = (_turned(st[x], st.get(x + "_weight"), row[..., :rd // 2], row[..., rd // 2:], rd,
                    c["interleaved"]).to(st[x].dtype) for x in ("q", "k"))
    page = st["table"].long()[seq, pos // c["page"]]
    st["k_cache"][page, :, pos % c["page"]] = k
    st["v_cache"][page, :, pos % c["page"]] = st["v"]
    return {"q": q, "k_cache": st["k_cache"], "v_cache": st["v_cache"]}


def _plain_attention(st):
    c = st["case"]
    q, n = st["q"], st["q"].shape[0]
    hq, hkv, d, rep = c["hq"], c["hkv"], c["d"], c["hq"] // c["hkv"]
    seqs, most_q, most_kv = c["seqs"], st["max_q"], st["max_kv"]
    kv, cu = st["kv_lens"].long(), st["cu_q"].long()
    pages = st["table"].long().clamp(min=0)
    k, v = (x[pages].transpose(1, 2).reshape(seqs, hkv, -1, d)[:, :, :most_kv].float()
            for x in (st["k_cache"], st["v_cache"]))
    i, j = torch.arange(most_q, device=q.device), torch.arange(most_kv, device=q.device)
    qlen = cu[1:] - cu[:-1]
    rows = q[(cu[:-1, None] + i).clamp(max=max(n - 1, 0))].float()                       # [S, Q, Hq, D]
    rows = rows.reshape(seqs, most_q, hkv, rep, d).permute(0, 2, 3, 1, 4).reshape(seqs, hkv, rep * most_q, d)
    seen = (j <= (kv - qlen)[:, None, None] + i[:, None]) & (i < qlen[:, None])[..., None]  # [S, Q, K]
    s = (rows * d ** -0.5) @ k.transpose(-1, -2)
    s = s.view(seqs, hkv, rep, most_q, most_kv)
    s.masked_fill_(~seen[:, None, None], -math.inf)
    top = s.amax(-1, keepdim=True)
    s.sub_(torch.where(top == -math.inf, 0.0, top)).exp_()
    total = s.sum(-1, keepdim=True)
    v = torch.where((j < kv[:, None])[:, None, :, None], v, 0.0)
    o = (s.view(seqs, hkv, rep * most_q, most_kv) @ v).view(seqs, hkv, rep, most_q, d)
    o = torch.where(total > 0, o / total, 0.0).permute(0, 3, 1, 2, 4).reshape(seqs, most_q, hq, d)
    seq, pos = _where(st, n)
    return o[seq, pos - (kv - qlen)[seq]].to(q.dtype)


def run(st):
    op = st["case"]["op"]
    if not own:
        return {"rope": _plain_rope, "append": _plain_append, "attention": _plain_attention}[op](st)
    from spruce_research_b200 import native

    if op == "rope":
        q, k = native.qk_norm_rope(st["q"], st["k"], st["rope"], q_weight=st.get("q_weight"),
                                   k_weight=st.get("k_weight"), eps=EPS, interleaved=st["case"]["interleaved"])
        return {"q": q, "k": k}
    if op == "append":
        q = native.paged_append(st["k"], st["v"], st["k_cache"], st["v_cache"], st["table"], st["cu_q"],
                                st["kv_lens"], q=st["q"], rope=st["rope"],
                                q_weight=st.get("q_weight"), k_weight=st.get("k_weight"), eps=EPS,
                                interleaved=st["case"]["interleaved"])
        return {"q": q, "k_cache": st["k_cache"], "v_cache": st["v_cache"]}
    return native.paged_attention(st["q"], st["k_cache"], st["v_cache"], st["table"], st["cu_q"], st["kv_lens"],
                                  max_q_len=st["max_q"], max_kv_len=st["max_kv"])


# ------------------------------------------------------------------ the definition in 64 bits
def _exact_turn(x, weight, angles, rd, interleaved):
    """x [..., D] doubles; each pair as a complex number times cos + i sin."""
    if weight is not None:
        x = x / (x.square().sum(-1, keepdim=True) / x.shape[-1] + EPS).sqrt() * weight.double()
    half = rd // 2
    unit = torch.complex(angles[..., :half].double(), angles[..., half:].double())
    first = slice(0, rd, 2) if interleaved else slice(0, half)
    second = slice(1, rd, 2) if interleaved else slice(half, rd)
    z = torch.complex(x[..., first], x[..., second]) * unit
    y = x.clone()
    y[..., first], y[..., second] = z.real, z.imag
    return y


def exact(case, seed):
    st = prepare(case, seed)
    if case["op"] == "rope":
        out = {}
        for x in ("q", "k"):
            y = torch.empty(st[x].shape, device="cuda", dtype=torch.float64)
            for h in range(st[x].shape[1]):
                y[:, h] = _exact_turn(st[x][:, h].double(), st.get(x + "_weight"), st["rope"], case["rd"],
                                      case["interleaved"])
            out[x] = y
        return out
    qlen, clen = _lengths(case)
    table, page = st["table"].tolist(), case["page"]
    if case["op"] == "append":
        q = torch.empty(st["q"].shape, device="cuda", dtype=torch.float64)
        kc, vc = st["k_cache"].double(), st["v_cache"].double()
        at = 0
        for s, (a, b) in enumerate(zip(qlen, clen)):
            if not a:
                continue
            angles = st["rope"][b:b + a, None]
            q[at:at + a] = _exact_turn(st["q"][at:at + a].double(), st.get("q_weight"), angles, case["rd"],
                                       case["interleaved"])
            k = _exact_turn(st["k"][at:at + a].double(), st.get("k_weight"), angles, case["rd"], case["interleaved"])
            v = st["v"][at:at + a].double()
            done = 0
            while done < a:
                p, r = divmod(b + done, page)
                m = min(page - r, a - done)
                kc[table[s][p], :, r:r + m] = k[done:done + m].transpose(0, 1)
                vc[table[s][p], :, r:r + m] = v[done:done + m].transpose(0, 1)
                done += m
            at += a
        return {"q": q, "k_cache": kc, "v_cache": vc}
    rep, d = case["hq"] // case["hkv"], case["d"]
    out = torch.zeros(st["q"].shape, device="cuda", dtype=torch.float64)
    at = 0
    for s, (a, b) in enumerate(zip(qlen, clen)):
        if a and a + b:
            pages = torch.tensor(table[s][:-(-(a + b) // page)], device="cuda")
            for g in range(case["hkv"]):
                k = st["k_cache"][pages, g].double().flatten(0, 1)[:a + b]
                v = st["v_cache"][pages, g].double().flatten(0, 1)[:a + b]
                for t in range(0, a, 512):
                    e = min(a, t + 512)
                    x = st["q"][at + t:at + e, g * rep:(g + 1) * rep].double()
                    z = torch.einsum("thd,kd->htk", x, k) / math.sqrt(d)
                    late = torch.arange(a + b, device="cuda") > torch.arange(b + t, b + e, device="cuda")[:, None]
                    p = torch.softmax(z.masked_fill(late, -math.inf), dim=-1)
                    out[at + t:at + e, g * rep:(g + 1) * rep] = torch.einsum("htk,kd->thd", p, v)
        at += a
    return out
