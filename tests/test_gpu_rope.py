"""Head norms and rotary positions, dense and into a paged cache, against 64-bit arithmetic.

Bounds, per element, with u the unit roundoff of the dtype (fp32 itself for float32) and e = 2^-24: the store rounds
by u |y|; the rotation's two products and sum add 3 e (|a cos| + |b sin|); with a norm the D-term sum of squares is off
by at most (D + 2) e relative, halved by the root, and the root, the division and two products add 5 e.  fp16 stores
below 2^-14 round by 2^-25 absolute.
"""
import pytest
import torch

from spruce_research_b200 import _lib, native
from spruce_research_b200.rope import rope_table

pytestmark = pytest.mark.gpu

U = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}
E = 2.0 ** -24


def turned(x, weight, rows, rd, interleaved, eps):
    """64-bit result and the bound on a kernel's error; x [..., D], rows [..., rd]."""
    u, D = U[x.dtype], x.shape[-1]
    x = x.double()
    rel = 0.0
    if weight is not None:
        x = x / (x.square().mean(-1, keepdim=True) + eps).sqrt() * weight.double()
        rel = (D / 2 + 6) * E
    y, mag = x.clone(), x.abs()
    if rd:
        a = slice(0, rd, 2) if interleaved else slice(0, rd // 2)
        b = slice(1, rd, 2) if interleaved else slice(rd // 2, rd)
        cos, sin = rows[..., :rd // 2].double(), rows[..., rd // 2:].double()
        xa, xb = x[..., a], x[..., b]
        y[..., a], y[..., b] = xa * cos - xb * sin, xb * cos + xa * sin
        mag[..., a] = (xa * cos).abs() + (xb * sin).abs()
        mag[..., b] = (xb * cos).abs() + (xa * sin).abs()
    return y, u * y.abs() + (rel + 3 * E) * (1 + u) * mag + 2.0 ** -25 * (u == 2.0 ** -11)


def check(got, want):
    y, bound = want
    assert got.shape == y.shape
    over = ((got.double() - y).abs() - bound).max().item() if y.numel() else 0.0
    assert over <= 0, f"error passes its bound by {over:.3e}"


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D,rd,interleaved,norm", [
    (128, 128, False, False), (128, 128, True, True), (128, 64, False, True), (64, 32, True, False), (64, 64, False, True),
    (96, 96, False, True), (80, 20, False, True), (80, 20, True, True), (256, 256, False, True), (6, 2, False, True),
    (2, 2, True, False), (100, 50, False, False), (16, 16, False, True), (128, 0, False, True)])
def test_norm_rope_matches_64_bits(dtype, D, rd, interleaved, norm):
    g = torch.Generator(device="cuda").manual_seed(D * 1000 + rd)
    B, Hq, Hkv, T = 2, 7, 3, 37
    # views of one fused projection; the head dim's stride is 1, the rest are not contiguous
    qk = torch.randn(B, T, Hq + Hkv, D, generator=g, device="cuda", dtype=dtype)
    q, k = qk[:, :, :Hq].transpose(1, 2), qk[:, :, Hq:].transpose(1, 2)
    table = torch.randn(50, rd, generator=g, device="cuda")       # any table: the kernel is linear in it
    pos = torch.randint(0, 50, (B, T), generator=g, device="cuda")
    wq = torch.randn(D, generator=g, device="cuda") if norm else None
    wk = torch.randn(D, generator=g, device="cuda") if norm else None
    status = torch.zeros(1, device="cuda", dtype=torch.int32)
    qo, ko = native.qk_norm_rope(q, k, table, pos, q_weight=wq, k_weight=wk, eps=1e-5, interleaved=interleaved,
                                 status=status)
    rows = table[pos][:, None]
    check(qo, turned(q, wq, rows, rd, interleaved, 1e-5))
    check(ko, turned(k, wk, rows, rd, interleaved, 1e-5))
    assert status.item() == 0 and qo.transpose(1, 2).is_contiguous()


@pytest.mark.parametrize("shift", [0, 1])
def test_in_place_unaligned_rows_and_a_weight_for_one_side(shift):
    """An odd base address takes scalar loads; outputs may be the inputs; only the keys have a norm here."""
    g = torch.Generator(device="cuda").manual_seed(3)
    B, Hq, Hkv, T, D = 1, 4, 2, 9, 64
    flat = torch.randn(T * (Hq + Hkv) * D + 8, generator=g, device="cuda", dtype=torch.bfloat16)
    qk = flat[shift:shift + T * (Hq + Hkv) * D].view(B, T, Hq + Hkv, D)
    q, k = qk[:, :, :Hq].transpose(1, 2), qk[:, :, Hq:].transpose(1, 2)
    table = rope_table(D, T, 1e6)
    wk = torch.rand(D, generator=g, device="cuda", dtype=torch.bfloat16)
    want_q, want_k = turned(q, None, table, D, False, 1e-6), turned(k, wk, table, D, False, 1e-6)
    guard = flat.clone()
    qo, ko = native.qk_norm_rope(q, k, table, k_weight=wk, q_out=q, k_out=k)
    assert qo is q and ko is k
    check(q, want_q)
    check(k, want_k)
    assert torch.equal(flat[:shift], guard[:shift])
    assert torch.equal(flat[shift + qk.numel():], guard[shift + qk.numel():])


def test_single_token_empty_and_positions_out_of_the_table():
    table = rope_table(64, 8)
    status = torch.zeros(1, device="cuda", dtype=torch.int32)
    q, k = torch.randn(1, 2, 1, 64, device="cuda"), torch.randn(1, 1, 1, 64, device="cuda")
    qo, _ = native.qk_norm_rope(q, k, table, torch.tensor([7], device="cuda"), status=status)
    check(qo, turned(q, None, table[7], 64, False, 0.0))
    assert status.item() == 0
    for bad, row in ((8, 7), (-1, 0)):        # the nearest row, and the status says so
        status.zero_()
        qo, _ = native.qk_norm_rope(q, k, table, torch.tensor([bad], device="cuda"), status=status)
        check(qo, turned(q, None, table[row], 64, False, 0.0))
        assert status.item() == _lib.STATUS_BAD_POSITION
    qo, ko = native.qk_norm_rope(q[:, :, :0], k[:, :, :0], table)
    assert qo.shape == (1, 2, 0, 64) and ko.shape == (1, 1, 0, 64)


def test_norm_of_zeros_infinities_and_nan_stay_in_their_rows():
    table = rope_table(64, 4)
    q = torch.randn(1, 2, 4, 64, device="cuda")
    q[0, 0, 0] = 0
    q[0, 0, 1, 5] = float("nan")
    q[0, 1, 2, 9] = float("inf")
    w = torch.ones(64, device="cuda")
    qo, ko = native.qk_norm_rope(q, torch.zeros_like(q[:, :1]), table, q_weight=w, k_weight=w)
    assert torch.all(ko == 0) and torch.all(qo[0, 0, 0] == 0)
    assert qo[0, 0, 1].isnan().all()
    clean = torch.ones(2, 4, dtype=torch.bool)
    clean[0, 1] = clean[1, 2] = False
    assert qo[0][clean.cuda()].isfinite().all()


def _batch(qlens, clens, page, seed):
    kv = [a + b for a, b in zip(qlens, clens)]
    need = [-(-x // page) for x in kv]
    order = torch.randperm(sum(need) + 2, generator=torch.Generator().manual_seed(seed)).int()
    table = torch.full((len(kv), max(1, max(need))), -1, dtype=torch.int32)
    at = 0
    for s, m in enumerate(need):
        table[s, :m] = order[at:at + m]
        at += m
    cu = torch.tensor([0] + qlens).cumsum(0).int()
    return table.cuda(), cu.cuda(), torch.tensor(kv, dtype=torch.int32).cuda(), sum(need) + 2


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("qlens,clens,page,D,rd,interleaved,norm,hnd", [
    ([1] * 5, [0, 15, 16, 63, 200], 16, 64, 64, False, True, True),        # decode: a page's last and first rows
    ([0, 3, 0, 70, 1, 0], [9, 0, 0, 30, 127, 0], 32, 128, 64, True, False, False),  # idle sequences, ragged chunks
    ([40], [0], 48, 80, 40, False, True, True),                            # pages of 48, head_dim 80
    ([5, 2], [1, 1], 16, 6, 2, False, True, False),                        # rows no vector fits
    ([17, 0], [3, 4], 64, 64, 0, False, False, True)])                     # no rotation: a copy
def test_append_matches_64_bits_and_touches_nothing_else(dtype, qlens, clens, page, D, rd, interleaved, norm, hnd):
    g = torch.Generator(device="cuda").manual_seed(7)
    Hq, Hkv, N = 6, 2, sum(qlens)
    table, cu, kv, pages = _batch(qlens, clens, page, 5)
    shape = (pages, Hkv, page, D) if hnd else (pages, page, Hkv, D)
    caches = [torch.randn(*shape, generator=g, device="cuda", dtype=dtype) for _ in range(2)]
    kc, vc = caches if hnd else [c.transpose(1, 2) for c in caches]
    before_k, before_v = kc.clone(), vc.clone()
    qkv = torch.randn(N, Hq + 2 * Hkv, D, generator=g, device="cuda", dtype=dtype)
    q, k, v = qkv[:, :Hq], qkv[:, Hq:Hq + Hkv], qkv[:, Hq + Hkv:]
    rope = torch.randn(512, rd, generator=g, device="cuda") if rd else None
    wq, wk = (torch.randn(D, generator=g, device="cuda") if norm else None for _ in range(2))
    status = torch.zeros(1, device="cuda", dtype=torch.int32)
    qo = native.paged_append(k, v, kc, vc, table, cu, kv, q=q, rope=rope, q_weight=wq, k_weight=wk, eps=1e-5,
                             interleaved=interleaved, status=status)
    assert status.item() == 0
    written = torch.zeros(pages, page, dtype=torch.bool, device="cuda")
    n = 0
    for s, (a, b) in enumerate(zip(qlens, clens)):
        for i in range(a):
            row = rope[b + i] if rd else None
            check(qo[n], turned(q[n], wq, row, rd, interleaved, 1e-5))
            p, r = int(table[s, (b + i) // page]), (b + i) % page
            check(kc[p, :, r], turned(k[n], wk, row, rd, interleaved, 1e-5))
            assert torch.equal(vc[p, :, r], v[n])
            written[p, r] = True
            n += 1
    keep = ~written[:, None, :, None].expand_as(kc)
    assert torch.equal(kc[keep], before_k[keep]) and torch.equal(vc[keep], before_v[keep])
    # without q and with positions of its own, the same cache
    kc2, vc2 = before_k, before_v
    pos = torch.tensor([b + i for a, b in zip(qlens, clens) for i in range(a)], device="cuda", dtype=torch.int32)
    assert native.paged_append(k, v, kc2, vc2, table, cu, kv, rope=rope, positions=pos if rd else None, k_weight=wk,
                               eps=1e-5, interleaved=interleaved) is None
    assert torch.equal(kc2, kc) and torch.equal(vc2, vc)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("D,rd,interleaved,sides", [
    (128, 64, False, "qk"), (64, 64, True, "q"), (80, 48, True, "k"), (96, 64, False, "")])
@pytest.mark.parametrize("Hq,Hkv", [(7, 3), (4, 5)])
def test_many_tokens_whose_heads_leave_part_of_a_group(dtype, D, rd, interleaved, sides, Hq, Hkv):
    """Enough tokens that a lane group takes four heads; the last group of each tensor is short; norms on either side."""
    g = torch.Generator(device="cuda").manual_seed(11)
    B, T = 2, 2003
    qkv = torch.randn(B, T, Hq + 2 * Hkv, D, generator=g, device="cuda", dtype=dtype)
    q, k, v = (x.transpose(1, 2) for x in qkv.split([Hq, Hkv, Hkv], 2))
    table = torch.randn(B * T, rd, generator=g, device="cuda")
    wq, wk = (torch.randn(D, generator=g, device="cuda") if side in sides else None for side in "qk")
    qo, ko = native.qk_norm_rope(q, k, table, q_weight=wq, k_weight=wk, eps=1e-5, interleaved=interleaved)
    check(qo, turned(q, wq, table[:T], rd, interleaved, 1e-5))
    check(ko, turned(k, wk, table[:T], rd, interleaved, 1e-5))
    # the same rows as one sequence of B * T tokens into pages
    flat = qkv.flatten(0, 1)
    q, k, v = flat.split([Hq, Hkv, Hkv], 1)
    pages, cu, kv, count = _batch([B * T], [0], 32, 5)
    kc, vc = (torch.zeros(count, Hkv, 32, D, device="cuda", dtype=dtype) for _ in range(2))
    qo = native.paged_append(k, v, kc, vc, pages, cu, kv, q=q, rope=table, q_weight=wq, k_weight=wk, eps=1e-5,
                             interleaved=interleaved)
    at = torch.arange(B * T, device="cuda")
    rows = pages[0, at // 32].long()
    check(qo, turned(q, wq, table[:, None], rd, interleaved, 1e-5))
    check(kc[rows, :, at % 32], turned(k, wk, table[:, None], rd, interleaved, 1e-5))
    assert torch.equal(vc[rows, :, at % 32], v)


def test_append_skips_bad_pages_and_lengths():
    D, page = 64, 16
    k = torch.randn(3, 1, D, device="cuda")
    cu, kv = (torch.tensor(x, device="cuda", dtype=torch.int32) for x in ([0, 1, 2, 3], [17, 5, 40]))
    table = torch.tensor([[0, 9], [1, -1], [0, 1]], device="cuda", dtype=torch.int32)
    kc, vc = torch.zeros(3, 1, page, D, device="cuda"), torch.zeros(3, 1, page, D, device="cuda")
    status = torch.zeros(1, device="cuda", dtype=torch.int32)
    native.paged_append(k, k, kc, vc, table, cu, kv, status=status)  # page 9 of 3; fine; position 39 of 32
    assert status.item() == _lib.STATUS_BAD_PAGE | _lib.STATUS_BAD_LENGTH
    assert torch.equal(kc[1, 0, 4], k[1, 0]) and (kc != 0).sum() == (k[1] != 0).sum()
    # more new tokens than the sequence holds: the ones before position 0 are left out
    status.zero_()
    kc.zero_()
    native.paged_append(k, k, kc, vc, table[1:2], torch.tensor([0, 3], device="cuda", dtype=torch.int32),
                        torch.tensor([2], device="cuda", dtype=torch.int32), status=status)
    assert status.item() == _lib.STATUS_BAD_LENGTH
    assert torch.equal(kc[1, 0, :2], k[1:, 0]) and (kc != 0).sum() == (k[1:] != 0).sum()
    # tokens past cu_q[-1] are left out
    kc.zero_()
    native.paged_append(k, k, kc, vc, table[1:2], torch.tensor([0, 1], device="cuda", dtype=torch.int32),
                        torch.tensor([1], device="cuda", dtype=torch.int32))
    assert torch.equal(kc[1, 0, 0], k[0, 0]) and (kc != 0).sum() == (k[0] != 0).sum()


def test_refusals():
    q = torch.zeros(1, 4, 8, 64, device="cuda", dtype=torch.bfloat16)
    k, table = q[:, :2], rope_table(64, 8)
    with pytest.raises(ValueError, match="share a dtype"):
        native.qk_norm_rope(q, k.float(), table)
    with pytest.raises(ValueError, match="rotary width"):
        native.qk_norm_rope(q, k, rope_table(128, 8))
    with pytest.raises(ValueError, match="as many positions"):
        native.qk_norm_rope(q, k, table[:7])
    with pytest.raises(ValueError, match="contiguous float32"):
        native.qk_norm_rope(q, k, table.half())
    with pytest.raises(ValueError, match="positions must be"):
        native.qk_norm_rope(q, k, table, torch.zeros(7, device="cuda", dtype=torch.int64))
    with pytest.raises(ValueError, match="integers"):
        native.qk_norm_rope(q, k, table, torch.zeros(8, device="cuda"))
    with pytest.raises(ValueError, match="q_weight"):
        native.qk_norm_rope(q, k, table, q_weight=torch.ones(32, device="cuda"))
    with pytest.raises(ValueError, match="an output must be"):
        native.qk_norm_rope(q, k, table, q_out=torch.empty_like(k))
    with pytest.raises(ValueError, match="dtype"):
        native.qk_norm_rope(q.double(), k.double(), table)
    with pytest.raises(RuntimeError, match="CUDA"):
        native.qk_norm_rope(q, k, table.cpu())
    x = torch.zeros(3, 2, 64, device="cuda", dtype=torch.bfloat16)
    cache = torch.zeros(4, 2, 16, 64, device="cuda", dtype=torch.bfloat16)
    bt, cu, kv = (torch.zeros(s, device="cuda", dtype=torch.int32) for s in ((1, 2), (2,), (1,)))
    with pytest.raises(ValueError, match="page_size"):
        native.paged_append(x, x, cache[:, :, :8], cache[:, :, :8], bt, cu, kv)
    with pytest.raises(ValueError, match="int32"):
        native.paged_append(x, x, cache, cache, bt.long(), cu, kv)
    with pytest.raises(ValueError, match="block_table"):
        native.paged_append(x, x, cache, cache, bt, cu[:1], kv)
    with pytest.raises(ValueError, match="new tokens' dtype"):
        native.paged_append(x, x, cache.half(), cache.half(), bt, cu, kv)
    with pytest.raises(ValueError, match="k and v must be"):
        native.paged_append(x[:, :1], x[:, :1], cache, cache, bt, cu, kv)
    with pytest.raises(ValueError, match="q must be"):
        native.paged_append(x, x, cache, cache, bt, cu, kv, q=x[:2])
    with pytest.raises(ValueError, match="q_out without q"):
        native.paged_append(x, x, cache, cache, bt, cu, kv, q_out=x)


@pytest.mark.parametrize("status", [torch.int64, torch.float32, None])
def test_a_status_of_another_type_or_without_an_element_is_refused(status):
    status = torch.zeros(int(status is not None), device="cuda", dtype=status or torch.int32)
    x = torch.zeros(3, 2, 64, device="cuda", dtype=torch.bfloat16)
    cache = torch.zeros(4, 2, 16, 64, device="cuda", dtype=torch.bfloat16)
    bt, cu, kv = (torch.zeros(s, device="cuda", dtype=torch.int32) for s in ((1, 2), (2,), (1,)))
    with pytest.raises(ValueError, match="status"):
        native.qk_norm_rope(x[None], x[None], rope_table(64, 8), status=status)
    with pytest.raises(ValueError, match="status"):
        native.paged_append(x, x, cache, cache, bt, cu, kv, status=status)
    with pytest.raises(ValueError, match="status"):
        native.paged_attention(x, cache, cache, bt, cu, kv, max_q_len=3, max_kv_len=3, status=status)
