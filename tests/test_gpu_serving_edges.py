"""The serving operators at the edges of their contract: tokens of no sequence, bounds below the lengths, scores that are
not finite, weights near the end of fp16's range, tensors at odd addresses."""
import pytest
import torch

from spruce_research_b200 import _lib, native
from spruce_research_b200.paged import PagedKVCache, PagedSparseLayer
from spruce_research_b200.pipeline import SparsePrefillLayer
from spruce_research_b200.synthetic import make_gate_weights

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("shift", [0, 1])          # an odd base address takes the scalar kernel
@pytest.mark.parametrize("with_q", [True, False])
def test_append_leaves_out_tokens_before_the_first_sequence(shift, with_q):
    """Two sequences of a larger batch, with all its packed tokens: cu_q starts at 3, tokens 0 to 2 and 7 to 8 belong to
    none.  Their q rows are not written, nor is any cache row but the four new ones."""
    g = torch.Generator(device="cuda").manual_seed(1)
    N, Hq, Hkv, D, page = 9, 4, 2, 64, 16
    flat = torch.randn(N * (Hq + 2 * Hkv) * D + 8, generator=g, device="cuda", dtype=torch.bfloat16)
    q, k, v = flat[shift:shift + N * (Hq + 2 * Hkv) * D].view(N, Hq + 2 * Hkv, D).split([Hq, Hkv, Hkv], 1)
    cu = torch.tensor([0, 3, 5, 7, 9], device="cuda", dtype=torch.int32)[1:4]
    kv = torch.tensor([10, 18], device="cuda", dtype=torch.int32)
    table = torch.tensor([[2, 3], [0, 1]], device="cuda", dtype=torch.int32)
    kc, vc = (torch.randn(4, Hkv, page, D, generator=g, device="cuda", dtype=torch.bfloat16) for _ in range(2))
    want_k, want_v = kc.clone(), vc.clone()
    for n, p, r in ((3, 2, 8), (4, 2, 9), (5, 1, 0), (6, 1, 1)):
        want_k[p, :, r], want_v[p, :, r] = k[n], v[n]
    status = torch.zeros(1, device="cuda", dtype=torch.int32)
    out = torch.full((N, Hq, D), 7.0, device="cuda", dtype=torch.bfloat16)
    native.paged_append(k, v, kc, vc, table, cu, kv, status=status, **(dict(q=q, q_out=out) if with_q else {}))
    assert status.item() == 0
    assert torch.equal(kc, want_k) and torch.equal(vc, want_v)
    if with_q:
        assert torch.equal(out[3:7], q[3:7]) and (out[:3] == 7).all() and (out[7:] == 7).all()


def _attend(q, k, v, page=16, **kw):
    """One sequence: q [Nq, Hq, D] are the last tokens of k, v [N, Hkv, D]."""
    N, Hkv, D = k.shape
    pages = -(-N // page)
    kc, vc = (torch.zeros(pages * page, Hkv, D, device="cuda", dtype=q.dtype) for _ in range(2))
    kc[:N], vc[:N] = k, v
    kc, vc = (x.view(pages, page, Hkv, D).transpose(1, 2).contiguous() for x in (kc, vc))
    table = torch.arange(pages, device="cuda", dtype=torch.int32)[None]
    cu, kv = (torch.tensor(x, device="cuda", dtype=torch.int32) for x in ([0, q.shape[0]], [N]))
    return native.paged_attention(q, kc, vc, table, cu, kv, **dict(max_q_len=q.shape[0], max_kv_len=N) | kw)


DTYPES = [torch.float32, torch.bfloat16, torch.float16]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("q", [1, 300])                    # single tokens and chunks are two kernels
@pytest.mark.parametrize("key", [28, 29, 30, 31, 190, 351, 383, 639])
@pytest.mark.parametrize("bad", ["nan", "inf"])
@pytest.mark.parametrize("heads", [2, 300])                # units split over CTAs and joined, or whole
def test_a_score_that_is_not_a_number_reaches_every_query_that_sees_it(dtype, q, key, bad, heads):
    """A NaN in a key, or a key that is so large that its scores are +inf, makes the rows that see it NaN, wherever in a
    tile it stands; rows before it are as they are without it."""
    g = torch.Generator(device="cuda").manual_seed(2)
    n = 700
    x, k, v = (torch.randn(m, heads, 128, generator=g, device="cuda").to(dtype) for m in (q, n, n))
    x[:, :, 3] = 1.0
    clean = _attend(x, k, v)
    k[key, :, 3] = float(bad)
    got = _attend(x, k, v)
    sees = torch.arange(n - q, n, device="cuda") >= key
    assert got[sees].isnan().all()
    assert torch.equal(got[~sees], clean[~sees]) and clean.isfinite().all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])     # fp16's largest products do not overflow fp32
@pytest.mark.parametrize("q", [1, 300])
@pytest.mark.parametrize("heads", [2, 300])
def test_rows_whose_scores_are_all_minus_infinity_are_zero(dtype, q, heads):
    """Scores that overflow to -inf weigh nothing, as masked ones: a row of nothing else is zero, and the rows of head 1,
    whose scores are ordinary, are as they are beside ordinary ones."""
    g = torch.Generator(device="cuda").manual_seed(3)
    n = 700
    x, k, v = (torch.randn(m, heads, 128, generator=g, device="cuda").to(dtype) for m in (q, n, n))
    low = torch.arange(heads, device="cuda") != 1
    ordinary = k[:, 1].clone(), x[:, 1].clone()
    k = k.abs() * 1e20 + 1e20
    x[:] = -1e20
    k[:, 1], x[:, 1] = ordinary
    got = _attend(x, k, v)
    assert (got[:, low] == 0).all()
    k[:, low] = 0
    assert torch.equal(got[:, 1], _attend(x, k, v)[:, 1]) and (got[:, 1] != 0).any()
    # -inf for the first half of the keys only: the second half decides
    k[:n // 2, low] = 1e20
    half = _attend(x, k, v)[:, low].double()
    total = v.double().cumsum(0)[:, low]
    mean = (total[n - q:] - total[n // 2 - 1]) / torch.arange(n - q - n // 2 + 1, n - n // 2 + 1, device="cuda")[:, None, None]
    # flat weights: the probabilities are 1 exactly, so the store rounds by u |o| and the sums by n 2^-24 of max |v|
    u = 2.0 ** -24 if dtype == torch.float32 else 2.0 ** -8
    assert ((half - mean).abs() <= u * mean.abs() + 2 * n * 2.0 ** -24 * v.abs().max()).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("heads", [4, 28])
def test_no_room_for_new_tokens_sets_the_status(dtype, heads):
    """max_q_len 0 while a sequence has new tokens: every one is cut off, which the status reports."""
    x = torch.randn(3, heads, 64, device="cuda").to(dtype)
    k = torch.randn(90, 4, 64, device="cuda").to(dtype)
    status = torch.zeros(1, device="cuda", dtype=torch.int32)
    out = torch.full_like(x, 5.0)
    _attend(x, k, k, max_q_len=0, out=out, status=status)
    assert status.item() == _lib.STATUS_BAD_LENGTH and (out == 5).all()
    _attend(x, k, k, max_q_len=0, out=out)
    assert (out == 5).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("q,cut", [(3, 1), (200, 1), (200, 100)])
def test_a_sequence_cut_to_the_bounds_keeps_its_positions(dtype, q, cut):
    """With max_q_len below its new tokens the first ones are computed and see what they saw; with max_kv_len below its
    length the keys past it are left out."""
    g = torch.Generator(device="cuda").manual_seed(4)
    n = 500
    x, k, v = (torch.randn(m, 4, 64, generator=g, device="cuda").to(dtype) for m in (q, n, n))
    want = _attend(x[:cut], k[:n - q + cut], v[:n - q + cut])
    status = torch.zeros(1, device="cuda", dtype=torch.int32)
    out = torch.full_like(x, 5.0)
    _attend(x, k, v, max_q_len=cut, out=out, status=status)
    assert status.item() == _lib.STATUS_BAD_LENGTH and (out[cut:] == 5).all()
    # the same sums in another split: see the bounds of the attention's tests, here at scores of order 1
    u = {torch.float32: 2.0 ** -18, torch.bfloat16: 2.0 ** -6, torch.float16: 2.0 ** -9}[dtype]
    assert (out[:cut].double() - want.double()).abs().max().item() <= u * v.abs().max().item()
    status.zero_()
    got = _attend(x, k, v, max_kv_len=n - q // 2, status=status)
    assert status.item() == _lib.STATUS_BAD_LENGTH
    seen = q - q // 2                                        # tokens whose keys all lie within the bound
    want = _attend(x[:seen], k[:n - q // 2], v[:n - q // 2])
    assert (got[:seen].double() - want.double()).abs().max().item() <= u * v.abs().max().item()


@pytest.mark.parametrize("q,n", [(1, 2000), (300, 20000)])
@pytest.mark.parametrize("gap", [17.0, 24.0, 25.5])
def test_fp16_keeps_many_small_weights(q, n, gap):
    """One key outweighs each other by 2^gap but holds zeros: what is left is the sum of the small weights, which has to
    be right relative to itself as long as each is above 2^-26 of the largest."""
    D = 128
    x = torch.zeros(q, 1, D, device="cuda", dtype=torch.float16)
    x[:, :, 0] = 1.0
    k = torch.zeros(n, 1, D, device="cuda", dtype=torch.float16)
    k[0] = gap * 0.6931471805599453 / D ** -0.5              # score gap ln 2
    v = torch.ones(n, 1, D, device="cuda", dtype=torch.float16)
    v[0] = 0
    score = k[0, 0, 0].double() * D ** -0.5
    got = _attend(x, k, v)[:, 0].double()
    small = torch.arange(n - q, n, device="cuda").double()[:, None]      # keys besides the first that the row sees
    want = small * torch.exp(-score) / (1 + small * torch.exp(-score))
    # each weight: rounded to fp16 (2^-11) and its exponential (1e-4 and the exponent's 2^-24 |x|); the store 2^-11, or
    # half of fp16's smallest step; sums n 2^-24
    rel = 2 * 2.0 ** -11 + 1e-4 + n * 2.0 ** -24 + 40 * 2.0 ** -23
    assert ((got - want).abs() <= rel * want + 2.0 ** -25).all()


@pytest.mark.parametrize("dtype", DTYPES)
def test_queries_at_an_odd_address_are_copied(dtype):
    """A contiguous q that does not begin on 16 bytes, or whose only token has any stride."""
    g = torch.Generator(device="cuda").manual_seed(5)
    flat = torch.randn(3 * 4 * 64 + 1, generator=g, device="cuda").to(dtype)
    k, v = (torch.randn(70, 2, 64, generator=g, device="cuda").to(dtype) for _ in range(2))
    q = flat[1:].view(3, 4, 64)
    assert q.is_contiguous()
    assert torch.equal(_attend(q, k, v), _attend(q.clone(), k, v))
    one = flat[:256].as_strided((1, 4, 64), (257, 64, 1))
    assert torch.equal(_attend(one, k, v), _attend(one.clone(memory_format=torch.contiguous_format), k, v))


@pytest.mark.parametrize("norm", [True, False])
def test_a_layer_without_a_rotation_table_prefills_as_with_angles_of_zero(norm):
    g = torch.Generator(device="cuda").manual_seed(6)
    n, Hq, Hkv, D = 200, 4, 2, 64
    q, k, v = torch.randn(n + 1, Hq + 2 * Hkv, D, generator=g, device="cuda", dtype=torch.bfloat16).split([Hq, Hkv, Hkv], 1)
    w = (1 + 0.1 * torch.randn(D, generator=g, device="cuda")) if norm else None
    gq, gk = make_gate_weights(1, D, D, seed=3, device="cuda")
    still = torch.cat([torch.ones(n + 1, D // 2), torch.zeros(n + 1, D // 2)], 1).cuda()      # cos 1, sin 0
    results = []
    for table in (None, still):
        cache = PagedKVCache(1, 20, 16, Hkv, D)
        layer = PagedSparseLayer(cache, 0, table, prefill=SparsePrefillLayer(gq[0], gk[0], 3), q_weight=w, k_weight=w)
        out, _ = layer.prefill(q[:n], k[:n], v[:n], cache.step([("a", n)]))
        results.append((out, layer.extend(q[n:], k[n:], v[n:], cache.step([("a", 1)]))))
    assert torch.equal(results[0][0], results[1][0]) and torch.equal(results[0][1], results[1][1])
