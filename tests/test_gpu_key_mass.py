"""The weight that cached keys receive, and the log-sums it is formed from, against 64-bit softmax arithmetic.

Bounds.  A score's fp32 dot of D products is off by at most D 2^-24 S with S = scale sum_d |q_d k_d|, and once more by as much
in its scaling.  The log-sum moves by the largest of these, by the exponentials' relative error E (16 bits: 1e-4 where a
polynomial of the attention serves; fp32: 2^-20), the sum's n 2^-24, and the roundings of a maximum plus a logarithm of at most
|lse| + 40.  A weight exp(s - lse) moves by the exponent's error (the score's, and four roundings at M = |s| + |lse|),
E' = 4e-6 in 16 bits and 2^-20 in fp32, and the sum's (rows + 2) 2^-24; terms under 2^-126 may be lost.
"""
import math

import pytest
import torch
from test_gpu_paged_attention import Batch

from spruce_research_b200 import _lib, native

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.bfloat16, torch.float16]
E_LSE = {torch.float32: 2.0 ** -20, torch.bfloat16: 1e-4, torch.float16: 1e-4}
E_MASS = {torch.float32: 2.0 ** -20, torch.bfloat16: 4e-6, torch.float16: 4e-6}


def scores(b, s, h, scale=None):
    """64-bit scores of sequence s, query head h (-inf where a token does not see a key), and the sums of magnitudes."""
    at, a, kv = sum(b.qlens[:s]), b.qlens[s], b.kvs[s]
    Hkv = b.k[s].shape[1]
    scale = b.q.shape[2] ** -0.5 if scale is None else scale
    q, k = b.q[at:at + a, h].double(), b.k[s][:, h // (b.q.shape[1] // Hkv)].double()
    late = torch.arange(kv, device="cuda") > torch.arange(kv - a, kv, device="cuda")[:, None]
    return (q @ k.T * scale).masked_fill(late, -math.inf), q.abs() @ k.abs().T * scale


def want_lse(b, scale=None):
    N, Hq, D = b.q.shape
    out, bound = (torch.zeros(N, Hq, device="cuda", dtype=torch.float64) for _ in range(2))
    at = 0
    for s, (a, kv) in enumerate(zip(b.qlens, b.kvs)):
        for h in range(Hq if a else 0):
            z, S = scores(b, s, h, scale)
            out[at:at + a, h] = lse = torch.logsumexp(z, -1) if kv else torch.full((a,), -math.inf, device="cuda")
            top = S.amax(-1) if kv else torch.zeros(a, device="cuda")
            bound[at:at + a, h] = (2 * D * 2.0 ** -24 * top + kv * 2.0 ** -24 + E_LSE[b.q.dtype]
                                   + 4 * 2.0 ** -24 * (lse.abs().nan_to_num(posinf=0.0) + 40))
        at += a
    return out, bound


def want_mass(b, lse, mass, decay, scale=None):
    """64-bit weights and bounds [pages, Hkv, page]; slots that no call writes are NaN."""
    N, Hq, D = b.q.shape
    out, bound = (torch.full(mass.shape, math.nan, device="cuda", dtype=torch.float64) for _ in range(2))
    page, Hkv, at = b.page, mass.shape[1], 0
    rep = Hq // Hkv
    for s, (a, kv) in enumerate(zip(b.qlens, b.kvs)):
        if a and kv:
            x = torch.arange(kv, device="cuda")
            pages = b.table[s].long()[x // page]
            for g in range(Hkv):
                total = torch.where(x < kv - a, decay * mass[pages, g, x % page].double(), 0.0) if decay else torch.zeros(
                    kv, device="cuda", dtype=torch.float64)
                slack = total.abs() * 2.0 ** -23
                for h in range(g * rep, (g + 1) * rep):
                    z, S = scores(b, s, h, scale)
                    r = lse[at:at + a, h].double()[:, None]
                    p = torch.exp(z - torch.where(r == -math.inf, math.inf, r))
                    M = S + r.abs().nan_to_num(posinf=0.0)
                    total = total + p.sum(0)
                    slack = slack + (p * (2 * D * 2.0 ** -24 * S + 4 * 2.0 ** -24 * M + E_MASS[b.q.dtype]
                                          + (rep * a + 2) * 2.0 ** -24)).sum(0) + a * 2.0 ** -120
                out[pages, g, x % page], bound[pages, g, x % page] = total, slack
        at += a
    return out, bound


def check(b, decay=1.0, scale=None, in_place=True, seed=5):
    """lse by the attention, weights by the key mass: both against 64 bits, slots of nobody as they were."""
    N, Hq, D = b.q.shape
    status = torch.zeros(1, device="cuda", dtype=torch.int32)
    lse = torch.full((N, Hq), 7.0, device="cuda")
    plain = b.call(scale=scale)
    out = b.call(scale=scale, lse=lse, status=status)
    assert torch.equal(out, plain)
    want, bound = want_lse(b, scale)
    same = (want == -math.inf) & (lse == -math.inf)
    assert (same | ((lse - want).abs() <= bound)).all(), (lse - want).abs().nan_to_num().max()
    mass = torch.rand(b.kc.shape[:3], generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda")
    if decay == 0:
        mass.fill_(math.nan)                                      # not read
    old = mass.clone()
    got = torch.full_like(mass, 3.0) if not in_place else mass
    kw = dict(max_q_len=max(b.qlens), max_kv_len=max(b.kvs), decay=decay, scale=scale, status=status)
    res = native.paged_key_mass(b.q, b.kc, mass, b.table, b.cu, b.kv, lse, out=None if in_place else got, **kw)
    assert res is got and status.item() == 0
    want, bound = want_mass(b, lse, old, decay, scale)
    named = ~want.isnan()
    assert ((got - want).abs() <= bound)[named].all(), ((got - want).abs() / bound)[named].max()
    left = old if in_place else torch.full_like(mass, 3.0)
    assert torch.equal(got[~named].nan_to_num(5.0), left[~named].nan_to_num(5.0))
    return lse, got


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("heads", [(28, 4, 128), (4, 2, 64), (3, 3, 64), (8, 1, 128)])
@pytest.mark.parametrize("qlens, kvs, page", [
    ([1], [1], 16), ([1, 1, 1], [15, 16, 17], 16), ([1, 0, 1, 1], [700, 40, 63, 1000], 64), ([2, 5], [130, 257], 32),
    ([9, 33], [64, 300], 48), ([70, 0, 1, 128], [70, 10, 129, 640], 64), ([200], [4000], 128), ([0, 1], [5, 0], 16),
    ([257, 3], [300, 3], 16)])
def test_weights_of_ragged_batches(dtype, heads, qlens, kvs, page):
    kvs = [max(a, b) for a, b in zip(qlens, kvs)] if 0 not in kvs else kvs
    if 0 in kvs:
        qlens = [0, 0]
        kvs = [5, 0]
    b = Batch(qlens, kvs, *heads, page, dtype, seed=len(kvs))
    check(b, decay=0.5)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("heads", [(130, 1, 64), (256, 2, 128), (65, 1, 64)])
def test_groups_of_more_heads_than_a_row_tile_has_rows(dtype, heads):
    check(Batch([3, 0, 1], [200, 9, 70], *heads, 32, dtype), decay=0.5)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_a_prompt_of_its_own_keys(dtype):
    """Few keys under many rows: a cluster shares an item, and the diagonal crosses every row tile."""
    check(Batch([1500], [1500], 8, 1, 128, 64, dtype), decay=0.0)
    check(Batch([700], [1300], 4, 2, 64, 16, dtype), decay=1.0)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("decay", [0.0, 0.75, 1.0])
@pytest.mark.parametrize("in_place", [True, False])
@pytest.mark.parametrize("q", [1, 40])
def test_old_weights_fade_and_new_slots_start_from_zero(dtype, decay, in_place, q):
    check(Batch([q, q, 0], [300, q, 50], 14, 2, 64, 32, dtype), decay=decay, in_place=in_place)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("q", [1, 8, 64])
def test_weights_over_a_long_cache(dtype, q):
    check(Batch([q], [20011], 28, 4, 128, 64, dtype), decay=0.0)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("q", [1, 50])
def test_a_cache_with_tokens_outside_heads_and_a_scale(dtype, q):
    check(Batch([q, 1], [200, 33], 8, 2, 64, 16, dtype, hnd=False), scale=0.3)
    check(Batch([q, 1], [200, 33], 8, 2, 128, 16, dtype), scale=0.0)


@pytest.mark.parametrize("q", [1, 40])
def test_strided_weights_and_queries(q):
    """Weights in a layout of their own ([Hkv, pages, page]), lse as rows of a wider tensor, q within a fused projection."""
    b = Batch([q, 2], [150, 77], 8, 4, 64, 16, torch.bfloat16)
    N = b.q.shape[0]
    lse, got = check(b, decay=0.5)
    fused = torch.zeros(N, 20, 64, device="cuda", dtype=torch.bfloat16)
    fused[:, 3:11] = b.q
    wide = torch.zeros(N, 30, device="cuda")
    wide[:, 5:13] = lse
    mass = torch.rand(b.kc.shape[:3], generator=torch.Generator(device="cuda").manual_seed(5), device="cuda")
    turned = mass.transpose(0, 1).contiguous().transpose(0, 1)
    native.paged_key_mass(fused[:, 3:11], b.kc, turned, b.table, b.cu, b.kv, wide[:, 5:13], max_q_len=max(b.qlens),
                          max_kv_len=max(b.kvs), decay=0.5)
    assert torch.equal(turned, got)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("q, kv", [(1, 90), (1, 9000), (60, 90), (300, 2500)])   # whole units and joined ones of each kernel
def test_log_sums_into_columns_of_a_wider_tensor(dtype, q, kv):
    """By strides, nothing beside them; rows of no sequence keep what they had."""
    b = Batch([q, 0, 2], [kv, 7, 2], 8, 2, 64, 16, dtype)
    lse = torch.empty(b.q.shape[:2], device="cuda")
    out = b.call(lse=lse)
    wide = torch.full((b.q.shape[0] + 3, 20), 7.0, device="cuda")
    padded = torch.cat([b.q, b.q[:3]])
    got = native.paged_attention(padded, b.kc, b.vc, b.table, b.cu, b.kv, max_q_len=max(q, 2), max_kv_len=kv,
                                 out=torch.full_like(padded, 7.0), lse=wide[:, 4:12])
    assert torch.equal(got[:-3], out) and (got[-3:] == 7).all()
    assert torch.equal(wide[:-3, 4:12], lse) and (wide[-3:] == 7).all() and (wide[:, :4] == 7).all() and (wide[:, 12:] == 7).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("q", [1, 60])
def test_rows_that_count_for_nothing_and_scores_that_are_not_finite(dtype, q):
    """An lse of -inf gives nothing.  What a masked place holds does not matter: rows past a sequence are NaN already, and a NaN key
    reaches only its own weight and that of rows whose lse it spoilt."""
    b = Batch([q], [100], 4, 2, 64, 16, dtype)
    lse = torch.full((q, 4), -math.inf, device="cuda")
    mass = torch.full(b.kc.shape[:3], 2.0, device="cuda")
    kw = dict(max_q_len=q, max_kv_len=100)
    native.paged_key_mass(b.q, b.kc, mass, b.table, b.cu, b.kv, lse, decay=1.0, **kw)
    x = torch.arange(100, device="cuda")
    pages = b.table[0].long()[x // 16]
    assert torch.equal(mass[pages, :, x % 16], torch.where(x < 100 - q, 2.0, 0.0)[:, None].expand(-1, 2))
    lse.fill_(1.0)
    b.kc[b.table[0, 2].long(), 1, 3] = math.nan                  # key 35 of head 1
    got = native.paged_key_mass(b.q, b.kc, mass, b.table, b.cu, b.kv, lse, decay=0.0, **kw)[pages, :, x % 16]
    assert got[35, 1].isnan() and got.isnan().sum() == 1
    if q > 1:                                                    # the last row is lost: every key that it sees
        lse[q - 1, 3] = math.nan
        got = native.paged_key_mass(b.q, b.kc, mass, b.table, b.cu, b.kv, lse, decay=0.0, **kw)[pages, :, x % 16]
        assert got[:, 1].isnan().all() and got[:, 0].isfinite().all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("q", [1, 60])
def test_bad_pages_and_lengths_are_reported(dtype, q):
    """Keys of a bad page get no weight; a sequence longer than the bounds is cut to them."""
    b = Batch([q, q], [200, 90], 4, 2, 64, 16, dtype)
    lse = torch.zeros(2 * q, 4, device="cuda")
    mass = torch.full(b.kc.shape[:3], 2.0, device="cuda")
    good = native.paged_key_mass(b.q, b.kc, mass, b.table, b.cu, b.kv, lse, max_q_len=q, max_kv_len=200,
                                 out=mass.clone(), decay=0.0)
    table = b.table.clone()
    table[0, 3], table[0, 5] = -1, b.kc.shape[0]
    status = torch.zeros(1, device="cuda", dtype=torch.int32)
    got = native.paged_key_mass(b.q, b.kc, mass, table, b.cu, b.kv, lse, max_q_len=q, max_kv_len=200, out=mass.clone(),
                                decay=0.0, status=status)
    assert status.item() == _lib.STATUS_BAD_PAGE
    want = good.clone()
    want[b.table[0, [3, 5]].long()] = 2.0
    assert torch.equal(got, want)
    status.zero_()
    got = native.paged_key_mass(b.q, b.kc, mass, b.table, b.cu, b.kv, lse, max_q_len=q, max_kv_len=100, out=mass.clone(),
                                decay=0.0, status=status)
    assert status.item() == _lib.STATUS_BAD_LENGTH
    x = torch.arange(112, 200, device="cuda")                    # slots 100 on are not seen; page 6 holds 96 to 111
    assert (got[b.table[0].long()[x // 16], :, x % 16] == 2.0).all()
    x = torch.arange(90, device="cuda")
    assert torch.equal(got[b.table[1].long()[x // 16], :, x % 16], good[b.table[1].long()[x // 16], :, x % 16])


@pytest.mark.parametrize("q", [1, 40])
def test_weights_replay_in_a_graph_and_on_another_stream(q):
    b = Batch([q, 1], [500, 90], 28, 4, 128, 64, torch.bfloat16)
    lse, want = check(b, decay=0.0, in_place=False)
    mass = torch.zeros(b.kc.shape[:3], device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    got = torch.zeros_like(lse)

    def step():
        b.call(lse=got)
        native.paged_key_mass(b.q, b.kc, mass, b.table, b.cu, b.kv, got, max_q_len=q, max_kv_len=500, decay=0.0)

    with torch.cuda.stream(side):
        step()
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    mass.zero_()
    graph.replay()
    torch.cuda.synchronize()
    named = want != 3.0
    assert torch.equal(mass[named], want[named]) and torch.equal(got, lse)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("heads", [(7, 1, 64), (28, 4, 128), (10, 2, 64), (40, 1, 64), (65, 1, 64), (4, 4, 128)])
@pytest.mark.parametrize("q", [1, 5, 40, 300])
def test_keys_whose_scores_are_minus_infinity_get_nothing(dtype, heads, q):
    """Zero rows that fill a tile up make no number with an infinite key, wherever in the tiles and the prompt it stands."""
    Hq, Hkv, D = heads
    b = Batch([q, q], [700 + q, 300 + q], Hq, Hkv, D, 16, dtype)
    b.q[..., 0] = 1.0
    b.kc[..., 0] = 0.0
    dead = torch.tensor([0, 3, 64, 127, 128, 200, 255, 290], device="cuda")
    for s in range(2):
        b.kc[b.table[s].long()[dead // 16], :, dead % 16, 0] = -math.inf
    batch, kw = (b.table, b.cu, b.kv), dict(max_q_len=q, max_kv_len=700 + q)
    lse, mass = torch.empty(2 * q, Hq, device="cuda"), torch.zeros(b.kc.shape[:3], device="cuda")
    native.paged_attention(b.q, b.kc, b.vc, *batch, lse=lse, **kw)
    native.paged_key_mass(b.q, b.kc, mass, *batch, lse, decay=0.0, **kw)
    for s, n in enumerate((700 + q, 300 + q)):
        j = torch.arange(n, device="cuda")
        got = mass[b.table[s].long()[j // 16], :, j % 16]
        # Each row gives 1 in all: its weights are good to 2 E, as its lse is, and the sum of q rep of them over n keys.
        assert (got[dead] == 0).all() and (got.sum(0).double() / (q * Hq // Hkv) - 1).abs().max() <= 1e-3
