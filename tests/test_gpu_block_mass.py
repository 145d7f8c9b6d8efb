"""The softmax weight of whole key blocks against 64-bit softmax attention.

Bound, relative to a block's weight: each probability moves by the errors of its score and of its row's total, twice D 2^-24 S and
four roundings at M = S + |total| each, by E = 4e-6 for the exponentials (fp32: 2^-20) twice, and the sums over 64 keys, the
blocks and the group's rows by (qb + 64 + 64 rep) 2^-24; weights under 2^-120 may be lost.
"""
import math

import pytest
import torch

from spruce_research_b200 import native

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.bfloat16, torch.float16]
E = {torch.float32: 2.0 ** -20, torch.bfloat16: 4e-6, torch.float16: 4e-6}


def make(B, Hq, Hkv, T, D, dtype, seed=0, scale=2.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    qk = torch.randn(B, T, Hq + Hkv, D, generator=g, device="cuda", dtype=dtype)
    qk[:, :, :Hq] *= scale
    return qk[:, :, :Hq].transpose(1, 2), qk[:, :, Hq:].transpose(1, 2)


def want(q, k, scale=None):
    B, Hq, T, D = q.shape
    Hkv, qb = k.shape[1], -(-T // 64)
    rep = Hq // Hkv
    scale = D ** -0.5 if scale is None else scale
    out, bound = (torch.zeros(B, Hkv, qb, qb, device="cuda", dtype=torch.float64) for _ in range(2))
    of = (torch.arange(T, device="cuda")[:, None] // 64 == torch.arange(qb, device="cuda")).double()
    late = torch.ones(T, T, device="cuda", dtype=torch.bool).triu(1)
    for b in range(B):
        for h in range(Hq):
            x, y = q[b, h].double(), k[b, h // rep].double()
            z = (x @ y.T * scale).masked_fill(late, -math.inf)
            S = (x.abs() @ y.abs().T * scale).masked_fill(late, 0.0).amax(-1, keepdim=True)
            total = torch.logsumexp(z, -1, keepdim=True)
            p = torch.exp(z - total)
            err = p * (4 * D * 2.0 ** -24 * S + 8 * 2.0 ** -24 * (S + total.abs() + 10) + 2 * E[q.dtype]
                       + (qb + 64 + 64 * rep) * 2.0 ** -24)
            out[b, h // rep] += of.T @ p @ of
            bound[b, h // rep] += of.T @ err @ of
    n = of.sum(0)[:, None] * rep
    return out / n, bound / n + 2.0 ** -120


def check(q, k, scale=None, **kw):
    status = torch.zeros(1, device="cuda", dtype=torch.int32)
    got = native.block_mass(q, k, scale=scale, status=status, **kw)
    w, bound = want(q, k, scale)
    assert status.item() == 0
    assert ((got - w).abs() <= bound).all(), ((got - w).abs() / bound).max()
    assert (got.triu(1) == 0).all()
    return got


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("heads", [(28, 4, 128), (4, 2, 64), (3, 3, 64), (8, 1, 128), (1, 1, 128)])
@pytest.mark.parametrize("T", [1, 63, 64, 65, 127, 128, 129, 192, 500, 1000])
def test_weights_of_blocks(dtype, heads, T):
    Hq, Hkv, D = heads
    got = check(*make(2 if T < 200 else 1, Hq, Hkv, T, D, dtype, seed=T))
    assert (got.sum(-1) - 1).abs().max() < 1e-4


@pytest.mark.parametrize("dtype", DTYPES)
def test_a_longer_prompt(dtype):
    check(*make(1, 4, 2, 4133, 128, dtype))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("scale", [0.0, 0.02, 1.0])
def test_scales_from_flat_rows_to_single_keys(dtype, scale):
    check(*make(1, 4, 2, 300, 64, dtype), scale=scale)


@pytest.mark.parametrize("dtype", DTYPES)
def test_scores_that_grow_along_the_row(dtype):
    """Each key outweighs those before it: the running maximum moves in every block; and the other way round."""
    q, k = make(1, 2, 1, 400, 64, dtype, scale=0.1)
    q, k = q.clone(), k.clone() * 0.1
    q[..., 0] = 16.0
    for sign in (1.0, -1.0):
        k[..., 0] = sign * torch.arange(400, device="cuda") / 8
        check(q, k)


@pytest.mark.parametrize("dtype", DTYPES)
def test_layouts(dtype):
    """[B, H, T, D] as such, a head that is shared by a stride, a batch of one with an odd stride, an odd address."""
    q, k = make(2, 4, 2, 150, 64, dtype)
    got = native.block_mass(q, k)
    assert torch.equal(got, native.block_mass(q.contiguous(), k.contiguous()))
    flat = torch.empty(q.numel() + 1, device="cuda", dtype=dtype)[1:].view(q.shape)
    flat.copy_(q)
    assert torch.equal(got, native.block_mass(flat, k))
    assert torch.equal(native.block_mass(q, k[:, :1].expand(-1, 2, -1, -1)), native.block_mass(q, k[:, :1]
                       .expand(-1, 2, -1, -1).contiguous()))
    assert torch.equal(got[1:], native.block_mass(q[1:], k[1:]))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("bad", ["nan", "inf"])
def test_scores_that_are_not_numbers(dtype, bad):
    """A NaN or an infinite key spoils the rows of the blocks that see it and no others."""
    q, k = make(1, 2, 1, 300, 64, dtype)
    q, k = q.clone(), k.clone()
    q[..., 3] = 1.0
    clean = native.block_mass(q, k)
    k[0, 0, 130, 3] = float(bad)
    got = native.block_mass(q, k)
    assert torch.equal(got[:, :, :2], clean[:, :, :2])
    assert got[0, 0, 2, :3].isnan().all() and got[0, 0, 3, :4].isnan().all() and (got.triu(1).nan_to_num() == 0).all()


def test_empty_shapes_and_a_workspace_of_ones_own():
    q, k = make(1, 4, 2, 300, 64, torch.bfloat16)
    assert native.block_mass(q[:, :, :0], k[:, :, :0]).shape == (1, 2, 0, 0)
    assert native.block_mass(q[:0], k[:0]).shape == (0, 2, 5, 5)
    ws = torch.full((1 << 22,), math.nan, device="cuda")
    out = torch.full((1, 2, 5, 5), math.nan, device="cuda")
    assert torch.equal(native.block_mass(q, k, workspace=ws, out=out), native.block_mass(q, k)) and out.isfinite().all()
    with pytest.raises(RuntimeError, match="workspace needs"):
        native.block_mass(q, k, workspace=ws[:64])


def test_a_graph_and_another_stream():
    q, k = make(1, 28, 4, 700, 128, torch.bfloat16)
    out = torch.empty(1, 4, 11, 11, device="cuda")
    want = native.block_mass(q, k)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = native.block_mass(q, k)
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        native.block_mass(q, k, out=out)
    out.zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, want) and torch.equal(other, want)


def want_without(q, k, gone):
    """`want`, the keys `gone` [T] having a score of -inf in every row; a row that sees no others gives nothing."""
    B, Hq, T, D = q.shape
    Hkv, qb = k.shape[1], -(-T // 64)
    rep = Hq // Hkv
    out, bound = (torch.zeros(B, Hkv, qb, qb, device="cuda", dtype=torch.float64) for _ in range(2))
    of = (torch.arange(T, device="cuda")[:, None] // 64 == torch.arange(qb, device="cuda")).double()
    hidden = torch.ones(T, T, device="cuda", dtype=torch.bool).triu(1) | gone
    for b in range(B):
        for h in range(Hq):
            x, y = q[b, h].double(), k[b, h // rep].double().masked_fill(gone[:, None], 0.0)
            z = (x @ y.T * D ** -0.5).masked_fill(hidden, -math.inf)
            S = (x.abs() @ y.abs().T * D ** -0.5).masked_fill(hidden, 0.0).amax(-1, keepdim=True)
            total = torch.logsumexp(z, -1, keepdim=True)
            p = torch.exp(z - total).masked_fill(hidden, 0.0)
            err = p * (4 * D * 2.0 ** -24 * S + 8 * 2.0 ** -24 * (S + total.abs() + 10) + 2 * E[q.dtype]
                       + (qb + 64 + 64 * rep) * 2.0 ** -24).masked_fill(hidden.all(-1, keepdim=True), 0.0)
            out[b, h // rep] += of.T @ p @ of
            bound[b, h // rep] += of.T @ err @ of
    n = of.sum(0)[:, None] * rep
    return out / n, bound / n + 2.0 ** -120


def check_without(q, k, gone):
    status = torch.zeros(1, device="cuda", dtype=torch.int32)
    got = native.block_mass(q, k, status=status)
    w, bound = want_without(q, k, gone)
    assert status.item() == 0
    assert ((got - w).abs() <= bound).all(), ((got - w).abs() / bound).max()
    return got


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("far", [0.0, -200.0])
@pytest.mark.parametrize("overflow", [False, True])
@pytest.mark.parametrize("dead", [(0,), (1,), (0, 1, 2, 3), (2, 3, 5), (0, 4)])
def test_blocks_whose_scores_are_all_minus_infinity(dtype, D, far, overflow, dead):
    """Whole blocks of -inf, by an infinite key or a product past fp32, ahead of scores near 0 and near -200: they weigh nothing."""
    if overflow and dtype == torch.float16:
        pytest.skip("products of fp16 do not leave fp32")
    q, k = make(1, 4, 2, 500, D, dtype, scale=0.5)
    q, k = q.clone(), k.clone()
    q[..., 0], k[..., 0] = 16.0, far * D ** 0.5 / 16
    q[..., 1], k[..., 1] = 1e30 if overflow else 1.0, 0.0
    gone = torch.isin(torch.arange(500, device="cuda") // 64, torch.tensor(dead, device="cuda"))
    k[:, :, gone, 1] = -1e30 if overflow else -math.inf
    got = check_without(q, k, gone)
    assert (got[..., list(dead)] == 0).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("T, dead", [(1, 0), (65, 0), (65, 64), (130, 129), (300, 100), (300, 0), (300, 299), (1000, 500)])
def test_a_key_of_minus_infinity_in_a_prompt_that_ends_inside_a_block(dtype, D, T, dead):
    """The rows of a tile past the prompt are zeros, and zero times an infinite key is not a number: it stays there."""
    q, k = make(2, 4, 2, T, D, dtype)
    q, k = q.clone(), k.clone()
    q[..., 0], k[..., 0] = 1.0, 0.0
    k[:, :, dead, 0] = -math.inf
    check_without(q, k, torch.arange(T, device="cuda") == dead)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("B, Hq, Hkv, T, D", [
    (3, 28, 4, 1100, 128),   # 384 units of mixed lengths on 148 CTAs, 216 items of the fp32 kernel
    (40, 12, 4, 300, 64),    # 800 units, the first 160 of a single tile: CTAs that take two such in a row; 800 items
    (5, 8, 2, 2100, 64),     # 340 units of up to 17 key tiles, 330 items
])
def test_ctas_that_take_several_units(dtype, B, Hq, Hkv, T, D):
    got = check(*make(B, Hq, Hkv, T, D, dtype, seed=T))
    assert (got.sum(-1) - 1).abs().max() < 1e-4
