"""Eviction from a paged cache by weight: nothing is computed, so everything has to be equal."""
import math

import pytest
import torch

from spruce_research_b200 import _lib, native

pytestmark = pytest.mark.gpu

DTYPES = [torch.float32, torch.bfloat16, torch.float16]


class Cache:
    """K, V and weights of sequences over shuffled pages; slots of no sequence hold a value that must stay."""

    def __init__(self, lens, Hkv, D, page, dtype, seed=0, weights=None, hnd=True, spare=2):
        g = torch.Generator(device="cuda").manual_seed(seed)
        need = [-(-x // page) for x in lens]
        n = sum(need) + spare
        order = torch.randperm(n, generator=torch.Generator().manual_seed(seed)).int()
        self.table = torch.full((len(lens), max(need, default=0) + 1), 1 << 30, dtype=torch.int32)   # never to be followed
        at = 0
        for s, m in enumerate(need):
            self.table[s, :m] = order[at:at + m]
            at += m
        self.table = self.table.cuda()
        shape = (n, Hkv, page, D) if hnd else (n, page, Hkv, D)
        self.k, self.v = (torch.randn(shape, generator=g, device="cuda").to(dtype) for _ in range(2))
        if not hnd:
            self.k, self.v = self.k.transpose(1, 2), self.v.transpose(1, 2)
        self.mass = torch.exp(2 * torch.randn(n, Hkv, page, generator=g, device="cuda"))
        if weights is not None:
            self.mass = weights(self.mass)
        self.lens, self.page, self.Hkv = lens, page, Hkv
        self.kv = torch.tensor(lens, dtype=torch.int32).cuda()

    def rows(self, x, s, n=None):
        j = torch.arange(self.lens[s] if n is None else n, device="cuda")
        return x[self.table[s].long()[j // self.page], :, j % self.page]

    def want(self, keep, sinks, recent):
        """Old slots kept, [S][Hkv] lists."""
        out = []
        for s, n in enumerate(self.lens):
            w = self.rows(self.mass, s).cpu()
            heads = []
            for h in range(self.Hkv):
                if n <= keep:
                    heads.append(list(range(n)))
                    continue
                lo = min(sinks, keep)
                hi = n - min(recent, keep - lo)
                def rank(j):
                    x = w[j, h].item()
                    return (-math.inf if math.isnan(x) else -x, j)
                # NaN above +inf: sorted first by itself
                mid = sorted(range(lo, hi), key=lambda j: (not math.isnan(w[j, h].item()), *rank(j)))
                heads.append(sorted(list(range(lo)) + mid[:keep - lo - (n - hi)] + list(range(hi, n))))
            out.append(heads)
        return out

    def check(self, keep, sinks=0, recent=0, into=False, most=None):
        kept = self.want(keep, sinks, recent)
        most = max(self.lens, default=0) if most is None else most
        status = torch.zeros(1, device="cuda", dtype=torch.int32)
        before = [x.clone() for x in (self.k, self.v, self.mass)]
        if into:
            to = Cache([min(n, keep) for n in self.lens], self.Hkv, self.k.shape[3], self.page, self.k.dtype, seed=99)
            args = dict(into=(to.k, to.v, to.mass, to.table))
        else:
            to, args = self, {}
        want = [x.clone() for x in (to.k, to.v, to.mass)]
        for s, heads in enumerate(kept):
            for h, slots in enumerate(heads):
                j, src = torch.arange(len(slots), device="cuda"), torch.tensor(slots, device="cuda", dtype=torch.long)
                for a, b in zip(before, want):
                    b[to.table[s].long()[j // self.page], h, j % self.page] = a[
                        self.table[s].long()[src // self.page], h, src % self.page]
        got, lens = native.paged_evict(self.k, self.v, self.mass, self.table, self.kv, keep, sinks=sinks, recent=recent,
                                       max_kv_len=most, status=status, **args)
        assert status.item() == 0
        assert lens.tolist() == [min(n, keep) for n in self.lens]
        assert got.shape == (len(self.lens), self.Hkv, min(keep, most))
        for s, heads in enumerate(kept):
            for h, slots in enumerate(heads):
                assert got[s, h].tolist() == slots + [-1] * (got.shape[2] - len(slots)), (s, h)
        for a, b, name in zip((to.k, to.v, to.mass), want, ("k", "v", "mass")):
            assert torch.equal(a.nan_to_num(5.0), b.nan_to_num(5.0)), name
        if into:
            for a, b in zip((self.k, self.v, self.mass), before):
                assert torch.equal(a.nan_to_num(5.0), b.nan_to_num(5.0))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("into", [False, True])
@pytest.mark.parametrize("lens, page, D", [([100], 16, 64), ([1, 0, 17, 64, 300], 16, 64), ([700, 33], 64, 128),
                                           ([1000], 48, 80), ([257, 256, 255], 128, 8)])
@pytest.mark.parametrize("keep, sinks, recent", [(32, 0, 0), (50, 4, 10), (33, 1, 32), (16, 30, 30), (1, 0, 0), (0, 0, 0),
                                                 (255, 3, 7), (2000, 4, 4)])
def test_kept_slots_and_their_rows(dtype, into, lens, page, D, keep, sinks, recent):
    Cache(lens, 3, D, page, dtype, seed=keep).check(keep, sinks, recent, into)


@pytest.mark.parametrize("into", [False, True])
@pytest.mark.parametrize("n, keep", [(5000, 1000), (5000, 4999), (20011, 4096), (70001, 9000)])
def test_long_sequences(into, n, keep):
    Cache([n, n // 3], 2, 64, 64, torch.bfloat16).check(keep, 16, 200, into)


def tied(m):
    return torch.randint(0, 3, m.shape, device="cuda", generator=torch.Generator(device="cuda").manual_seed(1)).float()


def signed_zero(m):
    return torch.where(tied(m) == 0, -0.0, 0.0)


def strange(m):
    x = tied(m)
    m = torch.where(x == 0, math.nan, m)
    return torch.where(x == 1, torch.where(m > 1, math.inf, -m), m)


@pytest.mark.parametrize("weights", [tied, signed_zero, strange, torch.zeros_like, lambda m: m * 1e-42])
@pytest.mark.parametrize("n, keep", [(90, 40), (3000, 1234)])
def test_ties_zeros_and_weights_that_are_not_numbers(weights, n, keep):
    """Equal weights (-0 and 0 are): the lowest slot stays.  NaN counts as the largest.  Subnormal weights differ."""
    Cache([n, n - 7], 2, 64, 16, torch.float16, weights=weights).check(keep, 2, 5)


@pytest.mark.parametrize("n, keep", [(100, 99), (3000, 2999), (2100, 2050)])
def test_rows_that_move_by_a_few_slots(n, keep):
    """The worst case of a move in place: almost every slot is read and written."""
    c = Cache([n], 2, 128, 64, torch.bfloat16, weights=lambda m: m)
    c.mass[c.table[0, 0].long(), :, 0] = 0.0
    c.check(keep, 0, 0)


def test_layouts_of_their_own():
    c = Cache([400, 90], 4, 64, 32, torch.bfloat16, hnd=False)
    c.mass = c.mass.transpose(0, 1).contiguous().transpose(0, 1)
    c.check(70, 3, 20)


def test_long_and_broken_sequences_are_reported():
    """A sequence past the bound, or of a negative length, is left as it is; a bad page's weights count as 0."""
    c = Cache([200, 60, 120], 2, 64, 16, torch.float32)
    status = torch.zeros(1, device="cuda", dtype=torch.int32)
    before = [x.clone() for x in (c.k, c.v, c.mass)]
    kv = c.kv.clone()
    kv[2] = -5
    kept, lens = native.paged_evict(c.k, c.v, c.mass, c.table, kv, 64, max_kv_len=150, status=status)
    assert status.item() == _lib.STATUS_BAD_LENGTH
    assert lens.tolist() == [200, 60, -5] and (kept[0] == -1).all() and (kept[2] == -1).all()
    assert kept[1, 0].tolist() == list(range(60)) + [-1] * 4
    for a, b in zip((c.k, c.v, c.mass), before):
        assert torch.equal(a, b)
    status.zero_()
    table = c.table.clone()
    table[0, 2], table[0, 4] = -1, c.k.shape[0]                       # slots 32 to 47 and 64 to 79
    kept, lens = native.paged_evict(c.k, c.v, c.mass, table, c.kv, 168, max_kv_len=200, status=status)
    assert status.item() == _lib.STATUS_BAD_PAGE and lens.tolist() == [168, 60, 120]
    lost = [*range(32, 48), *range(64, 80)]
    assert all(kept[0, h].tolist() == [j for j in range(200) if j not in lost] for h in range(2))


def test_the_same_cache_is_cut_twice_then_replayed_in_a_graph():
    c = Cache([500, 300], 2, 64, 16, torch.bfloat16)
    c.check(200, 4, 50)
    c.lens, c.kv = [200, 200], torch.tensor([200, 200], dtype=torch.int32).cuda()
    c.check(77, 4, 50)
    c = Cache([500, 300], 2, 64, 16, torch.bfloat16)
    to = Cache([128, 128], 2, 64, 16, torch.bfloat16, seed=3)
    want = [x.clone() for x in (to.k, to.v, to.mass)]
    kw = dict(sinks=1, recent=9, max_kv_len=500)
    kept, lens = native.paged_evict(c.k, c.v, c.mass, c.table, c.kv, 128, into=(*want, to.table), **kw)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kept2, lens2 = native.paged_evict(c.k, c.v, c.mass, c.table, c.kv, 128, into=(to.k, to.v, to.mass, to.table), **kw)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(kept, kept2) and torch.equal(lens, lens2)
    assert all(torch.equal(a, b) for a, b in zip(want, (to.k, to.v, to.mass)))
    assert native.paged_evict(c.k, c.v, c.mass, c.table[:0], c.kv[:0], 10, max_kv_len=5)[0].shape == (0, 2, 5)


@pytest.mark.parametrize("into", [False, True])
def test_pieces_of_more_slots_than_shared_memory_holds(into):
    """A million slots of one head: the weights past those that a CTA keeps are read again."""
    n, keep, page = 1_000_003, 5001, 64
    g = torch.Generator(device="cuda").manual_seed(1)
    pages = -(-n // page)
    table = torch.randperm(pages, generator=torch.Generator().manual_seed(1)).int()[None].cuda()
    k = torch.randn(pages, 1, page, 8, generator=g, device="cuda", dtype=torch.bfloat16)
    v, mass = k + 1, torch.rand(pages, 1, page, generator=g, device="cuda").mul_(4096).floor_()      # many ties
    kv = torch.tensor([n], device="cuda", dtype=torch.int32)
    flat = [x[:, 0][table[0].long()].reshape(pages * page, -1)[:n] for x in (k, v, mass[..., None])]
    w = flat[2][:, 0].clone()
    w[:3], w[n - 100:] = math.inf, math.inf
    want = torch.sort(w, descending=True, stable=True).indices[:keep].sort().values
    to = (torch.zeros(100, 1, page, 8, device="cuda", dtype=torch.bfloat16), torch.zeros(100, 1, page, 8, device="cuda", dtype=torch.bfloat16),
          torch.zeros(100, 1, page, device="cuda"), torch.arange(100, device="cuda", dtype=torch.int32)[None])
    kept, lens = native.paged_evict(k, v, mass, table, kv, keep, sinks=3, recent=100, max_kv_len=n, into=to if into else None)
    assert lens.item() == keep and torch.equal(kept[0, 0].long(), want)
    j = torch.arange(keep, device="cuda")
    at = (to[3] if into else table)[0].long()[j // page]
    for x, y in zip(to[:3] if into else (k, v, mass), flat):
        assert torch.equal(x[at, 0, j % page].reshape(keep, -1), y[want])


def test_heads_that_several_ctas_share_replay_in_a_graph():
    c = Cache([40000, 9000], 2, 64, 64, torch.bfloat16)
    to = Cache([3000, 3000], 2, 64, 64, torch.bfloat16, seed=3)
    kw = dict(sinks=1, recent=9, max_kv_len=40000, into=(to.k, to.v, to.mass, to.table))
    kept, lens = native.paged_evict(c.k, c.v, c.mass, c.table, c.kv, 3000, **kw)
    want = [x.clone() for x in (to.k, to.v, to.mass)]
    for s, heads in enumerate(c.want(3000, 1, 9)):
        for h, slots in enumerate(heads):
            assert kept[s, h].tolist() == slots
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kept2, lens2 = native.paged_evict(c.k, c.v, c.mass, c.table, c.kv, 3000, **kw)
    for x in (to.k, to.v, to.mass):
        x.zero_()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        graph.replay()
    side.synchronize()
    assert torch.equal(kept, kept2) and torch.equal(lens, lens2)
    j = torch.arange(3000, device="cuda")
    for s in range(2):
        at = to.table[s].long()[j // 64]
        for x, y in zip((to.k, to.v, to.mass), want):
            assert torch.equal(x[at, :, j % 64], y[at, :, j % 64])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("q", [1, 40])
def test_pages_past_the_32_bit_offset(dtype, q):
    """The last pages of a cache of more than 2^32 elements: weights, and rows evicted into a small cache, as from a small one."""
    Hkv, page, D, n = 4, 128, 128, 700
    pages = (1 << 32) // (Hkv * page * D) + 40
    g = torch.Generator(device="cuda").manual_seed(3)
    ids = torch.tensor([pages - 1 - 3 * i for i in range(6)], dtype=torch.int32, device="cuda")
    big = torch.empty(pages, Hkv, page, D, device="cuda", dtype=dtype)
    small = torch.randn(6, Hkv, page, D, generator=g, device="cuda").to(dtype)
    big[ids.long()] = small
    x = torch.randn(q, 8, D, generator=g, device="cuda").to(dtype)
    mass = torch.zeros(pages, Hkv, page, device="cuda")
    near = torch.zeros(6, Hkv, page, device="cuda")
    cu, kv = (torch.tensor(t, device="cuda", dtype=torch.int32) for t in ([0, q], [n]))
    order = torch.arange(6, device="cuda", dtype=torch.int32)[None]
    lse = torch.full((q, 8), 12.0, device="cuda")
    kw = dict(max_q_len=q, max_kv_len=n, decay=0.0)
    native.paged_key_mass(x, big, mass, ids[None], cu, kv, lse, **kw)
    native.paged_key_mass(x, small, near, order, cu, kv, lse, **kw)
    assert torch.equal(mass[ids.long()], near) and near.sum() > 0
    out = [[torch.zeros(2, Hkv, page, D, device="cuda", dtype=dtype) for _ in range(2)]
           + [torch.zeros(2, Hkv, page, device="cuda"), torch.arange(2, device="cuda", dtype=torch.int32)[None]] for _ in range(2)]
    a = native.paged_evict(big, big, mass, ids[None], kv, 200, sinks=1, recent=20, max_kv_len=n, into=out[0])
    b = native.paged_evict(small, small, near, order, kv, 200, sinks=1, recent=20, max_kv_len=n, into=out[1])
    assert all(torch.equal(s, t) for s, t in zip((*a, *out[0]), (*b, *out[1]))) and out[0][0].any()


@pytest.mark.parametrize("dtype, D", [(torch.bfloat16, 128), (torch.float16, 128), (torch.float32, 64), (torch.float32, 128)])
@pytest.mark.parametrize("keep", [40, 250, 699])
def test_many_heads_in_place(dtype, D, keep):
    """More CTAs of slices than the GPU holds at a time, so that each takes 64 bytes of a row; ragged lengths, moves of many and few slots."""
    lens = [700, 33, 251, 640, 1, 0, 412, 699, 250, 700]
    heads, row = 3 * len(lens), D * torch.empty(0, dtype=dtype).element_size()
    assert heads * (2 * (row // 32) + 1) > 2 * torch.cuda.get_device_properties(0).multi_processor_count
    c = Cache(lens, 3, D, 16, dtype, seed=keep)
    c.mass[c.table[0, 0].long(), :, 0] = 0.0       # its slot goes, so almost every row of the first sequence moves by one
    c.check(keep, 0, 1)


def test_long_heads_of_one_cta_each():
    """So many heads that none gets a second CTA, and more slots than a CTA's shared memory holds: the rest is read again."""
    lens, keep, heads = [49200, 50003], 2000, 40
    c = Cache(lens, heads, 8, 64, torch.bfloat16, weights=lambda m: (m * 64).floor())      # many ties
    assert 2 * heads * 2 > torch.cuda.get_device_properties(0).multi_processor_count
    before = [[c.rows(x, s).clone() for x in (c.k, c.v, c.mass)] for s in range(2)]
    kept, new = native.paged_evict(c.k, c.v, c.mass, c.table, c.kv, keep, sinks=3, recent=100, max_kv_len=max(lens))
    assert new.tolist() == [keep, keep]
    for s, n in enumerate(lens):
        w = before[s][2].clone()
        w[:3], w[n - 100:] = math.inf, math.inf
        want = torch.sort(w, dim=0, descending=True, stable=True).indices[:keep].sort(0).values
        assert torch.equal(kept[s].long(), want.T)
        for x, y in zip((c.k, c.v, c.mass), before[s]):
            at = want if y.dim() == 2 else want[..., None].expand(-1, -1, y.shape[2])
            assert torch.equal(c.rows(x, s, keep), y.gather(0, at))
