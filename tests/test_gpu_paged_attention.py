"""Attention of new tokens over a paged cache against 64-bit softmax attention, one sequence and head at a time.

Bound, per output element, with A = sum_j p_j |v_j| over the row's softmax and u the unit roundoff of the dtype:
the store rounds by u A at most and, in 16 bits, each probability once more (u); a score's fp32 dot is off by at most
D 2^-24 S with S = max_j scale sum_d |q_d k_d|, which moves p_j and the sum by that much each; exponentials
by 1e-4 in 16 bits (a polynomial takes part of them) and 2^-21 in fp32; the sums over n keys, taken in tiles and blocks,
by n 2^-24.
"""
import pytest
import torch

from spruce_research_b200 import _lib, native

pytestmark = pytest.mark.gpu

U = {torch.float32: 2.0 ** -24, torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11}


class Batch:
    """Packed queries, a shuffled page table and caches whose unused rows hold NaN."""

    def __init__(self, qlens, kvs, Hq, Hkv, D, page, dtype, seed=0, hnd=True, qscale=2.0):
        g = torch.Generator(device="cuda").manual_seed(seed)
        self.qlens, self.kvs, self.page = qlens, kvs, page
        need = [-(-x // page) for x in kvs]
        order = torch.randperm(sum(need) + 2, generator=torch.Generator().manual_seed(seed)).int()
        table = torch.full((len(kvs), max(1, max(need)) + 1), 1 << 30, dtype=torch.int32)  # never to be followed
        shape = (sum(need) + 2, Hkv, page, D) if hnd else (sum(need) + 2, page, Hkv, D)
        self.kc, self.vc = (torch.full(shape, float("nan"), device="cuda", dtype=dtype) for _ in range(2))
        if not hnd:
            self.kc, self.vc = self.kc.transpose(1, 2), self.vc.transpose(1, 2)
        self.k, self.v = [], []
        at = 0
        for s, n in enumerate(need):
            table[s, :n] = order[at:at + n]
            at += n
            self.k.append(torch.randn(kvs[s], Hkv, D, generator=g, device="cuda", dtype=dtype))
            self.v.append(torch.randn(kvs[s], Hkv, D, generator=g, device="cuda", dtype=dtype))
            for p in range(n):
                m = min(page, kvs[s] - p * page)
                self.kc[int(table[s, p]), :, :m] = self.k[s][p * page:p * page + m].transpose(0, 1)
                self.vc[int(table[s, p]), :, :m] = self.v[s][p * page:p * page + m].transpose(0, 1)
        self.table = table.cuda()
        self.cu = torch.tensor([0] + qlens).cumsum(0).int().cuda()
        self.kv = torch.tensor(kvs, dtype=torch.int32).cuda()
        self.q = torch.randn(sum(qlens), Hq, D, generator=g, device="cuda", dtype=dtype) * qscale

    def call(self, **kw):
        kw = dict(max_q_len=max(self.qlens), max_kv_len=max(self.kvs)) | kw
        return native.paged_attention(self.q, self.kc, self.vc, self.table, self.cu, self.kv, **kw)

    def want(self, scale=None):
        """64-bit outputs and bounds [N, Hq, D]."""
        N, Hq, D = self.q.shape
        scale = D ** -0.5 if scale is None else scale
        u = U[self.q.dtype]
        out = torch.zeros(N, Hq, D, device="cuda", dtype=torch.float64)
        bound = torch.zeros_like(out)
        at = 0
        for s, (a, kv) in enumerate(zip(self.qlens, self.kvs)):
            for h in range(Hq if a and kv else 0):
                g = h // (Hq // self.k[s].shape[1])
                k, v = self.k[s][:, g].double(), self.v[s][:, g].double()
                for t0 in range(0, a, 256):
                    t1 = min(a, t0 + 256)
                    q = self.q[at + t0:at + t1, h].double()
                    late = torch.arange(kv, device="cuda") > torch.arange(kv - a + t0, kv - a + t1, device="cuda")[:, None]
                    z = (q @ k.T * scale).masked_fill(late, float("-inf"))
                    p = torch.softmax(z, -1).nan_to_num(0.0)        # a row that sees nothing gives zeros
                    out[at + t0:at + t1, h] = p @ v
                    S = (q.abs() @ k.abs().T * abs(scale)).amax(-1, keepdim=True)
                    rel = 2 * D * 2.0 ** -24 * S + kv * 2.0 ** -24
                    rel = rel + (u + 2.0 ** -20 if u == 2.0 ** -24 else 2 * u + u * u + 2e-4)
                    bound[at + t0:at + t1, h] = rel * (p @ v.abs()) + 2.0 ** -25
            at += a
        return out, bound

    def check(self, scale=None, **kw):
        status = torch.zeros(1, device="cuda", dtype=torch.int32)
        got = self.call(status=status, scale=scale, **kw)
        out, bound = self.want(scale)
        assert got.shape == out.shape and got.dtype == self.q.dtype
        assert got.isfinite().all()
        over = ((got.double() - out).abs() - bound).max().item() if out.numel() else 0.0
        assert over <= 0, f"error passes its bound by {over:.3e}"
        assert status.item() == 0
        return got


DTYPES = [torch.float32, torch.bfloat16, torch.float16]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("qlens,kvs,Hq,Hkv,page", [
    ([1], [1], 28, 4, 64),                                    # one token, one key
    ([1, 1, 1, 1], [15, 16, 17, 1000], 28, 4, 16),            # decode around a page's end
    ([1] * 33, [64 * i + 63 for i in range(33)], 4, 2, 64),   # lengths of every residue of the key tiles' count
    ([1, 1], [129, 4000], 8, 8, 32),                          # no sharing of heads
    ([1] * 3, [300, 64, 129], 16, 1, 48),                     # one KV head; pages of 48
    ([2, 5, 1], [70, 5, 513], 28, 4, 64),                     # a few tokens each
    ([9, 4], [9, 700], 4, 2, 16),
    ([17], [129], 7, 1, 128),
    ([63, 0, 1, 130], [63, 40, 2, 257], 14, 2, 16),           # a chunk, an idle and a single-token sequence
    ([300], [1500], 28, 4, 64),
    ([256, 257], [256, 900], 4, 4, 256),
    ([37], [37], 3, 1, 80),                                   # a whole short prompt; rows of no power of two
    ([1] * 400, [1 + (37 * i) % 300 for i in range(400)], 4, 2, 16),             # more sequences than threads scan at once
    ([(11 * i) % 90 for i in range(41)], [(11 * i) % 90 + (53 * i) % 200 for i in range(41)], 4, 2, 16),
    ([1900], [1900], 4, 4, 64),                               # a prompt in one chunk: units of every length
    ([120, 120], [130, 1500], 8, 8, 64),                      # 65 to 128 rows: one tile of the pair
    ([40, 3], [600, 4000], 1, 1, 32)])                        # 33 to 64 rows
def test_matches_64_bits(dtype, D, qlens, kvs, Hq, Hkv, page):
    Batch(qlens, kvs, Hq, Hkv, D, page, dtype, seed=len(kvs) + page).check()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("q", [1, 3, 200])
def test_rows_that_see_nothing_are_zero(dtype, q):
    """Empty sequences and chunks longer than what the sequence holds, beside an ordinary one."""
    b = Batch([q, 1, q, q], [0, 0, q // 2, 77 + q], 6, 2, 64, 16, dtype, seed=1)
    got = b.check()
    assert (got[:q + 1] == 0).all() and (got[q + 1:2 * q + 1 - q // 2] == 0).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("q", [1, 70])
def test_strided_queries_outputs_and_caches(dtype, q):
    """Pages that keep their heads innermost, queries out of a fused projection, an output with a gap between tokens."""
    b = Batch([q, q], [90, 333], 4, 2, 64, 16, dtype, seed=2, hnd=False)
    wide = torch.randn(2 * q, 9, 64, device="cuda").to(dtype)
    wide[:, 2:6] = b.q
    b.q = wide[:, 2:6]
    assert not b.kc.is_contiguous()
    guard = torch.full((2 * q, 7, 64), 3.0, device="cuda", dtype=dtype)
    got = b.check(out=guard[:, 1:5])
    assert got.data_ptr() == guard[:, 1:5].data_ptr()
    assert (guard[:, 0] == 3).all() and (guard[:, 5:] == 3).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("q", [1, 40])
@pytest.mark.parametrize("scale", [1.0, 0.02, 0.0])
def test_scales_from_flat_to_one_key(dtype, q, scale):
    """scale 1: scores of a hundred and more, one key takes the row; 0: the plain mean of the keys seen."""
    Batch([q], [700], 4, 2, 128, 64, dtype, seed=3, qscale=3.0).check(scale=scale)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("q", [1, 150])
def test_scores_that_rise_along_the_keys(dtype, q):
    """Every key tile raises the maximum, by little and by much: the running sums are rescaled each time."""
    b = Batch([q], [900], 2, 2, 64, 16, dtype, seed=4)
    b.q.fill_(1.0)
    ramp = torch.arange(900, device="cuda")[:, None, None].double() / 900 * torch.tensor([2.0, 12.0], device="cuda").double()[:, None]
    b.k[0].copy_(ramp.expand(900, 2, 64))
    for p in range(-(-900 // 16)):
        m = min(16, 900 - 16 * p)
        b.kc[int(b.table[0, p]), :, :m] = b.k[0][16 * p:16 * p + m].transpose(0, 1)
    b.check()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("q", [1, 64])
def test_lowest_values_and_infinite_rows_of_other_sequences(dtype, q):
    """A sequence whose keys hold the type's lowest value and one with infinite values leave their neighbour alone."""
    b = Batch([q, q, q], [100, 130, 100], 4, 2, 64, 16, dtype, seed=5)
    low = torch.finfo(dtype).min
    b.kc[b.table[0, :6].long()] = low
    b.vc[b.table[2, :6].long()] = float("inf")
    got = b.call()
    out, bound = b.want()
    mid = slice(q, 2 * q)
    assert ((got.double() - out).abs() - bound)[mid].max().item() <= 0


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("q", [1, 33])
def test_a_cache_past_32_bit_offsets(dtype, q):
    """Pages beyond 2^31 elements (and 4 GB) into the cache: two heads of it are real, the pool is one large buffer."""
    if torch.cuda.mem_get_info()[0] < 40 << 30:
        pytest.skip("needs 40 GB of free device memory")
    b = Batch([q], [500], 4, 2, 128, 16, dtype, seed=6)
    pages = (1 << 31) // (2 * 16 * 128) + 1000
    big = [torch.empty(pages, 2, 16, 128, device="cuda", dtype=dtype) for _ in range(2)]
    ids = torch.arange(pages - 32, pages, device="cuda")
    for x, small in zip(big, (b.kc, b.vc)):
        x[ids] = small[b.table[0, :32].long()]
    b.kc, b.vc = big
    b.table[0, :32] = ids.int()
    b.check()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("q", [1, 6, 90])
def test_same_bits_every_time_with_any_workspace(dtype, q):
    """No atomics in the sums: two calls give the same bits, whatever the workspace held."""
    b = Batch([q] * 3, [2000, 31 + q, 700], 28, 4, 128, 64, dtype, seed=7)
    first = b.call()
    need = _lib.load().spruce_paged_attention_workspace_bytes(28, 4, 128, q, _lib.DTYPE_CODE[dtype])
    ws = torch.full((need,), 255, device="cuda", dtype=torch.uint8)
    for _ in range(3):
        assert torch.equal(b.call(workspace=ws), first)


@pytest.mark.parametrize("q", [1, 90])
def test_bounds_above_the_lengths_and_idle_tails(q):
    """max_q_len and max_kv_len are bounds; tokens past cu_q[-1] are not written; no sequence or token is fine."""
    b = Batch([q, 1], [500, 3], 4, 2, 64, 16, torch.bfloat16, seed=8)
    b.check(max_q_len=5 * q + 7, max_kv_len=100000)
    b.q = torch.cat([b.q, b.q[:3]])
    out = torch.full_like(b.q, 5.0)
    b.call(out=out)
    assert (out[q + 1:] == 5).all()
    none = native.paged_attention(b.q[:0], b.kc, b.vc, b.table[:0], b.cu[:1], b.kv[:0], max_q_len=0, max_kv_len=0)
    assert none.shape == (0, 4, 64)


@pytest.mark.parametrize("q", [1, 90])
def test_lengths_and_pages_out_of_bounds_set_the_status(q):
    """Lengths are cut to the bounds and bad page ids read zeros: reported, and nothing outside is touched."""
    b = Batch([q], [300], 4, 2, 64, 16, torch.bfloat16, seed=9)
    status = torch.zeros(1, device="cuda", dtype=torch.int32)
    b.call(max_kv_len=200, status=status)
    assert status.item() == _lib.STATUS_BAD_LENGTH
    if q > 1:
        status.zero_()
        b.call(max_q_len=q - 1, status=status)
        assert status.item() == _lib.STATUS_BAD_LENGTH
    for bad in (-1, b.kc.shape[0]):
        status.zero_()
        b.table[0, 3] = bad
        b.call(status=status)
        assert status.item() == _lib.STATUS_BAD_PAGE


def test_another_stream_and_a_graph():
    """A call belongs to the current stream, and a captured one follows lengths that change between replays."""
    b = Batch([1, 1], [100, 800], 28, 4, 128, 64, torch.bfloat16, seed=10)
    want = b.check()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = b.call()
        out = torch.empty_like(got)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            b.call(out=out)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)
    graph.replay()
    assert torch.equal(out, want)
    # after a copy and after an append, eager and captured: an attention that starts early still waits for them
    fresh = b.q.clone()
    k, v = torch.zeros(2, 4, 128, device="cuda", dtype=torch.bfloat16), torch.zeros(2, 4, 128, device="cuda", dtype=torch.bfloat16)
    last = [(b.kc[p, :, r].clone(), b.vc[p, :, r].clone()) for p, r in ((b.table[0, 1], 35), (b.table[1, 12], 31))]
    k.copy_(torch.stack([x[0] for x in last]))
    v.copy_(torch.stack([x[1] for x in last]))
    torch.cuda.synchronize()
    chain = torch.cuda.CUDAGraph()
    with torch.cuda.graph(chain):
        b.q.copy_(fresh)
        native.paged_append(k, v, b.kc, b.vc, b.table, b.cu, b.kv)
        b.call(out=out)
    for run in (chain.replay, lambda: (b.q.copy_(fresh), native.paged_append(k, v, b.kc, b.vc, b.table, b.cu, b.kv), b.call(out=out))):
        for _ in range(20):
            b.q.zero_()
            b.kc[b.table[0, 1], :, 35] = 0
            run()
            assert torch.equal(out, want)
    b.kvs = [37, 700]
    b.kv.copy_(torch.tensor(b.kvs))
    graph.replay()
    b.k, b.v = [x[:n] for x, n in zip(b.k, b.kvs)], [x[:n] for x, n in zip(b.v, b.kvs)]
    want, bound = b.want()
    assert ((out.double() - want).abs() - bound).max().item() <= 0


def test_refusals():
    b = Batch([2], [20], 4, 2, 64, 16, torch.bfloat16)
    call = dict(max_q_len=2, max_kv_len=20)
    with pytest.raises(ValueError, match="divisible by KV heads|bad paged attention shape"):
        native.paged_attention(b.q[:, :3], b.kc, b.vc, b.table, b.cu, b.kv, **call)
    with pytest.raises(ValueError, match="q must be"):
        native.paged_attention(b.q[..., :32], b.kc, b.vc, b.table, b.cu, b.kv, **call)
    with pytest.raises(ValueError, match="bad paged attention shape"):
        native.paged_attention(b.q[..., :32], b.kc[..., :32], b.vc[..., :32], b.table, b.cu, b.kv, **call)
    with pytest.raises(ValueError, match="page_size"):
        native.paged_attention(b.q, b.kc[:, :, :8], b.vc[:, :, :8], b.table, b.cu, b.kv, **call)
    with pytest.raises(ValueError, match="16-byte aligned"):
        odd = torch.zeros(b.kc.numel() + 8, device="cuda", dtype=torch.bfloat16)[1:1 + b.kc.numel()].view_as(b.kc)
        native.paged_attention(b.q, odd, b.vc, b.table, b.cu, b.kv, **call)
    with pytest.raises(ValueError, match="positive"):
        flat = b.kc[:, :1].expand(-1, 2, -1, -1)
        native.paged_attention(b.q, flat, flat, b.table, b.cu, b.kv, **call)
    with pytest.raises(ValueError, match="new tokens' dtype"):
        native.paged_attention(b.q.half(), b.kc, b.vc, b.table, b.cu, b.kv, **call)
    with pytest.raises(ValueError, match="int32"):
        native.paged_attention(b.q, b.kc, b.vc, b.table, b.cu.long(), b.kv, **call)
    with pytest.raises(ValueError, match="negative|bad paged attention shape"):
        native.paged_attention(b.q, b.kc, b.vc, b.table, b.cu, b.kv, max_q_len=-1, max_kv_len=20)
    with pytest.raises(ValueError, match="out must be"):
        native.paged_attention(b.q, b.kc, b.vc, b.table, b.cu, b.kv, out=b.q.float(), **call)
    with pytest.raises(RuntimeError, match="workspace"):
        native.paged_attention(b.q, b.kc, b.vc, b.table, b.cu, b.kv, workspace=b.q[:1].view(torch.uint8), **call)
    with pytest.raises(RuntimeError, match="CUDA"):
        native.paged_attention(b.q, b.kc, b.vc, b.table, b.cu.cpu(), b.kv, **call)
