// Eviction from a paged cache by weight: per (sequence, KV head) the first `sinks` slots, the last `recent` ones and the
// heaviest of those between stay, `keep` in all, and move in their order to slots 0 .. keep - 1.
//
// Selection: a cluster of CTAs a (sequence, head), a piece of its slots each, whose weights they read once and keep in shared
// memory as integers of the same order.  A radix select over 11, 11 and 10 bits, the CTAs' histograms read by all of them,
// finds the weight of the last one kept and how many of its equals stay (the lowest slots); the kept slots are then
// written in order, each warp's at a place that the counts before it give.
//
// Moving in place: slot j takes row kept[j] >= j, so going up in j a row is read before it is written over, if
// all rows of a round are read before any is written: one barrier a round.  Rows are cut into slices of columns, which
// never touch each other, so a (sequence, head) is spread over many CTAs that need not wait for one another.  Into other
// pages there is nothing to wait for: a warp takes 32 whole rows.
//
// On a B200 (4 KV heads of 128, bf16): one sequence of 131072 tokens cut to 16384 36 us, of which the selection, a chain of twelve
// cluster barriers (three a pass, three around them), takes about 20; 64 sequences of 300 to 8192 tokens cut to 2048 101 us, 82 of them the copy (5.9 TB/s).  In place
// 84 to 87 and 172 to 175 us: rounds of short pieces of scattered rows.
#include <algorithm>

#include "mass_common.cuh"

namespace spruce {

// Order of the weights as unsigned integers; NaN above all, -0 as +0.  kAlways, above that, is a slot that stays anyway.
constexpr uint32_t kAlways = 0xffffffffu, kNan = 0xfffffffeu;
__device__ __forceinline__ uint32_t weight_key(float w) {
  if (w != w) return kNan;
  const uint32_t b = __float_as_uint(w + 0.0f);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}

// n / page_size for 0 <= n < 2^31 by a product: exact, as d - 1 <= 2^l - 1 bounds the rounding of 2^(31 + l) / d.
struct PageDiv {
  uint32_t mul;
  int shift, size;
  __device__ __forceinline__ int page(int n) const {
    return static_cast<int>((static_cast<uint64_t>(static_cast<uint32_t>(n)) * mul) >> shift);
  }
};
static PageDiv page_div(int size) {
  PageDiv d;
  int l = 0;
  while ((int64_t(1) << l) < size) ++l;
  d.shift = 31 + l;
  d.mul = static_cast<uint32_t>(((uint64_t(1) << d.shift) + size - 1) / size);
  d.size = size;
  return d;
}

struct EvictSeq {
  int kv, keep;        // slots held and kept
  int sinks, tail;     // slots [0, sinks) and [tail, kv) always stay
};
__device__ __forceinline__ EvictSeq evict_seq(const EvictArgs& a, int s, bool report) {
  const int held = a.kv_lens[s];
  EvictSeq q;
  q.kv = held;
  if (held < 0 || held > a.cap) {  // left as it is
    if (report) raise_status(a.status, SPRUCE_STATUS_BAD_LENGTH);
    q.kv = 0;
  }
  q.keep = min(q.kv, a.keep);
  q.sinks = min(a.sinks, q.keep);
  q.tail = q.kv - min(a.recent, q.keep - q.sinks);
  return q;
}
__device__ __forceinline__ int evict_page(const int32_t* table, int index, int64_t pages, uint32_t* status) {
  const int page = table[index];
  if (page >= 0 && page < pages) return page;
  raise_status(status, SPRUCE_STATUS_BAD_PAGE);
  return -1;
}

// 256 threads measured 41 us and 1024 as much as 512 for one long sequence, 110 and 105 against 101 us for 64 (with the copies).
constexpr int kSelectThreads = 512, kSelectWarps = kSelectThreads / 32;
constexpr int kSelectBins = 2048, kSelectMostCtas = 16;
constexpr int kSelectCached = 48 * 1024;  // slots of a CTA whose weights fit in shared memory; longer pieces are read again

__device__ __forceinline__ uint32_t at_cta(const int* p, int cta) {
  uint32_t at;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(smem_u32(p)), "r"(cta));
  return at;
}
__device__ __forceinline__ int remote_int(const int* p, int cta) {
  int v;
  asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(v) : "r"(at_cta(p, cta)) : "memory");
  return v;
}
__device__ __forceinline__ void remote_store(int* p, int cta, int v) {
  asm volatile("st.shared::cluster.s32 [%0], %1;" ::"r"(at_cta(p, cta)), "r"(v) : "memory");
}
// All threads of the CTAs that share a head.
__device__ __forceinline__ void together(int ctas) {
  if (ctas > 1)
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
  else
    __syncthreads();
}

__global__ void __launch_bounds__(kSelectThreads, 2)
    evict_select_kernel(const EvictArgs a, const PageDiv pd, int ctas, int cached, bool vec) {
  extern __shared__ __align__(16) uint32_t keys[];  // [cached, to a multiple of 4]
  __shared__ int hist[kSelectBins];
  __shared__ int shares[kSelectMostCtas];
  __shared__ int sums[2][kSelectWarps];
  __shared__ int found[2];               // digit of the last one kept, and how many are left to take within it
  __shared__ int counts[2];              // of this CTA: above the last weight (or always kept), and equal to it
  const int sg = blockIdx.x / ctas, rank = blockIdx.x % ctas;
  const int s = sg / a.Hkv, g = sg % a.Hkv;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  for (int b = tid; b < kSelectBins; b += kSelectThreads) hist[b] = 0;
  let_next_kernel_start();
  wait_for_earlier_kernels();
  const EvictSeq q = evict_seq(a, s, g == 0 && rank == 0 && tid == 0);
  int32_t* kept = a.kept + (int64_t)sg * a.width;
  if (g == 0 && rank == 0 && tid == 0) a.new_lens[s] = q.kv == 0 ? a.kv_lens[s] : q.keep;
  for (int j = q.keep + rank * kSelectThreads + tid; j < a.width; j += ctas * kSelectThreads) kept[j] = -1;
  if (q.keep == q.kv) {  // of all CTAs of the head
    for (int j = rank * kSelectThreads + tid; j < q.keep; j += ctas * kSelectThreads) kept[j] = j;
    return;
  }
  // This CTA's slots.
  const int each = ((q.kv + ctas - 1) / ctas + 31) / 32 * 32;
  const int begin = min(rank * each, q.kv), n = min(each, q.kv - begin);
  const int32_t* table = a.table + s * a.table_stride;
  auto key = [&](int j, float w) { return j < q.sinks || j >= q.tail ? kAlways : weight_key(w); };
  auto read = [&](int j) {
    const int pi = pd.page(j), page = evict_page(table, pi, a.num_pages, a.status);
    return key(j, page < 0 ? 0.0f : a.mass[page * a.ms[0] + g * a.ms[1] + (j - pi * pd.size) * a.ms[2]]);
  };
  auto count = [&](int* h, uint32_t k, int digit) {
    if (k != kAlways) atomicAdd(&h[digit], 1);
  };
  together(ctas);  // the histograms are empty
  if (vec && n <= cached) {  // four slots a load; they lie in one page, and `begin` is a multiple of 32
#pragma unroll 4
    for (int i = 4 * tid; i < n; i += 4 * kSelectThreads) {
      const int j = begin + i, pi = pd.page(j), page = evict_page(table, pi, a.num_pages, a.status);
      float4 w = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      if (page >= 0) w = *reinterpret_cast<const float4*>(a.mass + page * a.ms[0] + g * a.ms[1] + (j - pi * pd.size));
      const uint4 k = make_uint4(key(j, w.x), key(j + 1, w.y), key(j + 2, w.z), key(j + 3, w.w));
      *reinterpret_cast<uint4*>(keys + i) = k;  // past the sequence's slots: those of the tail, kAlways
      count(hist, k.x, k.x >> 21);
      count(hist, k.y, k.y >> 21);
      count(hist, k.z, k.z >> 21);
      count(hist, k.w, k.w >> 21);
    }
  } else {
#pragma unroll 4
    for (int i = tid; i < n; i += kSelectThreads) {
      const uint32_t k = read(begin + i);
      if (i < cached) keys[i] = k;
      count(hist, k, k >> 21);
    }
    if (tid < 4 && n + tid < cached) keys[n + tid] = kAlways;
  }
  int left = q.keep - q.sinks - (q.kv - q.tail);  // to be taken between sinks and tail
  uint32_t prefix = left > 0 ? 0u : kNan, mask = 0;
#pragma unroll
  for (int pass = 0; pass < 3; ++pass) {
    const int shift = pass == 0 ? 21 : (pass == 1 ? 10 : 0), bins = pass == 2 ? 1024 : 2048;
    if (pass > 0 && left > 0) {
      auto look = [&](uint32_t k) {
        if ((k & mask) == prefix) count(hist, k, (k >> shift) & (bins - 1));
      };
      const int there = min(n, cached);
      for (int i = 4 * tid; i < there; i += 4 * kSelectThreads) {
        const uint4 k = *reinterpret_cast<const uint4*>(keys + i);
        look(k.x);
        if (i + 1 < there) look(k.y);
        if (i + 2 < there) look(k.z);
        if (i + 3 < there) look(k.w);
      }
      for (int i = cached + tid; i < n; i += kSelectThreads) look(read(begin + i));
    }
    together(ctas);
    // Bins from the highest down.  A CTA adds up an equal share of them over all CTAs; the shares' sums tell every CTA whose share
    // holds the last one kept, and that one finds it.  (All CTAs reading one CTA's totals took four times as long.)
    const int share = bins / ctas, top = bins - 1 - rank * share;
    const int bins_of = max(1, share / kSelectThreads);  // bins of a thread: 1, 2 or 4
    int c[4] = {0, 0, 0, 0}, inc = 0;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int b = bins_of * tid + k;
      if (k < bins_of && b < share) {
        if (ctas == 1) {
          c[k] = hist[top - b];
        } else {
#pragma unroll 16
          for (int x = 0; x < kSelectMostCtas; ++x)
            if (x < ctas) c[k] += remote_int(&hist[top - b], x);
        }
      }
      inc += c[k];
    }
    int before = -inc;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += y;
    }
    if (lane == 31) sums[0][warp] = inc;
    __syncthreads();
    before += inc + __reduce_add_sync(0xffffffffu, lane < warp ? sums[0][lane] : 0);
    bool here = true;
    if (ctas > 1) {
      const int all = __reduce_add_sync(0xffffffffu, lane < kSelectWarps ? sums[0][lane] : 0);
      if (warp == 0 && lane < ctas) remote_store(&shares[rank], lane, all);
      together(ctas);
      const int higher = __reduce_add_sync(0xffffffffu, lane < rank ? shares[lane] : 0);
      before += higher;
      here = higher < left && left <= higher + all;
    }
    if (left > 0 && here) {  // one thread of the head finds it
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        if (before < left && left <= before + c[k])
          for (int x = 0; x < ctas; ++x) {
            remote_store(&found[0], x, top - bins_of * tid - k);
            remote_store(&found[1], x, left - before);
          }
        before += c[k];
      }
    }
    for (int b = tid; b < kSelectBins; b += kSelectThreads) hist[b] = 0;
    together(ctas);
    if (left > 0) {
      prefix |= static_cast<uint32_t>(found[0]) << shift;
      left = found[1];
      mask |= static_cast<uint32_t>(bins - 1) << shift;
    }
  }
  // All above `prefix` stay and, of its equals, the first `left`.  128 slots a warp and step, four a lane.
  const int per = (n + kSelectWarps * 128 - 1) / (kSelectWarps * 128) * 128, w0 = min(warp * per, n), w1 = min(w0 + per, n);
  auto four = [&](int i) {
    uint4 k = make_uint4(0, 0, 0, 0);  // below all: neither above nor, as `prefix` is at least that of -inf, equal
    if (i + 3 < min(w1, cached)) {
      k = *reinterpret_cast<const uint4*>(keys + i);
    } else {
      if (i < w1) k.x = i < cached ? keys[i] : read(begin + i);
      if (i + 1 < w1) k.y = i + 1 < cached ? keys[i + 1] : read(begin + i + 1);
      if (i + 2 < w1) k.z = i + 2 < cached ? keys[i + 2] : read(begin + i + 2);
      if (i + 3 < w1) k.w = i + 3 < cached ? keys[i + 3] : read(begin + i + 3);
    }
    return k;
  };
  auto above = [&](const uint4& k) { return (k.x > prefix) + (k.y > prefix) + (k.z > prefix) + (k.w > prefix); };
  auto equal = [&](const uint4& k) { return (k.x == prefix) + (k.y == prefix) + (k.z == prefix) + (k.w == prefix); };
  int ups = 0, eqs = 0;
  for (int i = w0; i < w1; i += 128) {
    const uint4 k = four(i + 4 * lane);
    ups += above(k);
    eqs += equal(k);
  }
  ups = __reduce_add_sync(0xffffffffu, ups);
  eqs = __reduce_add_sync(0xffffffffu, eqs);
  if (lane == 0) {
    sums[0][warp] = ups;
    sums[1][warp] = eqs;
  }
  __syncthreads();
  {
    const int u = lane < kSelectWarps ? sums[0][lane] : 0, e = lane < kSelectWarps ? sums[1][lane] : 0;
    ups = __reduce_add_sync(0xffffffffu, lane < warp ? u : 0);
    eqs = __reduce_add_sync(0xffffffffu, lane < warp ? e : 0);
    if (ctas > 1) {
      const int all_u = __reduce_add_sync(0xffffffffu, u), all_e = __reduce_add_sync(0xffffffffu, e);
      if (tid == 0) {
        counts[0] = all_u;
        counts[1] = all_e;
      }
      together(ctas);
      const bool before = lane < rank;
      ups += __reduce_add_sync(0xffffffffu, before ? remote_int(&counts[0], lane) : 0);
      eqs += __reduce_add_sync(0xffffffffu, before ? remote_int(&counts[1], lane) : 0);
    }
  }
  for (int i = w0; i < w1; i += 128) {
    const uint4 k = four(i + 4 * lane);
    // Both counts in one scan: a step has at most 128 of each.
    const int mine = above(k) | equal(k) << 16;
    int inc = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += y;
    }
    const int all = __shfl_sync(0xffffffffu, inc, 31);
    int up = ups + ((inc - mine) & 0xffff), eq = eqs + ((inc - mine) >> 16);
    auto put = [&](uint32_t x, int j) {
      if (x > prefix) {
        kept[up + min(eq, left)] = j;
        ++up;
      } else if (x == prefix) {
        if (eq < left) kept[up + eq] = j;
        ++eq;
      }
    };
    const int j = begin + i + 4 * lane;
    put(k.x, j);
    put(k.y, j + 1);
    put(k.z, j + 2);
    put(k.w, j + 3);
    ups += all & 0xffff;
    eqs += all >> 16;
  }
  if (ctas > 1) together(ctas);  // the others read this CTA's shared memory
}

// In place: a CTA takes a slice of the columns of all rows, so that the rows' order is its own affair.  A round is kMoveRows rows a
// thread; the places of the next are looked up while this one's rows are on their way.
constexpr int kMoveThreads = 1024, kMoveRows = 4;
constexpr int kMoveSlice = 32;  // bytes of a row that a CTA takes, twice that where there are more CTAs than the GPU holds

template <typename V>
__device__ __forceinline__ void move_rows(const EvictArgs& a, const PageDiv& pd, const EvictSeq& q, int s, int g, char* data,
                                          const int64_t* st, int es, int lanes, int at) {
  const int32_t* kept = a.kept + ((int64_t)s * a.Hkv + g) * a.width;
  const int32_t* table = a.table + s * a.table_stride;
  const int r = threadIdx.x / lanes, c = threadIdx.x % lanes, per = kMoveThreads / lanes;
  data += g * st[1] * es + at + c * sizeof(V);
  int64_t from[kMoveRows], to[kMoveRows];  // -1: nothing to move
  auto look = [&](int base) {
    int src[kMoveRows];
#pragma unroll
    for (int u = 0; u < kMoveRows; ++u) {
      const int j = base + u * per + r;
      src[u] = j < q.keep ? kept[j] : -1;
    }
#pragma unroll
    for (int u = 0; u < kMoveRows; ++u) {
      const int j = base + u * per + r;
      from[u] = -1;
      if (src[u] < 0 || src[u] >= q.kv || src[u] == j) continue;
      const int i0 = pd.page(src[u]), i1 = pd.page(j);
      const int p0 = evict_page(table, i0, a.num_pages, a.status), p1 = evict_page(table, i1, a.num_pages, a.status);
      if (p0 < 0 || p1 < 0) continue;
      from[u] = (p0 * st[0] + (src[u] - i0 * pd.size) * st[2]) * es;
      to[u] = (p1 * st[0] + (j - i1 * pd.size) * st[2]) * es;
    }
  };
  look(0);
  for (int base = 0; base < q.keep; base += per * kMoveRows) {
    V v[kMoveRows];
    V* dst[kMoveRows];
#pragma unroll
    for (int u = 0; u < kMoveRows; ++u) {
      dst[u] = nullptr;
      if (from[u] < 0) continue;
      v[u] = *reinterpret_cast<const V*>(data + from[u]);
      dst[u] = reinterpret_cast<V*>(data + to[u]);
    }
    look(base + per * kMoveRows);
    __syncthreads();
#pragma unroll
    for (int u = 0; u < kMoveRows; ++u)
      if (dst[u] != nullptr) *dst[u] = v[u];
  }
}

// Blocks of a (sequence, head): `slices` of K, as many of V, and one of the weights.
__global__ void __launch_bounds__(kMoveThreads) evict_move_kernel(const EvictArgs a, const PageDiv pd, int slices, int lanes) {
  const int blocks = 2 * slices + 1, x = blockIdx.x % blocks;
  const int sg = blockIdx.x / blocks, s = sg / a.Hkv, g = sg % a.Hkv;
  let_next_kernel_start();
  wait_for_earlier_kernels();
  const EvictSeq q = evict_seq(a, s, false);
  if (q.keep == q.kv) return;
  const int at = x % slices * lanes * 16;
  if (x == 2 * slices)
    move_rows<float>(a, pd, q, s, g, reinterpret_cast<char*>(a.mass_out), a.ms, 4, 1, 0);
  else if (x < slices)
    move_rows<uint4>(a, pd, q, s, g, static_cast<char*>(a.k_out), a.ks, a.es, lanes, at);
  else
    move_rows<uint4>(a, pd, q, s, g, static_cast<char*>(a.v_out), a.vs, a.es, lanes, at);
}

// Into other pages: a warp takes 32 rows of a (sequence, head).  Each lane looks up the places of one, then all copy K and V
// rows 16 bytes a lane, eight loads in flight.
constexpr int kCopyThreads = 256, kCopyRows = 32, kCopyFlight = 8;

__global__ void __launch_bounds__(kCopyThreads) evict_copy_kernel(const EvictArgs a, const PageDiv pd, const PageDiv vecs, int chunks) {
  const int lane = threadIdx.x & 31;
  const int64_t at = (int64_t)blockIdx.x * (kCopyThreads / 32) + threadIdx.x / 32;
  let_next_kernel_start();
  wait_for_earlier_kernels();
  const int64_t sg = at / chunks;
  if (sg >= (int64_t)a.S * a.Hkv) return;
  const int s = static_cast<int>(sg / a.Hkv), g = static_cast<int>(sg % a.Hkv), j0 = static_cast<int>(at % chunks) * kCopyRows;
  const EvictSeq q = evict_seq(a, s, false);
  const int n = min(kCopyRows, q.keep - j0);
  if (n <= 0) return;
  // Places of this lane's row: pages and rows of them; -1: no such page.
  int p0 = -1, p1 = -1, r0 = 0, r1 = 0;
  if (lane < n) {
    const int src = a.kept[sg * a.width + j0 + lane];
    if (src >= 0 && src < q.kv) {
      const int i0 = pd.page(src), i1 = pd.page(j0 + lane);
      r0 = src - i0 * pd.size;
      r1 = j0 + lane - i1 * pd.size;
      p0 = evict_page(a.table + s * a.table_stride, i0, a.num_pages, a.status);
      p1 = evict_page(a.to_table + s * a.to_table_stride, i1, a.to_pages, a.status);
    }
  }
  const bool ok = p0 >= 0 && p1 >= 0;
  if (ok) a.mass_out[p1 * a.mos[0] + g * a.mos[1] + r1 * a.mos[2]] = a.mass[p0 * a.ms[0] + g * a.ms[1] + r0 * a.ms[2]];
  const unsigned rows_ok = __ballot_sync(0xffffffffu, ok);
#pragma unroll
  for (int kv = 0; kv < 2; ++kv) {
    const int64_t* fs = kv == 0 ? a.ks : a.vs;
    const int64_t* ts = kv == 0 ? a.kos : a.vos;
    const char* from = static_cast<const char*>(kv == 0 ? a.k : a.v) + g * fs[1] * a.es;
    char* to = static_cast<char*>(kv == 0 ? a.k_out : a.v_out) + g * ts[1] * a.es;
    const int64_t f = (p0 * fs[0] + r0 * fs[2]) * a.es, t = (p1 * ts[0] + r1 * ts[2]) * a.es;
    const int total = n * vecs.size;  // 16-byte pieces
    for (int i0 = 0; i0 < total; i0 += 32 * kCopyFlight) {
      uint4 v[kCopyFlight];
      char* dst[kCopyFlight];
#pragma unroll
      for (int u = 0; u < kCopyFlight; ++u) {
        const int i = i0 + 32 * u + lane, row = vecs.page(min(i, total - 1));
        const int64_t fr = __shfl_sync(0xffffffffu, f, row), tr = __shfl_sync(0xffffffffu, t, row);
        dst[u] = nullptr;
        if (i >= total || !(rows_ok >> row & 1)) continue;
        const int c = (i - row * vecs.size) * 16;
        v[u] = __ldcs(reinterpret_cast<const uint4*>(from + fr + c));
        dst[u] = to + tr + c;
      }
#pragma unroll
      for (int u = 0; u < kCopyFlight; ++u)
        if (dst[u] != nullptr) *reinterpret_cast<uint4*>(dst[u]) = v[u];
    }
  }
}

cudaError_t launch_evict(const EvictArgs& a, cudaStream_t stream) {
  const int64_t heads = (int64_t)a.S * a.Hkv;
  // CTAs of a head: as many as the GPU has room for, while each gets 2048 slots of the longest sequence allowed.
  int ctas = 1;
  while (ctas < kSelectMostCtas && heads * ctas * 2 <= sm_count() && a.cap / (ctas * 2) >= 2048) ctas *= 2;
  const int each = ((a.cap + ctas - 1) / ctas + 31) / 32 * 32, cached = std::min(each, kSelectCached);  // a multiple of 4
  static std::atomic<uint64_t> done{0};
  cudaError_t e = allow_smem(reinterpret_cast<const void*>(evict_select_kernel), kSelectCached * 4, done);
  if (e == cudaSuccess && ctas > 8)
    e = cudaFuncSetAttribute(evict_select_kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg{};
  cudaLaunchAttribute attr[2]{};
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = ctas;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.gridDim = dim3(static_cast<unsigned>(heads * ctas));
  cfg.blockDim = dim3(kSelectThreads);
  cfg.dynamicSmemBytes = cached * 4;
  cfg.stream = stream;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  const bool vec = a.ms[2] == 1 && a.ms[0] % 4 == 0 && a.ms[1] % 4 == 0 && (reinterpret_cast<uintptr_t>(a.mass) & 15u) == 0;
  const PageDiv pd = page_div(a.page_size);
  e = cudaLaunchKernelEx(&cfg, evict_select_kernel, a, pd, ctas, cached, vec);
  const int most = std::min(a.keep, a.cap);  // rows that a head keeps
  if (e != cudaSuccess || most == 0) return e;
  const int row = a.D * a.es;
  if (a.in_place) {
    // 256 threads of 8 rows, 32 bytes: 110 us for one sequence of 131072 tokens cut to 16384, 272 for 64 cut to 2048; 1024 threads of
    // 4 rows 87 and 213; 64 bytes 109 and 174.
    int slice = row % kMoveSlice == 0 ? kMoveSlice : 16;
    if (row % (2 * slice) == 0 && heads * (2 * (row / slice) + 1) > 2 * sm_count()) slice *= 2;
    return launch_early(evict_move_kernel, static_cast<int>(heads * (2 * (row / slice) + 1)), kMoveThreads, 0, stream, a, pd,
                        row / slice, slice / 16);
  }
  const int chunks = (most + kCopyRows - 1) / kCopyRows;
  const int64_t blocks = (heads * chunks + kCopyThreads / 32 - 1) / (kCopyThreads / 32);
  if (blocks > INT32_MAX) return cudaErrorInvalidConfiguration;
  return launch_early(evict_copy_kernel, static_cast<int>(blocks), kCopyThreads, 0, stream, a, pd, page_div(row / 16), chunks);
}

}  // namespace spruce
