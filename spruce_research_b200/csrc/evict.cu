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
// pages there is nothing to wait for: a CTA takes 128 whole rows.
#include <algorithm>

#include "mass_common.cuh"

namespace spruce {

// Order of the weights as unsigned integers; NaN above all, -0 as +0.
__device__ __forceinline__ uint32_t weight_key(float w) {
  if (w != w) return 0xffffffffu;
  const uint32_t b = __float_as_uint(w + 0.0f);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
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

constexpr int kSelectThreads = 1024, kSelectWarps = kSelectThreads / 32;
constexpr int kSelectBins = 2048, kSelectMostCtas = 8;
constexpr int kSelectCached = 48 * 1024;  // slots of a CTA whose weights fit in shared memory; longer pieces are read again

__device__ __forceinline__ int remote_int(const int* p, int cta) {
  uint32_t at;
  int v;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(smem_u32(p)), "r"(cta));
  asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(v) : "r"(at) : "memory");
  return v;
}
// All threads of the CTAs that share a head.
__device__ __forceinline__ void together(int ctas) {
  if (ctas > 1)
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
  else
    __syncthreads();
}

__global__ void __launch_bounds__(kSelectThreads, 1) evict_select_kernel(const EvictArgs a, int ctas, int cached) {
  extern __shared__ uint32_t keys[];  // [cached]
  __shared__ int hist[2][kSelectBins];
  __shared__ int sums[2][kSelectWarps];
  __shared__ int found[2];            // digit of the last one kept, and how many are left to take within it
  __shared__ int counts[2];           // of this CTA: above the last weight (or always kept), and equal to it
  const int sg = blockIdx.x / ctas, rank = blockIdx.x % ctas;
  const int s = sg / a.Hkv, g = sg % a.Hkv;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
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
  // This CTA's slots, a whole number of warps' steps.
  const int each = ((q.kv + ctas - 1) / ctas + 31) / 32 * 32;
  const int begin = min(rank * each, q.kv), n = min(each, q.kv - begin);
  const int32_t* table = a.table + s * a.table_stride;
  auto read = [&](int j) {
    const int page = evict_page(table, j / a.page_size, a.num_pages, a.status);
    return weight_key(page < 0 ? 0.0f : a.mass[page * a.ms[0] + g * a.ms[1] + j % a.page_size * a.ms[2]]);
  };
  auto key_of = [&](int i) { return i < cached ? keys[i] : read(begin + i); };
  auto always = [&](int j) { return j < q.sinks || j >= q.tail; };
  for (int b = tid; b < kSelectBins; b += kSelectThreads) hist[0][b] = 0;
  __syncthreads();
  int left = q.keep - q.sinks - (q.kv - q.tail);  // to be taken between sinks and tail
  uint32_t prefix = 0, mask = 0;
#pragma unroll
  for (int pass = 0; pass < 3; ++pass) {
    const int shift = pass == 0 ? 21 : (pass == 1 ? 10 : 0), bins = pass == 2 ? 1024 : 2048;
    int* const h = hist[pass & 1];
    if (pass == 0) {
#pragma unroll 4
      for (int i = tid; i < n; i += kSelectThreads) {
        const uint32_t k = read(begin + i);
        if (i < cached) keys[i] = k;
        if (!always(begin + i)) atomicAdd(&h[k >> 21], 1);
      }
    } else {
      for (int i = tid; i < n; i += kSelectThreads) {
        const uint32_t k = key_of(i);
        if ((k & mask) == prefix && !always(begin + i)) atomicAdd(&h[(k >> shift) & (bins - 1)], 1);
      }
    }
    together(ctas);
    // The other buffer was read by all before they came here.
    for (int b = tid; b < kSelectBins; b += kSelectThreads) hist[(pass + 1) & 1][b] = 0;
    // Bins from the highest down, two a thread.
    const int hi = bins - 1 - 2 * tid;
    int c0 = 0, c1 = 0;
    if (hi > 0) {
      if (ctas == 1) {
        c0 = h[hi];
        c1 = h[hi - 1];
      } else {
        for (int c = 0; c < ctas; ++c) {
          c0 += remote_int(&h[hi], c);
          c1 += remote_int(&h[hi - 1], c);
        }
      }
    }
    int inc = c0 + c1;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += y;
    }
    if (lane == 31) sums[0][warp] = inc;
    __syncthreads();
    int before = inc - c0 - c1;
    for (int w = 0; w < warp; ++w) before += sums[0][w];
    if (left > 0 && hi > 0) {  // one thread of the block finds it
      if (before < left && left <= before + c0) {
        found[0] = hi;
        found[1] = left - before;
      } else if (before + c0 < left && left <= before + c0 + c1) {
        found[0] = hi - 1;
        found[1] = left - before - c0;
      }
    }
    __syncthreads();
    if (left > 0) {
      prefix |= static_cast<uint32_t>(found[0]) << shift;
      left = found[1];
      mask |= static_cast<uint32_t>(bins - 1) << shift;
    }
  }
  // `left` slots of exactly the weight `prefix` stay, and all above it; none between sinks and tail where none is to be taken.
  const bool any = mask != 0;
  const int per = (n + kSelectWarps * 32 - 1) / (kSelectWarps * 32) * 32, w0 = min(warp * per, n), w1 = min(w0 + per, n);
  auto look = [&](int i, unsigned& above, unsigned& equal) {  // of 32 slots
    bool up = false, eq = false;
    if (i < w1) {
      const int j = begin + i;
      up = always(j);
      if (!up && any) {
        const uint32_t k = key_of(i);
        up = k > prefix;
        eq = k == prefix;
      }
    }
    above = __ballot_sync(0xffffffffu, up);
    equal = __ballot_sync(0xffffffffu, eq);
  };
  int ups = 0, eqs = 0;
  for (int i = w0; i < w1; i += 32) {
    unsigned above, equal;
    look(i + lane, above, equal);
    ups += __popc(above);
    eqs += __popc(equal);
  }
  if (lane == 0) {
    sums[0][warp] = ups;
    sums[1][warp] = eqs;
  }
  __syncthreads();
  int up0 = 0, eq0 = 0;
  for (int w = 0; w < kSelectWarps; ++w) {
    if (w == warp) {
      ups = up0;
      eqs = eq0;
    }
    up0 += sums[0][w];
    eq0 += sums[1][w];
  }
  if (ctas > 1) {
    if (tid == 0) {
      counts[0] = up0;
      counts[1] = eq0;
    }
    together(ctas);
    for (int c = 0; c < rank; ++c) {
      ups += remote_int(&counts[0], c);
      eqs += remote_int(&counts[1], c);
    }
  }
  for (int i = w0; i < w1; i += 32) {
    unsigned above, equal;
    look(i + lane, above, equal);
    const unsigned lower = (1u << lane) - 1;
    const int rank_eq = eqs + __popc(equal & lower);
    const int at = ups + __popc(above & lower) + min(rank_eq, left);
    if (((above >> lane & 1) || ((equal >> lane & 1) && rank_eq < left)) && at < q.keep) kept[at] = begin + i + lane;
    ups += __popc(above);
    eqs += __popc(equal);
  }
  if (ctas > 1) together(ctas);  // the others read this CTA's counts
}

// Bytes a thread moves of a row at a time, and rows that it holds.
constexpr int kMoveThreads = 256, kMoveRows = 8;
constexpr int kMoveSlice = 32;  // bytes of a row that a CTA of a move in place takes

// Rows [j0, j1) from their old slots: bytes [at, at + lanes * sizeof(V)) of each.
template <typename V>
__device__ __forceinline__ void move_rows(const EvictArgs& a, const EvictSeq& q, int s, int g, const void* from, const int64_t* fs,
                                          void* to, const int64_t* ts, int es, int lanes, int at, int j0, int j1) {
  const int32_t* kept = a.kept + ((int64_t)s * a.Hkv + g) * a.width;
  const int32_t* table = a.table + s * a.table_stride;
  const int32_t* to_table = a.to_table + s * a.to_table_stride;
  const int r = threadIdx.x / lanes, c = threadIdx.x % lanes, per = kMoveThreads / lanes;
  int src[kMoveRows];
  auto slots = [&](int base) {
#pragma unroll
    for (int u = 0; u < kMoveRows; ++u) {
      const int j = base + u * per + r;
      src[u] = r < per && j < j1 ? kept[j] : -1;
    }
  };
  slots(j0);
  for (int base = j0; base < j1; base += per * kMoveRows) {
    V v[kMoveRows];
    V* dst[kMoveRows];
#pragma unroll
    for (int u = 0; u < kMoveRows; ++u) {
      dst[u] = nullptr;
      const int j = base + u * per + r;
      if (src[u] < 0 || src[u] >= q.kv || (a.in_place && src[u] == j)) continue;
      const int p0 = evict_page(table, src[u] / a.page_size, a.num_pages, a.status);
      const int p1 = evict_page(to_table, j / a.page_size, a.to_pages, a.status);
      if (p0 < 0 || p1 < 0) continue;
      v[u] = *reinterpret_cast<const V*>(static_cast<const char*>(from) +
                                         (p0 * fs[0] + g * fs[1] + src[u] % a.page_size * fs[2]) * es + at + c * sizeof(V));
      dst[u] = reinterpret_cast<V*>(static_cast<char*>(to) + (p1 * ts[0] + g * ts[1] + j % a.page_size * ts[2]) * es + at +
                                    c * sizeof(V));
    }
    slots(base + per * kMoveRows);
    if (a.in_place) __syncthreads();
#pragma unroll
    for (int u = 0; u < kMoveRows; ++u)
      if (dst[u] != nullptr) *dst[u] = v[u];
  }
}

// In place: blocks of a (sequence, head) are `parts` slices of K, as many of V, and one of the weights.  Into other pages: `parts`
// pieces of `rows` rows of K with the weights, and as many of V.
__global__ void __launch_bounds__(kMoveThreads) evict_move_kernel(const EvictArgs a, int parts, int lanes, int rows) {
  const int blocks = a.in_place ? 2 * parts + 1 : 2 * parts, x = blockIdx.x % blocks;
  const int sg = blockIdx.x / blocks, s = sg / a.Hkv, g = sg % a.Hkv;
  let_next_kernel_start();
  wait_for_earlier_kernels();
  const EvictSeq q = evict_seq(a, s, false);
  if (a.in_place) {
    if (q.keep == q.kv) return;
    const int at = x % parts * lanes * 16;
    if (x == 2 * parts)
      move_rows<float>(a, q, s, g, a.mass, a.ms, a.mass_out, a.mos, 4, 1, 0, 0, q.keep);
    else if (x < parts)
      move_rows<uint4>(a, q, s, g, a.k, a.ks, a.k_out, a.kos, a.es, lanes, at, 0, q.keep);
    else
      move_rows<uint4>(a, q, s, g, a.v, a.vs, a.v_out, a.vos, a.es, lanes, at, 0, q.keep);
  } else {
    const int j0 = x % parts * rows, j1 = min(q.keep, j0 + rows);
    if (j0 >= j1) return;
    if (x < parts) {
      move_rows<float>(a, q, s, g, a.mass, a.ms, a.mass_out, a.mos, 4, 1, 0, j0, j1);
      move_rows<uint4>(a, q, s, g, a.k, a.ks, a.k_out, a.kos, a.es, lanes, 0, j0, j1);
    } else {
      move_rows<uint4>(a, q, s, g, a.v, a.vs, a.v_out, a.vos, a.es, lanes, 0, j0, j1);
    }
  }
}

cudaError_t launch_evict(const EvictArgs& a, cudaStream_t stream) {
  const int64_t heads = (int64_t)a.S * a.Hkv;
  // CTAs of a head: as many as the GPU has room for, while each gets 2048 slots of the longest sequence allowed.
  int ctas = 1;
  while (ctas < kSelectMostCtas && heads * ctas * 2 <= sm_count() && a.cap / (ctas * 2) >= 2048) ctas *= 2;
  const int each = ((a.cap + ctas - 1) / ctas + 31) / 32 * 32, cached = std::min(each, kSelectCached);
  static std::atomic<uint64_t> done{0};
  cudaError_t e = allow_smem(reinterpret_cast<const void*>(evict_select_kernel), kSelectCached * 4, done);
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
  e = cudaLaunchKernelEx(&cfg, evict_select_kernel, a, ctas, cached);
  const int most = std::min(a.keep, a.cap);  // rows that a head keeps
  if (e != cudaSuccess || most == 0) return e;
  const int row = a.D * a.es;
  int parts, lanes, rows = 0;
  if (a.in_place) {
    const int slice = row % kMoveSlice == 0 ? kMoveSlice : 16;
    parts = row / slice;
    lanes = slice / 16;
  } else {
    lanes = row / 16;
    rows = std::max(1, kMoveThreads / lanes) * kMoveRows;
    parts = (most + rows - 1) / rows;
  }
  const int64_t blocks = heads * (a.in_place ? 2 * parts + 1 : 2 * (int64_t)parts);
  if (blocks > INT32_MAX) return cudaErrorInvalidConfiguration;
  return launch_early(evict_move_kernel, static_cast<int>(blocks), kMoveThreads, 0, stream, a, parts, lanes, rows);
}

}  // namespace spruce
