// Eviction from a paged cache by weight: per (sequence, KV head) the first `sinks` slots, the last `recent` ones and the
// heaviest of those between stay, `keep` in all, and move in their order to slots 0 .. keep - 1.
//
// Selection: a radix select over the weights' order-preserving bits (four passes of 8 bits) finds the weight of the last
// one kept and how many of its equals stay (the lowest slots); one more pass writes the kept slots in order.
//
// Moving in place: slot j takes row kept[j] >= j, so going up in j a row is read before it is written over, if
// all rows of a round are read before any is written: one barrier a round.  Rows are cut into slices of columns, which
// never touch each other, so a (sequence, head) is spread over many CTAs that need not wait for one another.
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

constexpr int kSelectThreads = 1024;

__global__ void __launch_bounds__(kSelectThreads) evict_select_kernel(const EvictArgs a) {
  const int s = blockIdx.x / a.Hkv, g = blockIdx.x % a.Hkv;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  __shared__ int hist[256];
  __shared__ int counts[2][32];
  __shared__ uint32_t s_prefix;
  __shared__ int s_left;
  const EvictSeq q = evict_seq(a, s, g == 0 && tid == 0);
  int32_t* kept = a.kept + (int64_t)blockIdx.x * a.width;
  if (g == 0 && tid == 0) a.new_lens[s] = q.kv == 0 ? a.kv_lens[s] : q.keep;
  for (int j = q.keep + tid; j < a.width; j += kSelectThreads) kept[j] = -1;
  if (q.keep == q.kv) {
    for (int j = tid; j < q.keep; j += kSelectThreads) kept[j] = j;
    return;
  }
  const int32_t* table = a.table + s * a.table_stride;
  auto key_of = [&](int j) {
    const int page = evict_page(table, j / a.page_size, a.num_pages, a.status);
    return page < 0 ? 0u : weight_key(a.mass[page * a.ms[0] + g * a.ms[1] + j % a.page_size * a.ms[2]]);
  };
  int left = q.keep - q.sinks - (q.kv - q.tail);  // to be taken between sinks and tail
  uint32_t prefix = 0, mask = 0;
  for (int shift = 24; left > 0 && shift >= 0; shift -= 8) {
    if (tid < 256) hist[tid] = 0;
    __syncthreads();
    for (int j = q.sinks + tid; j < q.tail; j += kSelectThreads) {
      const uint32_t k = key_of(j);
      if ((k & mask) == prefix) atomicAdd(&hist[(k >> shift) & 255], 1);
    }
    __syncthreads();
    if (tid == 0) {
      int d = 255;
      while (d > 0 && hist[d] < left) left -= hist[d--];
      s_prefix = prefix | static_cast<uint32_t>(d) << shift;
      s_left = left;
    }
    __syncthreads();
    prefix = s_prefix;
    left = s_left;
    mask |= 255u << shift;
    __syncthreads();
  }
  // `left` slots of exactly the weight `prefix` stay, and all above it.
  const bool any = mask != 0;
  int taken = 0, equals = 0;
  for (int base = 0; base < q.kv; base += kSelectThreads) {
    const int j = base + tid;
    bool eq = false, in = j < q.sinks || (j >= q.tail && j < q.kv);
    if (any && j >= q.sinks && j < q.tail) {
      const uint32_t k = key_of(j);
      in = k > prefix;
      eq = k == prefix;
    }
    const unsigned eqs = __ballot_sync(0xffffffffu, eq);
    if (lane == 0) counts[0][warp] = __popc(eqs);
    __syncthreads();
    int before = 0, total = 0;
    for (int w = 0; w < 32; ++w) {
      before += w < warp ? counts[0][w] : 0;
      total += counts[0][w];
    }
    in = in || (eq && equals + before + __popc(eqs & ((1u << lane) - 1)) < left);
    equals += total;
    const unsigned ins = __ballot_sync(0xffffffffu, in);
    if (lane == 0) counts[1][warp] = __popc(ins);
    __syncthreads();
    before = total = 0;
    for (int w = 0; w < 32; ++w) {
      before += w < warp ? counts[1][w] : 0;
      total += counts[1][w];
    }
    const int at = taken + before + __popc(ins & ((1u << lane) - 1));
    if (in && at < q.keep) kept[at] = j;
    taken += total;
  }
}

// V: bytes a thread moves of a row; rows of V * lanes bytes.
constexpr int kMoveThreads = 256, kMoveRows = 8;

template <typename V>
__device__ __forceinline__ void move_rows(const EvictArgs& a, const EvictSeq& q, int s, int g, const void* from, const int64_t* fs,
                                          void* to, const int64_t* ts, int es, int lanes, int at) {
  const int32_t* kept = a.kept + ((int64_t)s * a.Hkv + g) * a.width;
  const int32_t* table = a.table + s * a.table_stride;
  const int32_t* to_table = a.to_table + s * a.to_table_stride;
  const int r = threadIdx.x / lanes, c = threadIdx.x % lanes, per = kMoveThreads / lanes;
  for (int base = 0; base < q.keep; base += per * kMoveRows) {
    V v[kMoveRows];
    V* dst[kMoveRows];
#pragma unroll
    for (int u = 0; u < kMoveRows; ++u) {
      dst[u] = nullptr;
      const int j = base + u * per + r;
      if (r >= per || j >= q.keep) continue;
      const int src = kept[j];
      if (src < 0 || src >= q.kv) continue;
      const int p0 = evict_page(table, src / a.page_size, a.num_pages, a.status);
      const int p1 = evict_page(to_table, j / a.page_size, a.to_pages, a.status);
      if (p0 < 0 || p1 < 0) continue;
      v[u] = *reinterpret_cast<const V*>(static_cast<const char*>(from) +
                                         (p0 * fs[0] + g * fs[1] + src % a.page_size * fs[2]) * es + at + c * sizeof(V));
      dst[u] = reinterpret_cast<V*>(static_cast<char*>(to) + (p1 * ts[0] + g * ts[1] + j % a.page_size * ts[2]) * es + at +
                                    c * sizeof(V));
    }
    __syncthreads();
#pragma unroll
    for (int u = 0; u < kMoveRows; ++u)
      if (dst[u] != nullptr) *dst[u] = v[u];
  }
}

// Blocks of a (sequence, head): `slices` of K, as many of V, one of the weights.
__global__ void __launch_bounds__(kMoveThreads) evict_move_kernel(const EvictArgs a, int slices, int slice_bytes) {
  const int parts = 2 * slices + 1, x = blockIdx.x % parts;
  const int sg = blockIdx.x / parts, s = sg / a.Hkv, g = sg % a.Hkv;
  const EvictSeq q = evict_seq(a, s, false);
  if (a.in_place && q.keep == q.kv) return;
  if (x == 2 * slices) {
    move_rows<float>(a, q, s, g, a.mass, a.ms, a.mass_out, a.mos, 4, 1, 0);
  } else if (x < slices) {
    move_rows<uint4>(a, q, s, g, a.k, a.ks, a.k_out, a.kos, a.es, slice_bytes / 16, x * slice_bytes);
  } else {
    move_rows<uint4>(a, q, s, g, a.v, a.vs, a.v_out, a.vos, a.es, slice_bytes / 16, (x - slices) * slice_bytes);
  }
}

cudaError_t launch_evict(const EvictArgs& a, cudaStream_t stream) {
  const int64_t heads = (int64_t)a.S * a.Hkv;
  evict_select_kernel<<<static_cast<unsigned>(heads), kSelectThreads, 0, stream>>>(a);
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess || a.width == 0) return e;
  const int row = a.D * a.es;
  const int slice = row % 64 == 0 ? 64 : 16;
  evict_move_kernel<<<static_cast<unsigned>(heads * (2 * (row / slice) + 1)), kMoveThreads, 0, stream>>>(a, row / slice, slice);
  return cudaGetLastError();
}

}  // namespace spruce
