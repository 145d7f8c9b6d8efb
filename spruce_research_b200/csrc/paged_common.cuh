// The split of paged attention's work over the GPU, shared by its kernels.
//
// A unit is (sequence, row tile, KV head): up to R query rows -- row r of a sequence is head r % rep of its token
// r / rep, so a tile has no padding heads -- against the keys its last token sees, in tiles of TK keys.  All units'
// key tiles are laid end to end and cut into equal runs, one a CTA: every SM gets the same work whatever the mix of
// lengths, and a long sequence is split over its keys as finely as the GPU is wide.  Lengths are read on the device
// (each CTA sums them itself, about a microsecond), so a call needs no host copy of them and can be captured in a graph.
//
// A run covers the end of one unit, some whole units and the start of another.  Whole units are written straight to
// the output.  A part (at most two a run: slot 0 begins with the run, slot 1 ends it) goes to the workspace as
// fp32 rows with their softmax maximum and sum; the CTA that holds a split unit's first part describes it, and a second
// kernel joins the parts in the order of the keys, so results do not depend on timing.
#pragma once

#include <atomic>
#include <utility>

#include "common.cuh"
#include "kernels.h"

namespace spruce {

struct PagedParams {
  PagedArgs a;
  int rep, row_tiles;     // Hq / Hkv; row tiles of the longest sequence allowed
  int kv_cap;             // keys a sequence may hold: min(max_kv, max_pages * page_size)
  int unit_cost;          // of starting and ending a unit, in key tiles
  int4* desc;             // [G] split unit whose first part is the run's last: {first token, qt, g, parts | slot << 12 | rows << 16}
  float2* part_ml;        // [2 G][R] softmax maximum (log2 units) and sum
  float* part_o;          // [2 G][R][D]
  float scale_log2;
  float inv_rep;
  float sum_log2;         // log2 of the factor that the kernel's sums carry
};

struct PagedSeq {
  int q0, qlen, kv, first;  // first token, new tokens, keys held, position of the first new token
};

__device__ __forceinline__ PagedSeq paged_seq(const PagedParams& p, int s) {
  const int c0 = p.a.cu_q[s], c1 = p.a.cu_q[s + 1], k = p.a.kv_lens[s];
  PagedSeq q;
  q.q0 = min(max(c0, 0), p.a.N);
  const int held = max(k, 0), added = min(max(c1, q.q0), p.a.N) - q.q0;
  q.qlen = min(added, p.a.max_q);
  q.kv = min(held, p.kv_cap);
  if (q.qlen != c1 - c0 || q.kv != k) raise_status(p.a.status, SPRUCE_STATUS_BAD_LENGTH);
  q.first = min(held, 1 << 30) - added;  // of the uncut lengths; positions stay ints
  return q;
}

// Keys that row tile qt sees (its last token's), and the tiles it counts as (an empty one still writes zeros):
// its key tiles and, after them, the fixed cost of a unit.
template <int R>
__device__ __forceinline__ int paged_keys(const PagedParams& p, const PagedSeq& q, int qt) {
  const int last_row = min((qt + 1) * R, q.qlen * p.rep) - 1;
  return min(max(q.first + last_row / p.rep + 1, 0), q.kv);
}
template <int R, int TK>
__device__ __forceinline__ int paged_weight(const PagedParams& p, const PagedSeq& q, int qt) {
  return max(1, (paged_keys<R>(p, q, qt) + TK - 1) / TK) + p.unit_cost;
}

// A piece of a unit that this CTA computes: key tiles [t0, t1) of n.
struct PagedPiece {
  PagedSeq q;
  int s, qt, g;
  int keys;         // keys the unit sees
  int t0, t1, n;
  int slot;         // of the partial result; -1: the whole unit
  int parts;        // > 0: the first part of a unit that this many runs share
};

constexpr int kMaxSms = 160, kPagedMaxRuns = 3 * kMaxSms;
static_assert(kPagedMaxRuns < 1 << 12, "parts of a unit fit their field");
__device__ __forceinline__ int4 paged_desc(const PagedPiece& x, int rows) {
  return make_int4(x.q.q0, x.qt, x.g, x.parts | x.slot << 12 | rows << 16);
}
__device__ __forceinline__ int paged_desc_parts(int w) { return w & 0xfff; }
__device__ __forceinline__ int paged_desc_slot(int w) { return (w >> 12) & 1; }
__device__ __forceinline__ int paged_desc_rows(int w) { return w >> 16; }

// Walks a run's pieces; every thread that calls next() with the same walker sees the same ones.
template <int R, int TK>
struct PagedWalk {
  int64_t left;     // tiles of the run not yet handed out
  int64_t run;      // tiles of a full run
  int s, qt, g, t;
  bool head;        // the next piece begins the run

  __device__ __forceinline__ bool next(const PagedParams& p, PagedPiece& x) {
    while (left > 0) {
      for (;;) {  // the next sequence with rows; one exists while tiles are left
        if (s >= p.a.S) return false;
        x.q = paged_seq(p, s);
        if (qt * R < x.q.qlen * p.rep) break;
        ++s;
        qt = 0;
      }
      x.s = s;
      x.qt = qt;
      x.g = g;
      x.keys = paged_keys<R>(p, x.q, qt);
      x.n = max(1, (x.keys + TK - 1) / TK);
      const int take = static_cast<int>(min((int64_t)(x.n + p.unit_cost), t + left)) - t;
      x.t0 = t;
      x.t1 = min(x.n, t + take);
      x.slot = x.t0 == 0 && x.t1 == x.n ? -1 : (head ? 0 : 1);
      x.parts = x.t0 == 0 && x.t1 < x.n ? 1 + static_cast<int>((x.n - x.t1 + run - 1) / run) : 0;
      left -= take;
      head = false;
      t = 0;
      if (++g == p.a.Hkv) {
        g = 0;
        ++qt;
      }
      if (x.t0 < x.n) return true;  // else the run begins in the unit's fixed cost: nothing to do
    }
    return false;
  }
};

// Sum of v over the block, and the sum over the threads before this one.  scratch: 33 int64.
template <int THREADS>
__device__ __forceinline__ int64_t block_scan(int64_t v, int64_t& before, int64_t* scratch) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  constexpr int WARPS = THREADS / 32;
  int64_t inc = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int64_t y = __shfl_up_sync(0xffffffffu, inc, o);
    if (lane >= o) inc += y;
  }
  if (lane == 31) scratch[warp] = inc;
  __syncthreads();
  int64_t base = 0, total = 0;
#pragma unroll
  for (int w = 0; w < WARPS; ++w) {
    const int64_t x = scratch[w];
    base += w < warp ? x : 0;
    total += x;
  }
  __syncthreads();
  before = base + inc - v;
  return total;
}

// This CTA's run.  Called by all THREADS threads (those of the block); returns false where the CTA has no work.
// scratch: 33 int64 of shared memory that stay untouched until the caller's next barrier.
template <int R, int TK, int THREADS>
__device__ __forceinline__ bool paged_run(const PagedParams& p, PagedWalk<R, TK>& w, int64_t* scratch) {
  const int G = gridDim.x, c = blockIdx.x;
  // Tiles of sequence s over all KV heads; several row tiles are summed by a group of lanes.
  const int gs = p.row_tiles == 1 ? 1 : (p.row_tiles <= 8 ? 8 : 32);
  const int per = THREADS / gs, sub = threadIdx.x % gs, mine = threadIdx.x / gs;
  auto weight = [&](int s) {  // on sub == 0 of the group, else 0; called by whole groups
    int64_t v = 0;
    if (s < p.a.S) {
      const PagedSeq q = paged_seq(p, s);
      const int tiles = (q.qlen * p.rep + R - 1) / R;
      for (int qt = sub; qt < tiles; qt += gs) v += paged_weight<R, TK>(p, q, qt);
    }
    for (int o = gs >> 1; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return sub == 0 ? v * p.a.Hkv : 0;
  };
  int64_t total = 0, before, w0 = 0, b0 = 0;
  for (int base = 0; base < p.a.S; base += per) {
    const int64_t v = weight(base + mine);
    total += block_scan<THREADS>(v, before, scratch);
    if (base == 0) {
      w0 = v;
      b0 = before;
    }
  }
  const int64_t run = max((int64_t)1, (total + G - 1) / G);
  const int64_t start = c * run;
  w.run = run;
  w.left = min(run, total - start);
  w.head = true;
  if (start >= total) return false;
  __shared__ int s_seq;
  __shared__ int64_t s_before;
  int64_t done = 0;
  for (int base = 0; base < p.a.S; base += per) {
    int64_t v = w0;
    before = b0;
    int64_t sum = total;
    if (p.a.S > per) {
      v = weight(base + mine);
      sum = block_scan<THREADS>(v, before, scratch);
    }
    if (start >= done + before && start < done + before + v) {  // one thread of the block
      s_seq = base + mine;
      s_before = done + before;
    }
    done += sum;
  }
  __syncthreads();
  w.s = s_seq;
  int64_t rest = start - s_before;
  const PagedSeq q = paged_seq(p, w.s);
  // The row tile that holds it: every warp looks at 32 of them at a time.
  const int lane = threadIdx.x & 31;
  const int tiles = (q.qlen * p.rep + R - 1) / R;
  w.qt = 0;
  for (int base = 0; base < tiles; base += 32) {
    const int64_t v = base + lane < tiles ? (int64_t)paged_weight<R, TK>(p, q, base + lane) * p.a.Hkv : 0;
    int64_t inc = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t y = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += y;
    }
    const unsigned past = __ballot_sync(0xffffffffu, rest < inc);
    if (past != 0) {
      const int at = __ffs(past) - 1;
      w.qt = base + at;
      rest -= __shfl_sync(0xffffffffu, inc - v, at);
      break;
    }
    rest -= __shfl_sync(0xffffffffu, inc, 31);
  }
  const int n = paged_weight<R, TK>(p, q, w.qt);
  w.g = static_cast<int>(rest / n);
  w.t = static_cast<int>(rest % n);
  return true;
}

// Tokens and heads of the rows of a tile: row r after row0 of sequence (q0 = its first token), KV head g.  One division a
// tile; within it (row and remainder under 2^21) the quotient by a rounded reciprocal is exact.
struct PagedRows {
  int tok0, rem0, head0, rep;
  int64_t q0;
  float inv;
  __device__ __forceinline__ PagedRows(const PagedParams& p, int first, int row0, int g)
      : tok0(row0 / p.rep), rem0(row0 - row0 / p.rep * p.rep), head0(g * p.rep), rep(p.rep), q0(first), inv(p.inv_rep) {}
  // Token of the sequence.
  __device__ __forceinline__ int token(int r) const { return tok0 + in_tile(r); }
  // Element offset in q or out.
  __device__ __forceinline__ int64_t offset(int r, int64_t token_stride, int64_t head_stride) const {
    const int t = in_tile(r);
    return (q0 + tok0 + t) * token_stride + (head0 + rem0 + r - t * rep) * head_stride;
  }

 private:
  __device__ __forceinline__ int in_tile(int r) const { return static_cast<int>((static_cast<float>(rem0 + r) + 0.5f) * inv); }
};

// Page of a key and the row in it; -1 (and a status) where the table names no page of the cache.
__device__ __forceinline__ int paged_page(const PagedParams& p, const int32_t* table, int index) {
  const int page = table[index];
  if (page >= 0 && page < p.a.num_pages) return page;
  raise_status(p.a.status, SPRUCE_STATUS_BAD_PAGE);
  return -1;
}

// log2 of the factor that all probabilities of a kernel carry until O / l cancels it.  P is rounded to the inputs' type for
// its product with V (the operand of the MMA), the sum l is of the fp32 values.  bf16 has fp32's range.  fp16 ends at 2^-24
// and loses bits below 2^-14: with the largest P at 1, weights under 2^-25 of it would be in l and not in O, and a long
// context has many of those.  With P up to 2^15 (fp16 holds 65504) a weight keeps all its bits down to 2^-29 of the largest.
template <typename T> struct PScale { static constexpr float log2 = 0.0f; };
template <> struct PScale<__half> { static constexpr float log2 = 15.0f; };

// Natural log of a row's softmax sum from its maximum (log2 units) and sum; -inf where nothing is above -inf.
__device__ __forceinline__ float paged_lse(const PagedParams& p, float m, float l) {
  return m == -INFINITY && !(l != l) ? -INFINITY : (m + (log2f(l) - p.sum_log2)) * 0.6931471805599453f;
}

// Opts a kernel into `bytes` of dynamic shared memory, once a device (`done` is the kernel's own mask of devices).
inline cudaError_t allow_smem(const void* kern, int bytes, std::atomic<uint64_t>& done) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess || dev < 0 || dev > 63 || (done.load() >> dev & 1)) {
    if (e == cudaSuccess && dev > 63) e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    return e;
  }
  e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e == cudaSuccess) done.fetch_or(uint64_t(1) << dev);
  return e;
}

// SMs of the current GPU (at most kMaxSms), asked for once (paged_attn.cu).
int sm_count();

// Launches a kernel that may start while the one before it in the stream ends; it waits (griddepcontrol) before it
// touches memory.
template <typename... Params, typename... Args>
cudaError_t launch_early(void (*kern)(Params...), int grid, int threads, int smem, cudaStream_t stream, Args&&... args) {
  cudaLaunchConfig_t cfg{};
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kern, std::forward<Args>(args)...);
}
// In a kernel: memory of the kernels before it is complete; the next kernel may start.
__device__ __forceinline__ void wait_for_earlier_kernels() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void let_next_kernel_start() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

// Tensor-core attention of chunks (paged_chunk_sm100.cu), on G CTAs.
constexpr int kPagedChunkRows = 256, kPagedChunkKeys = 128;
cudaError_t launch_paged_chunk(const PagedArgs& a, int dtype, int G, cudaStream_t stream);

// Warp-MMA attention of at most 32 query rows a unit, in 1 or 2 tiles of 16 (paged_rows_sm100.cu).
constexpr int kPagedRowsMax = 32, kPagedRowsKeys = 64, kPagedRowsPerSm = 2;
cudaError_t launch_paged_rows(const PagedArgs& a, int dtype, int tiles, int G, cudaStream_t stream);
// The cache's tensor maps, and the rows of a box of them, for key tiles of `tile` (paged_chunk_sm100.cu).
bool paged_cache_maps(const PagedArgs& a, int dtype, int box, CUtensorMap* mk, CUtensorMap* mv);
int paged_box(int page_size, int tile);

// Joins the parts of split units (paged_attn.cu).
template <typename T>
cudaError_t launch_paged_join(const PagedParams& p, int R, int G, int TK, cudaStream_t stream);

// Parameters of a launch with R-row tiles on at most G CTAs, its workspace carved up.
inline PagedParams paged_params(const PagedArgs& a, int R, int G, int unit_cost, float sum_log2 = 0.0f) {
  PagedParams p;
  p.sum_log2 = sum_log2;
  p.a = a;
  p.rep = a.Hq / a.Hkv;
  p.inv_rep = 1.0f / static_cast<float>(p.rep);
  p.row_tiles = static_cast<int>(((int64_t)a.max_q * p.rep + R - 1) / R);
  int64_t cap = (int64_t)a.max_pages * a.page_size;
  cap = cap < a.max_kv ? cap : a.max_kv;
  p.kv_cap = static_cast<int>(cap < (1 << 30) ? cap : 1 << 30);  // key indices stay ints with room for a tile more
  p.unit_cost = unit_cost;
  uint8_t* ws = static_cast<uint8_t*>(a.workspace);
  p.desc = reinterpret_cast<int4*>(ws);
  ws += ((int64_t)G * 16 + 255) / 256 * 256;
  p.part_ml = reinterpret_cast<float2*>(ws);
  ws += (int64_t)2 * G * R * 8;
  p.part_o = reinterpret_cast<float*>(ws);
  // Not 0: a masked score (-inf) times 0 is not a number.  1e-30 makes every finite score 0 as well.
  p.scale_log2 = a.scale > 0.0f ? a.scale * 1.4426950408889634f : 1e-30f;
  return p;
}
inline int64_t paged_params_bytes(int R, int G, int64_t D) {
  return ((int64_t)G * 16 + 255) / 256 * 256 + (int64_t)2 * G * R * (8 + 4 * D);
}

}  // namespace spruce
