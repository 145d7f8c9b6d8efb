// Attention of new tokens over a paged K/V cache: the fp32 CUDA-core kernel, the join of split units, and the
// choice of kernel.  The work's split is in paged_common.cuh.
//
// For a query row q at position i: o = sum_j p_j v_j / sum_j p_j, p_j = 2^(q.k_j scale log2(e) - m), j <= i, over
// key tiles in one pass with the running maximum m and sum.  Rows that see nothing are zero.  Cache rows at or past
// the sequence's length are never loaded.
#include <algorithm>

#include "attn_common.cuh"
#include "paged_common.cuh"

namespace spruce {

// SMs of the current GPU, asked for once.
static int sm_count() {
  static std::atomic<int> known[64];
  int dev = 0, v = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return 148;
  if (dev < 64 && (v = known[dev].load()) > 0) return v;
  if (cudaDeviceGetAttribute(&v, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || v < 1) return 148;
  v = std::min(v, kMaxSms);
  if (dev < 64) known[dev].store(v);
  return v;
}

__device__ __forceinline__ void copy16_or_zero(float* dst, const float* src, bool in) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(dst)), "l"(src), "r"(in ? 16 : 0)
               : "memory");
}

template <int D, int R, int TK, int STAGES>
struct F32Layout {
  static constexpr int TR = R == 64 ? 4 : 2, TC = R == 64 ? 4 : 2;  // rows and keys of a thread's scores
  static constexpr int NC = TK / TC;                               // threads along the keys, and along D
  static constexpr int THREADS = R / TR * NC;
  static constexpr int KP = D + 4;    // padded rows: float4 reads of adjacent keys hit distinct banks
  static constexpr int PP = TK + 4;
  static constexpr int STAGE = TK * KP + TK * D;
  // One stage: the probabilities take the place of the keys they were formed from.
  static constexpr int FLOATS = R * D + STAGES * STAGE + (STAGES == 1 ? 0 : R * PP);
  static_assert(STAGES > 1 || R * PP <= TK * KP, "probabilities fit over the keys");
  static_assert(NC == 16, "half a warp a row group");
};

// A CTA holds R query rows and STAGES tiles of TK keys in shared memory; a thread forms TR x TC scores, then TR rows x
// D / NC output dims.  Chunks are bound by the FMA pipe (4 x 4 scores a thread: 12 shared-memory wavefronts to 64
// FMAs), with two CTAs an SM one of which loads while the other computes.  Few rows are bound by HBM on paper and in
// practice by shared-memory reads (every key is read once a row group), so they take as few row groups as hold them,
// eight or sixteen rows, and keep two tiles in flight.  On a B200: 512 tokens over 8K (28 heads of 128) 1.66 ms, 37 TFLOP/s;
// one token over 32K 58 us, 2.3 TB/s.  At D = 128 the 64-row form spills 96 bytes of a thread's 128 registers.
template <int D, int R, int TK, int STAGES>
__global__ void __launch_bounds__(F32Layout<D, R, TK, STAGES>::THREADS) paged_attn_f32_kernel(const PagedParams p) {
  using L = F32Layout<D, R, TK, STAGES>;
  constexpr int TR = L::TR, TC = L::TC, NC = L::NC, KP = L::KP, PP = L::PP, THREADS = L::THREADS;
  constexpr int DV = D / (4 * NC);  // float4s of an output row a thread holds, 4 NC dims apart
  constexpr int CH = D / 4;
  extern __shared__ float fsm[];
  float* Qs = fsm;                   // [R][D]
  float* KVs = Qs + R * D;           // [STAGES]: [TK][KP], [TK][D]
  float* Ps = STAGES == 1 ? KVs : KVs + STAGES * L::STAGE;  // [R][PP]
  __shared__ int64_t scratch[33];

  const int tid = threadIdx.x;
  const int rg = tid / NC, cg = tid % NC;
  let_next_kernel_start();
  wait_for_earlier_kernels();
  PagedWalk<R, TK> walk;
  const bool any = paged_run<R, TK, THREADS>(p, walk, scratch);
  int4 mine = make_int4(0, 0, 0, 0);
  PagedPiece x;
  while (any && walk.next(p, x)) {
    const int rows = min(R, x.q.qlen * p.rep - x.qt * R);
    const int n = x.keys > 0 ? x.t1 - x.t0 : 0;
    const PagedRows row_at(p, x.q.q0, x.qt * R, x.g);
    const int32_t* table = p.a.block_table + x.s * p.a.table_stride;
    // Tile i of the piece into its stage: rows past the keys, or of no page, are zeros.
    auto load = [&](int i) {
      if (i < n) {
        float* ks = KVs + i % STAGES * L::STAGE;
        float* vs = ks + TK * KP;
        const int key0 = (x.t0 + i) * TK, d = tid % CH * 4;
#pragma unroll 1
        for (int r0 = 0; r0 < TK; r0 += 16) {  // sixteen keys lie in one page
          const int key = key0 + r0, pi = key / p.a.page_size;
          const int64_t page = key < x.keys ? paged_page(p, table, pi) : -1;
          const int64_t row = key - pi * p.a.page_size + tid / CH;
          const float* k = static_cast<const float*>(p.a.kc);
          const float* v = static_cast<const float*>(p.a.vc);
          if (page >= 0) {
            k += page * p.a.ks[0] + x.g * p.a.ks[1] + row * p.a.ks[2] + d;
            v += page * p.a.vs[0] + x.g * p.a.vs[1] + row * p.a.vs[2] + d;
          }
#pragma unroll
          for (int r = tid / CH; r < 16; r += THREADS / CH) {
            const bool in = page >= 0 && key + r < x.keys;
            copy16_or_zero(ks + (r0 + r) * KP + d, k, in);
            copy16_or_zero(vs + (r0 + r) * D + d, v, in);
            if (in) {
              k += THREADS / CH * p.a.ks[2];
              v += THREADS / CH * p.a.vs[2];
            }
          }
        }
      }
      asm volatile("cp.async.commit_group;" ::: "memory");
    };
    __syncthreads();
#pragma unroll
    for (int i = 0; i + 1 < STAGES; ++i) load(i);
    for (int e = tid; e < R * CH; e += THREADS) {
      const int r = e / CH, d = e % CH * 4;
      float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      if (r < rows) {
        v = *reinterpret_cast<const float4*>(static_cast<const float*>(p.a.q) + row_at.offset(r, p.a.qn, p.a.qh) + d);
      }
      *reinterpret_cast<float4*>(Qs + r * D + d) = v;
    }
    float4 o[TR][DV];
    float m[TR], l[TR];
    int seen[TR];  // keys the row sees
#pragma unroll
    for (int i = 0; i < TR; ++i) {
      m[i] = -INFINITY;
      l[i] = 0.0f;
      seen[i] = min(x.q.first + row_at.token(rg * TR + i) + 1, x.keys);
#pragma unroll
      for (int d = 0; d < DV; ++d) o[i][d] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    }
    for (int t = 0; t < n; ++t) {
      load(t + STAGES - 1);  // into the stage that the last tile's readers have left
      if constexpr (STAGES == 1) asm volatile("cp.async.wait_group 0;" ::: "memory");
      else asm volatile("cp.async.wait_group 1;" ::: "memory");
      __syncthreads();
      const float* Ks = KVs + t % STAGES * L::STAGE;
      const float* Vs = Ks + TK * KP;
      float s[TR][TC];
#pragma unroll
      for (int i = 0; i < TR; ++i)
#pragma unroll
        for (int j = 0; j < TC; ++j) s[i][j] = 0.0f;
#pragma unroll 4
      for (int d = 0; d < D; d += 4) {
        float4 qv[TR], kv[TC];
#pragma unroll
        for (int i = 0; i < TR; ++i) qv[i] = *reinterpret_cast<const float4*>(Qs + (rg * TR + i) * D + d);
#pragma unroll
        for (int j = 0; j < TC; ++j) kv[j] = *reinterpret_cast<const float4*>(Ks + (cg + j * NC) * KP + d);
#pragma unroll
        for (int i = 0; i < TR; ++i)
#pragma unroll
          for (int j = 0; j < TC; ++j)
            s[i][j] = fmaf(qv[i].x, kv[j].x,
                           fmaf(qv[i].y, kv[j].y, fmaf(qv[i].z, kv[j].z, fmaf(qv[i].w, kv[j].w, s[i][j]))));
      }
      if constexpr (STAGES == 1) __syncthreads();
#pragma unroll
      for (int i = 0; i < TR; ++i) {
        float mx = -INFINITY;
#pragma unroll
        for (int j = 0; j < TC; ++j) {
          s[i][j] = (x.t0 + t) * TK + cg + j * NC < seen[i] ? s[i][j] * p.scale_log2 : -INFINITY;
          mx = fmaxf(mx, s[i][j]);
        }
#pragma unroll
        for (int off = NC / 2; off > 0; off >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, off));
        const float m_new = fmaxf(m[i], mx);
        const float ref = m_new == -INFINITY ? 0.0f : m_new;
        const float alpha = exp2f(m[i] - ref);  // 0 while the row has seen nothing
        float sum = 0.0f;
#pragma unroll
        for (int j = 0; j < TC; ++j) {
          const float e = exp2f(s[i][j] - ref);
          Ps[(rg * TR + i) * PP + cg + j * NC] = e;
          sum += e;
        }
#pragma unroll
        for (int off = NC / 2; off > 0; off >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
        l[i] = l[i] * alpha + sum;
        m[i] = m_new;
#pragma unroll
        for (int d = 0; d < DV; ++d) {
          o[i][d].x *= alpha;
          o[i][d].y *= alpha;
          o[i][d].z *= alpha;
          o[i][d].w *= alpha;
        }
      }
      __syncwarp();  // a row's probabilities are written and read by the same NC lanes
#pragma unroll 2
      for (int j = 0; j < TK; j += 4) {
        float4 pr[TR];
#pragma unroll
        for (int i = 0; i < TR; ++i) pr[i] = *reinterpret_cast<const float4*>(Ps + (rg * TR + i) * PP + j);
#pragma unroll
        for (int jj = 0; jj < 4; ++jj)
#pragma unroll
          for (int d = 0; d < DV; ++d) {
            const float4 v = *reinterpret_cast<const float4*>(Vs + (j + jj) * D + (d * NC + cg) * 4);
#pragma unroll
            for (int i = 0; i < TR; ++i) {
              const float w = jj == 0 ? pr[i].x : (jj == 1 ? pr[i].y : (jj == 2 ? pr[i].z : pr[i].w));
              o[i][d].x = fmaf(w, v.x, o[i][d].x);
              o[i][d].y = fmaf(w, v.y, o[i][d].y);
              o[i][d].z = fmaf(w, v.z, o[i][d].z);
              o[i][d].w = fmaf(w, v.w, o[i][d].w);
            }
          }
      }
      __syncthreads();
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");
#pragma unroll
    for (int i = 0; i < TR; ++i) {
      const int r = rg * TR + i;
      if (r >= rows) continue;
      float* dst;
      float f = 1.0f;
      if (x.slot < 0) {
        dst = static_cast<float*>(p.a.out) + row_at.offset(r, p.a.on, p.a.oh);
        f = l[i] > 0.0f ? 1.0f / l[i] : 0.0f;
      } else {
        const int64_t at = (int64_t)(2 * blockIdx.x + x.slot) * R + r;
        if (cg == 0) p.part_ml[at] = make_float2(m[i], l[i]);
        dst = p.part_o + at * D;
      }
#pragma unroll
      for (int d = 0; d < DV; ++d)
        *reinterpret_cast<float4*>(dst + (d * NC + cg) * 4) =
            make_float4(o[i][d].x * f, o[i][d].y * f, o[i][d].z * f, o[i][d].w * f);
    }
    if (x.parts > 0) mine = paged_desc(x, rows);
  }
  if (tid == 0) p.desc[blockIdx.x] = mine;
}

// Joins the parts of split units: a row is the parts' rows weighted by 2^(m_i - max), taken in the order of the keys.
//
// Every CTA reads the G descriptions and deals the split units out as jobs: eight rows, a warp each,
// where a unit has few parts, else one row whose parts the eight warps share.  The launch is programmatic: its
// CTAs start while the attention's last ones run, and wait before they read.
constexpr int kJoinThreads = 256, kJoinWarps = kJoinThreads / 32, kJoinPerSm = 4;

template <typename T>
__global__ void __launch_bounds__(kJoinThreads) paged_join_kernel(const PagedParams p, int R, int G) {
  constexpr int PER = (kPagedMaxRuns + kJoinThreads - 1) / kJoinThreads;  // descriptions a thread
  __shared__ int4 desc[kPagedMaxRuns];
  __shared__ int first[kPagedMaxRuns + 1];  // jobs before each unit
  __shared__ int sums[kJoinWarps], job_s;
  __shared__ float l_s[kJoinWarps], o_s[kJoinWarps][128];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int D = p.a.D, dims = D / 32;  // 2 or 4 adjacent dims a lane
  let_next_kernel_start();
  wait_for_earlier_kernels();

  // Jobs of each unit, summed.
  int n[PER], inc = 0;
#pragma unroll
  for (int u = 0; u < PER; ++u) {
    n[u] = 0;
    if (PER * tid + u < G) {
      const int4 d = p.desc[PER * tid + u];
      desc[PER * tid + u] = d;
      const int parts = paged_desc_parts(d.w), rows = paged_desc_rows(d.w);
      n[u] = parts == 0 ? 0 : (parts <= kJoinWarps ? (rows + kJoinWarps - 1) / kJoinWarps : rows);
    }
    inc += n[u];
  }
  int before = -inc;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, inc, o);
    if (lane >= o) inc += y;
  }
  before += inc;
  if (lane == 31) sums[warp] = inc;
  __syncthreads();
  int jobs = 0;
#pragma unroll
  for (int w = 0; w < kJoinWarps; ++w) {
    before += w < warp ? sums[w] : 0;
    jobs += sums[w];
  }
#pragma unroll
  for (int u = 0; u < PER; ++u) {
    if (PER * tid + u < G) first[PER * tid + u] = before;
    before += n[u];
  }
  if (tid == 0) first[G] = jobs;
  __syncthreads();

  for (int job = blockIdx.x; job < jobs; job += gridDim.x) {
    for (int c = tid; c < G; c += kJoinThreads)
      if (first[c] <= job && job < first[c + 1]) job_s = c;
    __syncthreads();
    const int c = job_s;
    const int4 d = desc[c];
    const int parts = paged_desc_parts(d.w), rows = paged_desc_rows(d.w);
    const bool few = parts <= kJoinWarps;
    const int r = few ? (job - first[c]) * kJoinWarps + warp : job - first[c];
    const int step = few ? 1 : kJoinWarps, start = few ? 0 : warp;
    float acc[4] = {0.0f, 0.0f, 0.0f, 0.0f}, l = 0.0f;
    if (r < rows) {
      // Part i > 0 begins its run (slot 0); part 0 has the described slot.
      auto at = [&](int i) { return (int64_t)(2 * (c + i) + (i == 0 ? paged_desc_slot(d.w) : 0)) * R + r; };
      constexpr int U = 4;  // parts whose loads are in flight together
      float2 ml[U];
      float v[U][4];
      auto load = [&](int i0) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const int i = i0 + u * step;
          const bool in = i < parts;
          const int64_t row = at(in ? i : 0);
          ml[u] = in ? p.part_ml[row] : make_float2(-INFINITY, 0.0f);
          const float* o = p.part_o + row * D + lane * dims;
          v[u][2] = v[u][3] = 0.0f;
          if (dims == 4) {
            const float4 y = *reinterpret_cast<const float4*>(o);
            v[u][0] = y.x;
            v[u][1] = y.y;
            v[u][2] = y.z;
            v[u][3] = y.w;
          } else {
            const float2 y = *reinterpret_cast<const float2*>(o);
            v[u][0] = y.x;
            v[u][1] = y.y;
          }
        }
      };
      load(start);
      float top = -INFINITY;
      for (int i = lane; i < parts; i += 32) top = fmaxf(top, p.part_ml[at(i)].x);
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
      const float ref = top == -INFINITY ? 0.0f : top;
      for (int i0 = start; i0 < parts; i0 += U * step) {
        if (i0 > start) load(i0);
#pragma unroll
        for (int u = 0; u < U; ++u) {
          if (i0 + u * step >= parts) break;  // a repeated first part is not added
          const float w = exp2f(ml[u].x - ref);
          l = fmaf(ml[u].y, w, l);
#pragma unroll
          for (int k = 0; k < 4; ++k) acc[k] = fmaf(v[u][k], w, acc[k]);
        }
      }
    }
    if (!few) {  // the warps' sums share one maximum: add them in order
      if (lane == 0) l_s[warp] = l;
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (k < dims) o_s[warp][lane * dims + k] = acc[k];
      __syncthreads();
      if (warp == 0) {
        l = 0.0f;
        acc[0] = acc[1] = acc[2] = acc[3] = 0.0f;
        for (int w = 0; w < kJoinWarps; ++w) {
          l += l_s[w];
#pragma unroll
          for (int k = 0; k < 4; ++k)
            if (k < dims) acc[k] += o_s[w][lane * dims + k];
        }
      }
    }
    if (r < rows && (few || warp == 0)) {
      T* dst = static_cast<T*>(p.a.out) + PagedRows(p, d.x, d.y * R, d.z).offset(r, p.a.on, p.a.oh) + lane * dims;
      const float inv = l > 0.0f ? 1.0f / l : 0.0f;
      if constexpr (sizeof(T) == 4) {
        if (dims == 4)
          *reinterpret_cast<float4*>(dst) = make_float4(acc[0] * inv, acc[1] * inv, acc[2] * inv, acc[3] * inv);
        else
          *reinterpret_cast<float2*>(dst) = make_float2(acc[0] * inv, acc[1] * inv);
      } else {
        const uint32_t lo = Pack2<T>::pack(acc[0] * inv, acc[1] * inv);
        if (dims == 4)
          *reinterpret_cast<uint2*>(dst) = make_uint2(lo, Pack2<T>::pack(acc[2] * inv, acc[3] * inv));
        else
          *reinterpret_cast<uint32_t*>(dst) = lo;
      }
    }
    __syncthreads();
  }
}

template <typename T>
cudaError_t launch_paged_join(const PagedParams& p, int R, int G, int TK, cudaStream_t stream) {
  if (p.a.max_kv <= TK) return cudaSuccess;  // one key tile a unit: none is split
  return launch_early(paged_join_kernel<T>, kJoinPerSm * sm_count(), kJoinThreads, 0, stream, p, R, G);
}
template cudaError_t launch_paged_join<float>(const PagedParams&, int, int, int, cudaStream_t);
template cudaError_t launch_paged_join<__nv_bfloat16>(const PagedParams&, int, int, int, cudaStream_t);
template cudaError_t launch_paged_join<__half>(const PagedParams&, int, int, int, cudaStream_t);

// CTAs worth launching: all resident ones, or fewer where the tiles cannot be more.  One where there are none (no room for
// new tokens): it reports the sequences that have some.
static int grid_for(const PagedArgs& a, int R, int TK, int resident) {
  const int64_t rt = ((int64_t)a.max_q * (a.Hq / a.Hkv) + R - 1) / R;
  const int64_t kt = std::max<int64_t>(1, ((int64_t)a.max_kv + TK - 1) / TK);
  const __int128 tiles = (__int128)a.S * rt * kt * a.Hkv;
  return tiles < 1 ? 1 : (tiles < resident ? static_cast<int>(tiles) : resident);
}

constexpr int kF32Rows = 64, kF32PerSm = 2, kF32FewPerSm = 3;

template <int D, int R, int TK, int STAGES>
static cudaError_t launch_f32(const PagedArgs& a, int per_sm, cudaStream_t stream) {
  using L = F32Layout<D, R, TK, STAGES>;
  constexpr int smem = sizeof(float) * L::FLOATS;
  auto kern = paged_attn_f32_kernel<D, R, TK, STAGES>;
  static std::atomic<uint64_t> done{0};
  cudaError_t e = allow_smem(reinterpret_cast<const void*>(kern), smem, done);
  if (e != cudaSuccess) return e;
  const int G = grid_for(a, R, TK, sm_count() * per_sm);
  const PagedParams p = paged_params(a, R, G, 1);
  e = launch_early(kern, G, L::THREADS, smem, stream, p);
  return e != cudaSuccess ? e : launch_paged_join<float>(p, R, G, TK, stream);
}

template <int D>
static cudaError_t launch_f32_rows(const PagedArgs& a, cudaStream_t stream) {
  const int64_t rows = (int64_t)a.max_q * (a.Hq / a.Hkv);
  if (rows <= 8) return launch_f32<D, 8, 32, 2>(a, kF32FewPerSm, stream);
  if (rows <= 16) return launch_f32<D, 16, 32, 2>(a, kF32FewPerSm, stream);
  return launch_f32<D, kF32Rows, 64, 1>(a, kF32PerSm, stream);
}

static cudaError_t launch_paged_f32(const PagedArgs& a, cudaStream_t stream) {
  return a.D == 128 ? launch_f32_rows<128>(a, stream) : launch_f32_rows<64>(a, stream);
}

int64_t paged_workspace_bytes(int64_t Hq, int64_t Hkv, int64_t D, int64_t max_q, int dtype) {
  if (dtype == SPRUCE_DTYPE_F32)
    return std::max(paged_params_bytes(kF32Rows, kMaxSms * kF32PerSm, D), paged_params_bytes(16, kMaxSms * kF32FewPerSm, D));
  if (max_q * (Hq / Hkv) <= kPagedRowsMax) return paged_params_bytes(kPagedRowsMax, kMaxSms * kPagedRowsPerSm, D);
  return paged_params_bytes(kPagedChunkRows, kMaxSms, D);
}

cudaError_t launch_paged_attention(const PagedArgs& a, int dtype, cudaStream_t stream) {
  if (dtype == SPRUCE_DTYPE_F32) return launch_paged_f32(a, stream);
  const int64_t rows = (int64_t)a.max_q * (a.Hq / a.Hkv);
  if (rows <= kPagedRowsMax) {
    const int tiles = rows <= 16 ? 1 : 2;
    return launch_paged_rows(a, dtype, tiles, grid_for(a, 16 * tiles, kPagedRowsKeys, sm_count() * kPagedRowsPerSm),
                             stream);
  }
  return launch_paged_chunk(a, dtype, grid_for(a, kPagedChunkRows, kPagedChunkKeys, sm_count()), stream);
}

}  // namespace spruce
