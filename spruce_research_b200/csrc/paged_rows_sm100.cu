// Attention of single tokens and short drafts over a paged K/V cache (bf16 / fp16): up to 32 query rows a (sequence,
// KV head), bound by the HBM reads of K and V.
//
// The mathematics, the split of the work and its join are those of paged_common.cuh and paged_attn.cu.  Each byte of K
// and V meets 2 R flops a 16-bit value, far below the tensor cores' balance, so the tcgen05 path's 128-row tiles and their trip
// through TMEM would only add latency; warp-level MMAs (m16n8k16) on fragments from shared memory keep up with HBM.
//
// A CTA has one loader warp and four compute warps.  The loader keeps STAGES tiles of 64 keys (K and V) in flight by TMA,
// page by page, across the borders of units; page ids come 32 boxes at a time, one batch ahead.  MT = 1 or 2
// 16-row tiles (R = 16 MT) times 4 / MT slices of a tile's keys are dealt to the compute warps.  Each keeps its own
// running maximum, sum and output, so the warps meet only at the end of a piece, where slices are joined through
// shared memory.  Two CTAs an SM: one's joins and starts pass behind the other's loads.
//
// P is rounded to the inputs' type for its product with V, scaled as PScale says; sums, maxima and O are fp32.
//
// Cache rows past the sequence's end may hold anything: their scores are masked by selection and their V
// fragments cleared.
//
// Measured on a B200 (28 query / 4 KV heads, d = 128, bf16): 64 sequences of 300 to 8192 tokens 98 us (5.7 TB/s with the
// join), one of 131072 tokens 56 us (4.8 TB/s), pages of 16 or 64 tokens alike; CTAs on the slowest eighth of the SMs end
// 10-13% after the mean.  Four 16-row tiles (33 to 64 rows) took 59.8 us where the tcgen05 kernel takes 49.5.
// At d = 128 the 168 registers of two CTAs an SM leave 40 to 52 bytes of a thread spilled.
#include <algorithm>
#include <type_traits>

#include "attn_common.cuh"
#include "paged_common.cuh"

namespace spruce {

constexpr int kRowsThreads = 160;
constexpr int kRowsLoader = 4;
constexpr int kRowsKeys = kPagedRowsKeys;

template <int D>
struct RowsLayout {
  static constexpr int STAGES = D == 128 ? 3 : 6;
  static constexpr int NP = D / 64;
  static constexpr int PANEL = kRowsKeys * 128;
  static constexpr int TILE = NP * PANEL;            // K or V of a stage
  static constexpr int OFF_JOIN = STAGES * 2 * TILE;
  static constexpr int JOIN_ROW = 40;                // floats: 32 columns a round, rows 8 banks apart
  static constexpr int OFF_ML = OFF_JOIN + 64 * JOIN_ROW * 4;
  static constexpr int OFF_BAR = OFF_ML + 64 * 8;
  static constexpr int OFF_SCAN = OFF_BAR + 2 * STAGES * 8;
  static constexpr int OFF_MISC = OFF_SCAN + 33 * 8;
  static constexpr int BYTES = 1024 + OFF_MISC + 16;
};

__device__ __forceinline__ void ldmatrix4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldmatrix4t(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
template <typename T>
__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (std::is_same<T, __nv_bfloat16>::value)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

template <typename T, int D, int MT>
__global__ void __launch_bounds__(kRowsThreads, 2)
    paged_rows_sm100_kernel(const __grid_constant__ CUtensorMap tmk, const __grid_constant__ CUtensorMap tmv,
                            const PagedParams p, int box) {
  using L = RowsLayout<D>;
  constexpr int STAGES = L::STAGES;
  constexpr int R = 16 * MT, KS = 4 / MT, SLICE = kRowsKeys / KS;
  using Walk = PagedWalk<R, kRowsKeys>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  uint32_t* const status = p.a.status;
  uint64_t* full = reinterpret_cast<uint64_t*>(smem + L::OFF_BAR);
  uint64_t* empty = full + STAGES;
  int64_t* scan = reinterpret_cast<int64_t*>(smem + L::OFF_SCAN);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + L::OFF_MISC);

  if (threadIdx.x == 0) {
    *abort_flag = 0;
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 4);
    }
    fence_barrier_init();
    prefetch_tmap(&tmk);
    prefetch_tmap(&tmv);
  }
  let_next_kernel_start();
  wait_for_earlier_kernels();
  Walk walk;
  const bool any = paged_run<R, kRowsKeys, kRowsThreads>(p, walk, scan);
  __syncthreads();
  if (!any) walk.left = 0;
  PagedPiece x;

  if (warp == kRowsLoader) {
    // ------------------------------------------------------------ K and V
    const int nb = kRowsKeys / box;           // boxes of rows a tile: 1, 2 or 4
    const int pp = lane % L::NP, bi = lane / L::NP;
    const bool mine = lane < nb * L::NP;
    int j = 0;
    bool ok = true;
    while (ok && walk.next(p, x)) {
      if (x.keys == 0) continue;
      const int32_t* table = p.a.block_table + x.s * p.a.table_stride;
      // Page and row of the unit's box number k; past the keys (or the table): a page index that reads zeros.
      const int last = min(x.t1 * kRowsKeys, x.keys);
      auto page_of = [&](int k) {
        const int key = k * box;
        if (key >= last) return static_cast<int>(p.a.num_pages);
        const int page = paged_page(p, table, key / p.a.page_size);
        return page < 0 ? static_cast<int>(p.a.num_pages) : page;
      };
      int base = x.t0 * nb;
      int cur = page_of(base + lane), nxt = page_of(base + 32 + lane);
      for (int t = x.t0; t < x.t1; ++t, ++j) {
        if (t * nb - base == 32) {
          base += 32;
          cur = nxt;
          nxt = page_of(base + 32 + lane);
        }
        const int st = j % STAGES;
        if (j >= STAGES && !__all_sync(0xffffffffu, mbar_wait(&empty[st], ((j / STAGES) - 1) & 1, status, abort_flag))) {
          ok = false;
          break;
        }
        const int page = __shfl_sync(0xffffffffu, cur, (t * nb + bi - base) & 31);
        if (lane == 0) mbar_arrive_expect_tx(&full[st], 2 * L::TILE);
        __syncwarp();
        if (mine) {
          uint8_t* ks = smem + st * 2 * L::TILE + pp * L::PANEL + bi * box * 128;
          const int row = (t * kRowsKeys + bi * box) % p.a.page_size;
          tma_load_4d(ks, &tmk, &full[st], pp * 64, row, x.g, page);
          tma_load_4d(ks + L::TILE, &tmv, &full[st], pp * 64, row, x.g, page);
        }
      }
    }
    for (int i = max(0, j - STAGES); i < j; ++i) mbar_wait(&full[i % STAGES], (i / STAGES) & 1, status, nullptr);
    return;
  }

  // ------------------------------------------------------------ compute
  const int mt = warp % MT, ks = warp / MT;
  const int qr = lane >> 2, qc = lane & 3;  // fragment row and column pair
  float* join = reinterpret_cast<float*>(smem + L::OFF_JOIN);
  float2* ml = reinterpret_cast<float2*>(smem + L::OFF_ML);
  int4 mine = make_int4(0, 0, 0, 0);
  int j = 0;
  bool ok = true;
  while (walk.next(p, x)) {  // after a wait that ran out the warps still meet at the joins' barriers
    const int rows = min(R, x.q.qlen * p.rep - x.qt * R);
    if (x.parts > 0) mine = paged_desc(x, rows);
    const PagedRows row_at(p, x.q.q0, x.qt * R, x.g);
    uint32_t q[D / 16][4];
    int seen[2];  // keys that this thread's two rows see
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int r = mt * 16 + qr + 8 * i;
      const uint32_t* src = nullptr;
      if (r < rows) {
        src = reinterpret_cast<const uint32_t*>(static_cast<const T*>(p.a.q) + row_at.offset(r, p.a.qn, p.a.qh));
      }
      seen[i] = min(x.q.first + row_at.token(r) + 1, x.keys);
#pragma unroll
      for (int k = 0; k < D / 16; ++k) {
        q[k][i] = src != nullptr ? src[k * 8 + qc] : 0u;
        q[k][2 + i] = src != nullptr ? src[k * 8 + 4 + qc] : 0u;
      }
    }
    float o[D / 8][4];
#pragma unroll
    for (int n = 0; n < D / 8; ++n)
#pragma unroll
      for (int i = 0; i < 4; ++i) o[n][i] = 0.0f;
    float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f};

    const int n_tiles = x.keys == 0 ? 0 : x.t1 - x.t0;
    for (int i = 0; ok && i < n_tiles; ++i, ++j) {
      const int st = j % STAGES;
      ok = __all_sync(0xffffffffu, mbar_wait(&full[st], (j / STAGES) & 1, status, abort_flag));
      if (!ok) break;
      const uint32_t kb = smem_u32(smem + st * 2 * L::TILE), vb = kb + L::TILE;
#pragma unroll
      for (int sub = 0; sub < SLICE / 16; ++sub) {
        const int k0 = ks * SLICE + sub * 16;              // first of 16 keys of the tile
        const int key0 = (x.t0 + i) * kRowsKeys + k0;
        // S = Q K^T for 16 rows x 16 keys; two accumulators a key group shorten the chain.
        float s[2][2][4] = {};
        {
          const int key = k0 + (lane >> 4) * 8 + (lane & 7);
          const uint32_t row = kb + key * 128;
#pragma unroll
          for (int k = 0; k < D / 16; ++k) {
            const int chunk = 2 * k + ((lane >> 3) & 1);
            uint32_t b[4];
            ldmatrix4(b, row + (chunk >> 3) * L::PANEL + (((chunk & 7) ^ (key & 7)) << 4));
            mma16816<T>(s[k & 1][0], q[k], b[0], b[1]);
            mma16816<T>(s[k & 1][1], q[k], b[2], b[3]);
          }
        }
        float e[2][4];
        const bool whole = key0 + 16 <= min(seen[0], seen[1]);
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            e[n][c] = (s[0][n][c] + s[1][n][c]) * p.scale_log2;
            if (!whole && key0 + n * 8 + qc * 2 + (c & 1) >= seen[c >> 1]) e[n][c] = -INFINITY;
          }
        uint32_t pa[4];
        float alpha[2];
#pragma unroll
        for (int i2 = 0; i2 < 2; ++i2) {
          float mx = fmaxf(fmaxf(e[0][2 * i2], e[0][2 * i2 + 1]), fmaxf(e[1][2 * i2], e[1][2 * i2 + 1]));
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
          const float m_new = fmaxf(m[i2], mx);
          const float ref = m_new == -INFINITY ? 0.0f : m_new;
          alpha[i2] = fast_exp2(m[i2] - ref);
          m[i2] = m_new;
          const float low = ref - PScale<T>::log2;
          const float e0 = fast_exp2(e[0][2 * i2] - low), e1 = fast_exp2(e[0][2 * i2 + 1] - low);
          const float e2 = fast_exp2(e[1][2 * i2] - low), e3 = fast_exp2(e[1][2 * i2 + 1] - low);
          l[i2] = l[i2] * alpha[i2] + ((e0 + e1) + (e2 + e3));
          pa[i2] = Pack2<T>::pack(e0, e1);
          pa[2 + i2] = Pack2<T>::pack(e2, e3);
        }
        if (__any_sync(0xffffffffu, alpha[0] != 1.0f || alpha[1] != 1.0f)) {
#pragma unroll
          for (int n = 0; n < D / 8; ++n)
#pragma unroll
            for (int c = 0; c < 4; ++c) o[n][c] *= alpha[c >> 1];
        }
        // O += P V; V rows past the keys are cleared.
        const int left = x.keys - key0;  // keys of these 16 that exist
        uint32_t keep[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int a = h * 8 + qc * 2;
          keep[h] = (a < left ? 0x0000ffffu : 0u) | (a + 1 < left ? 0xffff0000u : 0u);
        }
        const int key = k0 + ((lane >> 3) & 1) * 8 + (lane & 7);
        const uint32_t row = vb + key * 128;
#pragma unroll
        for (int n = 0; n < D / 16; ++n) {
          const int chunk = 2 * n + (lane >> 4);
          uint32_t b[4];
          ldmatrix4t(b, row + (chunk >> 3) * L::PANEL + (((chunk & 7) ^ (key & 7)) << 4));
          if (left < 16) {
            b[0] &= keep[0];
            b[1] &= keep[1];
            b[2] &= keep[0];
            b[3] &= keep[1];
          }
          mma16816<T>(o[2 * n], pa, b[0], b[1]);
          mma16816<T>(o[2 * n + 1], pa, b[2], b[3]);
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&empty[st]);
    }

    // Join the key slices: factors to the rows' common maximum, then 32 columns a round through shared memory.
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      l[i] += __shfl_xor_sync(0xffffffffu, l[i], 1);
      l[i] += __shfl_xor_sync(0xffffffffu, l[i], 2);
      if (qc == 0) ml[warp * 16 + qr + 8 * i] = make_float2(m[i], l[i]);
    }
    named_barrier_sync(1, 128);
    const bool whole = x.slot < 0;
    const int64_t part = (int64_t)(2 * blockIdx.x + x.slot) * R;  // of the partial rows
    float f[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int r = mt * 16 + qr + 8 * i;
      float top = -INFINITY, sum = 0.0f;
#pragma unroll
      for (int w = 0; w < KS; ++w) top = fmaxf(top, ml[w * R + r].x);
      const float ref = top == -INFINITY ? 0.0f : top;
#pragma unroll
      for (int w = 0; w < KS; ++w) sum += ml[w * R + r].y * fast_exp2(ml[w * R + r].x - ref);
      f[i] = fast_exp2(m[i] - ref);
      if (whole) {
        f[i] *= sum > 0.0f ? 1.0f / sum : 0.0f;
        if (p.a.lse != nullptr && ks == 0 && qc == 0 && r < rows)
          p.a.lse[row_at.offset(r, p.a.ln, p.a.lh)] = paged_lse(p, top, sum);
      } else if (ks == 0 && qc == 0 && r < rows)
        p.part_ml[part + r] = make_float2(top, sum);
    }
    const int wr = threadIdx.x >> 3, wc = (threadIdx.x & 7) * 4;  // written by this thread: row of each 16, 4 columns
#pragma unroll
    for (int c0 = 0; c0 < D; c0 += 32) {
#pragma unroll
      for (int n = 0; n < 4; ++n) {
        float* dst = join + (warp * 16 + qr) * L::JOIN_ROW + n * 8 + qc * 2;
        const float (&v)[4] = o[c0 / 8 + n];
        *reinterpret_cast<float2*>(dst) = make_float2(v[0] * f[0], v[1] * f[0]);
        *reinterpret_cast<float2*>(dst + 8 * L::JOIN_ROW) = make_float2(v[2] * f[1], v[3] * f[1]);
      }
      named_barrier_sync(1, 128);
#pragma unroll 1
      for (int r = wr; r < rows; r += 16) {
        float4 sum = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
        for (int w = 0; w < KS; ++w) {
          const float4 v = *reinterpret_cast<const float4*>(join + (w * R + r) * L::JOIN_ROW + wc);
          sum.x += v.x;
          sum.y += v.y;
          sum.z += v.z;
          sum.w += v.w;
        }
        if (whole) {
          uint2 v;
          v.x = Pack2<T>::pack(sum.x, sum.y);
          v.y = Pack2<T>::pack(sum.z, sum.w);
          *reinterpret_cast<uint2*>(static_cast<T*>(p.a.out) + row_at.offset(r, p.a.on, p.a.oh) + c0 + wc) = v;
        } else {
          *reinterpret_cast<float4*>(p.part_o + (part + r) * D + c0 + wc) = sum;
        }
      }
      named_barrier_sync(1, 128);
    }
  }
  if (threadIdx.x == 0) p.desc[blockIdx.x] = mine;
}

template <typename T, int D, int MT>
static cudaError_t launch_rows(const PagedArgs& a, int dtype, int G, cudaStream_t stream) {
  using L = RowsLayout<D>;
  CUtensorMap mk, mv;
  const int box = paged_box(a.page_size, kRowsKeys);
  if (!paged_cache_maps(a, dtype, box, &mk, &mv)) return cudaErrorInvalidValue;
  auto kern = paged_rows_sm100_kernel<T, D, MT>;
  static std::atomic<uint64_t> done{0};
  cudaError_t e = allow_smem(reinterpret_cast<const void*>(kern), L::BYTES, done);
  if (e != cudaSuccess) return e;
  const PagedParams p = paged_params(a, 16 * MT, G, 1, PScale<T>::log2);
  e = launch_early(kern, G, kRowsThreads, L::BYTES, stream, mk, mv, p, box);
  return e != cudaSuccess ? e : launch_paged_join<T>(p, 16 * MT, G, kRowsKeys, stream);
}

template <typename T, int D>
static cudaError_t launch_rows_tiles(const PagedArgs& a, int dtype, int tiles, int G, cudaStream_t stream) {
  if (tiles == 1) return launch_rows<T, D, 1>(a, dtype, G, stream);
  return launch_rows<T, D, 2>(a, dtype, G, stream);
}

cudaError_t launch_paged_rows(const PagedArgs& a, int dtype, int tiles, int G, cudaStream_t stream) {
  if (dtype == SPRUCE_DTYPE_BF16)
    return a.D == 128 ? launch_rows_tiles<__nv_bfloat16, 128>(a, dtype, tiles, G, stream)
                      : launch_rows_tiles<__nv_bfloat16, 64>(a, dtype, tiles, G, stream);
  return a.D == 128 ? launch_rows_tiles<__half, 128>(a, dtype, tiles, G, stream)
                    : launch_rows_tiles<__half, 64>(a, dtype, tiles, G, stream);
}

}  // namespace spruce
