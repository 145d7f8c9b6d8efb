// Softmax weight of cached keys under few query rows: decode and drafts, bound by the HBM read of K.
//
// The formula is mass.cu's.  A warp takes 16 keys at a time as the A operand of m16n8k16 MMAs and the query rows of the
// (sequence, KV head), 8 or 16 or more of them, as B.  A dot product may take its dims in any order, so both operands are
// permuted alike: lane 4 r + c loads 16-byte chunks c, c + 4, ... of key r straight from the page into the registers that its
// fragments are (dims 8 c .. 8 c + 7 of a 32-dim step serve two MMAs), with no shared memory between; a warp load covers
// whole 64-byte pieces of 8 keys.  Q's fragments stay in registers while the warp walks its keys.
//
// Work is split as the attention's: all key tiles of the batch laid end to end, cut into equal runs, one a CTA; its warps
// take the run's tiles in turn.  A key belongs to one warp, so nothing is joined.  Bytes in flight come from the number of
// warps: a tile each of 24 warps an SM measured 50 us where two or three tiles each of 16 took 59 and 63 (CTAs of 128 or
// 256 threads alike).  Loads are marked to leave the caches first (62 -> 54 us).
//
// On a B200, 64 sequences of 300 to 8192 tokens, 28 query / 4 KV heads of 128 in bf16: 50 us, 5.7 TB/s.
#include <algorithm>
#include <type_traits>

#include "mass_common.cuh"

namespace spruce {

constexpr int kKrThreads = 128, kKrWarps = kKrThreads / 32;
constexpr int kKrTile = 16;

template <typename T>
__device__ __forceinline__ void kr_mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  if constexpr (std::is_same<T, __nv_bfloat16>::value)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// CTAs an SM: as many as the fragments of the query rows leave registers for.
template <int D, int NT> constexpr int kKrPerSm = D * NT <= 128 ? 6 : (D * NT == 512 ? 3 : 4);
constexpr int kKrPerSmF32 = 4;

// NT: tiles of 8 query rows.
template <typename T, int D, int NT>
__global__ void __launch_bounds__(kKrThreads, kKrPerSm<D, NT>) key_mass_rows_kernel(const KeyMassParams p) {
  constexpr int R = 8 * NT, CH = D / 32;  // 16-byte chunks of a row that a lane holds
  using Walk = PagedWalk<R, kKrTile>;
  __shared__ int64_t scratch[33];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, kr = lane >> 2, c = lane & 3;
  let_next_kernel_start();
  wait_for_earlier_kernels();
  Walk walk;
  if (!paged_run<R, kKrTile, kKrThreads>(p.v, walk, scratch)) return;
  PagedPiece x;
  while (walk.next(p.v, x)) {
    if (x.keys == 0) continue;
    // This lane's part of the query rows, as B fragments: row kr of each tile.
    const int rows = x.q.qlen * p.v.rep;
    const PagedRows row_at(p.v, x.q.q0, 0, x.g);
    uint4 q[NT][CH];
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int k = 0; k < CH; ++k) {
        q[t][k] = make_uint4(0, 0, 0, 0);
        if (8 * t + kr < rows)
          q[t][k] = *reinterpret_cast<const uint4*>(static_cast<const T*>(p.v.a.q) +
                                                    row_at.offset(8 * t + kr, p.v.a.qn, p.v.a.qh) + (4 * k + c) * 8);
      }
    // lse and the last key seen of the rows whose scores it holds: 2 c and 2 c + 1 of each tile.
    float lse[NT][2];
    int last[NT][2];
#pragma unroll
    for (int t = 0; t < NT; ++t)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int r = 8 * t + 2 * c + i;
        lse[t][i] = INFINITY;
        last[t][i] = -1;
        if (r < rows) {
          lse[t][i] = mass_row_lse(p.lse[row_at.offset(r, p.ln, p.lh)]);
          last[t][i] = x.q.first + row_at.token(r);
        }
      }
    const int32_t* table = p.v.a.block_table + x.s * p.v.a.table_stride;
    const T* kc = static_cast<const T*>(p.v.a.kc) + x.g * p.v.a.ks[1] + c * 8;
    struct Tile {
      uint4 k[2][CH];
      int page, slot;
      float old;  // kept of lane c's old weight
    };
    auto load = [&](int t, Tile& y) {  // sixteen keys lie in one page
      const int key = t * kKrTile;
      const int pi = key / p.v.a.page_size;
      y.slot = key - pi * p.v.a.page_size;
      y.page = paged_page(p.v, table, pi);
      if (y.page < 0) return;
      y.old = 0.0f;
      const int mine = key + kr + 8 * c;
      if (c < 2 && mine < x.q.first && p.decay != 0.0f)
        y.old = p.decay * __ldcs(p.mass + y.page * p.ms[0] + x.g * p.ms[1] + (y.slot + kr + 8 * c) * p.ms[2]);
      const T* src = kc + y.page * p.v.a.ks[0] + (y.slot + kr) * p.v.a.ks[2];
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int k = 0; k < CH; ++k) {
          y.k[i][k] = make_uint4(0, 0, 0, 0);
          if (key + kr + 8 * i < x.keys) y.k[i][k] = __ldcs(reinterpret_cast<const uint4*>(src + 8 * i * p.v.a.ks[2] + k * 32));
        }
    };
    auto use = [&](int t, const Tile& y) {
      if (y.page < 0) return;
      float sum[2] = {0.0f, 0.0f};
      const int key = t * kKrTile + kr;
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        float s[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int k = 0; k < CH; ++k) {
          kr_mma<T>(s, y.k[0][k].x, y.k[1][k].x, y.k[0][k].y, y.k[1][k].y, q[n][k].x, q[n][k].y);
          kr_mma<T>(s, y.k[0][k].z, y.k[1][k].z, y.k[0][k].w, y.k[1][k].w, q[n][k].z, q[n][k].w);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float e = fast_exp2(fmaf(s[i], p.v.scale_log2, -lse[n][i & 1]));
          sum[i >> 1] += key + 8 * (i >> 1) <= last[n][i & 1] ? e : 0.0f;
        }
      }
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        sum[i] += __shfl_xor_sync(0xffffffffu, sum[i], 1);
        sum[i] += __shfl_xor_sync(0xffffffffu, sum[i], 2);
      }
      // Lanes c = 0 and 1 store keys kr and kr + 8.
      const int mine = key + 8 * c;
      if (c < 2 && mine < x.keys)
        p.out[y.page * p.os[0] + x.g * p.os[1] + (y.slot + kr + 8 * c) * p.os[2]] = (c == 0 ? sum[0] : sum[1]) + y.old;
    };
    Tile a;
    for (int t = x.t0 + warp; t < x.t1; t += kKrWarps) {
      load(t, a);
      use(t, a);
    }
  }
}

// ------------------------------------------------------------------ fp32
// Eight lanes a key, each with D / 8 dims of it; the query rows come from shared memory.  Eight rows' partial dots are summed over the
// lanes by a transposing butterfly (7 shuffles), which leaves row c with lane c.  16 sequences of 2000 to 8000 tokens, 28 / 4 heads of
// 128: 36 us, 4.5 TB/s.
template <int D, int NT>
__global__ void __launch_bounds__(kKrThreads, kKrPerSmF32) key_mass_rows_f32_kernel(const KeyMassParams p) {
  constexpr int R = 8 * NT, CH = D / 32;
  using Walk = PagedWalk<R, kKrTile>;
  __shared__ __align__(16) float Q[R][D];
  __shared__ int64_t scratch[33];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, kr = lane >> 3, c = lane & 7;
  let_next_kernel_start();
  wait_for_earlier_kernels();
  Walk walk;
  if (!paged_run<R, kKrTile, kKrThreads>(p.v, walk, scratch)) return;
  PagedPiece x;
  while (walk.next(p.v, x)) {
    const int rows = x.q.qlen * p.v.rep;
    const PagedRows row_at(p.v, x.q.q0, 0, x.g);
    __syncthreads();
    for (int e = threadIdx.x; e < R * (D / 4); e += kKrThreads) {
      const int r = e / (D / 4), d = e % (D / 4) * 4;
      float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      if (r < rows) v = *reinterpret_cast<const float4*>(static_cast<const float*>(p.v.a.q) + row_at.offset(r, p.v.a.qn, p.v.a.qh) + d);
      *reinterpret_cast<float4*>(&Q[r][d]) = v;
    }
    __syncthreads();
    if (x.keys == 0) continue;
    float lse[NT];   // of row 8 t + c
    int last[NT];
#pragma unroll
    for (int t = 0; t < NT; ++t) {
      lse[t] = INFINITY;
      last[t] = -1;
      if (8 * t + c < rows) {
        lse[t] = mass_row_lse(p.lse[row_at.offset(8 * t + c, p.ln, p.lh)]);
        last[t] = x.q.first + row_at.token(8 * t + c);
      }
    }
    const int32_t* table = p.v.a.block_table + x.s * p.v.a.table_stride;
    const float* kc = static_cast<const float*>(p.v.a.kc) + x.g * p.v.a.ks[1] + c * 4;
    for (int tile = x.t0 + warp; tile < x.t1; tile += kKrWarps) {
      const int key0 = tile * kKrTile, pi = key0 / p.v.a.page_size, slot = key0 - pi * p.v.a.page_size;
      const int page = paged_page(p.v, table, pi);  // sixteen keys lie in one page
      if (page < 0) continue;
      float4 k[4][CH];
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < CH; ++j) {
          k[i][j] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
          if (key0 + 4 * i + kr < x.keys)
            k[i][j] = __ldcs(reinterpret_cast<const float4*>(kc + page * p.v.a.ks[0] + (slot + 4 * i + kr) * p.v.a.ks[2] + j * 32));
        }
      float old = 0.0f;  // of key 4 c + kr, which lanes c < 4 write
      const int mine = key0 + 4 * c + kr;
      if (c < 4 && mine < x.q.first && p.decay != 0.0f)
        old = p.decay * p.mass[page * p.ms[0] + x.g * p.ms[1] + (slot + 4 * c + kr) * p.ms[2]];
      float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        float s[4][8];
#pragma unroll
        for (int r = 0; r < 8; ++r) {
#pragma unroll
          for (int i = 0; i < 4; ++i) s[i][r] = 0.0f;
#pragma unroll
          for (int j = 0; j < CH; ++j) {
            const float4 q = *reinterpret_cast<const float4*>(&Q[8 * t + r][j * 32 + c * 4]);
#pragma unroll
            for (int i = 0; i < 4; ++i)
              s[i][r] = fmaf(q.x, k[i][j].x, fmaf(q.y, k[i][j].y, fmaf(q.z, k[i][j].z, fmaf(q.w, k[i][j].w, s[i][r]))));
          }
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
#pragma unroll
          for (int o = 4; o > 0; o >>= 1) {
            const bool up = c & o;
#pragma unroll
            for (int r = 0; r < o; ++r) {
              const float send = up ? s[i][r] : s[i][r + o], keep = up ? s[i][r + o] : s[i][r];
              s[i][r] = keep + __shfl_xor_sync(0xffffffffu, send, o);
            }
          }
          const float e = exp2f(s[i][0] * p.v.scale_log2 - lse[t]);
          sum[i] += key0 + 4 * i + kr <= last[t] ? e : 0.0f;
        }
      }
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int o = 4; o > 0; o >>= 1) sum[i] += __shfl_xor_sync(0xffffffffu, sum[i], o);
      if (c < 4 && mine < x.keys)
        p.out[page * p.os[0] + x.g * p.os[1] + (slot + 4 * c + kr) * p.os[2]] =
            (c == 0 ? sum[0] : (c == 1 ? sum[1] : (c == 2 ? sum[2] : sum[3]))) + old;
    }
  }
}

template <typename T, int D, int NT>
static cudaError_t launch(const KeyMassArgs& a, cudaStream_t stream) {
  KeyMassParams p = key_mass_params(a, kKrTile);
  p.v = paged_params(a.a, 8 * NT, 1, 4);
  const int64_t tiles = (int64_t)a.a.S * p.key_tiles * a.a.Hkv;
  const int64_t ctas = std::min<int64_t>((tiles + kKrWarps - 1) / kKrWarps, sm_count() * kKrPerSm<D, NT>);
  return launch_early(key_mass_rows_kernel<T, D, NT>, static_cast<int>(std::max<int64_t>(1, ctas)), kKrThreads, 0, stream, p);
}

template <typename T, int D>
static cudaError_t launch_tiles(const KeyMassArgs& a, cudaStream_t stream) {
  const int64_t rows = (int64_t)a.a.max_q * (a.a.Hq / a.a.Hkv);
  if (rows <= 8) return launch<T, D, 1>(a, stream);
  if (rows <= 16) return launch<T, D, 2>(a, stream);
  return launch<T, D, 4>(a, stream);
}

template <int D, int NT>
static cudaError_t launch_f32(const KeyMassArgs& a, cudaStream_t stream) {
  KeyMassParams p = key_mass_params(a, kKrTile);
  p.v = paged_params(a.a, 8 * NT, 1, 4);
  const int64_t tiles = (int64_t)a.a.S * p.key_tiles * a.a.Hkv;
  const int64_t ctas = std::min<int64_t>((tiles + kKrWarps - 1) / kKrWarps, sm_count() * kKrPerSmF32);
  return launch_early(key_mass_rows_f32_kernel<D, NT>, static_cast<int>(std::max<int64_t>(1, ctas)), kKrThreads, 0, stream, p);
}

cudaError_t launch_key_mass_rows(const KeyMassArgs& a, int dtype, cudaStream_t stream) {
  if (dtype == SPRUCE_DTYPE_F32) {
    const bool eight = (int64_t)a.a.max_q * (a.a.Hq / a.a.Hkv) <= 8;
    if (a.a.D == 128) return eight ? launch_f32<128, 1>(a, stream) : launch_f32<128, 2>(a, stream);
    return eight ? launch_f32<64, 1>(a, stream) : launch_f32<64, 2>(a, stream);
  }
  if (dtype == SPRUCE_DTYPE_BF16)
    return a.a.D == 128 ? launch_tiles<__nv_bfloat16, 128>(a, stream) : launch_tiles<__nv_bfloat16, 64>(a, stream);
  return a.a.D == 128 ? launch_tiles<__half, 128>(a, stream) : launch_tiles<__half, 64>(a, stream);
}

}  // namespace spruce
