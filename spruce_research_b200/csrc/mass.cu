// Softmax weight that keys receive, on the CUDA cores: of each cached key (spruce_paged_key_mass) and of whole key blocks
// (spruce_block_mass).
//
//   key mass:    out[j] = decay mass[j] + sum over rows r that see j of 2^(q_r.k_j scale log2(e) - lse_r log2(e))
//   block mass:  out[i][j] = mean over the rows r of query block i of sum_{u in block j} p_ru,  p_r = softmax of row r
//
// A row of the key mass is a (token, head of the group); its lse comes from the attention that it ran anyway, so one
// pass over the keys is enough, and a key's sum belongs to one CTA: no atomics, the order is fixed.  The block mass goes
// over the scores once as well: for every row and key block it keeps b = log2(sum of 2^s over the block), from which the
// row's total and then every weight 2^(b - total) follow, one exponential a (row, block) more.
//
// 16-bit inputs have tensor-core kernels (key_mass_rows.cu, key_mass_sm100.cu, block_mass_sm100.cu); these serve fp32, and key
// mass with more than 128 heads a group.  Bound by the FMA pipe and shared-memory reads (4 x 4 scores a thread: 8 wavefronts to 64
// FMAs).  On a B200 in fp32, 28 / 4 heads of 128: 64 tokens over 16K 280 us (26 TFLOP/s), block mass of 4000 tokens 3.1 ms
// (19 TFLOP/s).
#include <algorithm>

#include "mass_common.cuh"

namespace spruce {

constexpr int kTileKeys = 64, kTileRows = 64, kTileThreads = 256;

// Four elements of a row as floats.
template <typename T>
__device__ __forceinline__ float4 load4(const T* p) {
  if constexpr (sizeof(T) == 4) {
    return *reinterpret_cast<const float4*>(p);
  } else {
    const uint2 v = *reinterpret_cast<const uint2*>(p);
    const T* e = reinterpret_cast<const T*>(&v);
    return make_float4(Elem<T>::to_f(e[0]), Elem<T>::to_f(e[1]), Elem<T>::to_f(e[2]), Elem<T>::to_f(e[3]));
  }
}

// Scores of a tile: rows a0 .. of A (R of them, thread rows ra + 16 i) by 64 rows of B (4 a thread, 4 rb ..).
template <int D, int N, int M>
__device__ __forceinline__ void tile_scores(const float* A, int ra, const float* B, int rb, float (&s)[N][M]) {
  constexpr int P = D + 4;
#pragma unroll
  for (int i = 0; i < N; ++i)
#pragma unroll
    for (int j = 0; j < M; ++j) s[i][j] = 0.0f;
#pragma unroll 4
  for (int d = 0; d < D; d += 4) {
    float4 a[N], b[M];
#pragma unroll
    for (int i = 0; i < N; ++i) a[i] = *reinterpret_cast<const float4*>(A + (ra + 16 * i) * P + d);
#pragma unroll
    for (int j = 0; j < M; ++j) b[j] = *reinterpret_cast<const float4*>(B + (rb * M + j) * P + d);
#pragma unroll
    for (int i = 0; i < N; ++i)
#pragma unroll
      for (int j = 0; j < M; ++j)
        s[i][j] = fmaf(a[i].x, b[j].x, fmaf(a[i].y, b[j].y, fmaf(a[i].z, b[j].z, fmaf(a[i].w, b[j].w, s[i][j]))));
  }
}

// ------------------------------------------------------------------ key mass
// One (sequence, KV head, 64 keys) at a time; R query rows a step.
template <typename T, int D>
__global__ void __launch_bounds__(kTileThreads) key_mass_tile_kernel(const KeyMassParams p) {
  constexpr int R = kTileRows, P = D + 4, N = R / 16;
  extern __shared__ float sm[];
  float* Ks = sm;                      // [64][P]
  float* Qs = Ks + kTileKeys * P;      // [R][P]
  float* Ls = Qs + R * P;              // [R] lse in log2 units; +inf where a row counts for nothing
  int* Ts = reinterpret_cast<int*>(Ls + R);  // [R] last key the row sees
  __shared__ int pages[kTileKeys / 16];
  const int tid = threadIdx.x, rr = tid % 16, kk = tid / 16;
  const int64_t per_seq = (int64_t)p.key_tiles * p.v.a.Hkv, items = per_seq * p.v.a.S;
  for (int64_t item = blockIdx.x; item < items; item += gridDim.x) {
    const int s = static_cast<int>(item / per_seq), rest = static_cast<int>(item % per_seq);
    const int g = rest / p.key_tiles, key0 = rest % p.key_tiles * kTileKeys;
    const PagedSeq q = paged_seq(p.v, s);
    const int keys = mass_keys(q);
    if (q.qlen == 0 || key0 >= keys) continue;
    __syncthreads();
    if (tid < kTileKeys / 16) pages[tid] = mass_page(p, s, key0 + 16 * tid, keys);
    __syncthreads();
    for (int e = tid; e < kTileKeys * (D / 4); e += kTileThreads) {
      const int r = e / (D / 4), d = e % (D / 4) * 4, key = key0 + r, page = pages[r / 16];
      float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      if (page >= 0 && key < keys)
        v = load4(static_cast<const T*>(p.v.a.kc) + page * p.v.a.ks[0] + g * p.v.a.ks[1] + key % p.v.a.page_size * p.v.a.ks[2] + d);
      *reinterpret_cast<float4*>(Ks + r * P + d) = v;
    }
    float acc[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    const int rows = q.qlen * p.v.rep;
    // Tokens before the tile's first key do not see it.
    for (int r0 = max(0, key0 - q.first) * p.v.rep; r0 < rows; r0 += R) {
      const PagedRows row_at(p.v, q.q0, r0, g);
      __syncthreads();
      for (int e = tid; e < R * (D / 4); e += kTileThreads) {
        const int r = e / (D / 4), d = e % (D / 4) * 4;
        float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        if (r0 + r < rows) v = load4(static_cast<const T*>(p.v.a.q) + row_at.offset(r, p.v.a.qn, p.v.a.qh) + d);
        *reinterpret_cast<float4*>(Qs + r * P + d) = v;
      }
      if (tid < R) {
        Ls[tid] = INFINITY;
        Ts[tid] = -1;
        if (r0 + tid < rows) {
          Ls[tid] = mass_row_lse(p.lse[row_at.offset(tid, p.ln, p.lh)]);
          Ts[tid] = q.first + row_at.token(tid);
        }
      }
      __syncthreads();
      float sc[N][4];
      tile_scores<D, N, 4>(Qs, rr, Ks, kk, sc);
#pragma unroll
      for (int i = 0; i < N; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (key0 + kk * 4 + j <= Ts[rr + 16 * i]) acc[j] += exp2f(sc[i][j] * p.v.scale_log2 - Ls[rr + 16 * i]);
    }
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int o = 8; o > 0; o >>= 1) acc[j] += __shfl_xor_sync(0xffffffffu, acc[j], o);
    if (rr < 4) {
      const int key = key0 + kk * 4 + rr, page = pages[kk / 4];
      const float sum = rr == 0 ? acc[0] : (rr == 1 ? acc[1] : (rr == 2 ? acc[2] : acc[3]));
      if (page >= 0 && key < keys) mass_store(p, page, g, key % p.v.a.page_size, key < q.first, sum);
    }
  }
}

template <typename T, int D>
static cudaError_t launch_tile(const KeyMassArgs& a, int sms, cudaStream_t stream) {
  constexpr int R = kTileRows, smem = sizeof(float) * ((kTileKeys + R) * (D + 4) + 2 * R);
  auto kern = key_mass_tile_kernel<T, D>;
  static std::atomic<uint64_t> done{0};
  cudaError_t e = allow_smem(reinterpret_cast<const void*>(kern), smem, done);
  if (e != cudaSuccess) return e;
  const KeyMassParams p = key_mass_params(a, kTileKeys);
  const int64_t items = (int64_t)a.a.S * p.key_tiles * a.a.Hkv;
  kern<<<static_cast<int>(std::min<int64_t>(items, 16 * sms)), kTileThreads, smem, stream>>>(p);
  return cudaGetLastError();
}

template <typename T>
static cudaError_t launch_key_mass_t(const KeyMassArgs& a, int sms, cudaStream_t stream) {
  return a.a.D == 128 ? launch_tile<T, 128>(a, sms, stream) : launch_tile<T, 64>(a, sms, stream);
}

// fp32 rows by the lanes of a warp where they are few: 16 sequences of 2000 to 8000 tokens, 28 / 4 heads of 128: 7 rows 36 us, by tiles
// of 64 rows 223, 14 rows 52 and 226; one of 131000 54 and 336, 79 and 345.
// 16 bits by warp MMAs where rows are few, which read K at full rate: 64 sequences of 300 to 8191 tokens, 7 / 14 / 28 rows 50 / 59 / 76
// us, on tcgen05 100 / 95 / 97; one of 131000 28 / 32 / 41 and 44 / 44 / 46.  With one KV head and 24 or 32 rows the two are even on one
// long sequence (16.0 and 15.4, 16.4 and 15.3) and 25 to 37 us on 64.  Groups of more heads than a row tile has rows take the tiles.
cudaError_t launch_key_mass(const KeyMassArgs& a, int dtype, cudaStream_t stream) {
  const int sms = sm_count();
  if (key_mass_params(a, kTileKeys).key_tiles == 0) return cudaSuccess;
  const int rep = a.a.Hq / a.a.Hkv;
  const int64_t rows = (int64_t)a.a.max_q * rep;
  if (rows <= (dtype == SPRUCE_DTYPE_F32 ? kKmFewRowsF32 : kKmFewRows)) return launch_key_mass_rows(a, dtype, stream);
  if (dtype == SPRUCE_DTYPE_F32) return launch_key_mass_t<float>(a, sms, stream);
  if (rep <= 128) return launch_key_mass_sm100(a, dtype, stream);
  return dtype == SPRUCE_DTYPE_BF16 ? launch_key_mass_t<__nv_bfloat16>(a, sms, stream) : launch_key_mass_t<__half>(a, sms, stream);
}

// ------------------------------------------------------------------ block mass
// One (batch, KV head, query block) at a time: its heads one after another, 64 x 64 scores a step.
template <int D>
__global__ void __launch_bounds__(kTileThreads) block_mass_tile_kernel(const BlockMassArgs a, int qb) {
  constexpr int P = D + 4;
  extern __shared__ float sm[];
  float* Qs = sm;                       // [64][P]
  float* Ks = Qs + 64 * P;              // [64][P]
  float* Ls = Ks + 64 * P;              // [64] total of each row, log2 units
  const int tid = threadIdx.x, kk = tid % 16, rr = tid / 16;
  const int rep = a.Hq / a.Hkv;
  float* blocks = a.workspace + (int64_t)blockIdx.x * qb * 64;  // [key block][row]
  const int64_t items = (int64_t)a.B * a.Hkv * qb;
  for (int64_t item = blockIdx.x; item < items; item += gridDim.x) {
    const int i = qb - 1 - static_cast<int>(item / (a.B * a.Hkv));  // the longest first
    const int bg = static_cast<int>(item % (a.B * a.Hkv)), b = bg / a.Hkv, g = bg % a.Hkv;
    const int tokens = min(64, a.T - i * 64);
    float* out = a.out + ((int64_t)bg * qb + i) * qb;
    for (int h = 0; h < rep; ++h) {
      __syncthreads();
      const float* q = static_cast<const float*>(a.q) + b * a.qs[0] + (g * rep + h) * a.qs[1];
      for (int e = tid; e < 64 * (D / 4); e += kTileThreads) {
        const int r = e / (D / 4), d = e % (D / 4) * 4;
        float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        if (r < tokens) v = load4(q + (i * 64 + r) * a.qs[2] + d);
        *reinterpret_cast<float4*>(Qs + r * P + d) = v;
      }
      float m[4], l[4];
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        m[x] = -INFINITY;
        l[x] = 0.0f;
      }
      const float* k = static_cast<const float*>(a.k) + b * a.ks[0] + g * a.ks[1];
      for (int j = 0; j <= i; ++j) {
        __syncthreads();
        for (int e = tid; e < 64 * (D / 4); e += kTileThreads) {
          const int r = e / (D / 4), d = e % (D / 4) * 4;
          float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
          if (j * 64 + r < a.T) v = load4(k + (j * 64 + r) * a.ks[2] + d);
          *reinterpret_cast<float4*>(Ks + r * P + d) = v;
        }
        __syncthreads();
        float s[4][4];  // [key][row]: keys kk + 16 x, rows 4 rr + y
        tile_scores<D, 4, 4>(Ks, kk, Qs, rr, s);
#pragma unroll
        for (int y = 0; y < 4; ++y) {
          float top = -INFINITY;
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            s[x][y] = j < i || kk + 16 * x <= 4 * rr + y ? s[x][y] * a.scale_log2 : -INFINITY;
            top = fmaxf(top, s[x][y]);
          }
#pragma unroll
          for (int o = 8; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
          const float ref = top == -INFINITY ? 0.0f : top;
          float sum = 0.0f;
#pragma unroll
          for (int x = 0; x < 4; ++x) sum += exp2f(s[x][y] - ref);
#pragma unroll
          for (int o = 8; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
          const float up = fmaxf(m[y], top), at = up == -INFINITY ? 0.0f : up;
          l[y] = l[y] * exp2f(m[y] - at) + sum * exp2f(top - at);  // top, not ref: nothing times 2^(0 - at) may be no number
          m[y] = up;
          if (kk == 0) blocks[j * 64 + 4 * rr + y] = ref + log2f(sum);
        }
      }
#pragma unroll
      for (int y = 0; y < 4; ++y)
        if (kk == 0) Ls[4 * rr + y] = mass_total(m[y], l[y]);
      __syncthreads();
      const float share = 1.0f / static_cast<float>(tokens * rep);
      for (int j = tid / 32; j < qb; j += kTileThreads / 32) {
        float sum = 0.0f;
        if (j <= i) {
          const int r = tid % 32;
          if (r < tokens) sum = exp2f(blocks[j * 64 + r] - Ls[r]);
          if (r + 32 < tokens) sum += exp2f(blocks[j * 64 + r + 32] - Ls[r + 32]);
#pragma unroll
          for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        }
        if (tid % 32 == 0) {
          if (h > 0) sum += out[j];
          out[j] = h + 1 < rep ? sum : sum * share;
        }
      }
    }
  }
}

constexpr int kBlockTilePerSm = 2;

int64_t block_mass_workspace_bytes(int64_t B, int64_t Hq, int64_t Hkv, int64_t T, int64_t D, int dtype) {
  (void)D;
  if (dtype != SPRUCE_DTYPE_F32) return block_mass_sm100_workspace_bytes(B, Hq, Hkv, T);
  const int64_t qb = (T + 63) / 64;
  return std::min<int64_t>(B * Hkv * qb, kMaxSms * kBlockTilePerSm) * qb * 64 * 4;
}

template <int D>
static cudaError_t launch_block_tile(const BlockMassArgs& a, cudaStream_t stream) {
  constexpr int smem = sizeof(float) * (128 * (D + 4) + 64);
  auto kern = block_mass_tile_kernel<D>;
  static std::atomic<uint64_t> done{0};
  cudaError_t e = allow_smem(reinterpret_cast<const void*>(kern), smem, done);
  if (e != cudaSuccess) return e;
  const int qb = (a.T + 63) / 64;
  const int G = static_cast<int>(std::min<int64_t>((int64_t)a.B * a.Hkv * qb, sm_count() * kBlockTilePerSm));
  kern<<<G, kTileThreads, smem, stream>>>(a, qb);
  return cudaGetLastError();
}

cudaError_t launch_block_mass(const BlockMassArgs& a, int dtype, cudaStream_t stream) {
  if (dtype != SPRUCE_DTYPE_F32) return launch_block_mass_sm100(a, dtype, stream);
  return a.D == 128 ? launch_block_tile<128>(a, stream) : launch_block_tile<64>(a, stream);
}

}  // namespace spruce
