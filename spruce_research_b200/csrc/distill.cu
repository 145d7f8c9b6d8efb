// Distillation of a teacher's top entries: loss and gradient of rows of scores.
//
//   p = softmax_k(t_k / tau) over the row's teacher entries, q = softmax_j(s_j / tau) over its visible columns
//   loss = sum_k p_k (ln p_k - ln q_id(k))         d loss / d s_j = (q_j - sum_{k: id(k) = j} p_k) / tau
//
// The scores are read once (twice by a separate backward pass) and the gradient written once: HBM bounds the long rows.  Rows of up to 2048
// columns (a gate's) take a warp each, which holds the row in registers between the sums and the gradient.  Longer ones (a
// vocabulary's) take a CTA each, which keeps a running maximum and sum; its gradient pass reads the row again, mostly from L2 when
// both run in one call.  The teacher's columns are written again after the others,
// so that each element is rounded once.  A column named twice is found by a bitmap; only rows that have one search for it.
//
// On a B200: 4096 bf16 rows of 131072 columns, 64 entries each: forward 194 us (5.6 TB/s), backward 346 us (6.2 TB/s); 57344 fp32 rows
// of 512, half of them visible, loss and gradient in one call: 59 us, bound by instruction issue (75%) and the latency of a
// row's loads.  A warp that walks several rows and fetches the next one's entries ahead measured 68 to 90 us there.
#include <algorithm>

#include "mass_common.cuh"

namespace spruce {

constexpr int kRowWarps = 2;            // rows of a CTA of the warp kernel
constexpr int kShortRow = 24 << 10;    // bytes of the rows that the smallest CTAs take
constexpr int kRowMost = 2048, kRowEntries = 256;  // columns and teacher entries that it takes
constexpr int kRowBits = 64, kDistillBits = 1024;  // words of the bitmaps; columns share bits modulo their size
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

__device__ __forceinline__ float load_as_float(const void* p, int dtype, int64_t i) {
  if (dtype == SPRUCE_DTYPE_F32) return static_cast<const float*>(p)[i];
  if (dtype == SPRUCE_DTYPE_BF16) return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
  return __half2float(static_cast<const __half*>(p)[i]);
}

// A maximum and the sum of 2^((x - maximum) c) over it.  Differences are formed before they are scaled: the types' lowest
// values, as masks, stay finite.
__device__ __forceinline__ float2 join(float2 a, float2 b, float c) {
  const float m = fmaxf(a.x, b.x), ref = m == -INFINITY ? 0.0f : m;
  return make_float2(m, a.y * fast_exp2((a.x - ref) * c) + b.y * fast_exp2((b.x - ref) * c));
}
__device__ __forceinline__ float2 warp_join(float2 v, float c) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1)
    v = join(v, make_float2(__shfl_xor_sync(0xffffffffu, v.x, o), __shfl_xor_sync(0xffffffffu, v.y, o)), c);
  return v;
}
__device__ __forceinline__ float warp_max(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}
__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// Columns of the row that count.
__device__ __forceinline__ int row_seen(const DistillArgs& a, int64_t row, bool report) {
  if (a.visible == nullptr) return a.n;
  const int seen = a.visible[row];
  if (report && (seen < 0 || seen > a.n)) raise_status(a.status, SPRUCE_STATUS_BAD_LENGTH);
  return min(max(seen, 0), a.n);
}
// A teacher entry as it stands, and its column (-1: padding) and logit (-inf).
struct Entry {
  int64_t id;
  float logit;
};
__device__ __forceinline__ Entry row_entry(const DistillArgs& a, int64_t row, int k) {
  Entry e;
  e.id = a.ids64 ? static_cast<const int64_t*>(a.ids)[row * a.id_stride + k]
                 : static_cast<const int32_t*>(a.ids)[row * a.id_stride + k];
  e.logit = load_as_float(a.teacher, a.teacher_dtype, row * a.teacher_stride + k);
  return e;
}
__device__ __forceinline__ void use_entry(const DistillArgs& a, const Entry& e, int seen, int& column, float& logit) {
  if (e.id >= seen) raise_status(a.status, SPRUCE_STATUS_BAD_INDEX);
  const bool use = e.id >= 0 && e.id < seen;
  column = use ? static_cast<int>(e.id) : -1;
  logit = use ? e.logit : -INFINITY;
}
template <typename T>
__device__ __forceinline__ void unpack16(const uint4& v, float (&x)[16 / sizeof(T)]) {
  const T* e = reinterpret_cast<const T*>(&v);
#pragma unroll
  for (int i = 0; i < static_cast<int>(16 / sizeof(T)); ++i) x[i] = Elem<T>::to_f(e[i]);
}
template <typename T>
__device__ __forceinline__ uint4 pack16(const float (&x)[16 / sizeof(T)]) {
  uint4 v;
  T* e = reinterpret_cast<T*>(&v);
#pragma unroll
  for (int i = 0; i < static_cast<int>(16 / sizeof(T)); ++i) e[i] = Elem<T>::from_f(x[i]);
  return v;
}

// ------------------------------------------------------------------ a warp a row
// NV: 16-byte vectors of a lane.  Lane l holds columns V (32 i + l) ..; the order of the sums does not depend on alignment.
template <typename T, int NV>
__global__ void __launch_bounds__(32 * kRowWarps) distill_rows_kernel(const DistillArgs a, bool vec_in, bool vec_out) {
  constexpr int V = 16 / sizeof(T);
  extern __shared__ float sm[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  float* P = sm + warp * (3 * a.K + kRowBits);     // [K] teacher weights
  int* I = reinterpret_cast<int*>(P + a.K);        // [K] columns
  float* S = P + 2 * a.K;                          // [K] scores there
  uint32_t* bits = reinterpret_cast<uint32_t*>(S + a.K);
  const int64_t row = (int64_t)blockIdx.x * kRowWarps + warp;
  if (row >= a.R) return;
  const float c = a.inv_tau * kLog2e;
  const T* s = static_cast<const T*>(a.scores) + row * a.score_stride;
  // What does not hang on the visible columns is on its way first: the kernel is bound by the latency of its loads.
  Entry early{-1, 0.0f};
  if (lane < a.K) early = row_entry(a, row, lane);
  float w = 0.0f;
  if (a.grad != nullptr) w = a.weight[row * a.weight_stride] * a.inv_tau;
  float2 st;
  if (a.stats_in != nullptr) st = make_float2(a.stats_in[2 * row], a.stats_in[2 * row + 1]);
  const int seen = row_seen(a, row, lane == 0);
  float v[NV][V];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int col = (32 * i + lane) * V;
    if (vec_in && col + V <= seen) {
      unpack16<T>(*reinterpret_cast<const uint4*>(s + col), v[i]);
    } else if (32 * i * V < seen) {  // of the warp
#pragma unroll
      for (int e = 0; e < V; ++e) v[i][e] = col + e < seen ? Elem<T>::to_f(s[col + e]) : -INFINITY;
    } else {
#pragma unroll
      for (int e = 0; e < V; ++e) v[i][e] = -INFINITY;
    }
  }
  // Teacher.
  for (int b = lane; b < kRowBits; b += 32) bits[b] = 0;
  float tm = -INFINITY;
  __syncwarp();
  bool twice = false;
  for (int k = lane; k < a.K; k += 32) {
    int column;
    float logit;
    use_entry(a, k < 32 ? early : row_entry(a, row, k), seen, column, logit);
    I[k] = column;
    P[k] = logit;
    S[k] = column < 0 ? 0.0f : Elem<T>::to_f(s[column]);
    tm = fmaxf(tm, logit);
    if (a.grad != nullptr && column >= 0)
      twice = twice || (atomicOr(&bits[(column >> 5) % kRowBits], 1u << (column & 31)) >> (column & 31) & 1);
  }
  twice = __any_sync(0xffffffffu, twice);
  tm = warp_max(tm);
  const float tref = tm == -INFINITY ? 0.0f : tm;
  float tsum = 0.0f;
  for (int k = lane; k < a.K; k += 32) tsum += I[k] < 0 ? 0.0f : fast_exp2((P[k] - tref) * c);
  tsum = warp_sum(tsum);
  // Student.
  if (a.stats_in == nullptr) {
    float m = -INFINITY, l = 0.0f;
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int e = 0; e < V; ++e) m = fmaxf(m, v[i][e]);
    m = warp_max(m);
    const float ref = m == -INFINITY ? 0.0f : m;
#pragma unroll
    for (int i = 0; i < NV; ++i)
      if (32 * i * V < seen)
#pragma unroll
        for (int e = 0; e < V; ++e) l += fast_exp2((v[i][e] - ref) * c);
    st = make_float2(ref, __log2f(warp_sum(l)));  // -inf: nothing to see
  }
  const bool empty = st.y == -INFINITY || tsum == 0.0f;
  const float tlog = __log2f(tsum);
  float loss = 0.0f;
  for (int k = lane; k < a.K; k += 32) {
    if (I[k] < 0 || empty) continue;
    const float e = (P[k] - tref) * c - tlog, p = fast_exp2(e);
    if (a.loss != nullptr && p != 0.0f) loss += p * (e - ((S[k] - st.x) * c - st.y));
    P[k] = p;
  }
  if (a.loss != nullptr) {
    loss = warp_sum(loss) * kLn2;
    if (lane == 0) {
      a.loss[row] = empty ? 0.0f : loss;
      if (a.stats != nullptr) {
        a.stats[2 * row] = st.x;
        a.stats[2 * row + 1] = st.y;
      }
    }
  }
  if (a.grad == nullptr) return;
  T* grad = static_cast<T*>(a.grad) + row * a.grad_stride;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int col = (32 * i + lane) * V;
    float g[V];
    if (32 * i * V < seen && !empty) {  // of the warp
#pragma unroll
      for (int e = 0; e < V; ++e) g[e] = col + e < seen ? w * fast_exp2((v[i][e] - st.x) * c - st.y) : 0.0f;
    } else {
#pragma unroll
      for (int e = 0; e < V; ++e) g[e] = 0.0f;
    }
    if (vec_out && col + V <= a.n) {
      *reinterpret_cast<uint4*>(grad + col) = pack16<T>(g);  // not a streaming store: the teacher's columns follow (61.4 -> 59.4 us)
    } else {
#pragma unroll
      for (int e = 0; e < V; ++e)
        if (col + e < a.n) grad[col + e] = Elem<T>::from_f(g[e]);
    }
  }
  __syncwarp();
  for (int k = lane; k < a.K; k += 32) {
    const int j = I[k];
    if (j < 0 || empty) continue;
    float p = P[k];
    if (twice) {
      p = 0.0f;
      for (int x = 0; x < a.K; ++x) p += I[x] == j ? P[x] : 0.0f;
    }
    grad[j] = Elem<T>::from_f(w * (fast_exp2((S[k] - st.x) * c - st.y) - p));
  }
}

// ------------------------------------------------------------------ a CTA a row
template <int THREADS>
__device__ __forceinline__ float2 block_join(float2 v, float c, float2* red) {
  v = warp_join(v, c);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  v = red[0];
  for (int w = 1; w < THREADS / 32; ++w) v = join(v, red[w], c);
  return v;
}

// Columns [0, n) of a row: the 16-byte aligned middle by vectors, f(first column, pointer); the rest one by one, g(column).
template <typename T, int THREADS, typename F, typename G>
__device__ __forceinline__ void over_row(const T* s, int n, F f, G g) {
  constexpr int V = 16 / sizeof(T), U = 4;
  const int head = min(n, static_cast<int>((16 - (reinterpret_cast<uintptr_t>(s) & 15)) % 16 / sizeof(T)));
  const int vecs = (n - head) / V, rest = n - vecs * V;
  int i = threadIdx.x;
  for (; i + (U - 1) * THREADS < vecs; i += U * THREADS) {
    uint4 x[U];
#pragma unroll
    for (int u = 0; u < U; ++u) x[u] = *reinterpret_cast<const uint4*>(s + head + (i + u * THREADS) * V);
#pragma unroll
    for (int u = 0; u < U; ++u) f(head + (i + u * THREADS) * V, x[u]);
  }
  for (; i < vecs; i += THREADS) f(head + i * V, *reinterpret_cast<const uint4*>(s + head + i * V));
  for (int e = threadIdx.x; e < rest; e += THREADS) g(e < head ? e : vecs * V + e);
}

// CTAS an SM.
template <typename T, int THREADS, int CTAS>
__global__ void __launch_bounds__(THREADS, CTAS) distill_kernel(const DistillArgs a) {
  constexpr int V = 16 / sizeof(T);
  extern __shared__ float sm[];
  float* P = sm;                                  // [K] teacher weights
  int* I = reinterpret_cast<int*>(sm + a.K);      // [K] columns; -1: not used
  __shared__ uint32_t bits[kDistillBits];
  __shared__ float2 red[THREADS / 32];
  const int tid = threadIdx.x;
  const float c = a.inv_tau * kLog2e;
  for (int64_t row = blockIdx.x; row < a.R; row += gridDim.x) {
    const T* s = static_cast<const T*>(a.scores) + row * a.score_stride;
    const int seen = row_seen(a, row, tid == 0);
    __syncthreads();
    for (int b = tid; b < kDistillBits; b += THREADS) bits[b] = 0;
    __syncthreads();
    float2 t = make_float2(-INFINITY, 0.0f);
    bool mine = false;
    for (int k = tid; k < a.K; k += THREADS) {
      int column;
      float logit;
      use_entry(a, row_entry(a, row, k), seen, column, logit);
      I[k] = column;
      P[k] = logit;
      if (column < 0) continue;
      t = join(t, make_float2(logit, logit == -INFINITY ? 0.0f : 1.0f), c);
      if (a.grad != nullptr) mine = mine || (atomicOr(&bits[(column >> 5) % kDistillBits], 1u << (column & 31)) >> (column & 31) & 1);
    }
    const bool twice = __syncthreads_or(mine);
    t = block_join<THREADS>(t, c, red);
    const float tref = t.x == -INFINITY ? 0.0f : t.x, tsum = t.y;
    float2 st;  // maximum of the scores, log2 of the sum over it
    if (a.stats_in != nullptr) {
      st = make_float2(a.stats_in[2 * row], a.stats_in[2 * row + 1]);
    } else {
      float m = -INFINITY, l = 0.0f;
      auto more = [&](float top) {  // the running maximum moves
        if (top > m) {
          l *= fast_exp2((m - top) * c);
          m = top;
        }
      };
      over_row<T, THREADS>(s, seen,
                  [&](int, const uint4& y) {
                    float x[V];
                    unpack16<T>(y, x);
                    float top = x[0];
#pragma unroll
                    for (int e = 1; e < V; ++e) top = fmaxf(top, x[e]);
                    more(top);
                    const float ref = m == -INFINITY ? 0.0f : m;
#pragma unroll
                    for (int e = 0; e < V; ++e) l += fast_exp2((x[e] - ref) * c);
                  },
                  [&](int j) {
                    const float x = Elem<T>::to_f(s[j]);
                    more(x);
                    l += fast_exp2((x - (m == -INFINITY ? 0.0f : m)) * c);
                  });
      const float2 all = block_join<THREADS>(make_float2(m, l), c, red);
      st = make_float2(all.x == -INFINITY ? 0.0f : all.x, log2f(all.y));
    }
    const bool empty = st.y == -INFINITY || tsum == 0.0f;
    const float tlog = log2f(tsum), inv = 1.0f / tsum;
    float loss = 0.0f;
    for (int k = tid; k < a.K; k += THREADS) {
      if (I[k] < 0 || empty) continue;
      const float e = (P[k] - tref) * c, p = fast_exp2(e) * inv;
      if (a.loss != nullptr && p != 0.0f) loss += p * ((e - tlog) - ((Elem<T>::to_f(s[I[k]]) - st.x) * c - st.y));
      P[k] = p;
    }
    if (a.loss != nullptr) {
      loss = block_join<THREADS>(make_float2(0.0f, loss), c, red).y * kLn2;
      if (tid == 0) {
        a.loss[row] = empty ? 0.0f : loss;
        if (a.stats != nullptr) {
          a.stats[2 * row] = st.x;
          a.stats[2 * row + 1] = st.y;
        }
      }
    }
    if (a.grad == nullptr) continue;
    T* grad = static_cast<T*>(a.grad) + row * a.grad_stride;
    const float w = a.weight[row * a.weight_stride] * a.inv_tau;
    const bool same = ((reinterpret_cast<uintptr_t>(s) ^ reinterpret_cast<uintptr_t>(grad)) & 15) == 0;
    if (empty) {
      for (int j = tid; j < a.n; j += THREADS) grad[j] = Elem<T>::from_f(0.0f);
      continue;
    }
    auto value = [&](float x) { return w * fast_exp2((x - st.x) * c - st.y); };
    over_row<T, THREADS>(s, seen,
                [&](int j, const uint4& y) {
                  float x[V];
                  unpack16<T>(y, x);
#pragma unroll
                  for (int e = 0; e < V; ++e) x[e] = value(x[e]);
                  if (same) {
                    __stcs(reinterpret_cast<uint4*>(grad + j), pack16<T>(x));
                  } else {
#pragma unroll
                    for (int e = 0; e < V; ++e) grad[j + e] = Elem<T>::from_f(x[e]);
                  }
                },
                [&](int j) { grad[j] = Elem<T>::from_f(value(Elem<T>::to_f(s[j]))); });
    for (int j = seen + tid; j < a.n; j += THREADS) grad[j] = Elem<T>::from_f(0.0f);
    __syncthreads();
    for (int k = tid; k < a.K; k += THREADS) {
      const int j = I[k];
      if (j < 0) continue;
      float p = P[k];
      if (twice) {
        p = 0.0f;
        for (int x = 0; x < a.K; ++x) p += I[x] == j ? P[x] : 0.0f;
      }
      grad[j] = Elem<T>::from_f(w * (fast_exp2((Elem<T>::to_f(s[j]) - st.x) * c - st.y) - p));
    }
  }
}

template <typename T>
static cudaError_t launch_rows(const DistillArgs& a, cudaStream_t stream) {
  constexpr int V = 16 / sizeof(T);
  const int smem = kRowWarps * (3 * a.K + kRowBits) * 4;
  const unsigned G = static_cast<unsigned>((a.R + kRowWarps - 1) / kRowWarps);
  auto aligned = [](const void* p, int64_t stride) {
    return (reinterpret_cast<uintptr_t>(p) & 15u) == 0 && stride % V == 0;
  };
  const bool in = aligned(a.scores, a.score_stride), out = a.grad != nullptr && aligned(a.grad, a.grad_stride);
  const int vecs = (a.n + 32 * V - 1) / (32 * V);
  if (vecs <= 1) distill_rows_kernel<T, 1><<<G, 32 * kRowWarps, smem, stream>>>(a, in, out);
  else if (vecs <= 2) distill_rows_kernel<T, 2><<<G, 32 * kRowWarps, smem, stream>>>(a, in, out);
  else if (vecs <= 4) distill_rows_kernel<T, 4><<<G, 32 * kRowWarps, smem, stream>>>(a, in, out);
  else if (vecs <= 8) distill_rows_kernel<T, 8><<<G, 32 * kRowWarps, smem, stream>>>(a, in, out);
  else distill_rows_kernel<T, 64 / V><<<G, 32 * kRowWarps, smem, stream>>>(a, in, out);
  return cudaGetLastError();
}

template <typename T>
static cudaError_t launch(const DistillArgs& a, cudaStream_t stream) {
  constexpr int V = 16 / sizeof(T);
  const bool whole = (reinterpret_cast<uintptr_t>(a.scores) & 15u) == 0 && a.score_stride % V == 0 &&
                     (a.grad == nullptr || ((reinterpret_cast<uintptr_t>(a.grad) & 15u) == 0 && a.grad_stride % V == 0));
  // The warp kernel takes rows that are not 16-byte aligned element by element: long ones are better off with the other, which
  // takes their middle by vectors (15879 rows of 1316 columns in bf16: 130 us there).
  if (a.n <= (whole ? kRowMost : kRowMost / 2) && a.K <= kRowEntries && a.R < (int64_t(1) << 31)) return launch_rows<T>(a, stream);
  const unsigned G = static_cast<unsigned>(std::min<int64_t>(a.R, 1 << 20));
  // Short rows in small CTAs, whose barriers hold up fewer threads (49305 rows of 6352 columns in bf16, loss and gradient: 1274 /
  // 610 / 359 us with 512 / 256 / 128 threads; 3000 of 16000 in fp32: 79 us with 256, 103 with 128; 4096 of 131072 in bf16: 554 us
  // with 256, 574 with 512).  Fewer rows than SMs get 512 threads each: loss and gradient of 8 / 64 / 140 rows of 131072 in bf16 19 / 19 /
  // 20 us against 23 / 25 / 25 with 256, in fp32 25 / 25 / 44 against 31 / 32 / 61; 20 of 6000 in bf16 15.4 against 13.6 with 128.
  const int64_t bytes = (int64_t)a.n * sizeof(T);
  if (a.R < sm_count())
    distill_kernel<T, 512, 2><<<G, 512, a.K * 8, stream>>>(a);
  else if (bytes <= kShortRow)
    distill_kernel<T, 128, 10><<<G, 128, a.K * 8, stream>>>(a);
  else
    distill_kernel<T, 256, 5><<<G, 256, a.K * 8, stream>>>(a);
  return cudaGetLastError();
}

cudaError_t launch_distill(const DistillArgs& a, int dtype, cudaStream_t stream) {
  switch (dtype) {
    case SPRUCE_DTYPE_F32: return launch<float>(a, stream);
    case SPRUCE_DTYPE_BF16: return launch<__nv_bfloat16>(a, stream);
    default: return launch<__half>(a, stream);
  }
}

}  // namespace spruce
