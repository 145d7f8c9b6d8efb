// Distillation of a teacher's top entries: loss and gradient of rows of scores.
//
//   p = softmax_k(t_k / tau) over the row's teacher entries, q = softmax_j(s_j / tau) over its visible columns
//   loss = sum_k p_k (ln p_k - ln q_id(k))         d loss / d s_j = (q_j - sum_{k: id(k) = j} p_k) / tau
//
// One CTA a row.  The first pass keeps a running maximum and sum; the gradient's pass reads the row again (it is in L2 when
// both run in one call) and the columns of the teacher are written again after it, so that each element is rounded once.
#include <algorithm>

#include "mass_common.cuh"

namespace spruce {

constexpr int kDistillThreads = 256;
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

__device__ __forceinline__ float load_as_float(const void* p, int dtype, int64_t i) {
  if (dtype == SPRUCE_DTYPE_F32) return static_cast<const float*>(p)[i];
  if (dtype == SPRUCE_DTYPE_BF16) return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
  return __half2float(static_cast<const __half*>(p)[i]);
}

__device__ __forceinline__ float2 block_join(float m, float l, float2* red) {
  auto join = [](float2 a, float2 b) {
    const float m = fmaxf(a.x, b.x), ref = m == -INFINITY ? 0.0f : m;
    return make_float2(m, a.y * exp2f(a.x - ref) + b.y * exp2f(b.x - ref));
  };
  float2 v = make_float2(m, l);
  for (int o = 16; o > 0; o >>= 1)
    v = join(v, make_float2(__shfl_xor_sync(0xffffffffu, v.x, o), __shfl_xor_sync(0xffffffffu, v.y, o)));
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  v = red[0];
  for (int w = 1; w < kDistillThreads / 32; ++w) v = join(v, red[w]);
  return v;
}

template <typename T>
__global__ void __launch_bounds__(kDistillThreads) distill_kernel(const DistillArgs a) {
  extern __shared__ float sm[];
  float* P = sm;                                  // [K] teacher weights
  int* I = reinterpret_cast<int*>(sm + a.K);      // [K] columns; -1: not used
  __shared__ float2 red[kDistillThreads / 32];
  const int tid = threadIdx.x;
  const float c = a.inv_tau * kLog2e;
  for (int64_t row = blockIdx.x; row < a.R; row += gridDim.x) {
    const T* s = static_cast<const T*>(a.scores) + row * a.score_stride;
    int seen = a.n;
    if (a.visible != nullptr) {
      seen = a.visible[row];
      if ((seen < 0 || seen > a.n) && tid == 0) raise_status(a.status, SPRUCE_STATUS_BAD_LENGTH);
      seen = min(max(seen, 0), a.n);
    }
    __syncthreads();
    for (int k = tid; k < a.K; k += kDistillThreads) {
      const int64_t id = a.ids64 ? static_cast<const int64_t*>(a.ids)[row * a.id_stride + k]
                                 : static_cast<const int32_t*>(a.ids)[row * a.id_stride + k];
      if (id >= seen) raise_status(a.status, SPRUCE_STATUS_BAD_INDEX);
      const bool use = id >= 0 && id < seen;
      I[k] = use ? static_cast<int>(id) : -1;
      P[k] = use ? load_as_float(a.teacher, a.teacher_dtype, row * a.teacher_stride + k) : -INFINITY;
    }
    // Teacher: maximum and sum.
    float m = -INFINITY, l = 0.0f;
    for (int k = tid; k < a.K; k += kDistillThreads) m = fmaxf(m, P[k]);
    float tm = block_join(m, 0.0f, red).x;
    const float tref = tm == -INFINITY ? 0.0f : tm;
    for (int k = tid; k < a.K; k += kDistillThreads) l += I[k] < 0 ? 0.0f : exp2f((P[k] - tref) * c);
    const float tsum = block_join(0.0f, l, red).y;
    // Student.
    float2 st;
    if (a.stats_in != nullptr) {
      st = make_float2(a.stats_in[2 * row], a.stats_in[2 * row + 1]);
    } else {
      m = -INFINITY;
      for (int j = tid; j < seen; j += kDistillThreads) m = fmaxf(m, Elem<T>::to_f(s[j]));
      const float top = block_join(m, 0.0f, red).x, ref = top == -INFINITY ? 0.0f : top;
      l = 0.0f;
      for (int j = tid; j < seen; j += kDistillThreads) l += exp2f((Elem<T>::to_f(s[j]) - ref) * c);
      const float sum = block_join(0.0f, l, red).y;
      st = make_float2(ref, log2f(sum));  // -inf: nothing to see
    }
    const bool empty = st.y == -INFINITY || tsum == 0.0f;
    l = 0.0f;
    for (int k = tid; k < a.K; k += kDistillThreads) {
      if (I[k] < 0 || empty) continue;
      const float e = (P[k] - tref) * c, p = exp2f(e) / tsum;
      if (a.loss != nullptr && p != 0.0f)
        l += p * ((e - log2f(tsum)) - ((Elem<T>::to_f(s[I[k]]) - st.x) * c - st.y));
      P[k] = p;
    }
    if (a.loss != nullptr) {
      const float loss = block_join(0.0f, l, red).y * kLn2;
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
    for (int j = tid; j < a.n; j += kDistillThreads)
      grad[j] = Elem<T>::from_f(j < seen && !empty ? w * exp2f((Elem<T>::to_f(s[j]) - st.x) * c - st.y) : 0.0f);
    __syncthreads();
    for (int k = tid; k < a.K; k += kDistillThreads) {
      const int j = I[k];
      if (j < 0 || empty) continue;
      float p = 0.0f;
      for (int x = 0; x < a.K; ++x) p += I[x] == j ? P[x] : 0.0f;
      grad[j] = Elem<T>::from_f(w * (exp2f((Elem<T>::to_f(s[j]) - st.x) * c - st.y) - p));
    }
  }
}

cudaError_t launch_distill(const DistillArgs& a, int dtype, cudaStream_t stream) {
  const int smem = a.K * 8;
  const int G = static_cast<int>(std::min<int64_t>(a.R, 1 << 20));
  switch (dtype) {
    case SPRUCE_DTYPE_F32: distill_kernel<float><<<G, kDistillThreads, smem, stream>>>(a); break;
    case SPRUCE_DTYPE_BF16: distill_kernel<__nv_bfloat16><<<G, kDistillThreads, smem, stream>>>(a); break;
    default: distill_kernel<__half><<<G, kDistillThreads, smem, stream>>>(a); break;
  }
  return cudaGetLastError();
}

}  // namespace spruce
