// Head norms and rotary positions of queries and keys, dense or on the way into a paged K/V cache.
//
// For one row x (a token's head, D dims), in fp32 and rounded once at the store:
//   y = x * rsqrt(mean(x^2) + eps) * w            (where the head has a norm weight)
//   (a, b) -> (a cos t - b sin t, b cos t + a sin t)   for each pair of the first rd dims,
// pairs (i, i + rd/2) ("half") or (2i, 2i+1) ("interleaved"), cos t / sin t from row `position` of an fp32
// table [positions, cos(rd/2) | sin(rd/2)].  The table is made once in 64 bits: fp32 angle products lose 7e-3 rad at position
// 131072, and any scaling of the frequencies costs the kernel nothing.
//
// Bound: HBM bandwidth (every row read once, written once; ~10 flops an element).
//
// Layout: a row is held by LPR lanes (8 at D = 128 in 16 bits), each with two 16-byte vectors that hold whole pairs
// (half: one vector of each half; interleaved: adjacent vectors), so a rotation needs no exchange and the norm three
// shuffles.  A lane group takes HC heads of one token: the angles are loaded once for them and 2 HC loads are in flight
// per lane.  Shapes, strides or bases that 16-byte vectors do not fit take the same kernel with one element a load.
#include <algorithm>

#include "common.cuh"
#include "kernels.h"

namespace spruce {

constexpr int kRowThreads = 256;
constexpr int kHeadsPerGroup = 4;

template <typename T, int VN>
struct RowVec {
  T e[VN];
  __device__ __forceinline__ void load(const T* p) {
    if constexpr (VN * sizeof(T) == 16)
      *reinterpret_cast<uint4*>(e) = *reinterpret_cast<const uint4*>(p);  // not __ldg: the output may be the input
    else
      for (int i = 0; i < VN; ++i) e[i] = p[i];
  }
  __device__ __forceinline__ void store(T* p) const {
    if constexpr (VN * sizeof(T) == 16)
      *reinterpret_cast<uint4*>(p) = *reinterpret_cast<const uint4*>(e);
    else
      for (int i = 0; i < VN; ++i) p[i] = e[i];
  }
};

// Largest s with cu[s] <= n, for 0 <= n < cu[S] (cu non-decreasing).
__device__ __forceinline__ int seq_of_token(const int32_t* cu, int S, int n) {
  if (n < S && cu[n] == n && cu[n + 1] == n + 1) return n;  // single-token sequences
  int lo = 0, hi = S;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (cu[mid] <= n) lo = mid;
    else hi = mid;
  }
  return lo;
}

template <typename T, int VN, int ITERS, bool APPEND>
__global__ void __launch_bounds__(kRowThreads) norm_rope_kernel(const RowsArgs a, int lpr, int chunks) {
  constexpr int HC = kHeadsPerGroup;
  alignas(16) RowVec<T, VN> va[HC][ITERS], vb[HC][ITERS];
  const int l = threadIdx.x & (lpr - 1);
  const int64_t group = (int64_t)blockIdx.x * (kRowThreads / lpr) + threadIdx.x / lpr;
  const int64_t tokens = (int64_t)a.B * a.T;
  const bool live = group < tokens * chunks;
  const int64_t n = live ? group / chunks : 0;
  const int h0 = live ? static_cast<int>(group % chunks) * HC : 0;
  const int heads = a.Hq + (APPEND ? 2 : 1) * a.Hkv;  // query rows, key rows, (value rows)
  const int64_t b = n / a.T, t = n % a.T;
  const int items = a.D / (2 * VN);

  // Where the token's rotation and cache rows are.
  int64_t pos = t, page = 0;
  int slot = 0;
  bool write = live, cached = live;
  if constexpr (APPEND) {
    cached = write = live && n < a.cu_q[a.S];
    if (write) {
      const int s = seq_of_token(a.cu_q, a.S, static_cast<int>(n));
      pos = (int64_t)a.kv_lens[s] - (a.cu_q[s + 1] - n);
      const int64_t pi = pos >= 0 ? pos / a.page_size : -1;
      cached = pi >= 0 && pi < a.max_pages;
      if (!cached) raise_status(a.status, SPRUCE_STATUS_BAD_LENGTH);
      if (cached) {
        page = a.block_table[(int64_t)s * a.table_stride + pi];
        cached = page >= 0 && page < a.num_pages;
        if (!cached) raise_status(a.status, SPRUCE_STATUS_BAD_PAGE);
        slot = static_cast<int>(pos - pi * a.page_size);
      }
    }
  }
  const float* angles = nullptr;
  if (a.rd > 0) {
    if (a.positions != nullptr && write) pos = a.positions[b * a.pos_sb + t * a.pos_st];
    if (write && (pos < 0 || pos >= a.table_rows)) raise_status(a.status, SPRUCE_STATUS_BAD_POSITION);
    pos = pos < 0 ? 0 : (pos < a.table_rows ? pos : a.table_rows - 1);
    angles = a.rope + pos * a.rd;
  }

  // Vector offsets of this lane's pairs, and their angles.
  int oa[ITERS], ob[ITERS];
  bool in[ITERS], rot[ITERS];
  float cs[ITERS][VN], sn[ITERS][VN];
#pragma unroll
  for (int it = 0; it < ITERS; ++it) {
    const int item = l + it * lpr;
    const int nrot = a.rd / (2 * VN);
    in[it] = item < items;
    rot[it] = item < nrot;
    if (a.interleaved || !rot[it]) {
      oa[it] = 2 * item * VN;
      ob[it] = oa[it] + VN;
    } else {
      oa[it] = item * VN;
      ob[it] = a.rd / 2 + item * VN;
    }
    if (in[it] && rot[it]) {
      const float* c = angles + item * VN;
      const float* s = c + a.rd / 2;
      if constexpr (VN % 4 == 0) {
#pragma unroll
        for (int e = 0; e < VN; e += 4) {
          *reinterpret_cast<float4*>(&cs[it][e]) = __ldg(reinterpret_cast<const float4*>(c + e));
          *reinterpret_cast<float4*>(&sn[it][e]) = __ldg(reinterpret_cast<const float4*>(s + e));
        }
      } else {
#pragma unroll
        for (int e = 0; e < VN; ++e) {
          cs[it][e] = c[e];
          sn[it][e] = s[e];
        }
      }
    }
  }

  // All loads of the group's heads first.
  const T* src[HC];
#pragma unroll
  for (int i = 0; i < HC; ++i) {
    const int h = h0 + i;
    const bool isq = h < a.Hq, isk = h < a.Hq + a.Hkv;
    const Rows& r = isq ? a.q : (isk ? a.k : a.v);
    const int hh = isq ? h : (isk ? h - a.Hq : h - a.Hq - a.Hkv);
    src[i] = write && h < heads ? static_cast<const T*>(r.x) + b * r.sb + hh * r.sh + t * r.st : nullptr;
#pragma unroll
    for (int it = 0; it < ITERS; ++it)
      if (src[i] != nullptr && in[it]) {
        va[i][it].load(src[i] + oa[it]);
        vb[i][it].load(src[i] + ob[it]);
      }
  }

#pragma unroll
  for (int i = 0; i < HC; ++i) {
    const int h = h0 + i;
    const bool isq = h < a.Hq, isk = !isq && h < a.Hq + a.Hkv;
    const Rows& r = isq ? a.q : (isk ? a.k : a.v);
    const int hh = isq ? h : (isk ? h - a.Hq : h - a.Hq - a.Hkv);
    const float* w = isq ? a.q.weight : (isk ? a.k.weight : nullptr);
    // The norm's shuffles are executed by every lane; a row's lanes are adjacent.
    float inv = 1.0f;
    if (a.q.weight != nullptr || a.k.weight != nullptr) {
      float ss = 0.0f;
      if (src[i] != nullptr) {
#pragma unroll
        for (int it = 0; it < ITERS; ++it)
          if (in[it]) {
#pragma unroll
            for (int e = 0; e < VN; ++e) {
              const float x = Elem<T>::to_f(va[i][it].e[e]), y = Elem<T>::to_f(vb[i][it].e[e]);
              ss = fmaf(x, x, fmaf(y, y, ss));
            }
          }
      }
      for (int o = lpr >> 1; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
      inv = rsqrtf(ss / static_cast<float>(a.D) + a.eps);
    }
    if (src[i] == nullptr) continue;
    T* dst;
    if (APPEND && !isq) {
      if (!cached) continue;
      dst = static_cast<T*>(r.out) + page * r.ob + hh * r.oh + slot * r.ot;
    } else {
      dst = static_cast<T*>(r.out) + b * r.ob + hh * r.oh + t * r.ot;
    }
#pragma unroll
    for (int it = 0; it < ITERS; ++it) {
      if (!in[it]) continue;
      if (isq || isk) {
        float x[VN], y[VN];
#pragma unroll
        for (int e = 0; e < VN; ++e) {
          x[e] = Elem<T>::to_f(va[i][it].e[e]);
          y[e] = Elem<T>::to_f(vb[i][it].e[e]);
        }
        if (w != nullptr) {
#pragma unroll
          for (int e = 0; e < VN; ++e) {
            x[e] *= inv * w[oa[it] + e];
            y[e] *= inv * w[ob[it] + e];
          }
        }
        if (rot[it]) {
          if (VN > 1 && a.interleaved) {
#pragma unroll
            for (int e = 0; e + 1 < VN; e += 2) {
              const float c0 = cs[it][e / 2], s0 = sn[it][e / 2];
              const float c1 = cs[it][VN / 2 + e / 2], s1 = sn[it][VN / 2 + e / 2];
              const float x0 = x[e], x1 = x[e + 1], y0 = y[e], y1 = y[e + 1];
              x[e] = x0 * c0 - x1 * s0;
              x[e + 1] = x1 * c0 + x0 * s0;
              y[e] = y0 * c1 - y1 * s1;
              y[e + 1] = y1 * c1 + y0 * s1;
            }
          } else {
#pragma unroll
            for (int e = 0; e < VN; ++e) {
              const float x0 = x[e], y0 = y[e];
              x[e] = x0 * cs[it][e] - y0 * sn[it][e];
              y[e] = y0 * cs[it][e] + x0 * sn[it][e];
            }
          }
        }
#pragma unroll
        for (int e = 0; e < VN; ++e) {
          va[i][it].e[e] = Elem<T>::from_f(x[e]);
          vb[i][it].e[e] = Elem<T>::from_f(y[e]);
        }
      }
      va[i][it].store(dst + oa[it]);
      vb[i][it].store(dst + ob[it]);
    }
  }
}

template <typename T, int VN, int ITERS, bool APPEND>
static cudaError_t launch_rows_typed(const RowsArgs& a, cudaStream_t stream) {
  const int items = a.D / (2 * VN);
  int lpr = 1;
  while (lpr < items && lpr < 32) lpr *= 2;
  const int heads = a.Hq + (APPEND ? 2 : 1) * a.Hkv;
  const int chunks = (heads + kHeadsPerGroup - 1) / kHeadsPerGroup;
  const int64_t groups = (int64_t)a.B * a.T * chunks;
  const int per = kRowThreads / lpr;
  const int64_t ctas = (groups + per - 1) / per;
  if (ctas > 0x7fffffff) return cudaErrorInvalidValue;
  norm_rope_kernel<T, VN, ITERS, APPEND><<<(unsigned)ctas, kRowThreads, 0, stream>>>(a, lpr, chunks);
  return cudaGetLastError();
}

template <typename T>
static cudaError_t launch_rows_dtype(const RowsArgs& a, bool vec, cudaStream_t stream) {
  constexpr int V = 16 / sizeof(T);
  if (a.cu_q != nullptr)
    return vec ? launch_rows_typed<T, V, 1, true>(a, stream) : launch_rows_typed<T, 1, 4, true>(a, stream);
  return vec ? launch_rows_typed<T, V, 1, false>(a, stream) : launch_rows_typed<T, 1, 4, false>(a, stream);
}

cudaError_t launch_norm_rope(const RowsArgs& a, int dtype, cudaStream_t stream) {
  const int es = dtype == SPRUCE_DTYPE_F32 ? 4 : 2;
  const int V = 16 / es;
  // 16-byte vectors: pairs that fill them, and bases and strides that keep every one aligned.
  bool vec = a.D % (2 * V) == 0 && a.rd % (2 * V) == 0 && (reinterpret_cast<uintptr_t>(a.rope) & 15) == 0;
  auto fits = [&](const Rows& r) {
    return r.x == nullptr || ((reinterpret_cast<uintptr_t>(r.x) & 15) == 0 && (reinterpret_cast<uintptr_t>(r.out) & 15) == 0 &&
                              r.sb % V == 0 && r.sh % V == 0 && r.st % V == 0 && r.ob % V == 0 && r.oh % V == 0 &&
                              r.ot % V == 0);
  };
  vec = vec && fits(a.q) && fits(a.k) && fits(a.v);
  if (dtype == SPRUCE_DTYPE_F32) return launch_rows_dtype<float>(a, vec, stream);
  if (dtype == SPRUCE_DTYPE_BF16) return launch_rows_dtype<__nv_bfloat16>(a, vec, stream);
  return launch_rows_dtype<__half>(a, vec, stream);
}

}  // namespace spruce
