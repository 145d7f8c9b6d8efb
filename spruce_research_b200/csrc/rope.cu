// Head norms and rotary positions of queries and keys, dense or on the way into a paged K/V cache.
//
// For one row x (a token's head, D dims), in fp32 and rounded once at the store:
//   y = x * rsqrt(mean(x^2) + eps) * w            (where the head has a norm weight)
//   (a, b) -> (a cos t - b sin t, b cos t + a sin t)   for each pair of the first rd dims,
// pairs (i, i + rd/2) ("half") or (2i, 2i+1) ("interleaved"), cos t / sin t from row `position` of an fp32
// table [positions, cos(rd/2) | sin(rd/2)].  The table is made once in 64 bits: fp32 angle products lose 7e-3 rad at position
// 131072, and any scaling of the frequencies costs the kernel nothing.
//
// Bound: HBM bandwidth (every row read once, written once; ~10 flops an element).  On a B200 Q and K of a 131072-token
// layer (28 + 4 heads of 128, bf16, 2.2 GB) take 322 us, 6.9 TB/s; 16384 tokens with norms 45.3 us, 5.9 TB/s; 4097 tokens with
// norms 14.4 us; the append of 8.2K tokens 30.6 us, 5.3 TB/s.  fp32, 16384 tokens with norms: 84.2 us, 6.5 TB/s.  Rows that 16-byte
// vectors do not fit, a warp a row: 16384 tokens 202 us in bf16 (1.4 TB/s), 199 us in fp32 (2.7 TB/s), bound by element loads.
//
// Layout: a row is held by LPR lanes (8 at D = 128 in 16 bits), each with two 16-byte vectors that hold whole pairs (half
// pairs: the same place in each half of the rotated dims; interleaved: any vector), so a rotation needs no exchange and the
// norm three shuffles.  A lane group takes up to four heads of one token and one tensor: the angles and the norm's weights
// are loaded once for them, addresses advance by a stride, and their vectors are brought in by cp.async, 16 KB a CTA and
// 96 KB an SM in flight, which registers could not hold (register loads: 436 us at best for the layer; 256 threads or eight
// heads a group: 325-455 us, and slower at 4097 tokens).  Issue slots are the second bound: groups that ran over tensors'
// borders, with tensor, address and weights found anew for each head, took 285 instructions for a lane's 16 elements, and
// 50.6 us for the 16384 tokens, 18.5 us for the 4097.  Weights in registers want 78 of them: six CTAs an SM (five: 49.6 us;
// seven, with spills: 47.5 us).
#include "attn_common.cuh"
#include "paged_common.cuh"

namespace spruce {

constexpr int kRowThreads = 128;
constexpr int kHeadsPerGroup = 4;
constexpr int kRowCtasPerSm = 6;

__device__ __forceinline__ uint64_t unpack2(uint32_t v, __nv_bfloat16) {
  return f2_pack(__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u));
}
__device__ __forceinline__ uint64_t unpack2(uint32_t v, __half) {
  const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&v));
  return f2_pack(f.x, f.y);
}
// A 16-byte vector to and from packed fp32 pairs.
template <typename T, int NP>
__device__ __forceinline__ void unpack16(const uint4& v, uint64_t (&x)[NP]) {
  if constexpr (sizeof(T) == 4) {
    x[0] = f2_pack(__uint_as_float(v.x), __uint_as_float(v.y));
    x[1] = f2_pack(__uint_as_float(v.z), __uint_as_float(v.w));
  } else {
    x[0] = unpack2(v.x, T());
    x[1] = unpack2(v.y, T());
    x[2] = unpack2(v.z, T());
    x[3] = unpack2(v.w, T());
  }
}
template <typename T, int NP>
__device__ __forceinline__ uint4 pack16(const uint64_t (&x)[NP]) {
  float f[2 * NP];
#pragma unroll
  for (int i = 0; i < NP; ++i) f2_unpack(x[i], f[2 * i], f[2 * i + 1]);
  if constexpr (sizeof(T) == 4)
    return make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
  else
    return make_uint4(Pack2<T>::pack(f[0], f[1]), Pack2<T>::pack(f[2], f[3]), Pack2<T>::pack(f[4], f[5]),
                      Pack2<T>::pack(f[6], f[7]));
}
__device__ __forceinline__ void load_pairs(const float* p, uint64_t& a, uint64_t& b) {
  const float4 v = __ldg(reinterpret_cast<const float4*>(p));
  a = f2_pack(v.x, v.y);
  b = f2_pack(v.z, v.w);
}

__device__ __forceinline__ uint64_t load_pair(const float* p) {
  const float2 v = __ldg(reinterpret_cast<const float2*>(p));
  return f2_pack(v.x, v.y);
}

__device__ __forceinline__ void copy16(uint4* dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(dst)), "l"(src) : "memory");
}
// Until at most n of this thread's latest copy groups are under way (n a constant after unrolling).
__device__ __forceinline__ void wait_copies(int n) {
  switch (n) {
    case 0: asm volatile("cp.async.wait_group 0;" ::: "memory"); break;
    case 1: asm volatile("cp.async.wait_group 1;" ::: "memory"); break;
    case 2: asm volatile("cp.async.wait_group 2;" ::: "memory"); break;
    default: asm volatile("cp.async.wait_group 3;" ::: "memory"); break;
  }
}

// Interleaved pairs: x[e] holds (a, b) of one pair, its angle is number first + e of cs / sn.
template <int NP>
__device__ __forceinline__ void turn_pairs(uint64_t (&x)[NP], const uint64_t (&cs)[NP], const uint64_t (&sn)[NP], int first) {
#pragma unroll
  for (int e = 0; e < NP; ++e) {
    const int i = first + e;
    float c0, c1, s0, s1, u, v;
    f2_unpack(cs[i / 2], c0, c1);
    f2_unpack(sn[i / 2], s0, s1);
    f2_unpack(x[e], u, v);
    const float c = i & 1 ? c1 : c0, s = i & 1 ? s1 : s0;
    x[e] = f2_pack(u * c - v * s, v * c + u * s);
  }
}

// Where a token's rotation and cache rows are.
struct TokenPlace {
  const float* angles;  // its row of the table
  int64_t page;
  int slot;
  bool write, cached;   // the token is one of a sequence's; its cache row exists
};

template <bool APPEND>
__device__ __forceinline__ TokenPlace place_token(const RowsArgs& a, bool live, int n, int b, int t) {
  TokenPlace w{nullptr, 0, 0, live, live};
  int64_t pos = t;
  if constexpr (APPEND) {
    if (live) {
      // A sequence of one token most often: s == n.  These loads do not wait for one another.
      const int begin = a.cu_q[0], end = a.cu_q[a.S];
      int s = min(n, a.S - 1);
      const int first = a.cu_q[s];
      int next = a.cu_q[s + 1], kv = a.kv_lens[s];
      w.write = begin <= n && n < end;  // the search then ends at a sequence that holds n
      if (w.write && (first > n || next <= n)) {
        int lo = 0, hi = a.S;  // the largest s with cu_q[s] <= n
        while (hi - lo > 1) {
          const int mid = (lo + hi) >> 1;
          if (a.cu_q[mid] <= n) lo = mid;
          else hi = mid;
        }
        s = lo;
        next = a.cu_q[s + 1];
        kv = a.kv_lens[s];
      }
      pos = (int64_t)kv - next + n;
      const int p = pos >= 0 && pos < 0x7fffffff ? static_cast<int>(pos) : -1;
      const int pi = p >= 0 ? p / a.page_size : a.max_pages;
      w.cached = w.write && pi < a.max_pages;
      if (w.write && !w.cached) raise_status(a.status, SPRUCE_STATUS_BAD_LENGTH);
      if (w.cached) {
        w.page = a.block_table[(int64_t)s * a.table_stride + pi];
        w.cached = w.page >= 0 && w.page < a.num_pages;
        if (!w.cached) raise_status(a.status, SPRUCE_STATUS_BAD_PAGE);
        w.slot = p - pi * a.page_size;
      }
    }
  }
  if (a.rd > 0) {
    if (a.positions != nullptr && w.write) pos = a.positions[b * a.pos_sb + t * a.pos_st];
    if (w.write && (pos < 0 || pos >= a.table_rows)) raise_status(a.status, SPRUCE_STATUS_BAD_POSITION);
    pos = pos < 0 ? 0 : (pos < a.table_rows ? pos : a.table_rows - 1);
    w.angles = a.rope + pos * a.rd;
  }
  return w;
}

// The tensor a head belongs to, and its number there.
__device__ __forceinline__ const Rows& rows_of(const RowsArgs& a, int h, int& hh) {
  hh = h < a.Hq ? h : (h < a.Hq + a.Hkv ? h - a.Hq : h - a.Hq - a.Hkv);
  return h < a.Hq ? a.q : (h < a.Hq + a.Hkv ? a.k : a.v);
}

// 16-byte vectors.  Bound by instruction issue before HBM unless the arithmetic is packed: fp32 pairs throughout.
template <typename T, bool APPEND>
__global__ void __launch_bounds__(kRowThreads, kRowCtasPerSm)
    norm_rope_kernel(const RowsArgs a, int lpr, int hc, int chunks) {
  let_next_kernel_start();  // the attention over the cache sets up meanwhile, and waits for our end
  constexpr int HC = kHeadsPerGroup, VN = 16 / sizeof(T), NP = VN / 2;
  __shared__ uint4 stage[HC * 2][kRowThreads];  // a thread's own vectors: no barrier
  const int l = threadIdx.x & (lpr - 1);
  const unsigned block = blockIdx.x / chunks;
  // The CTA's heads, of one tensor: its chunks are the queries', then the keys' (then the values').
  int h0 = static_cast<int>(blockIdx.x - block * chunks) * hc;
  const int hq = (a.Hq + hc - 1) / hc * hc, hk = (a.Hkv + hc - 1) / hc * hc;
  const bool isq = h0 < hq, isv = h0 >= hq + hk;
  const Rows& r = isq ? a.q : (isv ? a.v : a.k);
  h0 -= isq ? 0 : (isv ? hq + hk : hq);
  const int rows = min(hc, (isq ? a.Hq : a.Hkv) - h0);
  const int64_t n = (int64_t)block * (kRowThreads / lpr) + threadIdx.x / lpr;
  const bool live = n < (int64_t)a.B * a.T;
  const int b = a.B == 1 ? 0 : static_cast<int>(n / a.T), t = static_cast<int>(n - (int64_t)b * a.T);
  const int rd = isv ? 0 : a.rd, items = a.D / (2 * VN), nrot = rd / (2 * VN);
  // This lane's two vectors.  Half pairs: the same place in each half of the rotated dims (or of the rest).  Interleaved:
  // of each half of the head, as a pair lies in one vector.  Adjacent lanes take adjacent vectors either way.
  const bool in = live && l < items;
  const bool rot = a.interleaved ? l * VN < rd : l < nrot;
  const int oa = a.interleaved || rot ? l * VN : rd + (l - nrot) * VN;
  const int ob = a.interleaved ? a.D / 2 + oa : (rot ? rd / 2 : (a.D - rd) / 2) + oa;
  const bool rot_b = a.interleaved ? ob < rd : rot;

  // The rows first: where they go and how they turn takes dependent loads of its own.
  const T* src = static_cast<const T*>(r.x) + b * r.sb + h0 * r.sh + t * r.st;
#pragma unroll
  for (int i = 0; i < HC; ++i) {
    if (in && i < rows) {
      copy16(&stage[2 * i][threadIdx.x], src + oa);
      copy16(&stage[2 * i + 1][threadIdx.x], src + ob);
      src += r.sh;
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  }
  const TokenPlace w = place_token<APPEND>(a, live, static_cast<int>(n), b, t);
  // cos and sin of the pairs (half), or of vector a's pairs and then vector b's (interleaved).
  uint64_t cs[NP], sn[NP];
  if constexpr (NP == 4) {
    if (rot && in) {
      const float* c = w.angles + (a.interleaved ? oa / 2 : oa);
      load_pairs(c, cs[0], cs[1]);
      load_pairs(c + rd / 2, sn[0], sn[1]);
    }
    if (rot_b && in) {
      const float* c = w.angles + (a.interleaved ? ob / 2 : oa + 4);
      load_pairs(c, cs[2], cs[3]);
      load_pairs(c + rd / 2, sn[2], sn[3]);
    }
  } else if (in) {
    if (a.interleaved) {
      if (rot) {
        cs[0] = load_pair(w.angles + oa / 2);
        sn[0] = load_pair(w.angles + rd / 2 + oa / 2);
      }
      if (rot_b) {
        cs[1] = load_pair(w.angles + ob / 2);
        sn[1] = load_pair(w.angles + rd / 2 + ob / 2);
      }
    } else if (rot) {
      load_pairs(w.angles + oa, cs[0], cs[1]);
      load_pairs(w.angles + rd / 2 + oa, sn[0], sn[1]);
    }
  }
  const bool norm = r.weight != nullptr, store = in && w.write && (!APPEND || isq || w.cached);
  const float per_dim = 1.0f / static_cast<float>(a.D);
  T* dst = static_cast<T*>(r.out) +
           (APPEND && !isq ? w.page * r.ob + h0 * r.oh + w.slot * r.ot : b * r.ob + h0 * r.oh + t * r.ot);
  uint64_t wa[NP], wb[NP];
  if (norm && in) {
#pragma unroll
    for (int e = 0; e < NP; e += 2) {
      load_pairs(r.weight + oa + 2 * e, wa[e], wa[e + 1]);
      load_pairs(r.weight + ob + 2 * e, wb[e], wb[e + 1]);
    }
  }

#pragma unroll
  for (int i = 0; i < HC; ++i) {
    wait_copies(HC - 1 - i);
    if (i >= rows) break;  // of the whole CTA
    uint4 ra = make_uint4(0, 0, 0, 0), rb = ra;
    if (in) {
      ra = stage[2 * i][threadIdx.x];
      rb = stage[2 * i + 1][threadIdx.x];
    }
    if (!isv) {
      uint64_t x[NP], y[NP];
      unpack16<T>(ra, x);
      unpack16<T>(rb, y);
      if (norm) {  // the shuffles are executed by every lane; a row's lanes are adjacent
        uint64_t s2 = f2_mul(x[0], x[0]);
#pragma unroll
        for (int e = 1; e < NP; ++e) s2 = f2_fma(x[e], x[e], s2);
#pragma unroll
        for (int e = 0; e < NP; ++e) s2 = f2_fma(y[e], y[e], s2);
        float s0, s1;
        f2_unpack(s2, s0, s1);
        float ss = s0 + s1;
        for (int o = lpr >> 1; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
        const float inv = rsqrtf(fmaf(ss, per_dim, a.eps));
        const uint64_t inv2 = f2_pack(inv, inv);
        if (in) {
#pragma unroll
          for (int e = 0; e < NP; ++e) {
            x[e] = f2_mul(x[e], f2_mul(wa[e], inv2));
            y[e] = f2_mul(y[e], f2_mul(wb[e], inv2));
          }
        }
      }
      if (rot) {
        if (a.interleaved) {
          // Angle i of cs is pair i of vector a, or pair i - NP of vector b.
          turn_pairs(x, cs, sn, 0);
          if (rot_b) turn_pairs(y, cs, sn, NP);
        } else {
#pragma unroll
          for (int e = 0; e < NP; ++e) {
            const uint64_t u = x[e], v = y[e];
            x[e] = f2_sub(f2_mul(u, cs[e]), f2_mul(v, sn[e]));
            y[e] = f2_fma(u, sn[e], f2_mul(v, cs[e]));
          }
        }
      }
      ra = pack16<T>(x);
      rb = pack16<T>(y);
    }
    if (store) {
      *reinterpret_cast<uint4*>(dst + oa) = ra;
      *reinterpret_cast<uint4*>(dst + ob) = rb;
    }
    dst += r.oh;
  }
}

// Rows that 16-byte vectors do not fit: a warp a row, one element a load; pairs l, l + 32, ... of at most 128.
template <typename T, bool APPEND>
__global__ void __launch_bounds__(kRowThreads) norm_rope_scalar_kernel(const RowsArgs a) {
  const int lane = threadIdx.x & 31;
  const int heads = a.Hq + (APPEND ? 2 : 1) * a.Hkv;
  const int64_t row = (int64_t)blockIdx.x * (kRowThreads / 32) + (threadIdx.x >> 5);
  const int64_t n = row / heads;
  const int h = static_cast<int>(row - n * heads);
  if (n >= (int64_t)a.B * a.T) return;
  const int b = static_cast<int>(n / a.T), t = static_cast<int>(n - (int64_t)b * a.T);
  const TokenPlace w = place_token<APPEND>(a, true, static_cast<int>(n), b, t);
  int hh;
  const Rows& r = rows_of(a, h, hh);
  const bool isq = h < a.Hq, isv = h >= a.Hq + a.Hkv;
  if (!w.write || (APPEND && !isq && !w.cached)) return;
  const T* src = static_cast<const T*>(r.x) + b * r.sb + hh * r.sh + t * r.st;
  T* dst = static_cast<T*>(r.out) +
           (APPEND && !isq ? w.page * r.ob + hh * r.oh + w.slot * r.ot : b * r.ob + hh * r.oh + t * r.ot);
  const int pairs = a.D / 2, nrot = isv ? 0 : a.rd / 2;
  T x[4], y[4];
  float ss = 0.0f;
#pragma unroll
  for (int it = 0; it < 4; ++it) {
    const int p = lane + 32 * it;
    if (p >= pairs) continue;
    const bool half = p < nrot && !a.interleaved;
    x[it] = src[half ? p : 2 * p];
    y[it] = src[half ? p + nrot : 2 * p + 1];
    const float u = Elem<T>::to_f(x[it]), v = Elem<T>::to_f(y[it]);
    ss = fmaf(u, u, fmaf(v, v, ss));
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
  const float inv = rsqrtf(ss / static_cast<float>(a.D) + a.eps);
#pragma unroll
  for (int it = 0; it < 4; ++it) {
    const int p = lane + 32 * it;
    if (p >= pairs) continue;
    const bool half = p < nrot && !a.interleaved;
    const int oa = half ? p : 2 * p, ob = half ? p + nrot : 2 * p + 1;
    if (isv) {
      dst[oa] = x[it];
      dst[ob] = y[it];
      continue;
    }
    float u = Elem<T>::to_f(x[it]), v = Elem<T>::to_f(y[it]);
    if (r.weight != nullptr) {
      u *= inv * r.weight[oa];
      v *= inv * r.weight[ob];
    }
    if (p < nrot) {
      const float c = w.angles[p], s = w.angles[nrot + p], u0 = u;
      u = u0 * c - v * s;
      v = v * c + u0 * s;
    }
    dst[oa] = Elem<T>::from_f(u);
    dst[ob] = Elem<T>::from_f(v);
  }
}

template <typename T, bool APPEND>
static cudaError_t launch_rows_typed(const RowsArgs& a, bool vec, cudaStream_t stream) {
  const int heads = a.Hq + (APPEND ? 2 : 1) * a.Hkv;
  const int64_t tokens = (int64_t)a.B * a.T;
  if (!vec) {
    const int64_t ctas = (tokens * heads + kRowThreads / 32 - 1) / (kRowThreads / 32);
    if (ctas > 0x7fffffff) return cudaErrorInvalidValue;
    norm_rope_scalar_kernel<T, APPEND><<<(unsigned)ctas, kRowThreads, 0, stream>>>(a);
    return cudaGetLastError();
  }
  const int items = a.D / (32 / (int)sizeof(T));
  int lpr = 1;
  while (lpr < items) lpr *= 2;
  const int per = kRowThreads / lpr;
  const int64_t blocks = (tokens + per - 1) / per;
  // Four rows a group keep enough bytes in flight; where that leaves SMs without work, one: 64 single tokens of 36 rows take
  // 4.2 us so, 5.3 us with two.
  auto chunks_of = [&](int hc) { return (a.Hq + hc - 1) / hc + (APPEND ? 2 : 1) * ((a.Hkv + hc - 1) / hc); };
  int hc = kHeadsPerGroup;
  if (blocks * chunks_of(hc) < 2 * 148) hc = 1;
  const int chunks = chunks_of(hc);
  if (blocks * chunks > 0x7fffffff) return cudaErrorInvalidValue;
  norm_rope_kernel<T, APPEND><<<(unsigned)(blocks * chunks), kRowThreads, 0, stream>>>(a, lpr, hc, chunks);
  return cudaGetLastError();
}

cudaError_t launch_norm_rope(const RowsArgs& a, int dtype, cudaStream_t stream) {
  const int V = dtype == SPRUCE_DTYPE_F32 ? 4 : 8;
  // 16-byte vectors: pairs that fill them, and bases and strides that keep every one aligned.
  auto at16 = [](const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; };
  auto fits = [&](const Rows& r) {
    return r.x == nullptr || (at16(r.x) && at16(r.out) && at16(r.weight) && r.sb % V == 0 && r.sh % V == 0 &&
                              r.st % V == 0 && r.ob % V == 0 && r.oh % V == 0 && r.ot % V == 0);
  };
  const bool vec = a.D % (2 * V) == 0 && a.rd % (2 * V) == 0 && at16(a.rope) && fits(a.q) && fits(a.k) && fits(a.v);
  const bool append = a.cu_q != nullptr;
  if (dtype == SPRUCE_DTYPE_F32)
    return append ? launch_rows_typed<float, true>(a, vec, stream) : launch_rows_typed<float, false>(a, vec, stream);
  if (dtype == SPRUCE_DTYPE_BF16)
    return append ? launch_rows_typed<__nv_bfloat16, true>(a, vec, stream)
                  : launch_rows_typed<__nv_bfloat16, false>(a, vec, stream);
  return append ? launch_rows_typed<__half, true>(a, vec, stream) : launch_rows_typed<__half, false>(a, vec, stream);
}

}  // namespace spruce
