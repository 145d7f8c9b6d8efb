// Softmax weight of whole key blocks on the tcgen05 tensor cores (bf16 / fp16).
//
// The formula is mass.cu's.  A row tile is 128 tokens of one head (two query blocks); the tiles of a (batch, KV head) in
// the order token tile, head are taken in pairs, so an odd group wastes none, and a pair shares its key tiles of 128:
//   S_t = Q_t K^T   M128 N128 K16, D / 16 MMAs.
// Nothing follows S: for each row and block of 64 keys the softmax warps form b = log2(sum 2^(s - m)) + m over the running
// maximum m, keep it in the workspace (written and read by the same thread) and add it to the row's total.  When a unit's
// keys are through, 2^(b - total) is summed over the 64 rows of a query block: 32 a round by a transposing butterfly, 31
// shuffles for 32 sums of a warp.  Heads are added by a second kernel in their order, so nothing depends on timing.
//
// Warps: 0-3 the first 64 keys of tile 0 (thread = row = TMEM lane), 4-7 the others, 8-15 likewise of tile 1, 16 and 17
// issue the MMAs of a tile each (a check of a barrier waits behind the MMAs that its warp has queued; one issuer for both:
// 4.55 ms where two take 4.48), 16 owns TMEM, 18 loads Q and K.  Four softmax warps a scheduler hide each other's latencies
// (two of 128 keys a row: 4.72 ms where these took 4.58).  Each S_t has two buffers, which fill TMEM: the tensor core runs
// a tile ahead of the exponentials, which are slower (16 a clock and SM, against 32 scores a clock of the MMAs at d =
// 128).  Part of them runs on the FMA pipe instead, as a polynomial of degree 4 with a relative error of 2.7e-6: a quarter
// (none, 1/8, 1/4, 3/8: 4.62, 4.53, 4.48, 4.78 ms; then the exponentials' pipe is 72% busy and issue 63%: neither is full, what
// is left is the latency of a block's chain of maximum, exponentials and sum).  Exponentials over
// an old maximum, without a pass for the block's own, measured 1.5% slower: the branch for a row that outgrows it keeps
// blocks from overlapping.
//
// On a B200, 28 query / 4 KV heads of 128 in bf16: 32768 tokens 4.5 to 4.7 ms, 825 to 850 TFLOP/s (the exponentials alone would
// take 2.4 ms with a quarter on the FMA pipe or 3.2 without, the MMAs 2.4); 131072 tokens 76 ms.
//
// Units go to the CTAs longest first, back and forth over them.
//
// Every wait is bounded (common.cuh).
#include <algorithm>
#include <type_traits>

#include "attn_common.cuh"
#include "mass_common.cuh"

namespace spruce {

constexpr int kBmThreads = 608, kBmMma = 16, kBmMma1 = 17, kBmLoad = 18;
constexpr int kBmKeys = 128;
constexpr int kBmMufu = 6;  // of 8 pairs of exponentials; the others by polynomial

template <int D>
struct BlockLayout {
  static constexpr int KST = D == 128 ? 4 : 6;
  static constexpr int NP = D / 64;
  static constexpr int PANEL = 128 * 128;
  static constexpr int TILE = NP * PANEL;
  static constexpr int OFF_Q = 0;
  static constexpr int OFF_K = 2 * TILE;
  static constexpr int OFF_SUM = OFF_K + KST * TILE;     // [8 pairs of warps][2][32] floats: sums handed to the other warp of a block
  static constexpr int OFF_ML = OFF_SUM + 8 * 2 * 32 * 4;  // [2][2 tiles][2 halves][128] maxima and sums
  static constexpr int OFF_BAR = OFF_ML + 2 * 512 * 8;
  // k_full[], k_empty[], q_full, q_empty, s_full[2][2], s_empty[2][2], drain[2]
  static constexpr int NBAR = 2 * KST + 2 + 4 + 4 + 2;
  static constexpr int OFF_MISC = OFF_BAR + NBAR * 8;
  static constexpr int BYTES = 1024 + OFF_MISC + 16;
  static_assert(BYTES <= 227 * 1024, "shared memory of a CTA");
};

struct BlockParams {
  BlockMassArgs a;
  int rep, tiles, qb, kbp;   // token tiles of 128; query blocks; key blocks rounded up to 64
  int pairs;                 // pairs of row tiles of a (batch, KV head)
  int units;
  float* blocks;             // [CTA][kbp][256]
  float* part;               // [B Hkv][tiles * rep][2 query blocks][2 halves][kbp / 2]
};

// 2^x of two values on the FMA pipe: n = round(x) by the 1.5 * 2^23 trick, 2^(x - n) by a polynomial fitted for minimal relative
// error on [-0.5, 0.5] (iterated weighted least squares; 2.7e-6 in fp32), n added to the exponent.  x <= 127; below -125 the
// result is 2^-125 (NaN too).
__device__ __forceinline__ void poly4_exp2_x2(float x0, float x1, float& e0, float& e1) {
  const float kRound = 12582912.0f;
  const uint64_t x = f2_pack(fmaxf(x0, -125.0f), fmaxf(x1, -125.0f));
  const uint64_t kr = f2_pack(kRound, kRound);
  const uint64_t t = f2_add(x, kr);
  const uint64_t f = f2_sub(x, f2_sub(t, kr));
  uint64_t q = f2_fma(f2_pack(0.009570102207362652f, 0.009570102207362652f), f, f2_pack(0.05591785907745361f, 0.05591785907745361f));
  q = f2_fma(q, f, f2_pack(0.240247443318367f, 0.240247443318367f));
  q = f2_fma(q, f, f2_pack(0.6931217908859253f, 0.6931217908859253f));
  q = f2_fma(q, f, f2_pack(0.9999992847442627f, 0.9999992847442627f));
  float q0, q1, t0, t1;
  f2_unpack(q, q0, q1);
  f2_unpack(t, t0, t1);
  e0 = __int_as_float(__float_as_int(q0) + (__float_as_int(t0) << 23));
  e1 = __int_as_float(__float_as_int(q1) + (__float_as_int(t1) << 23));
}

// max(a, b, c), NaN where one of them is.
__device__ __forceinline__ float bm_max3(float a, float b, float c) {
  float d;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

// A CTA's units, longest first.
struct BlockUnit {
  int bg, tile[2], keys[2];  // row tile (token tile * rep + head; -1: none) and its key tiles
};
__device__ __forceinline__ bool block_unit(const BlockParams& p, int round, BlockUnit& u) {
  const int G = gridDim.x, c = blockIdx.x;
  const int at = round * G + (round & 1 ? G - 1 - c : c);
  if (at >= p.units) return false;
  const int groups = p.a.B * p.a.Hkv;
  const int pair = p.pairs - 1 - at / groups;
  u.bg = at % groups;
#pragma unroll
  for (int t = 0; t < 2; ++t) {
    const int tile = 2 * pair + t;
    u.tile[t] = tile < p.tiles * p.rep ? tile : -1;
    u.keys[t] = u.tile[t] < 0 ? 0 : tile / p.rep + 1;
  }
  return true;
}

template <typename T, int D>
__global__ void __launch_bounds__(kBmThreads, 1)
    block_mass_sm100_kernel(const __grid_constant__ CUtensorMap tmq, const __grid_constant__ CUtensorMap tmk,
                            const __grid_constant__ BlockParams p) {
  using L = BlockLayout<D>;
  constexpr int KST = L::KST;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  uint32_t* const status = p.a.status;
  uint64_t* k_full = reinterpret_cast<uint64_t*>(smem + L::OFF_BAR);
  uint64_t* k_empty = k_full + KST;
  uint64_t* q_full = k_empty + KST;
  uint64_t* q_empty = q_full + 1;
  uint64_t* s_full = q_empty + 1;      // [tile * 2 + buffer]
  uint64_t* s_empty = s_full + 4;      // 256 arrivals
  uint64_t* drain = s_empty + 4;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + L::OFF_MISC);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + L::OFF_MISC + 4);

  if (warp == kBmLoad) {
    if (lane == 0) {
      *abort_flag = 0;
      for (int s = 0; s < KST; ++s) {
        mbar_init(&k_full[s], 1);
        mbar_init(&k_empty[s], 2);
      }
      mbar_init(q_full, 1);
      mbar_init(q_empty, 2);
      for (int s = 0; s < 4; ++s) {
        mbar_init(&s_full[s], 1);
        mbar_init(&s_empty[s], 256);
      }
      mbar_init(&drain[0], 1);
      mbar_init(&drain[1], 1);
      fence_barrier_init();
      prefetch_tmap(&tmq);
      prefetch_tmap(&tmk);
    }
    __syncwarp();
  } else if (warp == kBmMma) {
    tmem_alloc(tmem_slot, 512u);
    tmem_relinquish();
  }
  tc_fence_before();
  let_next_kernel_start();
  wait_for_earlier_kernels();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  BlockUnit u;

  if (warp == kBmLoad) {
    // ------------------------------------------------------------ Q and K
    const bool leader = elect_one();
    int st = 0, loaded = 0;
    uint32_t turn = 1;
    bool ok = true;
    for (int r = 0; ok && block_unit(p, r, u); ++r) {
      const int b = u.bg / p.a.Hkv, g = u.bg % p.a.Hkv;
      if (r > 0 && !(ok = __all_sync(0xffffffffu, mbar_wait(q_empty, (r - 1) & 1, status, abort_flag)))) break;
      if (leader) mbar_arrive_expect_tx(q_full, (u.tile[1] < 0 ? 1 : 2) * L::TILE);
      __syncwarp();
#pragma unroll
      for (int t = 0; t < 2; ++t)
        if (leader && u.tile[t] >= 0)
#pragma unroll
          for (int pp = 0; pp < L::NP; ++pp)
            tma_load_4d(smem + L::OFF_Q + t * L::TILE + pp * L::PANEL, &tmq, q_full, pp * 64,
                        g * p.rep + u.tile[t] % p.rep, u.tile[t] / p.rep * 128, b);
      __syncwarp();
      const int n = max(u.keys[0], u.keys[1]);
      for (int j = 0; j < n; ++j) {
        if (loaded >= KST && !(ok = __all_sync(0xffffffffu, mbar_wait(&k_empty[st], turn, status, abort_flag)))) break;
        if (leader) {
          mbar_arrive_expect_tx(&k_full[st], L::TILE);
#pragma unroll
          for (int pp = 0; pp < L::NP; ++pp)
            tma_load_4d(smem + L::OFF_K + st * L::TILE + pp * L::PANEL, &tmk, &k_full[st], pp * 64, g, j * kBmKeys, b);
        }
        __syncwarp();
        ++loaded;
        if (++st == KST) {
          st = 0;
          turn ^= 1;
        }
      }
      if (!ok || *abort_flag) mbar_wait(q_full, r & 1, status, nullptr);  // no copy may be in flight at the exit
    }
    for (int k = max(0, loaded - KST); k < loaded; ++k) mbar_wait(&k_full[k % KST], (k / KST) & 1, status, nullptr);
    __syncwarp();
  } else if (warp == kBmMma || warp == kBmMma1) {
    // ------------------------------------------------------------ MMA issuers, one a tile
    const bool leader = elect_one();
    const int t = warp - kBmMma;
    constexpr uint32_t idesc = idesc_f16(UmmaFormat<T>::value, 0, 0, 128, 128);
    const uint64_t dq0 = smem_desc(smem_u32(smem + L::OFF_Q + t * L::TILE), 16, 1024);
    const uint64_t dk0 = smem_desc(smem_u32(smem + L::OFF_K), 16, 1024);
    auto commit = [&](uint64_t* bar) {
      if (leader) umma_commit(bar);
      __syncwarp();
    };
    auto wait = [&](uint64_t* bar, uint32_t parity) {
      return __all_sync(0xffffffffu, mbar_wait(bar, parity, status, abort_flag));
    };
    int st = 0;
    uint32_t turn = 0, issued = 0;
    bool ok = true;
    for (int r = 0; ok && block_unit(p, r, u); ++r) {
      if (!(ok = wait(q_full, r & 1))) break;
      const int n = max(u.keys[0], u.keys[1]);
      for (int j = 0; j < n; ++j) {
        ok = wait(&k_full[st], turn);
        if (ok && j < u.keys[t]) {
          const uint32_t buf = issued & 1;
          if (issued >= 2) ok = wait(&s_empty[2 * t + buf], ((issued >> 1) - 1) & 1);
          if (!ok) break;
          ++issued;
          tc_fence_after();
#pragma unroll
          for (int ks = 0; ks < D / 16; ++ks) {
            const uint32_t off = ((ks >> 2) * L::PANEL + (ks & 3) * 32) >> 4;
            if (leader)
              umma_f16_ss(tmem + (2 * t + buf) * 128, dq0 + off, dk0 + ((st * L::TILE) >> 4) + off, idesc, ks > 0 ? 1u : 0u);
            __syncwarp();
          }
          commit(&s_full[2 * t + buf]);
        }
        if (!ok) break;
        commit(&k_empty[st]);
        if (++st == KST) {
          st = 0;
          turn ^= 1;
        }
      }
      if (ok) commit(q_empty);
    }
    commit(&drain[t]);  // no MMA may be in flight when TMEM is released
    mbar_wait(&drain[t], 0, status, nullptr);
    __syncwarp();
  } else {
    // ------------------------------------------------------------ softmax and sums
    const int t = warp >> 3, half = (warp >> 2) & 1;  // tile, and which 64 of its keys
    const uint32_t tS = tmem + (static_cast<uint32_t>((warp & 3) * 32) << 16) + t * 256 + half * 64;
    const int row = (warp & 3) * 32 + lane;
    float* const mine = p.blocks + ((int64_t)blockIdx.x * p.kbp + half) * 256 + t * 128 + row;  // [key tile] at stride 512
    float* const given = reinterpret_cast<float*>(smem + L::OFF_SUM) + (warp >> 1) * 64;        // [2][32] of this pair of warps
    float2* const ml = reinterpret_cast<float2*>(smem + L::OFF_ML) + t * 256 + row;             // [half] at stride 128
    const float sl2 = p.a.scale_log2;
    const uint64_t sl2x2 = f2_pack(sl2, sl2);
    uint32_t sj = 0, rounds = 0;
    bool ok = true;
    // After a wait that ran out the warps still meet at the barriers.
    for (int r = 0; block_unit(p, r, u); ++r) {
      const int n = u.keys[t];
      if (n == 0) continue;
      float m = -INFINITY, l = 0.0f;
      // 64 keys: b of the block, the total moved on.  lim: columns that the row sees.
      auto block = [&](const float (&s)[64], auto masked_c, int lim, int j) {
        constexpr bool masked = decltype(masked_c)::value;
        float z[64];
#pragma unroll
        for (int c = 0; c < 64; ++c) z[c] = masked && c >= lim ? -INFINITY : s[c];
        float mx[4];
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          mx[c] = bm_max3(z[c], z[c + 4], z[c + 8]);
#pragma unroll
          for (int i = 12; i < 60; i += 8) mx[c] = bm_max3(mx[c], z[c + i], z[c + i + 4]);
          mx[c] = bm_max3(mx[c], z[c + 60], z[c + 60]);
        }
        const float top = bm_max3(bm_max3(mx[0], mx[1], mx[2]), mx[3], mx[3]) * sl2;
        const float up = fmaxf(m, top);                        // a NaN is not taken over
        const float ref = up == -INFINITY ? 0.0f : up;
        // A score of NaN or +inf makes the sum NaN whichever column holds it (the polynomial takes NaN for a number).
        const float neg = top < INFINITY ? -ref : __int_as_float(0x7fffffff);
        const uint64_t neg2 = f2_pack(neg, neg);
        uint64_t sum2[2] = {f2_pack(0.0f, 0.0f), f2_pack(0.0f, 0.0f)};
#pragma unroll
        for (int k = 0; k < 32; ++k) {
          float x0, x1, e0, e1;
          f2_unpack(f2_fma(f2_pack(z[2 * k], z[2 * k + 1]), sl2x2, neg2), x0, x1);
          if (!masked && (k % 8) >= kBmMufu) {
            poly4_exp2_x2(x0, x1, e0, e1);
          } else {
            e0 = fast_exp2(x0);
            e1 = fast_exp2(x1);
          }
          sum2[k & 1] = f2_add(sum2[k & 1], f2_pack(e0, e1));
        }
        float a0, a1, a2, a3;
        f2_unpack(sum2[0], a0, a1);
        f2_unpack(sum2[1], a2, a3);
        // A block of -inf throughout weighs nothing: the polynomial does not go below 2^-125, which is not little to a row whose
        // total turns out far below.
        const float sum = top == -INFINITY ? 0.0f : (a0 + a1) + (a2 + a3);
        l = fmaf(l, fast_exp2(m - ref), sum);
        m = up;
        mine[(int64_t)j * 512] = ref + __log2f(sum);
      };
      for (int j = 0; ok && j < n; ++j, ++sj) {
        const uint32_t buf = sj & 1;
        ok = __all_sync(0xffffffffu, mbar_wait(&s_full[2 * t + buf], (sj >> 1) & 1, status, abort_flag));
        if (!ok) break;
        tc_fence_after();
        float s[64];
        tmem_ld32(tS + buf * 128, *reinterpret_cast<float(*)[32]>(s));
        tmem_ld32(tS + buf * 128 + 32, *reinterpret_cast<float(*)[32]>(s + 32));
        tmem_wait_ld();
        tc_fence_before();
        mbar_arrive(&s_empty[2 * t + buf]);
        if (j + 1 < n)
          block(s, std::false_type{}, 0, j);
        else  // the diagonal
          block(s, std::true_type{}, row + 1 - half * 64, j);
      }
      // The row's total over both halves.
      float2* const x = ml + (r & 1) * 512;
      x[half * 128] = make_float2(m, l);
      named_barrier_sync(9 + t, 256);
      const float2 other = x[128 - half * 128];
      const bool in = u.tile[t] / p.rep * 128 + row < p.a.T;
      const float top = fmaxf(m, other.x), ref = top == -INFINITY ? 0.0f : top;
      const float all = l * fast_exp2(m - ref) + other.y * fast_exp2(other.x - ref);
      // Rows past the prompt weigh nothing, though zero times an infinite key makes their scores NaN.
      const float total = !in || (top == -INFINITY && all == all) ? INFINITY : ref + __log2f(all);
      // Weights of this warp's 32 rows, summed, and those of the other warp of the query block.
      float* const out = p.part + (((int64_t)u.bg * p.tiles * p.rep + u.tile[t]) * 2 + ((warp >> 1) & 1)) * p.kbp +
                         half * (p.kbp / 2);
      for (int j0 = 0; j0 < n; j0 += 32, ++rounds) {
        float v[32];
#pragma unroll
        for (int k = 0; k < 32; ++k) v[k] = in && j0 + k < n ? mine[(int64_t)(j0 + k) * 512] : -INFINITY;
#pragma unroll
        for (int k = 0; k < 32; ++k) v[k] = fast_exp2(v[k] - total);
        // Halves of the values change sides with a lane half away, until lane k holds the sum of value k.
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
          const bool up = lane & o;
#pragma unroll
          for (int k = 0; k < o; ++k) {
            const float send = up ? v[k] : v[k + o], keep = up ? v[k + o] : v[k];
            v[k] = keep + __shfl_xor_sync(0xffffffffu, send, o);
          }
        }
        if (warp & 1) given[(rounds & 1) * 32 + lane] = v[0];
        named_barrier_sync(1 + (warp >> 1), 64);
        if (!(warp & 1)) out[j0 + lane] = v[0] + given[(rounds & 1) * 32 + lane];
      }
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == kBmMma) {
    tc_fence_after();
    tmem_dealloc(tmem, 512u);
  }
}

// Heads added in their order, rows scaled to a mean, zeros past the diagonal.
__global__ void __launch_bounds__(256) block_mass_join_kernel(const BlockParams p) {
  let_next_kernel_start();
  wait_for_earlier_kernels();
  const int i = blockIdx.x % p.qb, bg = blockIdx.x / p.qb;
  const float share = 1.0f / static_cast<float>(min(64, p.a.T - i * 64) * p.rep);
  const float* part = p.part + (((int64_t)bg * p.tiles + i / 2) * p.rep * 2 + (i & 1)) * p.kbp;
  float* out = p.a.out + ((int64_t)bg * p.qb + i) * p.qb;
  for (int j = threadIdx.x; j < p.qb; j += 256) {
    float sum = 0.0f;
    if (j <= i)
      for (int h = 0; h < p.rep; ++h) sum += part[(int64_t)h * 2 * p.kbp + (j & 1) * (p.kbp / 2) + j / 2];
    out[j] = sum * share;
  }
}

static BlockParams block_params(int64_t B, int64_t Hq, int64_t Hkv, int64_t T) {
  BlockParams p{};
  p.rep = static_cast<int>(Hq / Hkv);
  p.tiles = static_cast<int>((T + 127) / 128);
  p.qb = static_cast<int>((T + 63) / 64);
  p.kbp = (p.qb + 63) / 64 * 64;
  p.pairs = (p.tiles * p.rep + 1) / 2;
  p.units = static_cast<int>(B * Hkv * p.pairs);
  return p;
}

int64_t block_mass_sm100_workspace_bytes(int64_t B, int64_t Hq, int64_t Hkv, int64_t T) {
  const BlockParams p = block_params(B, Hq, Hkv, T);
  return (std::min<int64_t>(p.units, kMaxSms) * 256 + B * Hkv * p.tiles * p.rep * 2) * p.kbp * 4;
}

// Map over [B, H, T, D]: boxes of 64 dims x 128 tokens of one head; out-of-range rows read zeros.
static bool row_map(CUtensorMap* m, const void* base, CUtensorMapDataType dt, int B, int H, int T, int D, const int64_t* s) {
  EncodeTiledFn fn = encode_fn();
  if (fn == nullptr) return false;
  const cuuint64_t dims[4] = {(cuuint64_t)D, (cuuint64_t)H, (cuuint64_t)T, (cuuint64_t)B};
  // A dimension of one element never steps: any valid stride will do.
  const cuuint64_t row = (cuuint64_t)D * 2;
  const cuuint64_t strides[3] = {H > 1 ? (cuuint64_t)s[1] * 2 : row, T > 1 ? (cuuint64_t)s[2] * 2 : row,
                                 B > 1 ? (cuuint64_t)s[0] * 2 : row};
  const cuuint32_t box[4] = {64, 1, 128, 1};
  const cuuint32_t estr[4] = {1, 1, 1, 1};
  return fn(m, dt, 4, const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
            CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <typename T, int D>
static cudaError_t launch_block(const BlockMassArgs& a, CUtensorMapDataType dt, cudaStream_t stream) {
  using L = BlockLayout<D>;
  CUtensorMap mq, mk;
  if (!row_map(&mq, a.q, dt, a.B, a.Hq, a.T, D, a.qs) || !row_map(&mk, a.k, dt, a.B, a.Hkv, a.T, D, a.ks))
    return cudaErrorInvalidValue;
  auto kern = block_mass_sm100_kernel<T, D>;
  static std::atomic<uint64_t> done{0};
  cudaError_t e = allow_smem(reinterpret_cast<const void*>(kern), L::BYTES, done);
  if (e != cudaSuccess) return e;
  BlockParams p = block_params(a.B, a.Hq, a.Hkv, a.T);
  p.a = a;
  const int G = std::min(p.units, sm_count());
  p.blocks = a.workspace;
  p.part = a.workspace + (int64_t)G * 256 * p.kbp;
  e = launch_early(kern, G, kBmThreads, L::BYTES, stream, mq, mk, p);
  return e != cudaSuccess ? e : launch_early(block_mass_join_kernel, a.B * a.Hkv * p.qb, 256, 0, stream, p);
}

cudaError_t launch_block_mass_sm100(const BlockMassArgs& a, int dtype, cudaStream_t stream) {
  if (dtype == SPRUCE_DTYPE_BF16)
    return a.D == 128 ? launch_block<__nv_bfloat16, 128>(a, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, stream)
                      : launch_block<__nv_bfloat16, 64>(a, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, stream);
  return a.D == 128 ? launch_block<__half, 128>(a, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, stream)
                    : launch_block<__half, 64>(a, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, stream);
}

}  // namespace spruce
