// Softmax weight of cached keys under many query rows, on the tcgen05 tensor cores (bf16 / fp16).
//
// The formula is mass.cu's.  Scores are formed as S^T, keys by rows: M = 128 keys are the lanes of TMEM, so the sum over
// the rows runs along a thread's own columns and nothing crosses lanes:
//   S^T_t = K_t Q^T   M128 N128 K16, D / 16 MMAs     sum_j += sum_r 2^(S^T_jr c - lse_r).
// An item is 256 keys (two tiles) of a (sequence, KV head); the query rows that see them stream by in tiles of as many whole
// tokens as fit 128 rows, each a TMA box of (token, head of the group) rows.  Items go to the CTAs round robin; where a
// cluster of CTAs can be had for each, it shares the item's rows and its first CTA adds the sums up in their order.
//
// Warps: 0-3 the first 64 rows of tile 0 (thread = key = TMEM lane), 4-7 the others, 8-15 likewise of tile 1, 16 and 17
// issue the MMAs of a tile each (a check of a barrier waits behind the MMAs that its warp has queued: one warp's checks
// would leave the tensor core idle), 16 owns TMEM, 18 loads K (an item ahead) and Q, 19 works the items out and brings the
// rows' lse and limits.  Each S^T_t has two buffers.
//
// Bound by the softmax warps: 16 exponentials a clock and SM (2048 clocks a step of 256 keys x 128 rows) and their issue, which
// took 2460 of a step's 2960 clocks; the MMAs take 1100 and K comes from HBM behind them.  All exponentials are the hardware's: a
// polynomial on the FMA pipe, which takes NaN for a number, would need the steps with a NaN lse set apart, and was not built.
// Where a tile is filled up with zero rows (groups of 7 heads: 2 of 128), its last 32 go by their limits: 95 -> 97 us, so that a key
// at -inf gets 0.
// On a B200, 28 query / 4 KV heads of 128 in bf16: 64 tokens over 131072 97 to 105 us (570 to 620 TFLOP/s); a ragged fp16 batch of 9
// sequences of up to 3000 tokens and 300 new ones 16 us.
//
// Every wait is bounded (common.cuh).
#include <algorithm>
#include <type_traits>

#include "attn_common.cuh"
#include "mass_common.cuh"

namespace spruce {

constexpr int kKmThreads = 640, kKmMma = 16, kKmMma1 = 17, kKmLoad = 18, kKmLse = 19;
constexpr int kKmKeys = 256;

template <int D>
struct KeyMassLayout {
  static constexpr int QST = D == 128 ? 2 : 4, LST = 4;
  static constexpr int NP = D / 64;
  static constexpr int PANEL = 128 * 128;
  static constexpr int TILE = NP * PANEL;
  static constexpr int OFF_K = 0;                       // [2 items][2 tiles]
  static constexpr int OFF_Q = OFF_K + 4 * TILE;
  static constexpr int OFF_ROW = OFF_Q + QST * TILE;    // [LST]: 128 times -lse, 128 limits
  static constexpr int OFF_SUM = OFF_ROW + LST * 1024;  // [4][256] sums handed over
  static constexpr int OFF_ITEM = OFF_SUM + 4 * 1024;   // [4] what the softmax warps need of an item
  static constexpr int OFF_PART = OFF_ITEM + 4 * 64;   // [8 CTAs][256] sums of a cluster
  static constexpr int OFF_BAR = OFF_PART + 8 * 1024;
  // k_full[2], k_empty[2], q_full[], q_empty[], l_full[], l_empty[], s_full[4], s_empty[4], drain[2], i_full[4], i_empty[4],
  // g_full[2][4]
  static constexpr int NBAR = 4 + 2 * QST + 2 * LST + 8 + 2 + 8 + 8;
  static constexpr int OFF_MISC = OFF_BAR + NBAR * 8;
  static constexpr int BYTES = 1024 + OFF_MISC + 16;
  static_assert(BYTES <= 227 * 1024, "shared memory of a CTA");
};

// An item of a CTA: its keys, and its share of the rows that see them.
struct KeyMassItem {
  PagedSeq q;
  int s, g, key0, keys;  // keys: of the sequence, that its new tokens see
  int tok0, steps;  // first token of this CTA's rows, and its row tiles
};

// An item as the softmax warps take it; steps < 0 after the last.
struct KeyMassTask {
  int s, g, key0, keys, first, steps;
  int open0, open1;  // row tiles whose tokens are all the sequence's and see all the item's keys
  int left;          // query rows from this CTA's first on
};
static_assert(sizeof(KeyMassTask) <= 64, "fits its slot");

// Walks a CTA's items: those of its number, and every `stride` further.
struct KeyMassWalk {
  int s, rest, per, ds, dr;  // sequence, item in it, items of a sequence; the step
  __device__ __forceinline__ KeyMassWalk(const KeyMassParams& p, int first, int stride) {
    per = p.key_tiles * p.v.a.Hkv;
    s = first / per;
    rest = first - s * per;
    ds = stride / per;
    dr = stride - ds * per;
  }
  __device__ __forceinline__ bool more(const KeyMassParams& p) const { return s < p.v.a.S; }
  __device__ __forceinline__ void next() {
    s += ds;
    rest += dr;
    if (rest >= per) {
      rest -= per;
      ++s;
    }
  }
  // False where there is nothing to write.
  __device__ __forceinline__ bool item(const KeyMassParams& p, int ntok, int rank, int parts, KeyMassItem& x) const {
    x.s = s;
    const int tile = rest / p.v.a.Hkv;
    x.g = rest - tile * p.v.a.Hkv;
    x.key0 = tile * kKmKeys;
    x.q = paged_seq(p.v, s);
    x.keys = mass_keys(x.q);
    if (x.q.qlen == 0 || x.key0 >= x.keys) return false;
    // Tokens before the item's first key do not see it.
    const int lo = min(max(x.key0 - x.q.first, 0), x.q.qlen);
    const int tiles = (x.q.qlen - lo + ntok - 1) / ntok, each = (tiles + parts - 1) / parts;
    x.tok0 = lo + rank * each * ntok;
    x.steps = max(0, min(each, tiles - rank * each));
    return true;
  }
};

// All threads of the cluster's CTAs.
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

template <typename T, int D>
__global__ void __launch_bounds__(kKmThreads, 1)
    key_mass_sm100_kernel(const __grid_constant__ CUtensorMap tmq, const __grid_constant__ CUtensorMap tmk,
                          const __grid_constant__ KeyMassParams p, int box, int ntok, int parts) {
  using L = KeyMassLayout<D>;
  constexpr int QST = L::QST, LST = L::LST;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  uint32_t* const status = p.v.a.status;
  uint64_t* k_full = reinterpret_cast<uint64_t*>(smem + L::OFF_BAR);
  uint64_t* k_empty = k_full + 2;      // 2 arrivals: a tile's MMAs each
  uint64_t* q_full = k_empty + 2;
  uint64_t* q_empty = q_full + QST;    // likewise
  uint64_t* l_full = q_empty + QST;    // 32 arrivals
  uint64_t* l_empty = l_full + LST;    // 16: a lane of each softmax warp
  uint64_t* s_full = l_empty + LST;    // [tile * 2 + buffer]
  uint64_t* s_empty = s_full + 4;      // 256 arrivals
  uint64_t* drain = s_empty + 4;       // [tile]
  uint64_t* i_full = drain + 2;
  uint64_t* i_empty = i_full + 4;      // 16: a lane of each softmax warp
  uint64_t* g_full = i_empty + 4;      // [tile * 4 + item % 4], 128 arrivals: the second half's sums are there
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + L::OFF_MISC);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + L::OFF_MISC + 4);
  const int rank = blockIdx.x % parts;
  const int first = blockIdx.x / parts, stride = gridDim.x / parts;
  const int rows = ntok * p.v.rep;     // of a row tile that a box fills

  if (warp == kKmLoad) {
    if (lane == 0) {
      *abort_flag = 0;
      for (int i = 0; i < 2; ++i) {
        mbar_init(&k_full[i], 1);
        mbar_init(&k_empty[i], 2);
        mbar_init(&drain[i], 1);
      }
      for (int i = 0; i < QST; ++i) {
        mbar_init(&q_full[i], 1);
        mbar_init(&q_empty[i], 2);
      }
      for (int i = 0; i < LST; ++i) {
        mbar_init(&l_full[i], 32);
        mbar_init(&l_empty[i], 16);
      }
      for (int i = 0; i < 4; ++i) {
        mbar_init(&s_full[i], 1);
        mbar_init(&s_empty[i], 256);
        mbar_init(&i_full[i], 1);
        mbar_init(&i_empty[i], 16);
        mbar_init(&g_full[i], 128);
        mbar_init(&g_full[4 + i], 128);
      }
      fence_barrier_init();
      prefetch_tmap(&tmq);
      prefetch_tmap(&tmk);
    }
    __syncwarp();
  } else if (warp == kKmMma) {
    tmem_alloc(tmem_slot, 512u);
    tmem_relinquish();
  }
  // Rows of a stage that no box fills stay zero; what they multiply into is not summed.
  for (int e = threadIdx.x; e < QST * L::NP * (128 - rows) * 8; e += kKmThreads) {
    const int c = e % 8, r = rows + e / 8 % (128 - rows), panel = e / 8 / (128 - rows);
    *reinterpret_cast<uint4*>(smem + L::OFF_Q + panel * L::PANEL + r * 128 + c * 16) = make_uint4(0, 0, 0, 0);
  }
  fence_proxy_async_smem();
  tc_fence_before();
  let_next_kernel_start();
  wait_for_earlier_kernels();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  if (parts > 1) cluster_sync();       // the others' shared memory is there
  KeyMassItem x;
  float* to = nullptr;                 // where a sum that the cluster shares goes
  float old_part = 0.0f;

  if (warp == kKmLoad) {
    // ------------------------------------------------------------ K and Q
    const bool leader = elect_one();
    const int boxes = kKmKeys / box;  // at most 16
    int kn = 0, st = 0, qn = 0;
    bool ok = true;
    KeyMassItem y;
    // The keys of the next item that has some; called an item ahead of its rows, so that they are there in time.
    auto load_keys = [&](KeyMassWalk& w) {
      for (; w.more(p); w.next()) {
        if (!w.item(p, ntok, rank, parts, y) || y.steps == 0) continue;
        const int key = y.key0 + lane * box;
        int page = static_cast<int>(p.v.a.num_pages);  // reads zeros
        if (lane < boxes && key < y.keys) {
          page = paged_page(p.v, p.v.a.block_table + y.s * p.v.a.table_stride, key / p.v.a.page_size);
          if (page < 0) page = static_cast<int>(p.v.a.num_pages);
        }
        const int kb = kn & 1;
        if (kn >= 2 && !(ok = __all_sync(0xffffffffu, mbar_wait(&k_empty[kb], ((kn >> 1) - 1) & 1, status, abort_flag)))) return;
        if (leader) mbar_arrive_expect_tx(&k_full[kb], 2 * L::TILE);
        __syncwarp();
        int row = y.key0 % p.v.a.page_size;  // of the next box in its page
        for (int b = 0; b < boxes; ++b) {
          const int pb = __shfl_sync(0xffffffffu, page, b);
          const int r = b * box;  // of the item's keys
          if (leader)
#pragma unroll
            for (int pp = 0; pp < L::NP; ++pp)
              tma_load_4d(smem + L::OFF_K + (2 * kb + (r >> 7)) * L::TILE + pp * L::PANEL + (r & 127) * 128, &tmk, &k_full[kb],
                          pp * 64, row, y.g, pb);
          __syncwarp();
          row += box;
          if (row == p.v.a.page_size) row = 0;
        }
        ++kn;
        w.next();
        return;
      }
    };
    KeyMassWalk ahead(p, first, stride);
    load_keys(ahead);
    for (KeyMassWalk at(p, first, stride); ok && at.more(p); at.next()) {
      if (!at.item(p, ntok, rank, parts, x) || x.steps == 0) continue;
      for (int i = 0; ok && i < x.steps; ++i) {
        if (qn >= QST && !(ok = __all_sync(0xffffffffu, mbar_wait(&q_empty[st], ((qn / QST) - 1) & 1, status, abort_flag)))) break;
        if (leader) {
          mbar_arrive_expect_tx(&q_full[st], L::NP * rows * 128);
#pragma unroll
          for (int pp = 0; pp < L::NP; ++pp)
            tma_load_4d(smem + L::OFF_Q + st * L::TILE + pp * L::PANEL, &tmq, &q_full[st], pp * 64, x.g * p.v.rep,
                        x.q.q0 + x.tok0 + i * ntok, 0);
        }
        __syncwarp();
        ++qn;
        if (++st == QST) st = 0;
        // The next item's keys, whose place the last item leaves: after the rows that this item starts with, or the tensor core
        // would wait for those at every item.
        if (i == min(QST, x.steps) - 1) load_keys(ahead);
      }
    }
    // No copy may be in flight when the CTA exits.
    for (int i = max(0, kn - 2); i < kn; ++i) mbar_wait(&k_full[i & 1], (i >> 1) & 1, status, nullptr);
    for (int i = max(0, qn - QST); i < qn; ++i) mbar_wait(&q_full[i % QST], (i / QST) & 1, status, nullptr);
    __syncwarp();
  } else if (warp == kKmLse) {
    // ------------------------------------------------------------ lse and limits of the rows
    int ln = 0, in = 0;
    bool ok = true;
    auto tell = [&](const KeyMassTask& y) {
      if (in >= 4 && !(ok = __all_sync(0xffffffffu, mbar_wait(&i_empty[in & 3], ((in >> 2) - 1) & 1, status, abort_flag)))) return;
      if (lane == 0) {
        *reinterpret_cast<KeyMassTask*>(smem + L::OFF_ITEM + (in & 3) * 64) = y;
        mbar_arrive(&i_full[in & 3]);
      }
      __syncwarp();
      ++in;
    };
    KeyMassTask y{};
    for (KeyMassWalk at(p, first, stride); ok && at.more(p); at.next()) {
      if (!at.item(p, ntok, rank, parts, x)) continue;
      y.s = x.s;
      y.g = x.g;
      y.key0 = x.key0;
      y.keys = x.keys;
      y.first = x.q.first;
      y.steps = x.steps;
      y.open0 = (max(0, x.key0 + kKmKeys - 1 - x.q.first - x.tok0) + ntok - 1) / ntok;
      y.open1 = (x.q.qlen - x.tok0) / ntok;
      y.left = (x.q.qlen - x.tok0) * p.v.rep;
      tell(y);
      for (int i = 0; ok && i < x.steps; ++i, ++ln) {
        const int st = ln % LST, tok = x.tok0 + i * ntok;
        float v[4];
        int lim[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const int r = lane + 32 * k;
          const int t = static_cast<int>((static_cast<float>(r) + 0.5f) * p.v.inv_rep), h = r - t * p.v.rep;
          v[k] = INFINITY;
          lim[k] = -1;
          if (r < rows && tok + t < x.q.qlen) {
            v[k] = mass_row_lse(p.lse[(int64_t)(x.q.q0 + tok + t) * p.ln + (int64_t)(x.g * p.v.rep + h) * p.lh]);
            lim[k] = x.q.first + tok + t - x.key0;
          }
        }
        if (ln >= LST && !(ok = __all_sync(0xffffffffu, mbar_wait(&l_empty[st], ((ln / LST) - 1) & 1, status, abort_flag)))) break;
        float* dst = reinterpret_cast<float*>(smem + L::OFF_ROW + st * 1024);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          dst[lane + 32 * k] = -v[k];
          reinterpret_cast<int*>(dst)[128 + lane + 32 * k] = lim[k];
        }
        mbar_arrive(&l_full[st]);
      }
    }
    y.steps = -1;
    if (ok) tell(y);
  } else if (warp == kKmMma || warp == kKmMma1) {
    // ------------------------------------------------------------ MMA issuers, one a tile
    const bool leader = elect_one();
    const int t = warp - kKmMma;
    constexpr uint32_t idesc = idesc_f16(UmmaFormat<T>::value, 0, 0, 128, 128);
    const uint64_t dq0 = smem_desc(smem_u32(smem + L::OFF_Q), 16, 1024);
    const uint64_t dk0 = smem_desc(smem_u32(smem + L::OFF_K + t * L::TILE), 16, 1024);
    auto commit = [&](uint64_t* bar) {
      if (leader) umma_commit(bar);
      __syncwarp();
    };
    auto wait = [&](uint64_t* bar, uint32_t parity) {
      return __all_sync(0xffffffffu, mbar_wait(bar, parity, status, abort_flag));
    };
    int kn = 0, qn = 0;
    bool ok = true;
    for (KeyMassWalk at(p, first, stride); ok && at.more(p); at.next()) {
      if (!at.item(p, ntok, rank, parts, x) || x.steps == 0) continue;
      if (!(ok = wait(&k_full[kn & 1], (kn >> 1) & 1))) break;
      for (int i = 0; i < x.steps; ++i, ++qn) {
        const int st = qn % QST;
        const uint32_t buf = qn & 1;
        ok = wait(&q_full[st], (qn / QST) & 1) && (qn < 2 || wait(&s_empty[2 * t + buf], ((qn >> 1) - 1) & 1));
        if (!ok) break;
        tc_fence_after();
#pragma unroll
        for (int ks = 0; ks < D / 16; ++ks) {
          const uint32_t off = ((ks >> 2) * L::PANEL + (ks & 3) * 32) >> 4;
          if (leader)
            umma_f16_ss(tmem + (2 * t + buf) * 128, dk0 + ((2 * (kn & 1) * L::TILE) >> 4) + off,
                        dq0 + ((st * L::TILE) >> 4) + off, idesc, ks > 0 ? 1u : 0u);
          __syncwarp();
        }
        commit(&s_full[2 * t + buf]);
        commit(&q_empty[st]);
      }
      if (ok) commit(&k_empty[kn & 1]);
      ++kn;
    }
    commit(&drain[t]);  // no MMA may be in flight when TMEM is released
    mbar_wait(&drain[t], 0, status, nullptr);
    __syncwarp();
  } else {
    // ------------------------------------------------------------ weights and sums
    const int t = warp >> 3, half = (warp >> 2) & 1;  // tile, and which 64 of the rows
    const uint32_t tS = tmem + (static_cast<uint32_t>((warp & 3) * 32) << 16) + t * 256 + half * 64;
    const int key = t * 128 + (warp & 3) * 32 + lane;  // of the item
    float* const given = reinterpret_cast<float*>(smem + L::OFF_SUM);
    const float sl2 = p.v.scale_log2;
    const uint64_t sl2x2 = f2_pack(sl2, sl2);
    int qn = 0;
    bool ok = true;
    for (int done = 0; ok; ++done) {
      ok = __all_sync(0xffffffffu, mbar_wait(&i_full[done & 3], (done >> 2) & 1, status, abort_flag));
      if (!ok) break;
      const KeyMassTask* const y = reinterpret_cast<const KeyMassTask*>(smem + L::OFF_ITEM + (done & 3) * 64);
      const int steps = y->steps;
      if (steps < 0) break;
      const int open0 = y->open0, open1 = y->open1, left = y->left - half * 64;
      // Where the sum goes, and the old weight, fetched while the rows stream by: the page first, what hangs on it a step later.
      float* dst = nullptr;
      float old = 0.0f;
      const int pos = y->key0 + key;
      const bool writes = half == 0 && rank == 0 && pos < y->keys;
      const int pi = pos / p.v.a.page_size;
      int page = -1;
      if (writes) page = p.v.a.block_table[y->s * p.v.a.table_stride + pi];
      auto place = [&] {
        if (!writes) return;
        if (page < 0 || page >= p.v.a.num_pages) {
          raise_status(status, SPRUCE_STATUS_BAD_PAGE);
          return;
        }
        const int slot = pos - pi * p.v.a.page_size;
        dst = p.out + page * p.os[0] + y->g * p.os[1] + slot * p.os[2];
        if (pos < y->first && p.decay != 0.0f) old = p.mass[page * p.ms[0] + y->g * p.ms[1] + slot * p.ms[2]];
      };
      uint64_t sum2[2] = {f2_pack(0.0f, 0.0f), f2_pack(0.0f, 0.0f)};
      // Sixteen rows; those of the other tiles have limits.
      auto rows_of = [&](const float* s, const float* lse, auto masked_c) {
        constexpr bool masked = decltype(masked_c)::value;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const float4 v = *reinterpret_cast<const float4*>(lse + 4 * k);
          float x0, x1, x2, x3;
          f2_unpack(f2_fma(f2_pack(s[4 * k], s[4 * k + 1]), sl2x2, f2_pack(v.x, v.y)), x0, x1);
          f2_unpack(f2_fma(f2_pack(s[4 * k + 2], s[4 * k + 3]), sl2x2, f2_pack(v.z, v.w)), x2, x3);
          float e0 = fast_exp2(x0), e1 = fast_exp2(x1), e2 = fast_exp2(x2), e3 = fast_exp2(x3);
          if constexpr (masked) {
            const int4 lim = *reinterpret_cast<const int4*>(lse + 128 + 4 * k);
            e0 = key <= lim.x ? e0 : 0.0f;
            e1 = key <= lim.y ? e1 : 0.0f;
            e2 = key <= lim.z ? e2 : 0.0f;
            e3 = key <= lim.w ? e3 : 0.0f;
          }
          sum2[0] = f2_add(sum2[0], f2_pack(e0, e1));
          sum2[1] = f2_add(sum2[1], f2_pack(e2, e3));
        }
      };
      for (int i = 0; ok && i < steps; ++i, ++qn) {
        const uint32_t buf = qn & 1;
        ok = __all_sync(0xffffffffu, mbar_wait(&l_full[qn % LST], (qn / LST) & 1, status, abort_flag) &&
                                         mbar_wait(&s_full[2 * t + buf], (qn >> 1) & 1, status, abort_flag));
        if (!ok) break;
        tc_fence_after();
        const float* lse = reinterpret_cast<const float*>(smem + L::OFF_ROW + (qn % LST) * 1024) + half * 64;
        const int there = min(left - i * rows, rows - half * 64);  // rows of this half
        const bool open = i >= open0 && i < open1;
#pragma unroll
        for (int r = 0; r < 64; r += 32) {  // 64 scores at once would not fit the registers of five warps a scheduler
          float s[32];
          tmem_ld32(tS + buf * 128 + r, s);
          tmem_wait_ld();
          if (r == 32) {
            tc_fence_before();
            mbar_arrive(&s_empty[2 * t + buf]);
          }
          // Zero rows that fill a tile up are kept out by their limits: times an infinite key they are not numbers.
          if (open && r + 32 <= there) {
            rows_of(s, lse + r, std::false_type{});
            rows_of(s + 16, lse + r + 16, std::false_type{});
          } else {
            if (r < there) rows_of(s, lse + r, std::true_type{});
            if (r + 16 < there) rows_of(s + 16, lse + r + 16, std::true_type{});
          }
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&l_empty[qn % LST]);
        if (i == 0) place();
      }
      if (steps == 0) place();
      float a0, a1, a2, a3;
      f2_unpack(sum2[0], a0, a1);
      f2_unpack(sum2[1], a2, a3);
      float sum = (a0 + a1) + (a2 + a3);
      // The second half hands its sum over and goes on; its place is free again when all are done with the item.
      float* const mine = given + (done & 3) * 256;
      if (half == 1) {
        mine[key] = sum;
        mbar_arrive(&g_full[t * 4 + (done & 3)]);
      } else {
        ok = __all_sync(0xffffffffu, mbar_wait(&g_full[t * 4 + (done & 3)], (done >> 2) & 1, status, abort_flag)) && ok;
        sum += mine[key];
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&i_empty[done & 3]);
      old *= p.decay;
      if (parts == 1) {
        if (dst != nullptr) *dst = sum + old;
      } else if (half == 0) {  // the only item: to the cluster's first CTA
        uint32_t there;
        asm("mapa.shared::cluster.u32 %0, %1, %2;"
            : "=r"(there)
            : "r"(smem_u32(smem + L::OFF_PART) + static_cast<uint32_t>(rank * 256 + key) * 4), "r"(0));
        asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(there), "f"(sum) : "memory");
        to = dst;
        old_part = old;
      }
    }
  }

  if (parts > 1) {
    cluster_sync();
    if (to != nullptr) {  // half 0 of the first CTA
      const float* const part = reinterpret_cast<const float*>(smem + L::OFF_PART) + (warp >> 3) * 128 + (warp & 3) * 32 + lane;
      float sum = 0.0f;
      for (int c = 0; c < parts; ++c) sum += part[c * 256];
      *to = sum + old_part;
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == kKmMma) {
    tc_fence_after();
    tmem_dealloc(tmem, 512u);
  }
}

// q as [N][Hq][D]: boxes of 64 dims x the heads of a group x `ntok` tokens, whose rows are those of a row tile in order.
static bool rows_map(CUtensorMap* m, const KeyMassArgs& x, CUtensorMapDataType dt, int ntok) {
  EncodeTiledFn fn = encode_fn();
  if (fn == nullptr) return false;
  const PagedArgs& a = x.a;
  const cuuint64_t dims[4] = {(cuuint64_t)a.D, (cuuint64_t)a.Hq, (cuuint64_t)a.N, 1};
  // A dimension of one element never steps: any valid stride will do.
  const cuuint64_t row = (cuuint64_t)a.D * 2;
  const cuuint64_t strides[3] = {a.Hq > 1 ? (cuuint64_t)a.qh * 2 : row, a.N > 1 ? (cuuint64_t)a.qn * 2 : row, row};
  const cuuint32_t b[4] = {64, (cuuint32_t)(a.Hq / a.Hkv), (cuuint32_t)ntok, 1};
  const cuuint32_t estr[4] = {1, 1, 1, 1};
  return fn(m, dt, 4, const_cast<void*>(a.q), dims, strides, b, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
            CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <typename T, int D>
static cudaError_t launch_rows(const KeyMassArgs& a, int dtype, cudaStream_t stream) {
  using L = KeyMassLayout<D>;
  const int ntok = 128 / (a.a.Hq / a.a.Hkv), box = paged_box(a.a.page_size, 128);
  CUtensorMap mq, mk, mv;
  if (!rows_map(&mq, a, dtype == SPRUCE_DTYPE_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, ntok) ||
      !paged_cache_maps(a.a, dtype, box, &mk, &mv))
    return cudaErrorInvalidValue;
  auto kern = key_mass_sm100_kernel<T, D>;
  static std::atomic<uint64_t> done{0};
  cudaError_t e = allow_smem(reinterpret_cast<const void*>(kern), L::BYTES, done);
  if (e != cudaSuccess) return e;
  const KeyMassParams p = key_mass_params(a, kKmKeys);
  const int64_t items = (int64_t)a.a.S * p.key_tiles * a.a.Hkv;
  if ((int64_t)p.key_tiles * a.a.Hkv > (1 << 30)) return cudaErrorInvalidValue;
  const int sms = sm_count();
  // CTAs of an item: as many as leave one item each, and a row tile each of the longest sequence allowed.
  int parts = 1;
  while (parts < 8 && items * parts * 2 <= sms && 2 * parts * ntok <= a.a.max_q) parts *= 2;
  cudaLaunchConfig_t cfg{};
  cudaLaunchAttribute attr[2]{};
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = parts;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.gridDim = dim3(static_cast<unsigned>(parts * std::min<int64_t>(items, sms / parts)));
  cfg.blockDim = dim3(kKmThreads);
  cfg.dynamicSmemBytes = L::BYTES;
  cfg.stream = stream;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  return cudaLaunchKernelEx(&cfg, kern, mq, mk, p, box, ntok, parts);
}

cudaError_t launch_key_mass_sm100(const KeyMassArgs& a, int dtype, cudaStream_t stream) {
  if (dtype == SPRUCE_DTYPE_BF16)
    return a.a.D == 128 ? launch_rows<__nv_bfloat16, 128>(a, dtype, stream) : launch_rows<__nv_bfloat16, 64>(a, dtype, stream);
  return a.a.D == 128 ? launch_rows<__half, 128>(a, dtype, stream) : launch_rows<__half, 64>(a, dtype, stream);
}

}  // namespace spruce
