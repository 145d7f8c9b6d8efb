// Attention of chunks of new tokens over a paged K/V cache on the tcgen05 tensor cores (bf16 / fp16).
//
// The mathematics, the split of the work and its join are those of paged_common.cuh and paged_attn.cu.  A unit has R = 256
// query rows -- two M = 128 tiles of (token, head of the group) rows, so a group of 7 heads fills its tiles as well as one of
// 8 -- and its keys come in tiles of 128:
//   S_t = Q_t K^T   M128 N128 K16, D / 16 MMAs      O_t += P_t V   M128 N = D K16, 8 MMAs.
// A CTA per SM walks its run of key tiles, from unit to unit, with the loads running ahead across the units' border.
//
// Warps: 0-3 softmax and epilogue of tile 0 (thread = row = TMEM lane), 4-7 of tile 1, 8 issues the MMAs and owns TMEM,
// 9 loads K, 10 loads V, 11 only fills its warpgroup.  The softmax warps also bring in their own Q rows (once a unit).
// O_0 O_1 S_0 S_1 fill TMEM's columns; P_t is written over the first half of S_t.  One thread issues PV_0(j) QK_0(j+1)
// PV_1(j) QK_1(j+1) ..., in whose order they execute, so QK_t(j+1) overwrites P_t(j) after PV_t(j) has read it, and while
// one tile's softmax runs the tensor core works for the other.  P is announced in halves of 64 keys, so PV starts on the
// first while the second is exponentiated.  O is rescaled only when the running maximum grew by more than 8 (log2 units;
// fp16: 2), which O / l cancels.  P is rounded to the input type (the MMA's operand) and stays below 2^8 in bf16; in fp16 it
// carries 2^13 and stays below 2^15, so weights keep all their bits down to 2^-27 of the row's largest.  The sum l is of the
// unrounded fp32 values.
//
// Pages: one TMA box of a page's rows (or of 128 of them, or of its largest power-of-two divisor) lands as rows of the
// 128-byte-swizzled tile.  Boxes past the sequence's end take a page index past the cache, which reads zeros; the rows of
// the last page past the end may hold anything, so the loader clears them in V (their scores are masked by selection)
// before the MMA issuer may read the tile.
//
// Measured on a B200 (28 query / 4 KV heads, d = 128, bf16): 2048 tokens over 64K 1.62-1.65 ms in short runs from idle (1,150
// TFLOP/s), 1.80 ms in runs of a hundred under the power cap, 1.90 ms in longer ones (995 TFLOP/s); fp16 1.76 and 1.92 ms in the
// first two.  A 16K prompt in one chunk 1.65 ms, 512 tokens over 32K 224 us, 247 us in long runs.  A key tile of both M-tiles was
// traced at 3,210 cycles, the MMAs alone 2,880 (90 each, not the 64 of their rate: Q and K are both read from shared
// memory), a tile's softmax 1,900.  The registers go to the softmax (208 a thread by setmaxnreg: with 168 it ran a sixth
// slower; 200, 192 and 216 with what is left for the other warps 1-5% slower).
//
// Every wait is bounded (common.cuh).
#include <algorithm>
#include <type_traits>

#include "attn_common.cuh"
#include "paged_common.cuh"

namespace spruce {

// Starting and ending a unit takes about 16,000 cycles, five or six of the 3,200 a key tile takes (swept 2 - 8: a 16K
// prompt, whose first units have one tile, 2.01 / 1.82 / 1.66 / 1.59 / 1.58 ms at 2 / 3 / 4 / 5 / 6; nothing else moves).
constexpr int kChunkUnitCost = 6;
constexpr int kChunkThreads = 384;
constexpr int kChunkMma = 8;
constexpr int kChunkLoadK = 9;
constexpr int kChunkLoadV = 10;
constexpr int kChunkRows = kPagedChunkRows;
constexpr int kChunkKeys = kPagedChunkKeys;

constexpr int kChunkRoleBytes = 144;

template <int D>
struct ChunkLayout {
  static constexpr int KST = D == 128 ? 3 : 5, VST = D == 128 ? 2 : 5;  // tiles of K and of V in flight
  static constexpr int NP = D / 64;           // 128-byte panels along the head dim
  static constexpr int PANEL = 128 * 128;     // 128 rows x 128 B
  static constexpr int TILE = NP * PANEL;
  static constexpr int OFF_Q = 0;
  static constexpr int OFF_K = 2 * TILE;
  static constexpr int OFF_V = OFF_K + KST * TILE;
  static constexpr int OFF_BAR = OFF_V + VST * TILE;
  // q_full[2], k_full[], k_empty[], v_full[], v_empty[], v_tail, s_full[2], p_full[2][2], o_done[2], drain
  static constexpr int NBAR = 2 + 2 * (KST + VST) + 1 + 2 + 4 + 2 + 1;
  static constexpr int OFF_MISC = OFF_BAR + NBAR * 8;
  static constexpr int OFF_SCAN = (OFF_MISC + 16 + 15) / 16 * 16;
  static constexpr int OFF_ROLE = OFF_SCAN;   // a ChunkRole for each warp with a part, once the scan is done
  static constexpr int BYTES = 1024 + OFF_ROLE + 11 * kChunkRoleBytes;
  static_assert(BYTES + 16 <= 227 * 1024, "shared memory of a CTA");
  static constexpr int COL_S = 2 * D;         // S_t (and P_t) at COL_S + 128 t
};

// 32 lanes x 32 bit, 16 consecutive columns per thread.
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, float (&v)[16]) {
  uint32_t r[16];
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr));
#pragma unroll
  for (int i = 0; i < 16; ++i) v[i] = __uint_as_float(r[i]);
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const float (&v)[16]) {
  uint32_t r[16];
#pragma unroll
  for (int i = 0; i < 16; ++i) r[i] = __float_as_uint(v[i]);
  tmem_st16u(taddr, r);
}

// max(a, b, c), NaN where one of them is.
__device__ __forceinline__ float fmax3_nan(float a, float b, float c) {
  float d;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

// A warp's place in the CTA's run.  It lives in shared memory so that the softmax's inner loop, which wants every
// register, does not carry it.
struct ChunkRole {
  PagedWalk<kChunkRows, kChunkKeys> walk;
  PagedPiece x;
};
static_assert(sizeof(ChunkRole) <= kChunkRoleBytes, "fits its slot");
__device__ __forceinline__ bool next_piece(const PagedParams& p, ChunkRole* r) {
  PagedWalk<kChunkRows, kChunkKeys> w = r->walk;
  PagedPiece x;
  const bool more = w.next(p, x);
  __syncwarp();
  if ((threadIdx.x & 31) == 0) {
    r->walk = w;
    r->x = x;
  }
  __syncwarp();
  return more;
}

template <typename T, int D>
__global__ void __launch_bounds__(kChunkThreads, 1)
    paged_chunk_sm100_kernel(const __grid_constant__ CUtensorMap tmk, const __grid_constant__ CUtensorMap tmv,
                             const __grid_constant__ PagedParams p, int box) {
  using L = ChunkLayout<D>;
  constexpr int KST = L::KST, VST = L::VST;
  using Walk = PagedWalk<kChunkRows, kChunkKeys>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  uint32_t* const status = p.a.status;

  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + L::OFF_BAR);
  uint64_t* q_full = bars;                // [tile]: its Q rows are in shared memory (128 arrivals)
  uint64_t* k_full = q_full + 2;
  uint64_t* k_empty = k_full + KST;
  uint64_t* v_full = k_empty + KST;
  uint64_t* v_empty = v_full + VST;
  uint64_t* v_tail = v_empty + VST;       // the loader's own: a V tile whose tail it clears has landed
  uint64_t* s_full = v_tail + 1;          // [tile]: S_t(j) written
  uint64_t* p_full = s_full + 2;          // [tile * 2 + half]: that half of P_t(j) written (128 arrivals)
  uint64_t* o_done = p_full + 4;          // [tile]: the piece's last PV_t complete
  uint64_t* drain = o_done + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + L::OFF_MISC);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(smem + L::OFF_MISC + 4);
  int64_t* scan = reinterpret_cast<int64_t*>(smem + L::OFF_SCAN);

  if (warp == kChunkLoadK) {
    if (lane == 0) {
      *abort_flag = 0;
      for (int s = 0; s < 2 * KST; ++s) mbar_init(&k_full[s], 1);  // and k_empty
      for (int s = 0; s < 2 * VST; ++s) mbar_init(&v_full[s], 1);  // and v_empty
      for (int t = 0; t < 2; ++t) {
        mbar_init(&q_full[t], 128);
        mbar_init(&s_full[t], 1);
        mbar_init(&p_full[2 * t], 128);
        mbar_init(&p_full[2 * t + 1], 128);
        mbar_init(&o_done[t], 1);
      }
      mbar_init(v_tail, 1);
      mbar_init(drain, 1);
      fence_barrier_init();
      prefetch_tmap(&tmk);
      prefetch_tmap(&tmv);
    }
    __syncwarp();
  } else if (warp == kChunkMma) {
    tmem_alloc(tmem_slot, 512u);
    tmem_relinquish();
  }
  tc_fence_before();
  let_next_kernel_start();
  wait_for_earlier_kernels();
  Walk walk;
  const bool any = paged_run<kChunkRows, kChunkKeys, kChunkThreads>(p, walk, scan);
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  if (!any) walk.left = 0;
  ChunkRole* const role = reinterpret_cast<ChunkRole*>(smem + L::OFF_ROLE + min(warp, 10) * kChunkRoleBytes);
  if (lane == 0 && warp < 11) role->walk = walk;
  __syncwarp();
  const PagedPiece& x = role->x;

  // All warps of a warpgroup execute the same setmaxnreg, the idle one included, before their roles part.
  if (warp >= kChunkMma) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 88;");
    if (warp == kChunkLoadK || warp == kChunkLoadV) {
      // ------------------------------------------------------------ K or V
      const bool v = warp == kChunkLoadV;
      const CUtensorMap* const map = v ? &tmv : &tmk;
      uint8_t* const base = smem + (v ? L::OFF_V : L::OFF_K);
      uint64_t* const full = v ? v_full : k_full;
      uint64_t* const empty = v ? v_empty : k_empty;
      const int stages = v ? VST : KST;
      const int boxes = kChunkKeys / box;  // of a tile's rows: at most 8
      const bool leader = elect_one();
      int st = 0, loaded = 0;              // the next tile's stage; tiles loaded
      uint32_t turn = 1, tails = 0;        // parity of the stage's last release (none before the first round)
      bool ok = true;
      while (ok && next_piece(p, role)) {
        if (x.keys == 0) continue;
        const int keys = x.keys, t1 = x.t1, g = x.g;
        const int32_t* table = p.a.block_table + x.s * p.a.table_stride;
        // Lane b: page of box b of tile t; past the keys (or the table) a page index that reads zeros.
        auto page_of = [&](int t) {
          const int key = t * kChunkKeys + lane * box;
          if (lane >= boxes || t >= t1 || key >= keys) return static_cast<int>(p.a.num_pages);
          const int page = paged_page(p, table, key / p.a.page_size);
          return page < 0 ? static_cast<int>(p.a.num_pages) : page;
        };
        int page = page_of(x.t0);
        int row = (x.t0 * kChunkKeys) % p.a.page_size;       // of the next box in its page
        for (int t = x.t0; t < t1; ++t) {
          if (loaded >= stages && !(ok = __all_sync(0xffffffffu, mbar_wait(&empty[st], turn, status, abort_flag)))) break;
          uint8_t* dst = base + st * L::TILE;
          const int valid = keys - t * kChunkKeys;           // keys of this tile that exist
          const bool tail = v && valid < kChunkKeys && valid % box != 0;
          uint64_t* const bar = tail ? v_tail : &full[st];
          if (leader) mbar_arrive_expect_tx(bar, L::TILE);
          __syncwarp();
          for (int b = 0; b < boxes; ++b) {
            const int pb = __shfl_sync(0xffffffffu, page, b);
            if (leader) {
#pragma unroll
              for (int pp = 0; pp < L::NP; ++pp)
                tma_load_4d(dst + pp * L::PANEL + b * box * 128, map, bar, pp * 64, row, g, pb);
            }
            __syncwarp();
            row += box;
            if (row == p.a.page_size) row = 0;
          }
          page = page_of(t + 1);  // its latency passes behind the wait for the next stage
          if (tail) {
            ok = __all_sync(0xffffffffu, mbar_wait(v_tail, tails & 1, status, abort_flag));
            ++tails;
            // Rows past the end, to the end of their box (whole 16-byte chunks: any swizzle).
            const int end = min(kChunkKeys, (valid / box + 1) * box);
            for (int e = lane; e < (end - valid) * 8 * L::NP; e += 32) {
              const int panel = e / ((end - valid) * 8), c = e % ((end - valid) * 8);
              *reinterpret_cast<uint4*>(dst + panel * L::PANEL + (valid + c / 8) * 128 + c % 8 * 16) = make_uint4(0, 0, 0, 0);
            }
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(&full[st]);
          }
          ++loaded;
          if (++st == stages) {
            st = 0;
            turn ^= 1;
          }
          if (!ok) break;
        }
      }
      // No copy may be in flight when the CTA exits.
      for (int k = max(0, loaded - stages); k < loaded; ++k)
        mbar_wait(&full[k % stages], (k / stages) & 1, status, nullptr);
      __syncwarp();
    } else if (warp == kChunkMma) {
      // ------------------------------------------------------------ MMA issuer
      const bool leader = elect_one();
      constexpr uint32_t fmt = UmmaFormat<T>::value;
      constexpr uint32_t idesc_qk = idesc_f16(fmt, 0, 0, 128, 128);
      constexpr uint32_t idesc_pv = idesc_f16(fmt, 0, 1, D, 128);
      const uint64_t dq0 = smem_desc(smem_u32(smem + L::OFF_Q), 16, 1024);
      const uint64_t dk0 = smem_desc(smem_u32(smem + L::OFF_K), 16, 1024);
      const uint64_t dv0 = smem_desc(smem_u32(smem + L::OFF_V), L::PANEL, 1024);
      auto commit = [&](uint64_t* bar) {
        if (leader) umma_commit(bar);
        __syncwarp();
      };
      auto wait = [&](uint64_t* bar, uint32_t parity) {
        return __all_sync(0xffffffffu, mbar_wait(bar, parity, status, abort_flag));
      };
      // A descriptor's address is in its low word, which alone is stepped, where an MMA is issued (the asm statements below
      // see to that): all steps kept ahead of the loop spill at 88 registers, and 64-bit additions cost 2.8% of a long chunk.
      auto at_address = [](uint64_t d, uint32_t low) { return (d & 0xffffffff00000000ull) | low; };
      auto issue_qk = [&](int t, int st) {
        const uint32_t d = tmem + L::COL_S + 128 * t;
        uint32_t qa = static_cast<uint32_t>(dq0) + ((t * L::TILE) >> 4);
        uint32_t kb = static_cast<uint32_t>(dk0) + ((st * L::TILE) >> 4);
        asm volatile("" : "+r"(qa), "+r"(kb));
#pragma unroll
        for (int ks = 0; ks < D / 16; ++ks) {
          const uint32_t off = ((ks >> 2) * L::PANEL + (ks & 3) * 32) >> 4;
          if (leader) umma_f16_ss(d, at_address(dq0, qa + off), at_address(dk0, kb + off), idesc_qk, ks > 0 ? 1u : 0u);
          __syncwarp();
        }
        commit(&s_full[t]);
      };
      uint32_t pvs[2] = {0, 0};  // PVs issued for each tile
      auto pv_half = [&](int t, int st, int h, bool first) {
        if (!wait(&p_full[2 * t + h], pvs[t] & 1)) return false;
        tc_fence_after();
        const uint32_t a = tmem + L::COL_S + 128 * t;
        uint32_t vb = static_cast<uint32_t>(dv0) + ((st * L::TILE) >> 4);
        asm volatile("" : "+r"(vb));
#pragma unroll
        for (int kk = 0; kk < 4; ++kk) {
          const int ks = 4 * h + kk;
          if (leader)
            umma_f16_ts(tmem + t * D, a + ks * 8, at_address(dv0, vb + ((ks * 2048) >> 4)), idesc_pv,
                        (!first || ks > 0) ? 1u : 0u);
          __syncwarp();
        }
        if (h == 1) ++pvs[t];
        return true;
      };
      uint32_t pieces[2] = {0, 0};
      int kst = 0, vst = 0;            // stages of the next K and V tile, and the parities of their turns
      uint32_t kturn = 0, vturn = 0;
      bool ok = true;
      auto next_k = [&] {
        if (++kst == KST) {
          kst = 0;
          kturn ^= 1;
        }
      };
      while (ok && next_piece(p, role)) {
        const bool two = x.q.qlen * p.rep - x.qt * kChunkRows > 128;
        if (x.keys == 0) continue;
        const int n = x.t1 - x.t0;
        ok = wait(&q_full[0], pieces[0]++ & 1) && (!two || wait(&q_full[1], pieces[1]++ & 1)) &&
             wait(&k_full[kst], kturn);
        if (!ok) break;
        tc_fence_after();
        issue_qk(0, kst);
        if (two) issue_qk(1, kst);
        commit(&k_empty[kst]);
        next_k();
        for (int i = 0; i < n; ++i) {
          // A check of a barrier waits behind this warp's queued MMAs, so what PV_t(i) and QK_t(i+1) need is checked
          // before them and they are issued without a pause.
          const bool more = i + 1 < n;
          if (!(ok = wait(&v_full[vst], vturn) && (!more || wait(&k_full[kst], kturn)))) break;
          if (!(ok = pv_half(0, vst, 0, i == 0) && pv_half(0, vst, 1, i == 0))) break;
          if (more)
            issue_qk(0, kst);
          else
            commit(&o_done[0]);
          if (two) {
            if (!(ok = pv_half(1, vst, 0, i == 0) && pv_half(1, vst, 1, i == 0))) break;
            if (more)
              issue_qk(1, kst);
            else
              commit(&o_done[1]);
          }
          commit(&v_empty[vst]);  // every MMA reading these stages is issued before this
          if (++vst == VST) {
            vst = 0;
            vturn ^= 1;
          }
          if (more) {
            commit(&k_empty[kst]);
            next_k();
          }
        }
      }
      commit(drain);  // no MMA may be in flight when TMEM is released
      mbar_wait(drain, 0, status, nullptr);
      __syncwarp();
    }
  } else {
    // ------------------------------------------------------------ softmax + epilogue
    asm volatile("setmaxnreg.inc.sync.aligned.u32 208;");
    const int t = warp >> 2;
    const int row = (warp & 3) * 32 + lane;  // TMEM lane == tile row
    const uint32_t lane_off = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const uint32_t tO = tmem + lane_off + t * D;
    const uint32_t tS = tmem + lane_off + L::COL_S + 128 * t;
    const float sl2 = p.scale_log2;
    if (threadIdx.x == 0) p.desc[blockIdx.x] = make_int4(0, 0, 0, 0);
    uint32_t sj = 0, pieces = 0;  // tiles and pieces of this M-tile so far
    bool ok = true;
    while (ok && next_piece(p, role)) {
      if (x.parts > 0 && threadIdx.x == 0)
        p.desc[blockIdx.x] = paged_desc(x, min(kChunkRows, x.q.qlen * p.rep - x.qt * kChunkRows));
      const int rows = min(128, x.q.qlen * p.rep - x.qt * kChunkRows - t * 128);
      if (rows <= 0) continue;
      const int r0 = x.qt * kChunkRows + t * 128;  // the tile's first row in the sequence
      const int n = x.keys == 0 ? 0 : x.t1 - x.t0;
      const PagedRows row_at(p, x.q.q0, r0, x.g);
      if (n > 0) {
        // This warp's 32 rows of Q into the swizzled layout (rows past the end: zeros), all its loads in flight at once.
        constexpr int CH = D / 8;  // 16-byte chunks of a row
        uint8_t* qs = smem + L::OFF_Q + t * L::TILE;
        const int c = lane % CH;
        uint4 v[CH];
#pragma unroll
        for (int e = 0; e < CH; ++e) {
          const int r = (warp & 3) * 32 + e * (32 / CH) + lane / CH;
          v[e] = make_uint4(0, 0, 0, 0);
          if (r < rows) {
            v[e] = *reinterpret_cast<const uint4*>(static_cast<const T*>(p.a.q) + row_at.offset(r, p.a.qn, p.a.qh) + c * 8);
          }
        }
#pragma unroll
        for (int e = 0; e < CH; ++e) {
          const int r = (warp & 3) * 32 + e * (32 / CH) + lane / CH;
          *reinterpret_cast<uint4*>(qs + (c >> 3) * L::PANEL + r * 128 + (((c & 7) ^ (r & 7)) << 4)) = v[e];
        }
        fence_proxy_async_smem();
        mbar_arrive(&q_full[t]);
      }
      // Columns of the piece's first key tile that this row sees; each tile further leaves 128 fewer.
      int lim = min(x.q.first + row_at.token(row) + 1, x.keys) - x.t0 * kChunkKeys;
      // Growth of the maximum that O is not rescaled for, and the factor of P: together P's range.
      constexpr float kLag = std::is_same<T, __half>::value ? 2.0f : 8.0f;
      constexpr float kScale = PScale<T>::log2 > 0.0f ? PScale<T>::log2 - kLag : 0.0f;
      float m_used = -INFINITY;  // reference max (log2 units) the exponentials use
      float l = 0.0f;
      // One key tile.  Masked tiles are a unit's last ones; they have a body of their own because a branch within the
      // exponentials keeps the compiler from interleaving them (measured: 3680 -> 3110 cycles a step of both tiles).
      auto softmax_tile = [&](auto masked_c, bool first) {
        constexpr bool masked = decltype(masked_c)::value;
        float s[4][32];  // s[q][c] = column 32q + c
#pragma unroll
        for (int q = 0; q < 4; ++q) tmem_ld32(tS + 32 * q, s[q]);
        tmem_wait_ld();
        if constexpr (masked) {
#pragma unroll
          for (int q = 0; q < 4; ++q)
#pragma unroll
            for (int c = 0; c < 32; ++c)
              if (32 * q + c >= lim) s[q][c] = -INFINITY;
        }
        float mx8[8];
#pragma unroll
        for (int u = 0; u < 8; ++u) {
          float a = fmax3_nan(s[0][u], s[0][u + 8], s[0][u + 16]);
          a = fmax3_nan(a, s[0][u + 24], s[1][u]);
          a = fmax3_nan(a, s[1][u + 8], s[1][u + 16]);
          a = fmax3_nan(a, s[1][u + 24], s[2][u]);
          a = fmax3_nan(a, s[2][u + 8], s[2][u + 16]);
          a = fmax3_nan(a, s[2][u + 24], s[3][u]);
          a = fmax3_nan(a, s[3][u + 8], s[3][u + 16]);
          mx8[u] = fmax3_nan(a, s[3][u + 24], a);
        }
        const float mx = fmax3_nan(fmax3_nan(mx8[0], mx8[1], mx8[2]), fmax3_nan(mx8[3], mx8[4], mx8[5]), fmax3_nan(mx8[6], mx8[7], mx8[7]));
        const float top = mx * sl2;
        const float m_new = fmaxf(m_used, top);  // a NaN is not taken over
        const bool rescale = m_new > m_used + kLag;  // the first tile's too
        if (__any_sync(0xffffffffu, rescale)) {
          // PV_t(j-1) is complete and PV_t(j) waits for this tile's P.
          const float alpha = rescale ? fast_exp2(m_used - m_new) : 1.0f;
          if (rescale) m_used = m_new;
          l *= alpha;
          if (!first) {
#pragma unroll 1
            for (int cc = 0; cc < D; cc += 16) {
              float o[16];
              tmem_ld16(tO + cc, o);
              tmem_wait_ld();
#pragma unroll
              for (int e = 0; e < 16; ++e) o[e] *= alpha;
              tmem_st16(tO + cc, o);
            }
          }
        }
        // A tile with a score of NaN or +inf makes the row NaN whichever column holds it: the polynomial, whose clamp takes NaN
        // for a number, would lose it in the columns that it serves.
        const float lost = __int_as_float(0x7fffffff);
        const float neg_ref = top < INFINITY ? (m_used == -INFINITY ? 0.0f : kScale - m_used) : lost;
        uint64_t sum2[2] = {f2_pack(0.0f, 0.0f), f2_pack(0.0f, 0.0f)};
        const uint64_t sl2x2 = f2_pack(sl2, sl2), nref2 = f2_pack(neg_ref, neg_ref);
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          uint32_t pk[16];
#pragma unroll
          for (int k = 0; k < 16; ++k) {
            float x0, x1, e0, e1;
            f2_unpack(f2_fma(f2_pack(s[q][2 * k], s[q][2 * k + 1]), sl2x2, nref2), x0, x1);
            if (!masked && k == 15) {  // a sixteenth by polynomial, which does not give 0 for -inf
              poly_exp2_x2(x0, x1, e0, e1);
            } else {
              e0 = fast_exp2(x0);
              e1 = fast_exp2(x1);
            }
            sum2[k & 1] = f2_add(sum2[k & 1], f2_pack(e0, e1));
            pk[k] = Pack2<T>::pack(e0, e1);
          }
          tmem_st16u(tS + 16 * q, pk);
          if (q & 1) {  // those 64 keys of P are written
            tmem_wait_st();
            tc_fence_before();
            mbar_arrive(&p_full[2 * t + q / 2]);
          }
        }
        float part[4];
        f2_unpack(sum2[0], part[0], part[1]);
        f2_unpack(sum2[1], part[2], part[3]);
        l += (part[0] + part[1]) + (part[2] + part[3]);
      };
      for (int j = 0; j < n; ++j, ++sj, lim -= kChunkKeys) {
        ok = __all_sync(0xffffffffu, mbar_wait(&s_full[t], sj & 1, status, abort_flag));
        if (!ok) break;
        tc_fence_after();
        if (__any_sync(0xffffffffu, lim < kChunkKeys))
          softmax_tile(std::true_type{}, j == 0);
        else
          softmax_tile(std::false_type{}, j == 0);
      }
      if (!ok) break;
      if (n > 0) {
        ok = __all_sync(0xffffffffu, mbar_wait(&o_done[t], pieces & 1, status, abort_flag));
        ++pieces;
        if (!ok) break;
        tc_fence_after();
      }
      // The rows leave through this warp's rows of the Q tile, whose MMAs are complete: 128 bytes of each row a round,
      // written row by thread and read back row by eight lanes, so that a store covers whole lines.
      const bool whole = x.slot < 0;
      // No maximum: no key, or scores of -inf alone, of which the polynomial's columns made 2^-126.
      const float inv = l > 0.0f && m_used > -INFINITY ? 1.0f / l : 0.0f;
      uint8_t* dst = nullptr;  // this row in the output, or among the parts
      if (row < rows) {
        if (whole) {
          dst = reinterpret_cast<uint8_t*>(static_cast<T*>(p.a.out) +
                                           PagedRows(p, x.q.q0, r0, x.g).offset(row, p.a.on, p.a.oh));
        } else {
          const int64_t at = (int64_t)(2 * blockIdx.x + x.slot) * kChunkRows + t * 128 + row;
          p.part_ml[at] = make_float2(m_used, l);
          dst = reinterpret_cast<uint8_t*>(p.part_o + at * D);
        }
      }
      uint8_t* const stage = smem + L::OFF_Q + t * L::TILE + (warp & 3) * 32 * 128;
      float o[D];
      if (n > 0) {
#pragma unroll
        for (int cc = 0; cc < D / 32; ++cc) tmem_ld32(tO + cc * 32, *reinterpret_cast<float(*)[32]>(o + cc * 32));
        tmem_wait_ld();
      } else {  // no key seen: O was not written
#pragma unroll
        for (int d = 0; d < D; ++d) o[d] = 0.0f;
      }
      auto send = [&](int round, const uint4 (&v)[8]) {
#pragma unroll
        for (int e = 0; e < 8; ++e)
          *reinterpret_cast<uint4*>(stage + lane * 128 + ((e ^ (lane & 7)) << 4)) = v[e];
        __syncwarp();
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const int r = e * 4 + (lane >> 3);
          const uint4 y = *reinterpret_cast<const uint4*>(stage + r * 128 + (((lane & 7) ^ (r & 7)) << 4));
          uint8_t* const to = reinterpret_cast<uint8_t*>(
              __shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(dst), r));
          if (to != nullptr) *reinterpret_cast<uint4*>(to + round * 128 + (lane & 7) * 16) = y;
        }
        __syncwarp();
      };
      uint4 v[8];
      if (whole) {
#pragma unroll
        for (int round = 0; round < D / 64; ++round) {
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const float* f = o + round * 64 + e * 8;
            v[e] = make_uint4(Pack2<T>::pack(f[0] * inv, f[1] * inv), Pack2<T>::pack(f[2] * inv, f[3] * inv),
                              Pack2<T>::pack(f[4] * inv, f[5] * inv), Pack2<T>::pack(f[6] * inv, f[7] * inv));
          }
          send(round, v);
        }
      } else {
#pragma unroll
        for (int round = 0; round < D / 32; ++round) {
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            const float* f = o + round * 32 + e * 4;
            v[e] = make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
          }
          send(round, v);
        }
      }
      tc_fence_before();  // O and S are read before the next piece's MMAs, which wait for its Q
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == kChunkMma) {
    tc_fence_after();
    tmem_dealloc(tmem, 512u);
  }
}

// Tensor map of a cache [pages, Hkv, page_size, D]: boxes of 64 dims x `box` rows of one head's page.
static bool cache_map(CUtensorMap* m, const void* base, CUtensorMapDataType dt, const PagedArgs& a, const int64_t* s,
                      int box) {
  EncodeTiledFn fn = encode_fn();
  if (fn == nullptr) return false;
  const cuuint64_t dims[4] = {(cuuint64_t)a.D, (cuuint64_t)a.page_size, (cuuint64_t)a.Hkv, (cuuint64_t)a.num_pages};
  // A dimension of one element never steps: any valid stride will do.
  const cuuint64_t row = (cuuint64_t)a.D * 2;
  const cuuint64_t strides[3] = {(cuuint64_t)s[2] * 2, a.Hkv > 1 ? (cuuint64_t)s[1] * 2 : row,
                                 a.num_pages > 1 ? (cuuint64_t)s[0] * 2 : row};
  const cuuint32_t b[4] = {64, (cuuint32_t)box, 1, 1};
  const cuuint32_t estr[4] = {1, 1, 1, 1};
  return fn(m, dt, 4, const_cast<void*>(base), dims, strides, b, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
            CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// Rows of a TMA box: a page's, where they divide the tile; else the largest power of two that divides them.
int paged_box(int page_size, int tile) {
  int box = 16;
  while (box < tile && page_size % (2 * box) == 0) box *= 2;
  return box;
}

bool paged_cache_maps(const PagedArgs& a, int dtype, int box, CUtensorMap* mk, CUtensorMap* mv) {
  const CUtensorMapDataType dt =
      dtype == SPRUCE_DTYPE_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
  return cache_map(mk, a.kc, dt, a, a.ks, box) && cache_map(mv, a.vc, dt, a, a.vs, box);
}

template <typename T, int D>
static cudaError_t launch_chunk(const PagedArgs& a, int dtype, int G, cudaStream_t stream) {
  using L = ChunkLayout<D>;
  CUtensorMap mk, mv;
  const int box = paged_box(a.page_size, kChunkKeys);
  if (!paged_cache_maps(a, dtype, box, &mk, &mv)) return cudaErrorInvalidValue;
  auto kern = paged_chunk_sm100_kernel<T, D>;
  static std::atomic<uint64_t> done{0};
  cudaError_t e = allow_smem(reinterpret_cast<const void*>(kern), L::BYTES, done);
  if (e != cudaSuccess) return e;
  const PagedParams p = paged_params(a, kChunkRows, G, kChunkUnitCost);
  // An early start saves short calls two microseconds (512-token prompt 26.7 -> 23.8 us, 8 x 64 tokens over 1000 41.2 -> 38.3)
  // and costs calls whose CTAs take several units some (4K prompt 168 -> 180 us, 16K prompt 1.62 -> 1.65 ms).
  if ((int64_t)a.S * p.row_tiles * a.Hkv <= G) {
    e = launch_early(kern, G, kChunkThreads, L::BYTES, stream, mk, mv, p, box);
  } else {
    kern<<<G, kChunkThreads, L::BYTES, stream>>>(mk, mv, p, box);
    e = cudaGetLastError();
  }
  return e != cudaSuccess ? e : launch_paged_join<T>(p, kChunkRows, G, kChunkKeys, stream);
}

cudaError_t launch_paged_chunk(const PagedArgs& a, int dtype, int G, cudaStream_t stream) {
  if (dtype == SPRUCE_DTYPE_BF16)
    return a.D == 128 ? launch_chunk<__nv_bfloat16, 128>(a, dtype, G, stream)
                      : launch_chunk<__nv_bfloat16, 64>(a, dtype, G, stream);
  return a.D == 128 ? launch_chunk<__half, 128>(a, dtype, G, stream) : launch_chunk<__half, 64>(a, dtype, G, stream);
}

}  // namespace spruce
