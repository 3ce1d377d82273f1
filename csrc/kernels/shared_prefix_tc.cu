// Attention of many rows over shared tokens: the queries of all sequences of a group for one KV head, 256 rows a CTA, on the 5th-generation tensor cores.
//
// A CTA goes through its run of units (128 tokens each; see shared_prefix.cuh) with two tiles of 128 rows, A and B, that share every tile of keys and values.  TMEM holds
// S_A, S_B (128 fp32 columns each) and the accumulators O_A, O_B (a head's columns each).  For unit j one thread issues
//     PV(j, A)  O_A += P_A V_j   (P from TMEM, V_j row by row from shared memory),   QK(j + 1, A)  S_A = Q_A K_j+1^T,   PV(j, B),   QK(j + 1, B),
// so that the tensor cores work for one tile while the other tile's softmax runs, one row per thread.  Where all rows fit one tile, A takes the run's even units and B the
// odd ones with the same queries, and a part has two sums.  A row keeps its maximum until a new one is more than 2^8 larger, O
// stays in TMEM meanwhile.  Pages come by TMA, a copy per page and 64 columns, into rings of stages that go on from one part of the run to the next; the next part's
// queries are loaded as soon as the last product that reads the old ones is done.  A part's sums leave as they are, fp32 with the row's maximum and
// sum, for the join (shared_prefix.cu).
//
// Tokens behind a group's shared ones lie in the same pages, or in none: the last unit's scores are masked, and the rows of its V tile behind the last
// token are set to zero, since a weight of zero times what they hold need not be zero.
//
// The sequences' own tokens are read in the same launch by CTAs of their own, three runs of four warps each (shared_prefix_split.cuh): one part of the GPU is bound by products and
// exponentials while the other waits for memory.  From a captured graph, one after the other they took 145 us, beside one another 133, 122 to 124 with all later steps, as calls among
// others, where the clock is lower, 137 (256 sequences with 4 rows each for 8 KV heads of 128, 16384 shared and 16 to 512 own
// tokens); 73.5, 71.7 and 72 for 12 groups of 8; 54.6, 50.8 and 49 for one document of 32771 tokens and 16 sequences.  Every CTA finds from the lengths how many CTAs each kind gets.
//
// Bound by the softmax's exponentials and the products where there are 256 rows, by the keys' and values' bytes where there are few.
#define RB_INLINE_WAITS                 // registers are reallocated between warp groups
#include <string.h>

#include <type_traits>

#include "shared_prefix_split.cuh"

namespace rb {

constexpr int kStThreads = 384;          // warps 0-7 softmax, 8, 10 and 11 TMA, 9 MMA
constexpr int kStTile = 128;
constexpr float kStRescale = 8.f;        // log2 units
// Sequences whose totals, tokens and spans fit beside 192 KB of tiles.  One more and a batch has tiles of 32 rows on mma.sync: one group over 4000 shared and 100 own tokens, 32 heads
// (8 KV) of 128, 704 sequences 137 us, 705 478.
constexpr int kStMostBatch = 704;
constexpr int kStRuns = 3;               // of a CTA that has sequences' own tokens
// What a unit of 128 tokens takes a CTA, relative to one another: with two tiles of rows, with one, and of a sequence's own.  When they were set the first case above took 133 us
// with 5 : 3 : 2, 146 with 6 : 3 : 2 and 143 with 4 : 3 : 2; the second 71.7, or 73.7 with 5 : 2 : 2 and 79 with 5 : 4 : 2.  Both are bf16, 8 KV heads of 128 and pages of 16: other
// shapes get the same shares, unmeasured.
constexpr int kStTwo = 5, kStOne = 3, kStOwn = 2;

__device__ __forceinline__ void st_ld32(uint32_t taddr, uint32_t* r) { tmem_ld_32x32(taddr, *reinterpret_cast<uint32_t(*)[32]>(r)); }
__device__ __forceinline__ void st_st32(uint32_t taddr, const uint32_t* r) {
  tmem_st_32x16(taddr, *reinterpret_cast<const uint32_t(*)[16]>(r));
  tmem_st_32x16(taddr + 16, *reinterpret_cast<const uint32_t(*)[16]>(r + 16));
}

__device__ __forceinline__ float st_max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

template <int D>
struct StSmem {
  static constexpr int kStages = D == 64 ? 4 : 2;                // of K, and of V
  static constexpr int kHalf = kStTile * 128;                    // one 64-column swizzle atom: 128 rows x 128 B
  static constexpr int kTileBytes = (D / 64) * kHalf;
  static constexpr int kQ = 0;                                   // two tiles
  static constexpr int kK = kQ + 2 * kTileBytes;
  static constexpr int kV = kK + kStages * kTileBytes;
  static constexpr int kStage = kV + kStages * kTileBytes;       // 2 KB for each softmax warp: 16 columns of its rows' sums
  static constexpr int kBar = kStage + 8 * 2048;
  static constexpr int kNumBars = 3 + 4 * kStages + 8;           // q, q free, tail; full and empty per K and V stage; s_full[2], o_ready[2], p_full[2][2]
  static constexpr int kInts = kBar + kNumBars * 8;              // TMEM address, abort flag
  static constexpr int kTotal = (kInts + 8 + 15) / 16 * 16;      // then what is held of the lists
};

struct StMaps {
  CUtensorMap q, k, v, own_k, own_v;
};

template <typename T, int D>
__global__ void __launch_bounds__(kStThreads, 1)
shared_tc_kernel(const __grid_constant__ StMaps maps, const SpParams p, unsigned int* status RB_BOUNDS_PARAM) {
  using L = StSmem<D>;
  constexpr int kStages = L::kStages;
  extern __shared__ __align__(1024) uint8_t st_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(st_raw) + 1023) & ~uintptr_t(1023));
  __shared__ int warp_sums[kStThreads / 32];
  __shared__ unsigned long long work;
  __shared__ uint64_t own_bars[2 * kStThreads / 32];
  const uint32_t sbase = smem_u32(smem), sQ = sbase + L::kQ, sK = sbase + L::kK, sV = sbase + L::kV;
  const uint32_t b0 = sbase + L::kBar;
  const uint32_t bar_q = b0, bar_qfree = b0 + 8, bar_tail = b0 + 16;
  const uint32_t bar_kfull = b0 + 24, bar_kempty = bar_kfull + 8 * kStages, bar_vfull = bar_kempty + 8 * kStages, bar_vempty = bar_vfull + 8 * kStages;
  const uint32_t bar_sfull = bar_vempty + 8 * kStages, bar_oready = bar_sfull + 16, bar_pfull = bar_oready + 16;
  uint32_t* tmem_ptr = reinterpret_cast<uint32_t*>(smem + L::kInts);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_ptr + 1);
  const SpList& list = p.prefix;
  int* const own_totals = reinterpret_cast<int*>(smem + L::kTotal);
  int* const totals = own_totals + p.batch + 1;
  const SpHeld own = {own_totals, totals + p.batch + 1, totals + 2 * p.batch + 1, reinterpret_cast<uint32_t*>(totals + 3 * p.batch + 1), totals + 4 * p.batch + 1};
  const SpHeld held = {totals, nullptr, own.shared, own.span, nullptr};
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  constexpr uint32_t kTmemCols = 512;

  if (threadIdx.x == 0) {
    mbar_init(bar_q, 1);
    mbar_init(bar_qfree, 1);
    mbar_init(bar_tail, 1);
    for (int s = 0; s < kStages; ++s) {
      mbar_init(bar_kfull + 8 * s, 1);
      mbar_init(bar_kempty + 8 * s, 1);
      mbar_init(bar_vfull + 8 * s, 1);
      mbar_init(bar_vempty + 8 * s, 1);
    }
    for (int t = 0; t < 2; ++t) {
      mbar_init(bar_sfull + 8 * t, 1);
      mbar_init(bar_pfull + 16 * t, 4);
      mbar_init(bar_pfull + 16 * t + 8, 4);
      mbar_init(bar_oready + 8 * t, 1);
    }
    for (int i = 0; i < 2 * kStThreads / 32; ++i) mbar_init(smem_u32(own_bars + i), 1);
    *abort_flag = 0;
    fence_mbar_init();
    tma_prefetch_desc(&maps.q);
    tma_prefetch_desc(&maps.k);
    tma_prefetch_desc(&maps.v);
    tma_prefetch_desc(&maps.own_k);
    tma_prefetch_desc(&maps.own_v);
  }
  if (warp == 9) {
    tmem_alloc(smem_u32(tmem_ptr), kTmemCols);
    tmem_relinquish();
  }
  pdl_wait();
  pdl_launch();
  sp_prepare(p, own, warp_sums, totals, &work, kStOne, kStTwo);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_ptr;
  const int total = held.totals[list.entries] * list.virtual_heads;
  // ---- the last CTAs, as many as their units' share of the work, have the sequences' own tokens
  const int ctas = gridDim.x;
  const unsigned long long w_own = static_cast<unsigned long long>(own_totals[p.batch]) * p.list.virtual_heads * kStOwn, w_all = w_own + work * list.virtual_heads;
  int n_own = w_all == 0 ? 0 : static_cast<int>((ctas * w_own + w_all / 2) / w_all);
  if (w_own > 0 && n_own == 0) n_own = 1;
  if (w_own < w_all && n_own == ctas) n_own = ctas - 1;
  const int n_shared = ctas - n_own;
  if (blockIdx.x == 0) {
    sp_keep_totals(list, totals, n_shared);
    sp_keep_totals(p.list, own_totals, n_own * kStRuns);
  }
  const int u_begin = n_shared ? sp_run(total, n_shared, blockIdx.x) : 0, u_end = n_shared ? sp_run(total, n_shared, blockIdx.x + 1) : 0;
  const int half = list.half;                                  // sequences of one of the two tiles
  const int tile_rows = half * list.per;

  if (static_cast<int>(blockIdx.x) >= n_shared) {
    const int run = warp / kSpWarps;
    const SpTma tma = {&maps.own_k, &maps.own_v, smem_u32(own_bars) + run * kSpWarps * 16, abort_flag, status};
    sp_split<T, D, 1, true>(p, p.list, own, smem + run * SpSmem<D, 1>::kRun, (blockIdx.x - n_shared) * kStRuns + run, n_own * kStRuns, threadIdx.x % (kSpWarps * 32), 1 + run, tma RB_BOUNDS_PASS);
  } else if (warp >= 8) {
    setmaxnreg_dec<104>();
    if (warp == 8 || warp == 10) {
      // ---------------------------------------------------------------- TMA producers, all lanes: warp 8 keys, warp 10 values
      const bool values = warp == 10;
      const CUtensorMap* map = values ? &maps.v : &maps.k;
      const uint32_t tiles = values ? sV : sK, full = values ? bar_vfull : bar_kfull, empty = values ? bar_vempty : bar_kempty;
      const int bs = p.block_size, size = min(bs, kSpUnit);    // rows of a copy
      bool ok = true;
      int it = 0, tails = 0;
      for (int u = u_begin; u < u_end && ok;) {
        const SpPart s = sp_next(p, list, held, u, u_end);
        const int shared = s.shared;
        // pages of a unit: lane i has the i-th (one of 128 rows, from `row` on, where pages are larger); looked up a unit ahead
        auto page_of = [&](int unit) {
          const int at = unit * kSpUnit + lane * size;
          return unit < s.u1 && lane * size < kSpUnit && at < shared ? s.table[at / bs] : 0;
        };
        int page = page_of(s.u0);
        for (int unit = s.u0; unit < s.u1; ++unit, ++it) {
          const int st = it % kStages, first = unit * kSpUnit, valid = min(kSpUnit, shared - first), pages = (valid + size - 1) / size;
          int blk = page;
          if (lane < pages && (blk < 0 || blk >= p.num_blocks)) {      // corrupt tables read block 0 instead of faulting
            RB_BOUNDS_HIT(104);
            blk = 0;
          }
          page = page_of(unit + 1);
          const int row = first % bs * (bs > kSpUnit);
          const uint32_t tile = tiles + st * L::kTileBytes;
          const bool tail = values && valid < kSpUnit;
          const uint32_t bar = tail ? bar_tail : full + 8 * st;
          ok = mbar_wait(empty + 8 * st, (it / kStages & 1) ^ 1, abort_flag, status, 52 + values);
          if (!__all_sync(0xffffffffu, ok)) { ok = false; break; }
          if (lane == 0) mbar_arrive_expect_tx(bar, pages * size * 128 * (D / 64));
          __syncwarp();
          if (lane < pages) {
#pragma unroll
            for (int hf = 0; hf < D / 64; ++hf) tma_load_4d(tile + hf * L::kHalf + lane * size * 128, map, hf * 64, s.vh, row, blk, bar);
          }
          if (tail) {
            // the copies land, then the rows behind the last token become zero, then the tile is full
            ok = mbar_wait(bar_tail, tails & 1, abort_flag, status, 54);
            ++tails;
            if (!__all_sync(0xffffffffu, ok)) { ok = false; break; }
            uint8_t* rows = smem + L::kV + st * L::kTileBytes + valid * 128;
            for (int i = lane; i < (kSpUnit - valid) * 8; i += 32)
#pragma unroll
              for (int hf = 0; hf < D / 64; ++hf) *reinterpret_cast<uint4*>(rows + hf * L::kHalf + i * 16) = make_uint4(0u, 0u, 0u, 0u);
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(full + 8 * st);
          }
        }
      }
    } else if (warp == 11) {
      // ---------------------------------------------------------------- queries of a part, behind the last product of the part in front
      bool ok = true;
      int part = 0;
      for (int u = u_begin; u < u_end && ok; ++part) {
        const SpPart s = sp_next(p, list, held, u, u_end);
        if (part > 0) ok = mbar_wait(bar_qfree, (part - 1) & 1, abort_flag, status, 51);
        if (ok && lane == 0) {
          const int n = s.n > half ? 2 : 1;
          mbar_arrive_expect_tx(bar_q, n * tile_rows * 128 * (D / 64));
          for (int t = 0; t < n; ++t)
#pragma unroll
            for (int hf = 0; hf < D / 64; ++hf)
              tma_load_4d(sQ + t * L::kTileBytes + hf * L::kHalf, &maps.q, hf * 64, s.vh * list.per, s.b + t * half, 0, bar_q);
        }
      }
    } else if (warp == 9) {
      if (elect_one()) {
        // ---------------------------------------------------------------- MMA issuer
        const uint64_t dQ = umma_smem_desc_sw128(sQ, 16, 1024), dK = umma_smem_desc_sw128(sK, 16, 1024), dV = umma_smem_desc_sw128(sV, L::kHalf, 1024);
        constexpr bool kBf16 = sizeof(T) == sizeof(__nv_bfloat16) && !std::is_same<T, __half>::value;
        constexpr uint32_t drop = kBf16 ? 0u : (1u << 7) | (1u << 10);       // operand formats: 1 bf16, 0 f16
        constexpr uint32_t idesc_qk = umma_idesc_bf16(128, 128, 0, 0) & ~drop;
        constexpr uint32_t idesc_pv = umma_idesc_bf16(128, D, 0, 1) & ~drop; // A = P (TMEM), B = V, rows along the sum
        bool ok = true;
        int it = 0, part = 0, done[2] = {0, 0};
        // S_t = Q_tile K_i^T
        auto issue_qk = [&](int i, int t, int tile) -> bool {
          const int st = i % kStages;
          if (!mbar_wait(bar_kfull + 8 * st, (i / kStages) & 1, abort_flag, status, 55)) return false;
          tc_fence_after();
          const uint64_t q = dQ + tile * (L::kTileBytes / 16), k = dK + st * (L::kTileBytes / 16);
#pragma unroll
          for (int ks = 0; ks < D / 16; ++ks) {
            const uint64_t off = (ks >> 2) * (L::kHalf / 16) + (ks & 3) * 2;
            umma_bf16_ss(tmem_base + t * 128, q + off, k + off, idesc_qk, ks != 0 ? 1u : 0u);
          }
          umma_commit(bar_sfull + 8 * t);
          return true;
        };
        // O_t (+)= P_t V_i, each half of the unit's tokens once P_t has it
        auto issue_pv = [&](int i, int t, bool add) -> bool {
          const uint32_t tmem_p = tmem_base + t * 128, tmem_o = tmem_base + 256 + t * 128;
          const uint64_t v = dV + (i % kStages) * (L::kTileBytes / 16);
#pragma unroll
          for (int ks = 0; ks < kSpUnit / 16; ++ks) {
            if (ks % (kSpUnit / 32) == 0) {
              if (!mbar_wait(bar_pfull + 16 * t + (ks ? 8 : 0), done[t] & 1, abort_flag, status, 58)) return false;
              tc_fence_after();
            }
            umma_bf16_ts(tmem_o, tmem_p + ks * 8, v + ks * (2048 / 16), idesc_pv, (add || ks != 0) ? 1u : 0u);
          }
          ++done[t];
          umma_commit(bar_oready + 8 * t);
          return true;
        };
        for (int u = u_begin; u < u_end && ok; ++part) {
          const SpPart s = sp_next(p, list, held, u, u_end);
          const int n = s.u1 - s.u0;
          ok = mbar_wait(bar_q, part & 1, abort_flag, status, 56);
          if (s.n > half) {                                      // two tiles of rows
            for (int t = 0; t < 2 && ok; ++t) ok = issue_qk(it, t, t);
            if (!ok) break;
            umma_commit(bar_kempty + 8 * (it % kStages));
            if (n == 1) umma_commit(bar_qfree);
            for (int j = 0; j < n && ok; ++j) {
              const int i = it + j, st = i % kStages;
              if (!mbar_wait(bar_vfull + 8 * st, (i / kStages) & 1, abort_flag, status, 57)) { ok = false; break; }
              for (int t = 0; t < 2; ++t) {
                if (!issue_pv(i, t, j > 0)) { ok = false; break; }
                if (j + 1 < n && !issue_qk(i + 1, t, t)) { ok = false; break; }   // overwrites S_t / P_t: ordered behind PV(j, t)
              }
              if (!ok) break;
              umma_commit(bar_vempty + 8 * st);
              if (j + 1 < n) umma_commit(bar_kempty + 8 * ((i + 1) % kStages));
              if (j + 2 == n) umma_commit(bar_qfree);            // the last products that read the queries have been issued
            }
          } else {                                               // one: units in turn with the S and O of A and of B
            for (int j = 0; j < 2 && j < n && ok; ++j) {
              ok = issue_qk(it + j, j, 0);
              if (!ok) break;
              umma_commit(bar_kempty + 8 * ((it + j) % kStages));
              if (j + 1 == n) umma_commit(bar_qfree);
            }
            for (int j = 0; j < n && ok; ++j) {
              const int i = it + j, st = i % kStages;
              if (!mbar_wait(bar_vfull + 8 * st, (i / kStages) & 1, abort_flag, status, 57) || !issue_pv(i, j & 1, j > 1)) { ok = false; break; }
              umma_commit(bar_vempty + 8 * st);
              if (j + 2 < n) {
                if (!issue_qk(i + 2, j & 1, 0)) { ok = false; break; }
                umma_commit(bar_kempty + 8 * ((i + 2) % kStages));
                if (j + 3 == n) umma_commit(bar_qfree);
              }
            }
          }
          it += n;
        }
      }
    }
  } else {
    setmaxnreg_inc<200>();
    // ------------------------------------------------------------------ softmax, one row per thread
    const int t = warp >> 2, wq = warp & 3;
    const uint32_t lane_off = static_cast<uint32_t>(wq * 32) << 16;
    const uint32_t tmem_s = tmem_base + t * 128 + lane_off, tmem_o = tmem_base + 256 + t * 128 + lane_off;
    const float sl2 = p.scale * kSpLog2e;
    bool ok = true;
    int done = 0;
    uint8_t* stage = smem + L::kStage + warp * 2048;
    for (int u = u_begin; u < u_end && ok;) {
      const SpPart s = sp_next(p, list, held, u, u_end);
      const bool twin = s.n <= half;                           // one tile of rows: A has the part's even units, B the odd ones
      const int shared = s.shared, step = twin ? 2 : 1, j0 = s.u0 + (twin ? t : 0);
      const int tile_seqs = twin ? s.n : t == 0 ? half : s.n - half;
      const bool busy = wq * 32 < tile_seqs * list.per;        // this warp has rows
      float m_run = -INFINITY, l_run = 0.f;
      for (int j = j0; j < s.u1; j += step, ++done) {
        if (!mbar_wait(bar_sfull + 8 * t, done & 1, abort_flag, status, 59)) { ok = false; break; }
        tc_fence_after();
        if (busy) {
          const int valid = shared - j * kSpUnit;
          // 64 scores of the row, those behind the last token -infinity
          auto scores = [&](int c, uint32_t (&r)[64]) {
            st_ld32(tmem_s + c * 64, r);
            st_ld32(tmem_s + c * 64 + 32, r + 32);
            tmem_ld_wait();
            if (valid < kSpUnit) {
#pragma unroll
              for (int i = 0; i < 64; ++i)
                if (c * 64 + i >= valid) r[i] = 0xff800000u;
            }
          };
          float mx0 = -INFINITY, mx1 = -INFINITY, mx2 = -INFINITY, mx3 = -INFINITY;
#pragma unroll 1
          for (int c = 0; c < 2; ++c) {
            uint32_t r[64];
            scores(c, r);
#pragma unroll
            for (int i = 0; i < 64; i += 8) {
              mx0 = st_max3(mx0, __uint_as_float(r[i]), __uint_as_float(r[i + 1]));
              mx1 = st_max3(mx1, __uint_as_float(r[i + 2]), __uint_as_float(r[i + 3]));
              mx2 = st_max3(mx2, __uint_as_float(r[i + 4]), __uint_as_float(r[i + 5]));
              mx3 = st_max3(mx3, __uint_as_float(r[i + 6]), __uint_as_float(r[i + 7]));
            }
          }
          const float mx = fmaxf(fmaxf(mx0, mx1), fmaxf(mx2, mx3));
          const bool grow = mx > m_run && ((mx - m_run) * sl2 > kStRescale || m_run == -INFINITY);
          float alpha = 1.f;
          if (grow) {
            alpha = m_run == -INFINITY ? 0.f : wm_ex2((m_run - mx) * sl2);
            m_run = mx;
            l_run *= alpha;
          }
          if (j > j0 && __any_sync(0xffffffffu, grow)) {
            // O has the sum over the units in front once their last product is done; the next one cannot start before P is there
            if (!mbar_wait(bar_oready + 8 * t, (done - 1) & 1, abort_flag, status, 60)) { ok = false; break; }
            tc_fence_after();
#pragma unroll 1
            for (int c = 0; c < D / 32; ++c) {
              uint32_t o[32];
              st_ld32(tmem_o + c * 32, o);
              tmem_ld_wait();
#pragma unroll
              for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * alpha);
              st_st32(tmem_o + c * 32, o);
            }
          }
          const float msc = (m_run == -INFINITY ? 0.f : m_run) * sl2;
          float rs0 = 0.f, rs1 = 0.f, rs2 = 0.f, rs3 = 0.f;
          // P takes the columns of scores that have been read.  64 at a time, not all: the loops' code is met for the first time in every launch, and unrolled over a row of 128 that took
          // 6500 cycles, twice a unit's time
#pragma unroll 1
          for (int c = 0; c < 2; ++c) {
            uint32_t r[64];
            scores(c, r);
            uint32_t packed[32];
#pragma unroll
            for (int i = 0; i < 64; i += 4) {
              const float p0 = wm_ex2(fmaf(__uint_as_float(r[i]), sl2, -msc)), p1 = wm_ex2(fmaf(__uint_as_float(r[i + 1]), sl2, -msc));
              const float p2 = wm_ex2(fmaf(__uint_as_float(r[i + 2]), sl2, -msc)), p3 = wm_ex2(fmaf(__uint_as_float(r[i + 3]), sl2, -msc));
              rs0 += p0;
              rs1 += p1;
              rs2 += p2;
              rs3 += p3;
              packed[i / 2] = sp_pack<T>(p0, p1);
              packed[i / 2 + 1] = sp_pack<T>(p2, p3);
            }
            st_st32(tmem_s + c * 32, packed);
            tmem_st_wait();
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(bar_pfull + 16 * t + 8 * c);          // the products of the first half run beside the second's exponentials
          }
          l_run += (rs0 + rs1) + (rs2 + rs3);
        } else if (lane == 0) {
          mbar_arrive(bar_pfull + 16 * t);
          mbar_arrive(bar_pfull + 16 * t + 8);
        }
      }
      if (!ok) break;
      // ---- the part's sums, 16 columns at a time through shared memory: rows of 512 bytes by threads of their own would be 32 sectors a store
      const bool some = j0 < s.u1;
      if (some && !mbar_wait(bar_oready + 8 * t, (done - 1) & 1, abort_flag, status, 61)) break;
      tc_fence_after();
      if (busy) {
        const long long to = sp_row(list, s.vh, s.e, blockIdx.x, s.u0 == 0) + (twin ? 0 : t * tile_rows) + wq * 32 + (twin && t ? list.rows : 0);
        const int rows = min(32, tile_seqs * list.per - wq * 32);
        if (lane < rows) list.ml[to + lane] = make_float2(m_run * sl2, l_run);
        if (some) {                                            // a part of one unit: B has none
#pragma unroll 1
          for (int c = 0; c < D / 16; ++c) {
            // piece i (16 bytes) of row `lane` to place i ^ lane / 2 of 4: no two of eight rows meet in a bank
            uint32_t o[16];
            tmem_ld_32x16(tmem_o + c * 16, o);
            tmem_ld_wait();
#pragma unroll
            for (int i = 0; i < 4; ++i) *reinterpret_cast<uint4*>(stage + (lane * 4 + ((i ^ lane >> 1) & 3)) * 16) = make_uint4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]);
            __syncwarp();
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const int r = i * 8 + (lane >> 2), k = lane & 3;
              const uint4 v = *reinterpret_cast<const uint4*>(stage + (r * 4 + ((k ^ r >> 1) & 3)) * 16);
              if (r < rows) *reinterpret_cast<uint4*>(list.acc + (to + r) * D + c * 16 + k * 4) = v;
            }
            __syncwarp();
          }
        }
      }
      tc_fence_before();                                       // the next part's first product overwrites O behind the next arrival
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 9) {
    if (*abort_flag) {
      // a wait gave up: let copies and products in flight land before the accumulators are released
      const unsigned long long t0 = globaltimer_ns();
      while (globaltimer_ns() - t0 < 200000ull) __nanosleep(1000);
    }
    tc_fence_after();
    tmem_dealloc(tmem_base, kTmemCols);
  }
}

}  // namespace rb

namespace {

template <typename T, int D>
int launch(const rb::SpParams& p, cudaStream_t stream) {
  const rb::SpList& l = p.prefix;
  int err = 0;
  const uint64_t q_dims[4] = {(uint64_t)D, (uint64_t)p.heads, (uint64_t)p.batch, 1}, q_str[3] = {(uint64_t)D * 2, (uint64_t)p.ld_q * 2, (uint64_t)p.ld_q * 2 * p.batch};
  const uint32_t q_box[4] = {64, (uint32_t)l.per, (uint32_t)(rb::kStTile / l.per), 1};
  const uint64_t dims[4] = {(uint64_t)D, (uint64_t)p.kv_heads, (uint64_t)p.block_size, (uint64_t)p.num_blocks};
  const uint64_t token = (uint64_t)D * p.kv_heads * 2, str[3] = {(uint64_t)D * 2, token, token * p.block_size};
  const uint32_t box[4] = {64, 1, (uint32_t)(p.block_size < rb::kSpUnit ? p.block_size : rb::kSpUnit), 1};
  rb::StMaps maps;
  const CUtensorMap* m = rbhost::get_tmap_4d(p.q, 2, q_dims, q_str, q_box, 1, &err);
  if (!m) return err ? err : -7;
  maps.q = *m;
  m = rbhost::get_tmap_4d(p.k, 2, dims, str, box, 1, &err);
  if (!m) return err ? err : -7;
  maps.k = *m;
  m = rbhost::get_tmap_4d(p.v, 2, dims, str, box, 1, &err);
  if (!m) return err ? err : -7;
  maps.v = *m;
  // of the sequences' own tokens: 64 columns, tokens of all pages, the halves of a head, heads
  const int grain = 1 << p.list.log_grain;
  const uint64_t own_dims[4] = {64, (uint64_t)p.num_blocks * p.block_size, D / 64, (uint64_t)p.kv_heads}, own_str[3] = {token, 128, (uint64_t)D * 2};
  const uint32_t own_box[4] = {64, (uint32_t)grain, D / 64, 1};
  m = rbhost::get_tmap_4d(p.k, 2, own_dims, own_str, own_box, 1, &err);
  if (!m) return err ? err : -7;
  maps.own_k = *m;
  m = rbhost::get_tmap_4d(p.v, 2, own_dims, own_str, own_box, 1, &err);
  if (!m) return err ? err : -7;
  maps.own_v = *m;
  auto smem_of = [](int batch, int groups) { return rb::StSmem<D>::kTotal + (5 * static_cast<size_t>(batch) + 2 + groups) * 4 + 1024; };
  constexpr size_t kMostSmem = rb::StSmem<D>::kTotal + (6 * static_cast<size_t>(rb::kStMostBatch) + 2) * 4 + 1024;
  static_assert(kMostSmem + 1024 <= 227 * 1024 && rb::kStRuns * rb::SpSmem<D, 1>::kRun <= rb::StSmem<D>::kBar && rb::kStRuns * rb::kSpWarps * 32 == rb::kStThreads, "shared memory");
  static bool configured[64] = {false};
  const int dev = rbhost::device_slot();
  if (!configured[dev]) {
    const cudaError_t e = cudaFuncSetAttribute(rb::shared_tc_kernel<T, D>, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(kMostSmem));
    if (e != cudaSuccess) return static_cast<int>(e);
    configured[dev] = true;
  }
  const size_t smem = smem_of(p.batch, p.groups);
  return static_cast<int>(rbhost::launch_pdl(rb::shared_tc_kernel<T, D>, dim3(l.ctas), dim3(rb::kStThreads), smem, stream, 1, maps, p,
                                             rbhost::status_ptr() RB_BOUNDS_ARG));
}

}  // namespace

namespace rbhost {

// Pages that a unit of 128 tokens (and a warp's 32 of a sequence's own) has a whole number of, or that have a whole number of units; every sequence's rows of a KV head in one tile.
bool shared_tc_takes(int batch, int heads, int kv_heads, int block_size, int most) {
  return batch <= rb::kStMostBatch && heads / kv_heads <= rb::kStTile && most >= 1 &&
         (block_size % rb::kSpUnit == 0 || (block_size >= 8 && rb::kSpUnit % block_size == 0)) && block_size < (1 << 20);
}
rb::SpList shared_tc_list(int batch, int heads, int kv_heads) {
  rb::SpList l;
  memset(&l, 0, sizeof(l));
  l.entries = l.own = batch;
  l.per = heads / kv_heads;
  l.parts = 1;
  l.virtual_heads = kv_heads;
  l.seqs = rb::kStTile / l.per * 2;
  l.ctas = device_sm_count();
  l.half = l.seqs / 2;
  l.rows = sp_list_rows(l);
  return l;
}
int shared_tc_runs() { return device_sm_count() * rb::kStRuns; }
int shared_tc(const rb::SpParams& p, int type, int head_dim, cudaStream_t stream) {
  if (type == 0) return head_dim == 64 ? launch<__nv_bfloat16, 64>(p, stream) : launch<__nv_bfloat16, 128>(p, stream);
  return head_dim == 64 ? launch<__half, 64>(p, stream) : launch<__half, 128>(p, stream);
}

}  // namespace rbhost
