// A run of units by four warps, for few rows (up to 16, or 32): the rows are one or two m16n8k16 tiles, a warp takes 32 of a unit's tokens, keys and values come by 16-byte asynchronous
// copies into tiles of its own.
#pragma once
#include "shared_prefix.cuh"

namespace rb {

constexpr int kSpWarps = 4;

template <typename T>
__device__ __forceinline__ void sp_mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1);
template <>
__device__ __forceinline__ void sp_mma<__nv_bfloat16>(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) { wm_mma(c, a, b0, b1); }
template <>
__device__ __forceinline__ void sp_mma<__half>(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <int D, int MT>
struct SpSmem {
  static constexpr int kTile = 32 * D;           // a warp's tile of K or V (elements)
  static constexpr int kQ = kSpWarps * 2 * kTile * 2;                    // byte offsets
  static constexpr int kMl = kQ + 16 * MT * D * 2;
  static constexpr int kHeld = kMl + kSpWarps * 16 * MT * 8;
  static constexpr int kRun = (kHeld + 1023) / 1024 * 1024;              // of one of several runs that a CTA has
};
// Tensor maps of the caches (boxes of up to 32 rows of a page), for runs whose keys and values come by TMA, and such a run's two barriers for each of its warps.
struct SpTma {
  const CUtensorMap* k;
  const CUtensorMap* v;
  uint32_t bars;
  volatile int* abort_flag;
  unsigned int* status;
};
// Byte offset of 16-byte piece c of row r in a tile of D columns: pieces of eight neighbouring rows, which ldmatrix takes at a time, lie in different banks.
template <int D>
__device__ __forceinline__ uint32_t sp_piece(int r, int c) { return (r * (D / 8) + (c ^ (r & 7))) * 16; }
// A unit of a run: where it is in the list of its virtual KV head.
struct SpUnit {
  int vh, hk, at, e, upto;                       // upto: the entry's end
};
__device__ __forceinline__ void sp_advance(const SpList& l, const SpHeld& held, int all, SpUnit& c) {
  if (++c.at < c.upto) return;
  if (c.at == all) {
    c.at = 0;
    c.e = -1;
    ++c.vh;
    c.hk = l.parts == 1 ? c.vh : c.vh / l.parts;
  }
  do c.upto = held.totals[++c.e + 1];
  while (c.upto <= c.at);
}

// The copies go on from one part to the next: the next unit's keys, whichever part they are of, are asked for as soon as this unit's scores are formed, its values behind this unit's
// product, and its places in the cache are looked up a unit earlier (looked up when they were needed they took 4300 of a unit's 7000 cycles).  Bound by the chain of these steps, 4500 cycles
// for a unit with three runs on an SM, of which waits for memory are a tenth.  The warps' sums are joined in the memory of
// their V tiles (two m-tiles: of K and V, and the next part's keys are asked for behind the join).
//
// Warps 4 * n .. 4 * n + 3 of a CTA, tid: a thread's number among them, `bar`: the barrier they meet at.  TMA: pages of 8, 16 or a multiple of 32 tokens; a copy by asynchronous
// accesses of 16 bytes took 4000 of a unit's 6600 cycles with three runs on an SM.  An entry's tokens then begin with the first of a page, or of 32 of a page, that it shares with the
// tokens in front (list.grain); those are masked, and like the rows behind the last token their values become zero: a weight of zero times what is there need not be zero.
template <typename T, int D, int MT, bool TMA>
__device__ __forceinline__ void sp_split(const SpParams& p, const SpList& list, const SpHeld& held, uint8_t* sp_mem, int run, int runs, int tid, int bar, const SpTma& tma RB_BOUNDS_PARAM) {
  // TMA writes a tile page by page, a page's 64 columns behind one another in rows of 128 bytes, in which the pieces lie as sp_piece has them.  Row r begins at row_at(r).
  const int size = 1 << list.log_grain;          // tokens of a copy by TMA
  auto row_at = [&](int r) { return (r >> list.log_grain) * size * D * 2 + (r & (size - 1)) * 128; };
  const int far = size * 128;                    // from 64 columns to the next
  auto sync = [&]() { asm volatile("bar.sync %0, %1;" ::"r"(bar), "n"(kSpWarps * 32) : "memory"); };
  using L = SpSmem<D, MT>;
  constexpr int NT = D / 8, LP = D / 8, kRows = 16 * MT, kQPieces = kRows * LP / (kSpWarps * 32);
  constexpr bool kAhead = MT == 1;
  const int warp = tid >> 5, lane = tid & 31, gq = lane >> 2, tq = lane & 3;
  float2* ml_sh = reinterpret_cast<float2*>(sp_mem + L::kMl);           // [warp][row]: maximum, sum
  const uint32_t q_u32 = smem_u32(sp_mem + L::kQ), k_u32 = smem_u32(sp_mem) + warp * 2 * L::kTile * 2, v_u32 = k_u32 + L::kTile * 2;
  uint8_t* const v_tile = sp_mem + warp * 2 * L::kTile * 2 + L::kTile * 2;
  uint32_t k_rows[2], v_rows[2];                 // this lane's rows for ldmatrix
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    k_rows[i] = k_u32 + row_at(i * 16 + (lane & 7) + ((lane >> 4) << 3));
    v_rows[i] = v_u32 + row_at(i * 16 + (lane & 7) + ((lane >> 3) & 1) * 8);
  }
  // fp32 [rows][D] of a warp's sums
  float* mine = reinterpret_cast<float*>(sp_mem + warp * 2 * L::kTile * 2 + (kAhead ? L::kTile * 2 : 0));
  const int all = held.totals[list.entries], total = all * list.virtual_heads, group = p.heads / p.kv_heads;
  const int u_begin = sp_run(total, runs, run);
  int left = sp_run(total, runs, run + 1) - u_begin;        // units of the run from this one on
  if (left <= 0) return;
  const T* K = static_cast<const T*>(p.k);
  const T* V = static_cast<const T*>(p.v);
  const float scale2 = p.scale * kSpLog2e;

  SpUnit c0;                                     // this unit
  c0.vh = u_begin / all;
  c0.at = u_begin - c0.vh * all;
  c0.e = 0;
  for (int hi = list.entries; hi - c0.e > 1;) {  // the last entry that begins at or in front of it
    const int mid = (c0.e + hi) >> 1;
    if (held.totals[mid] <= c0.at) c0.e = mid;
    else hi = mid;
  }
  c0.hk = c0.vh / list.parts;
  c0.upto = held.totals[c0.e + 1];
  // runs whose keys and values come by TMA have entries of sequences' own tokens only
  auto is_own = [&](int e) { return TMA || e >= list.own; };
  auto first_of = [&](int e) { return TMA ? e : e >= list.own ? e - list.own : e; };
  auto rows_of = [&](int e) {
    if (is_own(e)) return list.per;
    return min(list.seqs, static_cast<int>(held.span[e] >> 16) - e) * list.per;
  };
  // ---- rows of queries: loaded into registers, stored when the last part's have been read
  uint4 q_next[kQPieces];
  int q_seq[kQPieces], q_head[kQPieces];
#pragma unroll
  for (int i = 0; i < kQPieces; ++i) {
    const int r = (i * kSpWarps * 32 + tid) / LP;
    q_seq[i] = r / list.per;
    q_head[i] = r - q_seq[i] * list.per;
  }
  auto load_q = [&](const SpUnit& c) {
    const int head0 = (c.vh - c.hk * list.parts) * list.per, real = min(list.per, group - head0);
    const int b = first_of(c.e), seqs = is_own(c.e) ? 1 : min(list.seqs, static_cast<int>(held.span[c.e] >> 16) - c.e);
#pragma unroll
    for (int i = 0; i < kQPieces; ++i) {
      const int piece = (i * kSpWarps * 32 + tid) % LP;
      q_next[i] = make_uint4(0u, 0u, 0u, 0u);
      if (q_seq[i] < seqs && q_head[i] < real)
        q_next[i] = *reinterpret_cast<const uint4*>(static_cast<const T*>(p.q) + (b + q_seq[i]) * p.ld_q + static_cast<long long>(c.hk * group + head0 + q_head[i]) * D + piece * 8);
    }
  };
  auto store_q = [&]() {
#pragma unroll
    for (int i = 0; i < kQPieces; ++i) {
      const int at = i * kSpWarps * 32 + tid, r = at / LP, piece = at - r * LP;
      *reinterpret_cast<uint4*>(sp_mem + L::kQ + sp_piece<D>(r, piece)) = q_next[i];
    }
  };
  auto page_of = [&](int token) { return p.log_block >= 0 ? token >> p.log_block : token / p.block_size; };
  // ---- places of a unit's keys and values: looked up, then asked for
  struct Places {
    int blk, off, n, hk, lead;                   // of the lane's token or page: block and place in it; the warp's tokens (0 and less: none), the first `lead` of them others'
  };
  auto look_up = [&](const SpUnit& c) {
    Places w;
    const bool own = is_own(c.e);
    const int shared = held.shared[c.e], at = (c.at - held.totals[c.e]) * kSpUnit + warp * 32;
    w.n = min(32, held.count[c.e] - at);
    w.hk = c.hk;
    w.blk = w.off = 0;
    w.lead = 0;
    const int* table = p.tables + static_cast<long long>(own ? first_of(c.e) : static_cast<int>(held.span[c.e] & 0xffffu)) * p.width;
    if (TMA) {                                   // of the lane's page
      if (at == 0) w.lead = shared & (size - 1); // the first tokens of an entry may be others'
      if (lane * size < w.n) {
        const int token = (shared & -size) + at + lane * size, page = page_of(token);
        w.off = token - page * p.block_size;
        w.blk = table[page];
      }
    } else if (lane < w.n) {
      const int token = (own ? shared : 0) + at + lane, page = page_of(token);
      w.off = token - page * p.block_size;
      w.blk = table[page];
    }
    return w;
  };
  auto request = [&](const T* cache, uint32_t tile, const Places& w) {
    if (TMA) {
      if (w.n > 0) {
        const bool values = tile == v_u32, mine_too = lane * size < w.n;
        const CUtensorMap* map = values ? tma.v : tma.k;
        const uint32_t full = tma.bars + warp * 16 + values * 8;
        int blk = w.blk;
        if (mine_too && (blk < 0 || blk >= p.num_blocks)) {
          RB_BOUNDS_HIT(104);
          blk = 0;
        }
        if (lane == 0) mbar_arrive_expect_tx(full, (w.n + size - 1 & -size) * D * 2);
        __syncwarp();
        if (mine_too) {
          tma_load_4d(tile + lane * size * D * 2, map, 0, blk * p.block_size + w.off, 0, w.hk, full);       // the host bounds num_blocks * block_size below 2^31
        }
      }
      return;
    }
    if (w.n > 0) {
      int blk = w.blk;
      if (blk < 0 || blk >= p.num_blocks) {                            // corrupt tables read block 0 instead of faulting
        RB_BOUNDS_HIT(104);
        blk = 0;
      }
      const int slot = blk * p.block_size + w.off;                     // the host bounds num_blocks * block_size below 2^31
#pragma unroll
      for (int i = 0; i < LP; ++i) {
        const int idx = i * 32 + lane, r = idx / LP, piece = idx - r * LP;
        const int s = __shfl_sync(0xffffffffu, slot, r);
        wm_cp16(tile + sp_piece<D>(r, piece), r < w.n ? cache + (static_cast<long long>(s) * p.kv_heads + w.hk) * D + piece * 8 : cache, r < w.n);
      }
    }
    wm_cp_commit();
  };

  Places w0 = look_up(c0);
  SpUnit c1 = c0;                                // the next unit, if there is one
  if (left > 1) sp_advance(list, held, all, c1);
  Places w1 = look_up(c1);
  load_q(c0);
  request(K, k_u32, w0);
  request(V, v_u32, w0);
  store_q();
  sync();
  bool begins = c0.at == held.totals[c0.e];      // this part begins its entry
  float m[MT][2], l[MT][2], acc[MT][NT][4];
  auto clear = [&]() {
#pragma unroll
    for (int t = 0; t < MT; ++t) {
      m[t][0] = m[t][1] = -INFINITY;
      l[t][0] = l[t][1] = 0.f;
#pragma unroll
      for (int n = 0; n < NT; ++n) acc[t][n][0] = acc[t][n][1] = acc[t][n][2] = acc[t][n][3] = 0.f;
    }
  };
  clear();
  uint32_t phase = 0;                            // of this warp's two barriers
  for (;; --left) {
    const int n_tok = w0.n, rows = rows_of(c0.e);
    const int lead = TMA ? w0.lead : 0;
    const bool more = left > 1, last = !more || c1.e != c0.e || c1.vh != c0.vh;
    if (!TMA) wm_cp_wait<1>();                   // this unit's K tile has landed (V may be on its way)
    else if (n_tok > 0) mbar_wait(tma.bars + warp * 16, phase, tma.abort_flag, tma.status, 62);
    __syncwarp();
    float s[MT][4][4];
#pragma unroll
    for (int t = 0; t < MT; ++t)
#pragma unroll
      for (int n = 0; n < 4; ++n) s[t][n][0] = s[t][n][1] = s[t][n][2] = s[t][n][3] = 0.f;
    if (n_tok > 0) {
#pragma unroll
      for (int k0 = 0; k0 < D / 8; k0 += 2) {    // pieces of 8 columns
        uint32_t bk[2][4];
#pragma unroll
        for (int np = 0; np < 2; ++np) {
          const int r = np * 16 + (lane & 7) + ((lane >> 4) << 3), c = k0 + ((lane >> 3) & 1);
          wm_ldsm_x4(TMA ? k_rows[np] + (k0 >> 3) * far + (((c & 7) ^ (lane & 7)) << 4) : k_u32 + sp_piece<D>(r, c), bk[np]);
        }
#pragma unroll
        for (int t = 0; t < MT; ++t) {
          if (t > 0 && rows <= t * 16) continue;
          uint32_t a[4];
          wm_ldsm_x4(q_u32 + sp_piece<D>(t * 16 + (lane & 15), k0 + (lane >> 4)), a);
#pragma unroll
          for (int np = 0; np < 2; ++np) {
            sp_mma<T>(s[t][2 * np], a, bk[np][0], bk[np][1]);
            sp_mma<T>(s[t][2 * np + 1], a, bk[np][2], bk[np][3]);
          }
        }
      }
    }
    __syncwarp();                                // every lane has read its K fragments
    // ---- the next unit's keys, and a look at the one behind it
    if (!more) w1.n = 0;
    if (kAhead || !last) request(K, k_u32, w1);
    else if (!TMA) wm_cp_commit();
    if (last && more) load_q(c1);
    SpUnit c2 = c1;
    if (left > 2) sp_advance(list, held, all, c2);
    const Places w2 = look_up(c2);
    if (n_tok > 0) {
      uint32_t pf[MT][2][4];
#pragma unroll
      for (int t = 0; t < MT; ++t) {
        if (t > 0 && rows <= t * 16) continue;
#pragma unroll
        for (int i = 0; i < 2; ++i) {            // rows gq and gq + 8
          if (TMA && i == 1 && rows <= 8) {      // there are none of the second kind
            pf[t][0][1] = pf[t][0][3] = pf[t][1][1] = pf[t][1][3] = 0u;
            continue;
          }
          float mx = -INFINITY;
#pragma unroll
          for (int n = 0; n < 4; ++n)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              float& x = s[t][n][2 * i + j];
              x = static_cast<uint32_t>(n * 8 + j + 2 * tq - lead) < static_cast<uint32_t>(n_tok - lead) ? x * scale2 : -INFINITY;
              mx = fmaxf(mx, x);
            }
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
          const float mn = fmaxf(m[t][i], mx), from = mn == -INFINITY ? 0.f : mn;       // scores of minus infinity
          const float al = wm_ex2(m[t][i] - from);
          float sum = 0.f;
#pragma unroll
          for (int n = 0; n < 4; ++n) {
            const float p0 = wm_ex2(s[t][n][2 * i] - from), p1 = wm_ex2(s[t][n][2 * i + 1] - from);
            sum += p0 + p1;
            pf[t][n >> 1][(n & 1) * 2 + i] = sp_pack<T>(p0, p1);
          }
          l[t][i] = fmaf(l[t][i], al, sum);      // of this lane's tokens
          m[t][i] = mn;
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            acc[t][n][2 * i] *= al;
            acc[t][n][2 * i + 1] *= al;
          }
        }
      }
      if (!TMA) {
        wm_cp_wait<1>();                         // this unit's V tile has landed
      } else {
        mbar_wait(tma.bars + warp * 16 + 8, phase, tma.abort_flag, tma.status, 63);
        phase ^= 1;
        if (n_tok < 32 || lead > 0) {
          const int r = lane;
          if (r < lead || r >= n_tok) {
#pragma unroll
            for (int c = 0; c < LP; ++c) *reinterpret_cast<uint4*>(v_tile + row_at(r) + (c >> 3) * far + ((c + lane) & 7) * 16) = make_uint4(0u, 0u, 0u, 0u);
          }
          fence_proxy_async_smem();              // ahead of the next copy
        }
      }
      __syncwarp();
#pragma unroll
      for (int ks = 0; ks < 2; ++ks)
#pragma unroll
        for (int n2 = 0; n2 < NT / 2; ++n2) {
          uint32_t bv[4];
          const int r = ks * 16 + (lane & 7) + ((lane >> 3) & 1) * 8, c = n2 * 2 + (lane >> 4);
          wm_ldsm_x4_t(TMA ? v_rows[ks] + (n2 >> 2) * far + (((c & 7) ^ (lane & 7)) << 4) : v_u32 + sp_piece<D>(r, c), bv);
#pragma unroll
          for (int t = 0; t < MT; ++t) {
            if (t > 0 && rows <= t * 16) continue;
            sp_mma<T>(acc[t][2 * n2], pf[t][ks], bv[0], bv[1]);
            sp_mma<T>(acc[t][2 * n2 + 1], pf[t][ks], bv[2], bv[3]);
          }
        }
      __syncwarp();                              // every lane has read its V fragments
    }
    if (last) {
      // ---- the part's sums
      if (!TMA) wm_cp_wait<kAhead ? 1 : 0>();    // nothing is on its way into the memory that the sums take
      __syncwarp();
#pragma unroll
      for (int t = 0; t < MT; ++t) {
        if (t > 0 && rows <= t * 16) continue;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          if (TMA && i == 1 && rows <= 8) continue;
          const int r = t * 16 + gq + i * 8;
          l[t][i] += __shfl_xor_sync(0xffffffffu, l[t][i], 1);
          l[t][i] += __shfl_xor_sync(0xffffffffu, l[t][i], 2);
          if (tq == 0) ml_sh[warp * kRows + r] = make_float2(m[t][i], l[t][i]);
#pragma unroll
          for (int n = 0; n < NT; ++n) *reinterpret_cast<float2*>(mine + r * D + ((n * 8) ^ ((r & 7) * 8)) + 2 * tq) = make_float2(acc[t][n][2 * i], acc[t][n][2 * i + 1]);
        }
      }
      sync();
      const long long row0 = sp_row(list, c0.vh, c0.e, run, begins);
      for (int i = tid; i < rows * (D / 4); i += kSpWarps * 32) {
        const int r = i / (D / 4), c = (i - r * (D / 4)) * 4;
        float mx = -INFINITY;
#pragma unroll
        for (int w = 0; w < kSpWarps; ++w) mx = fmaxf(mx, ml_sh[w * kRows + r].x);
        float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
        float den = 0.f;
#pragma unroll
        for (int w = 0; w < kSpWarps; ++w) {
          const float2 ml = ml_sh[w * kRows + r];
          const float f = ml.x == -INFINITY ? 0.f : wm_ex2(ml.x - mx);
          const float4 x = *reinterpret_cast<const float4*>(reinterpret_cast<const float*>(sp_mem + w * 2 * L::kTile * 2 + (kAhead ? L::kTile * 2 : 0)) + r * D + (c ^ ((r & 7) * 8)));
          sum.x = fmaf(x.x, f, sum.x); sum.y = fmaf(x.y, f, sum.y); sum.z = fmaf(x.z, f, sum.z); sum.w = fmaf(x.w, f, sum.w);
          den = fmaf(ml.y, f, den);
        }
        *reinterpret_cast<float4*>(list.acc + (row0 + r) * D + c) = sum;
        if (c == 0) list.ml[row0 + r] = make_float2(mx, den);
      }
      if (!more) return;
      if (TMA) fence_proxy_async_smem();         // sums that were written, ahead of the copies into their memory
      sync();                           // sums and queries have been read
      store_q();
      if (!kAhead) request(K, k_u32, w1);
      sync();
      clear();
      begins = true;                             // what follows in a run begins at its entry's first unit
    }
    request(V, v_u32, w1);
    c0 = c1;
    w0 = w1;
    c1 = c2;
    w1 = w2;
  }
}

}  // namespace rb
