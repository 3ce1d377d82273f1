// Decode attention for sequences that share their first tokens (beams and samples of one prompt, requests behind one system prompt).
//
// Alone, every sequence of a group reads the shared keys and values again: n sequences, n times the bytes.  Here the queries of all of a group's
// sequences for one KV head are the rows of one product over the shared tokens, which are read once; each sequence's own tokens follow as in any decode
// attention, and a last launch joins the parts of a row by their maxima and sums:
//     out = sum_i 2^(m_i - M) acc_i / sum_i 2^(m_i - M) l_i,   M = max_i m_i.
//
// Work is a list of entries (a tile of a group's rows over its shared tokens, a sequence's rows over its own), cut into units of 128 tokens; the units of all entries,
// one behind the other, are dealt in equal runs to CTAs that stay.  An entry's rows are accumulated over all units of a run, so there are at most (entries +
// CTAs) parts: the one that begins an entry has a place of the entry's own, one that goes on with it is the first of its CTA's run and has the CTA's.  Every CTA forms the
// list of running totals itself from the lengths.
//
// This file's split kernel is for few rows (up to 32): the rows are one or two m16n8k16 tiles, a warp takes 32 of a unit's tokens, keys and values come
// by 16-byte asynchronous copies into tiles of its own.  It is bound by these reads.
#include "shared_prefix.h"

#include <string.h>

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
};
// Byte offset of 16-byte piece c of row r in a tile of D columns: pieces of eight neighbouring rows, which ldmatrix takes at a time, lie in different banks.
template <int D>
__device__ __forceinline__ uint32_t sp_piece(int r, int c) { return (r * (D / 8) + (c ^ (r & 7))) * 16; }

// A unit of a run: where it is in the list of its virtual KV head.
struct SpUnit {
  int vh, at, e;
};
__device__ __forceinline__ void sp_advance(const SpList& l, const SpHeld& held, SpUnit& c) {
  if (++c.at == held.totals[l.entries]) {
    c.at = c.e = 0;
    ++c.vh;
  }
  while (held.totals[c.e + 1] <= c.at) ++c.e;
}

// The copies go on from one part to the next: the next unit's keys, whichever part they are of, are asked for as soon as this unit's scores are formed, its values behind this unit's
// product, and its places in the cache are looked up a unit earlier (looked up when they were needed they took 4300 of a unit's 7000 cycles).  The warps' sums are joined in the memory of
// their V tiles (two m-tiles: of K and V, and the next part's keys are asked for behind the join).
template <typename T, int D, int MT>
__global__ void __launch_bounds__(kSpWarps * 32, MT == 1 ? 3 : 2)
shared_split_kernel(const SpParams p RB_BOUNDS_PARAM) {
  pdl_wait();
  pdl_launch();
  using L = SpSmem<D, MT>;
  constexpr int NT = D / 8, LP = D / 8, kRows = 16 * MT, kQPieces = kRows * LP / (kSpWarps * 32);
  constexpr bool kAhead = MT == 1;
  extern __shared__ __align__(128) uint8_t sp_mem[];
  __shared__ int warp_sums[kSpWarps];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, gq = lane >> 2, tq = lane & 3;
  float2* ml_sh = reinterpret_cast<float2*>(sp_mem + L::kMl);           // [warp][row]: maximum, sum
  const uint32_t q_u32 = smem_u32(sp_mem + L::kQ), k_u32 = smem_u32(sp_mem) + warp * 2 * L::kTile * 2, v_u32 = k_u32 + L::kTile * 2;
  // fp32 [rows][D] of a warp's sums
  float* mine = reinterpret_cast<float*>(sp_mem + warp * 2 * L::kTile * 2 + (kAhead ? L::kTile * 2 : 0));
  const SpList& list = p.list;
  const SpHeld held = sp_held(list, reinterpret_cast<int*>(sp_mem + L::kHeld));
  sp_prepare(p, list, held, warp_sums);
  const int all = held.totals[list.entries], total = all * list.virtual_heads, group = p.heads / p.kv_heads;
  const int u_begin = sp_run(total, list.ctas, blockIdx.x);
  int left = sp_run(total, list.ctas, blockIdx.x + 1) - u_begin;        // units of the run from this one on
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
  auto rows_of = [&](int e) {
    if (e >= list.own) return list.per;
    return min(list.seqs, static_cast<int>(held.span[e] >> 16) - e) * list.per;
  };
  // ---- rows of queries: loaded into registers, stored when the last part's have been read
  uint4 q_next[kQPieces];
  auto load_q = [&](const SpUnit& c) {
    const int hk = c.vh / list.parts, head0 = (c.vh - hk * list.parts) * list.per, real = min(list.per, group - head0), rows = rows_of(c.e);
    const int b = c.e >= list.own ? c.e - list.own : c.e;
#pragma unroll
    for (int i = 0; i < kQPieces; ++i) {
      const int at = i * kSpWarps * 32 + tid, r = at / LP, piece = at - r * LP, seq = r / list.per, h = r - seq * list.per;
      q_next[i] = make_uint4(0u, 0u, 0u, 0u);
      if (r < rows && h < real)
        q_next[i] = *reinterpret_cast<const uint4*>(static_cast<const T*>(p.q) + (b + seq) * p.ld_q + static_cast<long long>(hk * group + head0 + h) * D + piece * 8);
    }
  };
  auto store_q = [&]() {
#pragma unroll
    for (int i = 0; i < kQPieces; ++i) {
      const int at = i * kSpWarps * 32 + tid, r = at / LP, piece = at - r * LP;
      *reinterpret_cast<uint4*>(sp_mem + L::kQ + sp_piece<D>(r, piece)) = q_next[i];
    }
  };
  // ---- places of a unit's keys and values: looked up, then asked for
  struct Places {
    int blk, off, n, hk;                         // of the lane's token: block and place in it; the warp's tokens (0 and less: none)
  };
  auto look_up = [&](const SpUnit& c) {
    Places w;
    const bool own = c.e >= list.own;
    const int shared = held.shared[c.e], at = (c.at - held.totals[c.e]) * kSpUnit + warp * 32;
    w.n = min(32, held.count[c.e] - at);
    w.hk = c.vh / list.parts;
    w.blk = w.off = 0;
    if (lane < w.n) {
      const int token = (own ? shared : 0) + at + lane, page = token / p.block_size;
      w.off = token - page * p.block_size;
      w.blk = p.tables[static_cast<long long>(own ? c.e - list.own : static_cast<int>(held.span[c.e] & 0xffffu)) * p.width + page];
    }
    return w;
  };
  auto request = [&](const T* cache, uint32_t tile, const Places& w) {
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
  if (left > 1) sp_advance(list, held, c1);
  Places w1 = look_up(c1);
  load_q(c0);
  request(K, k_u32, w0);
  request(V, v_u32, w0);
  store_q();
  __syncthreads();
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
  for (;; --left) {
    const int n_tok = w0.n, rows = rows_of(c0.e);
    const bool more = left > 1, last = !more || c1.e != c0.e || c1.vh != c0.vh;
    wm_cp_wait<1>();                             // this unit's K tile has landed (V may be on its way)
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
        for (int np = 0; np < 2; ++np) wm_ldsm_x4(k_u32 + sp_piece<D>(np * 16 + (lane & 7) + ((lane >> 4) << 3), k0 + ((lane >> 3) & 1)), bk[np]);
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
    else wm_cp_commit();
    if (last && more) load_q(c1);
    SpUnit c2 = c1;
    if (left > 2) sp_advance(list, held, c2);
    const Places w2 = look_up(c2);
    if (n_tok > 0) {
      uint32_t pf[MT][2][4];
#pragma unroll
      for (int t = 0; t < MT; ++t) {
        if (t > 0 && rows <= t * 16) continue;
#pragma unroll
        for (int i = 0; i < 2; ++i) {            // rows gq and gq + 8
          float mx = -INFINITY;
#pragma unroll
          for (int n = 0; n < 4; ++n)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
              float& x = s[t][n][2 * i + j];
              x = n * 8 + 2 * tq + j < n_tok ? x * scale2 : -INFINITY;
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
          sum += __shfl_xor_sync(0xffffffffu, sum, 1);
          sum += __shfl_xor_sync(0xffffffffu, sum, 2);
          l[t][i] = fmaf(l[t][i], al, sum);
          m[t][i] = mn;
#pragma unroll
          for (int n = 0; n < NT; ++n) {
            acc[t][n][2 * i] *= al;
            acc[t][n][2 * i + 1] *= al;
          }
        }
      }
      wm_cp_wait<1>();                           // this unit's V tile has landed
      __syncwarp();
#pragma unroll
      for (int ks = 0; ks < 2; ++ks)
#pragma unroll
        for (int n2 = 0; n2 < NT / 2; ++n2) {
          uint32_t bv[4];
          wm_ldsm_x4_t(v_u32 + sp_piece<D>(ks * 16 + (lane & 7) + ((lane >> 3) & 1) * 8, n2 * 2 + (lane >> 4)), bv);
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
      wm_cp_wait<kAhead ? 1 : 0>();              // nothing is on its way into the memory that the sums take
      __syncwarp();
#pragma unroll
      for (int t = 0; t < MT; ++t) {
        if (t > 0 && rows <= t * 16) continue;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int r = t * 16 + gq + i * 8;
          if (tq == 0) ml_sh[warp * kRows + r] = make_float2(m[t][i], l[t][i]);
#pragma unroll
          for (int n = 0; n < NT; ++n) *reinterpret_cast<float2*>(mine + r * D + ((n * 8) ^ ((r & 7) * 8)) + 2 * tq) = make_float2(acc[t][n][2 * i], acc[t][n][2 * i + 1]);
        }
      }
      __syncthreads();
      const long long row0 = sp_row(list, c0.vh, c0.e, blockIdx.x, begins);
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
      __syncthreads();                           // sums and queries have been read
      store_q();
      if (!kAhead) request(K, k_u32, w1);
      __syncthreads();
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

// out[b, head] from the parts of its row.  A CTA has some heads of a sequence and KV head; a row's parts are summed by `share` warps, and
// lanes own D / 32 neighbouring columns.  Grid (batch, KV heads, parts of a KV head's query heads).
constexpr int kSpJoinWarps = 8;
template <typename T, int D>
__global__ void __launch_bounds__(kSpJoinWarps * 32)
shared_join_kernel(const SpParams p, const int share) {
  constexpr int C = D / 32;
  __shared__ float sum_sh[kSpJoinWarps][D + 2];  // a warp's columns, maximum and sum
  const int b = blockIdx.x, hk = blockIdx.y, group = p.heads / p.kv_heads;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int2 span = p.span_of[b];                // older than the launches in front
  const bool any = sp_length(p, b) > 0;          // a sequence without tokens gets zeros
  pdl_wait();
  pdl_launch();
  const int tile = b - (b - span.x) % p.prefix.seqs;
  // parts of an entry that one of two tiles of rows had alone come in twos (see shared_prefix_tc.cu)
  const int twin = p.prefix.half > 0 && min(p.prefix.seqs, span.y - tile) <= p.prefix.half ? 2 : 1;
  // lanes 0, 1: first and last unit over shared tokens, lanes 2, 3: the sequence's own
  const SpList& look = lane & 2 ? p.list : p.prefix;
  const int all = look.totals[look.entries], t0 = look.totals[lane & 2 ? look.own + b : tile], t1 = look.totals[(lane & 2 ? look.own + b : tile) + 1];
  {
    const int h = blockIdx.z * (kSpJoinWarps / share) + warp / share, which = warp % share;
    const bool mine = h < group;
    float mx = -INFINITY, den = 0.f, acc[C];
#pragma unroll
    for (int c = 0; c < C; ++c) acc[c] = 0.f;
    if (mine && any) {
      // parts over shared tokens, then the sequence's own: how many CTAs, the first, and the rows where its part and those of CTA 0 are
      const int k_look = h / look.per, u = (hk * look.parts + k_look) * all + (lane & 1 ? t1 - 1 : t0);
      const int cta = t1 > t0 ? sp_cta_of(all * look.virtual_heads, look.ctas, u) : lane & 1 ? -1 : 0;
      int n[2], c0[2];
      long long row[2], later[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const SpList& l = i == 0 ? p.prefix : p.list;
        const int e = i == 0 ? tile : l.own + b, k = h / l.per, vh = hk * l.parts + k, r = (i == 0 ? b - tile : 0) * l.per + h - k * l.per;
        c0[i] = __shfl_sync(0xffffffffu, cta, 2 * i);
        n[i] = __shfl_sync(0xffffffffu, cta, 2 * i + 1) - c0[i] + 1;
        row[i] = sp_row(l, vh, e, 0, true) + r;
        later[i] = sp_row(l, vh, e, 0, false) + r;
      }
      n[0] *= twin;
      const int parts = n[0] + n[1];
      for (int s0 = which; s0 < parts; s0 += 32 * share) {
        // a lane looks up one part
        const int s = s0 + lane * share;
        const float* columns = nullptr;
        float2 ml = make_float2(-INFINITY, 0.f);
        if (s < parts) {
          const int i = s >= n[0] ? 1 : 0, j = i ? s - n[0] : twin == 2 ? s >> 1 : s;
          const SpList& l = i ? p.list : p.prefix;
          long long at = j == 0 ? row[i] : later[i] + static_cast<long long>(c0[i] + j) * l.seqs * l.per;
          if (!i && twin == 2 && (s & 1)) at += l.rows;
          ml = l.ml[at];
          columns = l.acc + at * D;
        }
        const float top = fmaxf(mx, warp_max(ml.x)), from = top == -INFINITY ? 0.f : top, again = wm_ex2(mx - from);
        const float f = wm_ex2(ml.x - from);
        den = fmaf(den, again, ml.y * f);
#pragma unroll
        for (int c = 0; c < C; ++c) acc[c] *= again;
        mx = top;
        const int m = min(32, (parts - s0 + share - 1) / share);
#pragma unroll 8
        for (int k = 0; k < m; ++k) {
          const float fk = __shfl_sync(0xffffffffu, f, k);
          const float* x = reinterpret_cast<const float*>(__shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(columns), k)) + lane * C;
          if (fk != 0.f) {                       // a part without tokens has no sums
            if (C == 4) {
              const float4 v = *reinterpret_cast<const float4*>(x);
              acc[0] = fmaf(v.x, fk, acc[0]); acc[1] = fmaf(v.y, fk, acc[1]); acc[2 % C] = fmaf(v.z, fk, acc[2 % C]); acc[3 % C] = fmaf(v.w, fk, acc[3 % C]);
            } else {
              const float2 v = *reinterpret_cast<const float2*>(x);
              acc[0] = fmaf(v.x, fk, acc[0]); acc[1] = fmaf(v.y, fk, acc[1]);
            }
          }
        }
      }
      den = warp_sum(den);
    }
    if (share > 1) {
#pragma unroll
      for (int c = 0; c < C; ++c) sum_sh[warp][lane * C + c] = acc[c];
      if (lane == 0) {
        sum_sh[warp][D] = mx;
        sum_sh[warp][D + 1] = den;
      }
      __syncthreads();
      if (mine && which == 0) {
        float top = mx;
        for (int w = 1; w < share; ++w) top = fmaxf(top, sum_sh[warp + w][D]);
        const float from = top == -INFINITY ? 0.f : top, f0 = wm_ex2(mx - from);
        den *= f0;
#pragma unroll
        for (int c = 0; c < C; ++c) acc[c] *= f0;
        for (int w = 1; w < share; ++w) {
          const float f = wm_ex2(sum_sh[warp + w][D] - from);
          den = fmaf(sum_sh[warp + w][D + 1], f, den);
#pragma unroll
          for (int c = 0; c < C; ++c) acc[c] = fmaf(sum_sh[warp + w][lane * C + c], f, acc[c]);
        }
      }
      __syncthreads();
    }
    if (mine && which == 0) {
      const float inv = any ? 1.f / den : 0.f;
      T* o = static_cast<T*>(p.out) + b * p.ld_o + static_cast<long long>(hk * group + h) * D + lane * C;
      uint32_t w[C / 2];
#pragma unroll
      for (int c = 0; c < C / 2; ++c) w[c] = sp_pack<T>(acc[2 * c] * inv, acc[2 * c + 1] * inv);
      if (C == 4) *reinterpret_cast<uint2*>(o) = make_uint2(w[0], w[1 % (C / 2)]);
      else *reinterpret_cast<uint32_t*>(o) = w[0];
    }
  }
}

}  // namespace rb

namespace {

struct Plan {
  rb::SpList list, prefix;
  size_t smem;
  int tiles;                                     // m-tiles of the split kernel
  int share;                                     // warps of a row of the join
  bool tc;
};
// Shared tokens of groups with more than 16 rows go to the tcgen05 kernel, which takes 256 at a time; the split kernel has one m-tile, or two where rows need them.
Plan plan_of(int batch, int groups, int heads, int kv_heads, int head_dim, int block_size, int most, bool positive) {
  Plan p;
  memset(&p, 0, sizeof(p));
  const int group = heads / kv_heads;
  p.tc = static_cast<long long>(most) * group > 16 && positive && rbhost::shared_tc_takes(batch, heads, kv_heads, block_size, most);
  p.tiles = static_cast<long long>(p.tc ? 1 : most) * group > 16 ? 2 : 1;
  const int rows = 16 * p.tiles;
  rb::SpList& l = p.list;
  l.parts = (group + rows - 1) / rows;
  l.per = (group + l.parts - 1) / l.parts;
  l.parts = (group + l.per - 1) / l.per;
  l.seqs = rows / l.per;
  l.virtual_heads = kv_heads * l.parts;
  l.own = p.tc ? 0 : batch;
  l.entries = l.own + batch;
  const size_t tiles = head_dim == 64 ? (p.tiles == 1 ? rb::SpSmem<64, 1>::kHeld : rb::SpSmem<64, 2>::kHeld)
                                      : (p.tiles == 1 ? rb::SpSmem<128, 1>::kHeld : rb::SpSmem<128, 2>::kHeld);
  p.smem = tiles + rb::sp_held_bytes(l.entries, groups);
  const int resident = static_cast<int>((228 * 1024) / (p.smem + 1024 + 64)), most_resident = p.tiles == 1 ? 3 : 2;
  l.ctas = rbhost::device_sm_count() * (resident < 1 ? 1 : resident < most_resident ? resident : most_resident);
  l.rows = rbhost::sp_list_rows(l);
  p.prefix = p.tc ? rbhost::shared_tc_list(batch, heads, kv_heads) : l;
  // parts of a row over shared tokens, if these are long: about four for a warp
  const int tiles_of = (batch + p.prefix.seqs - 1) / p.prefix.seqs, entries = groups > tiles_of ? groups : tiles_of;
  const long long parts = p.prefix.ctas / (static_cast<long long>(entries) * p.prefix.virtual_heads) * (p.tc ? 2 : 1);
  p.share = parts >= 24 ? 8 : parts >= 12 ? 4 : parts >= 6 ? 2 : 1;
  return p;
}
// Puts a list's arrays at `at` (NULL: only counts) and returns their size.
long long place(rb::SpList& l, char* at, int head_dim) {
  const long long totals = ((l.entries + 1) * 4ll + 15) / 16 * 16, rows = l.rows * (l.half > 0 ? 2 : 1), ml = (rows * 8 + 15) / 16 * 16;
  if (at) {
    l.totals = reinterpret_cast<int*>(at);
    l.ml = reinterpret_cast<float2*>(at + totals);
    l.acc = reinterpret_cast<float*>(at + totals + ml);
  }
  return totals + ml + rows * head_dim * 4;
}
bool sound(int batch, int heads, int kv_heads, int head_dim, int block_size) {
  return batch >= 0 && batch <= 4096 && kv_heads >= 1 && kv_heads <= 65535 && heads >= kv_heads && heads % kv_heads == 0 && (head_dim == 64 || head_dim == 128) &&
         block_size >= 1;
}

template <typename T, int D, int MT>
cudaError_t split(const rb::SpParams& p, const Plan& l, cudaStream_t s) {
  static size_t configured[64] = {0};
  const int dev = rbhost::device_slot();
  if (configured[dev] < l.smem) {
    const cudaError_t e = cudaFuncSetAttribute(rb::shared_split_kernel<T, D, MT>, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(l.smem));
    if (e != cudaSuccess) return e;
    configured[dev] = l.smem;
  }
  return rbhost::launch_pdl(rb::shared_split_kernel<T, D, MT>, dim3(l.list.ctas), dim3(rb::kSpWarps * 32), l.smem, s, 1, p RB_BOUNDS_ARG);
}
// The sequences' own tokens, the shared ones where they have a kernel of their own, and the join.  Neither of the first two reads what the other writes: the second begins as the first
// one's CTAs leave the SMs.
template <typename T, int D>
int launch(const rb::SpParams& p, const Plan& l, int type, cudaStream_t s) {
  cudaError_t e = l.tiles == 1 ? split<T, D, 1>(p, l, s) : split<T, D, 2>(p, l, s);
  if (e != cudaSuccess) return static_cast<int>(e);
  if (l.tc) {
    const int code = rbhost::shared_tc(p, type, D, s);
    if (code) return code;
  }
  const int rows = rb::kSpJoinWarps / l.share, group = p.heads / p.kv_heads;
  return static_cast<int>(rbhost::launch_pdl(rb::shared_join_kernel<T, D>, dim3(p.batch, p.kv_heads, (group + rows - 1) / rows), dim3(rb::kSpJoinWarps * 32), 0, s, 1, p, l.share));
}

}  // namespace

RB_API long long rb_shared_prefix_scratch_bytes(int batch, int groups, int heads, int kv_heads, int head_dim, int block_size, int most_rows) {
  if (!sound(batch, heads, kv_heads, head_dim, block_size) || batch == 0) return 16;
  long long most = 0;
  for (int positive = 0; positive < 2; ++positive) {
    Plan l = plan_of(batch, groups, heads, kv_heads, head_dim, block_size, most_rows, positive != 0);
    const long long n = place(l.list, nullptr, head_dim) + (l.tc ? place(l.prefix, nullptr, head_dim) : 0);
    if (n > most) most = n;
  }
  return most;
}

RB_API int rb_shared_prefix(const RbSharedPrefixArgs* a, void* stream) {
  if (!a || !sound(a->batch, a->heads, a->kv_heads, a->head_dim, a->block_size)) return -1;
  if (a->batch == 0) return 0;
  if (!a->q || !a->out || !a->k_cache || !a->v_cache || !a->block_tables || !a->context_lens || !a->shared_lens || !a->group_of || !a->span_of || reinterpret_cast<unsigned long long>(a->span_of) % 8 || !a->scratch ||
      a->groups < 1 || a->groups > a->batch || a->max_blocks < 1 || a->num_blocks < 1 || a->type < 0 || a->type > 1 || a->most_rows < 1 || a->most_rows > a->batch)
    return -1;
  if ((reinterpret_cast<unsigned long long>(a->q) | reinterpret_cast<unsigned long long>(a->out) | reinterpret_cast<unsigned long long>(a->k_cache) |
       reinterpret_cast<unsigned long long>(a->v_cache)) & 15 || a->ld_q % 8 || a->ld_o % 8)
    return -2;
  Plan l = plan_of(a->batch, a->groups, a->heads, a->kv_heads, a->head_dim, a->block_size, a->most_rows, a->scale > 0.f);
  const long long cap = static_cast<long long>(a->max_blocks) * a->block_size;
  if (a->num_blocks * a->block_size > 0x7fffffffll || cap > (1ll << 30) ||
      2ll * a->batch * ((cap + rb::kSpUnit - 1) / rb::kSpUnit) * l.list.virtual_heads > 0x7fffffffll || l.smem > 227 * 1024)
    return -3;
  rb::SpParams p;
  memset(&p, 0, sizeof(p));
  p.q = a->q; p.out = a->out; p.k = a->k_cache; p.v = a->v_cache;
  p.tables = a->block_tables; p.lens = a->context_lens; p.shared = a->shared_lens; p.group_of = a->group_of;
  p.span_of = reinterpret_cast<const int2*>(a->span_of);
  p.ld_q = a->ld_q; p.ld_o = a->ld_o; p.num_blocks = a->num_blocks;
  p.batch = a->batch; p.groups = a->groups; p.width = a->max_blocks; p.block_size = a->block_size; p.heads = a->heads; p.kv_heads = a->kv_heads;
  p.cap = static_cast<int>(cap); p.scale = a->scale;
  char* at = static_cast<char*>(a->scratch);
  at += place(l.list, at, a->head_dim);
  if (l.tc) place(l.prefix, at, a->head_dim);
  else l.prefix = l.list;
  p.list = l.list;
  p.prefix = l.prefix;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  int e;
  if (a->type == 0) e = a->head_dim == 64 ? launch<__nv_bfloat16, 64>(p, l, 0, s) : launch<__nv_bfloat16, 128>(p, l, 0, s);
  else e = a->head_dim == 64 ? launch<__half, 64>(p, l, 1, s) : launch<__half, 128>(p, l, 1, s);
  return e;
}
