// Decode attention for sequences that share their first tokens (beams and samples of one prompt, requests behind one system prompt).
//
// Alone, every sequence of a group reads the shared keys and values again: n sequences, n times the bytes.  Here the queries of all of a group's
// sequences for one KV head are the rows of one product over the shared tokens, which are read once; each sequence's own tokens follow as in any decode
// attention, and a last launch joins the parts of a row by their maxima and sums:
//     out = sum_i 2^(m_i - M) acc_i / sum_i 2^(m_i - M) l_i,   M = max_i m_i.
//
// Work is a list of entries (a tile of a group's rows over its shared tokens, a sequence's rows over its own), cut into units of 128 tokens; the units of all entries, one behind the other, are
// dealt in equal runs.  An entry's rows are accumulated over all units of a run, so there are at most (entries + runs) parts: the one that begins an entry has a place of the entry's
// own, one that goes on with it is the first of its run and has the run's.  Every CTA forms the list of running totals itself from the lengths: the host knows none, and a captured
// graph may be replayed with others.
//
// Up to 16 rows of a group, one list and one kernel (here) that is bound by its launch or by the reads: 4 beams over 300 tokens, 12 KV heads of 64, 11 us with the join; 4 over 4000,
// 8 KV heads of 128, 18 us.  More rows, two lists in one launch (shared_prefix_tc.cu).
#include "shared_prefix.h"

#include <string.h>

#include "shared_prefix_split.cuh"

namespace rb {

template <typename T, int D, int MT>
__global__ void __launch_bounds__(kSpWarps * 32, MT == 1 ? 3 : 2)
shared_split_kernel(const SpParams p RB_BOUNDS_PARAM) {
  pdl_wait();
  pdl_launch();
  extern __shared__ __align__(128) uint8_t sp_mem[];
  __shared__ int warp_sums[kSpWarps];
  const SpHeld held = sp_held(p.list, reinterpret_cast<int*>(sp_mem + SpSmem<D, MT>::kHeld));
  sp_prepare(p, held, warp_sums);
  if (blockIdx.x == 0) sp_keep_totals(p.list, held.totals, p.list.ctas);
  sp_split<T, D, MT, false>(p, p.list, held, sp_mem, blockIdx.x, p.list.ctas, threadIdx.x, 0, SpTma() RB_BOUNDS_PASS);
}

// out[b, head] from the parts of its row.  A CTA has some heads of a sequence and KV head; a row's parts are summed by `share` warps, and
// lanes own D / 32 neighbouring columns.  Grid (batch, KV heads, parts of a KV head's query heads).
constexpr int kSpJoinWarps = 8;
template <typename T, int D>
__global__ void __launch_bounds__(kSpJoinWarps * 32)
shared_join_kernel(const SpParams p, const int log_share) {
  constexpr int C = D / 32;
  const int share = 1 << log_share;
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
  const int all = look.totals[look.entries], runs = look.totals[look.entries + 1], t0 = look.totals[lane & 2 ? look.own + b : tile], t1 = look.totals[(lane & 2 ? look.own + b : tile) + 1];
  {
    const int h = (blockIdx.z * (blockDim.x >> 5) + warp) >> log_share, which = warp & (share - 1);
    const bool mine = h < group;
    float mx = -INFINITY, den = 0.f, acc[C];
#pragma unroll
    for (int c = 0; c < C; ++c) acc[c] = 0.f;
    if (mine && any) {
      // parts over shared tokens, then the sequence's own: how many CTAs, the first, and the rows where its part and those of CTA 0 are
      const int k_look = look.parts == 1 ? 0 : h / look.per, u = (hk * look.parts + k_look) * all + (lane & 1 ? t1 - 1 : t0);
      const int cta = t1 > t0 ? sp_cta_of(all * look.virtual_heads, runs, u) : lane & 1 ? -1 : 0;
      int n[2], c0[2];
      long long row[2], later[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const SpList& l = i == 0 ? p.prefix : p.list;
        const int e = i == 0 ? tile : l.own + b, k = l.parts == 1 ? 0 : h / l.per, vh = hk * l.parts + k, r = (i == 0 ? b - tile : 0) * l.per + h - k * l.per;
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
        const int m = min(32, (parts - s0 + share - 1) >> log_share);
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
  int log_share;                                 // 2^log_share warps of a row of the join
  bool tc;
};
// Groups with more than 16 rows go to the tcgen05 kernel, which takes 256 at a time where pages, batch and scale allow
// (256 sequences with 4 rows each for 8 KV heads over 16384 shared tokens took 456 us with tiles of 32 rows on mma.sync, 124 now); else this file's has one m-tile, or two where rows need them.
Plan plan_of(int batch, int groups, int heads, int kv_heads, int head_dim, int block_size, int most, bool positive) {
  Plan p;
  memset(&p, 0, sizeof(p));
  const int group = heads / kv_heads;
  p.tc = static_cast<long long>(most) * group > 16 && positive && rbhost::shared_tc_takes(batch, heads, kv_heads, block_size, most);
  p.tiles = !p.tc && static_cast<long long>(most) * group > 16 ? 2 : 1;
  const int rows = 16 * p.tiles;
  rb::SpList& l = p.list;
  l.parts = (group + rows - 1) / rows;
  l.per = (group + l.parts - 1) / l.parts;
  l.parts = (group + l.per - 1) / l.per;
  l.seqs = rows / l.per;
  for (l.log_grain = 0; p.tc && l.log_grain < 5 && (block_size >> l.log_grain & 1) == 0;) ++l.log_grain;
  l.virtual_heads = kv_heads * l.parts;
  l.own = p.tc ? 0 : batch;
  l.entries = l.own + batch;
  const size_t tiles = head_dim == 64 ? (p.tiles == 1 ? rb::SpSmem<64, 1>::kHeld : rb::SpSmem<64, 2>::kHeld)
                                      : (p.tiles == 1 ? rb::SpSmem<128, 1>::kHeld : rb::SpSmem<128, 2>::kHeld);
  p.smem = tiles + rb::sp_held_bytes(l.entries, groups);
  const int resident = static_cast<int>((228 * 1024) / (p.smem + 1024 + 64)), most_resident = p.tiles == 1 ? 3 : 2;
  l.ctas = p.tc ? rbhost::shared_tc_runs() : rbhost::device_sm_count() * (resident < 1 ? 1 : resident < most_resident ? resident : most_resident);
  l.rows = rbhost::sp_list_rows(l);
  p.prefix = p.tc ? rbhost::shared_tc_list(batch, heads, kv_heads) : l;
  // parts of a row over shared tokens, if these are long: up to about five for a warp, which looks every row's up first
  const int tiles_of = (batch + p.prefix.seqs - 1) / p.prefix.seqs, entries = groups > tiles_of ? groups : tiles_of;
  const long long parts = p.prefix.ctas / (static_cast<long long>(entries) * p.prefix.virtual_heads) * (p.prefix.half > 0 && most <= p.prefix.half ? 2 : 1);
  p.log_share = parts >= 24 ? 3 : parts >= 12 ? 2 : parts >= 6 ? 1 : 0;
  return p;
}
// Puts a list's arrays at `at` (NULL: only counts) and returns their size.
long long place(rb::SpList& l, char* at, int head_dim) {
  const long long totals = ((l.entries + 2) * 4ll + 15) / 16 * 16, rows = l.rows * (l.half > 0 ? 2 : 1), ml = (rows * 8 + 15) / 16 * 16;
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
// All tokens, then the join.
template <typename T, int D>
int launch(const rb::SpParams& p, const Plan& l, int type, cudaStream_t s) {
  const int code = l.tc ? rbhost::shared_tc(p, type, D, s) : static_cast<int>(l.tiles == 1 ? split<T, D, 1>(p, l, s) : split<T, D, 2>(p, l, s));
  if (code) return code;
  const int group = p.heads / p.kv_heads, warps = (group << l.log_share) < rb::kSpJoinWarps ? group << l.log_share : rb::kSpJoinWarps, rows = warps >> l.log_share;
  return static_cast<int>(rbhost::launch_pdl(rb::shared_join_kernel<T, D>, dim3(p.batch, p.kv_heads, (group + rows - 1) / rows), dim3(warps * 32), 0, s, 1, p, l.log_share));
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
  p.log_block = -1;
  for (int i = 0; i < 31; ++i)
    if (a->block_size == 1 << i) p.log_block = i;
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
