// What the kernels of decode attention over a shared prefix have in common: the list of units, its division among CTAs, and the places of partial
// results (shared_prefix.cu, shared_prefix_tc.cu).
#pragma once
#include <cuda_fp16.h>
#include <limits.h>

#include "pdl.cuh"
#include "warp_mma.cuh"

namespace rb {

#ifdef RB_BOUNDS
#define RB_BOUNDS_PASS , rb_bounds_status
#else
#define RB_BOUNDS_PASS
#endif

constexpr int kSpUnit = 128;                     // tokens
constexpr float kSpLog2e = 1.4426950408889634f;

// Entries and their units.  A list has the tiles of rows over shared tokens (tiles: entry b is the tile that begins with sequence b, if one does), the sequences' own tokens
// (own: one entry a sequence), or both, tiles first.  The units of all entries, for each of the virtual KV heads one after the other, are dealt in equal runs, `ctas` at most, to CTAs or parts of them.
struct SpList {
  int* totals;                                   // [entries + 2] running totals of units, then the number of runs
  float2* ml;                                    // maximum (base 2) and sum of every row's part
  float* acc;                                    // [part][head_dim]
  int entries, own;                              // own: the first entry of a sequence's own tokens
  int per, parts, virtual_heads;                 // a KV head's query heads in `parts` equal parts of `per`, so that a sequence's rows fit a tile
  int ctas, seqs;                                // seqs: sequences of a tile
  int log_grain;                                 // an entry's own tokens begin at a multiple of this power of two, the last not behind the first that no other has
  int half;                                      // > 0: parts of entries of at most so many sequences come in twos, the second `rows` behind the first
  long long rows;                                // of parts
};
struct SpParams {
  const void* q;
  void* out;
  const void* k;
  const void* v;
  const int* tables;
  const int* lens;
  const int* shared;
  const int* group_of;                           // [batch]
  const int2* span_of;                           // [batch] first sequence of the sequence's group and of the next
  long long ld_q, ld_o, num_blocks;
  int batch, groups, width, block_size, heads, kv_heads;
  int log_block;                                 // of the block size, -1: no power of two
  int cap;                                       // tokens of a table's row
  float scale;
  SpList list, prefix;                           // prefix: where the parts over shared tokens are; the same list, or that of the launch in front
};

__device__ __forceinline__ int sp_length(const SpParams& p, int b) { return min(max(p.lens[b], 0), p.cap); }
// What a CTA's shared memory holds of a list: running totals of the entries' units, and of every entry its tokens, the tokens that its group shares and the first sequences of its group
// and of the next.
struct SpHeld {
  int* totals;                                   // [entries + 1]
  int* count;                                    // [entries]
  int* shared;                                   // [entries]
  uint32_t* span;                                // [entries]: two numbers of 16 bits
  int* least;                                    // [groups], while the list is formed
};
__host__ __device__ constexpr size_t sp_held_bytes(int entries, int groups) { return (4 * static_cast<size_t>(entries) + 1 + groups) * 4; }
__device__ __forceinline__ SpHeld sp_held(const SpList& l, int* at) {
  const int n = l.entries;
  return {at, at + n + 1, at + 2 * n + 1, reinterpret_cast<uint32_t*>(at + 3 * n + 1), at + 4 * n + 1};
}
// Forms them, all threads of a CTA.  `totals`: of p.prefix, where that is a list of tiles beside p.list of as many sequences; then `work` gets the sum of its units, those of two tiles of rows
// times `two`, else times `one`.
//
// What a group's sequences read together are no more tokens than the shortest of them has, those without tokens aside, so that all rows of a tile see all of its tokens.  Tiles of rows
// begin at every `seqs`-th sequence of a group.  The loads of the first sequences of a thread go out together: the chain of latencies is what this costs.
__device__ __forceinline__ void sp_prepare(const SpParams& p, const SpHeld& held, int* warp_sums, int* totals = nullptr, unsigned long long* work = nullptr, int one = 0, int two = 0) {
  const SpList& l = p.list;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  int* least = held.least;
  const int b0 = min(static_cast<int>(threadIdx.x), p.batch - 1), g0 = min(static_cast<int>(threadIdx.x), p.groups - 1);
  const int length0 = sp_length(p, b0), group0 = p.group_of[b0], said0 = p.shared[g0];
  const int2 span0 = p.span_of[b0];
  for (int g = threadIdx.x; g < p.groups; g += blockDim.x) least[g] = INT_MAX;
  if (threadIdx.x == 0) {
    held.totals[0] = 0;
    if (totals) {
      totals[0] = 0;
      *work = 0;
    }
  }
  __syncthreads();
  for (int b = threadIdx.x; b < p.batch; b += blockDim.x) {
    const bool first = b == static_cast<int>(threadIdx.x);
    const int n = first ? length0 : sp_length(p, b);
    if (n > 0) atomicMin(&least[first ? group0 : p.group_of[b]], n);
  }
  __syncthreads();
  for (int g = threadIdx.x; g < p.groups; g += blockDim.x) {
    const int n = least[g];
    least[g] = n == INT_MAX ? 0 : min(n, max(g == static_cast<int>(threadIdx.x) ? said0 : p.shared[g], 0));
  }
  __syncthreads();
  // running totals of the units that `units` says of an entry
  auto sum = [&](int entries, int* to, auto units) {
    int before = 0;
    for (int e0 = 0; e0 < entries; e0 += blockDim.x) {
      const int e = e0 + threadIdx.x;
      int upto = e < entries ? units(e) : 0;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += v;
      }
      if (lane == 31) warp_sums[warp] = upto;
      __syncthreads();
      int all = 0;
      for (int w = 0; w < warps; ++w) {
        const int s = warp_sums[w];
        if (w < warp) upto += s;
        all += s;
      }
      if (e < entries) to[e + 1] = before + upto;
      before += all;
      __syncthreads();
    }
  };
  sum(l.entries, held.totals, [&](int e) {
    const bool own = e >= l.own;
    const int b = own ? e - l.own : e;
    const bool first = b == static_cast<int>(threadIdx.x);
    const int shared = least[first ? group0 : p.group_of[b]];
    const int2 span = first ? span0 : p.span_of[b];
    held.shared[e] = shared;
    held.span[e] = static_cast<uint32_t>(span.x) | static_cast<uint32_t>(span.y) << 16;
    const int mine = (first ? length0 : sp_length(p, b)) - shared;
    const int count = own ? (mine > 0 ? mine + (shared & ((1 << l.log_grain) - 1)) : 0) : (b - span.x) % l.seqs == 0 ? shared : 0;
    held.count[e] = count;
    return (count + kSpUnit - 1) / kSpUnit;
  });
  if (totals)
    sum(p.batch, totals, [&](int b) {            // this thread wrote what it reads
      const int from = static_cast<int>(held.span[b] & 0xffffu), upto = static_cast<int>(held.span[b] >> 16);
      const int units = (b - from) % p.prefix.seqs == 0 ? (held.shared[b] + kSpUnit - 1) / kSpUnit : 0;
      if (units) atomicAdd(work, static_cast<unsigned long long>(units) * (upto - b > p.prefix.half ? two : one));
      return units;
    });
}
// A list's running totals and the number of its runs, for the join.
__device__ __forceinline__ void sp_keep_totals(const SpList& l, const int* totals, int runs) {
  for (int i = threadIdx.x; i <= l.entries; i += blockDim.x) l.totals[i] = totals[i];
  if (threadIdx.x == 0) l.totals[l.entries + 1] = runs;
}
// First unit of CTA c's run, and the CTA that has unit u.
__device__ __forceinline__ int sp_run(int total, int ctas, int c) {
  const int share = total / ctas, over = total - share * ctas;
  return c * share + min(c, over);
}
__device__ __forceinline__ int sp_cta_of(int total, int ctas, int u) {
  const int share = total / ctas, over = total - share * ctas, wide = over * (share + 1);
  return u < wide ? u / (share + 1) : over + (u - wide) / share;
}
// A part of an entry: units u0 .. u1 - 1 of it, for one virtual KV head.
struct SpPart {
  int vh, e, u0, u1;
  int b, n;                                      // first sequence, sequences of the tile
  int shared;                                    // tokens that the group shares
  const int* table;
  bool own;
};
// The part that a run u .. u_end begins with; u goes behind it.  Every thread that calls it gets the same.
__device__ __forceinline__ SpPart sp_next(const SpParams& p, const SpList& l, const SpHeld& held, int& u, int u_end) {
  SpPart s;
  const int all = held.totals[l.entries];
  s.vh = u / all;
  const int at = u - s.vh * all;
  int e = 0;
  for (int hi = l.entries; hi - e > 1;) {        // the last entry that begins at or in front of the unit
    const int mid = (e + hi) >> 1;
    if (held.totals[mid] <= at) e = mid;
    else hi = mid;
  }
  s.e = e;
  s.u0 = at - held.totals[e];
  s.u1 = min(held.totals[e + 1], at + u_end - u) - held.totals[e];
  s.own = e >= l.own;
  s.b = s.own ? e - l.own : e;
  s.shared = held.shared[e];
  const uint32_t span = held.span[e];
  s.n = s.own ? 1 : min(l.seqs, static_cast<int>(span >> 16) - s.b);
  s.table = p.tables + static_cast<long long>(s.own ? s.b : static_cast<int>(span & 0xffffu)) * p.width;
  u += s.u1 - s.u0;
  return s;
}
// Where a part's row 0 goes, rows (sequence, head) one behind the other.  A part that begins its entry has places of the entry's own; one that goes on with it is the
// first of its CTA's run and has the CTA's.
__device__ __forceinline__ long long sp_row(const SpList& l, int vh, int e, int cta, bool begins) {
  const long long heads = static_cast<long long>(l.entries) * l.per;
  return begins ? vh * heads + static_cast<long long>(e) * l.per : l.virtual_heads * heads + static_cast<long long>(cta) * l.seqs * l.per;
}

template <typename T>
__device__ __forceinline__ uint32_t sp_pack(float lo, float hi);
template <>
__device__ __forceinline__ uint32_t sp_pack<__nv_bfloat16>(float lo, float hi) { return pack_bf16x2(lo, hi); }
template <>
__device__ __forceinline__ uint32_t sp_pack<__half>(float lo, float hi) {
  __half2 v = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<uint32_t*>(&v);
}

}  // namespace rb

namespace rbhost {
// Rows of partial results of a list.
inline long long sp_list_rows(const rb::SpList& l) {
  return static_cast<long long>(l.virtual_heads) * l.entries * l.per + static_cast<long long>(l.ctas) * l.seqs * l.per;
}
// shared_prefix_tc.cu: the parts over shared tokens with tcgen05
bool shared_tc_takes(int batch, int heads, int kv_heads, int block_size, int most);
rb::SpList shared_tc_list(int batch, int heads, int kv_heads);
int shared_tc_runs();                            // of the sequences' own tokens, at most
int shared_tc(const rb::SpParams& p, int type, int head_dim, cudaStream_t stream);
}  // namespace rbhost
