// Eviction from a paged cache in e4m3: which tokens of a sequence stay, by their attention weight, and their move to the front.
#include <cooperative_groups.h>

#include "pdl.cuh"
#include "paged_e4m3.cuh"

namespace rb {

namespace cg = cooperative_groups;

constexpr int kE4SelectThreads = 1024, kE4SelectWarps = kE4SelectThreads / 32;
constexpr int kE4SelectKeys = 16384;                 // keys that a CTA holds

// order-preserving: larger weights have larger keys, -0 is 0, a NaN is largest
__device__ __forceinline__ uint32_t e4_key(float w) {
  if (!(w == w)) return 0xffffffffu;
  const uint32_t u = __float_as_uint(w + 0.f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// The places that stay, for a sequence and KV head.  The `take`-th largest key of the tokens that may go is found by radix selection over keys in shared
// memory, 11 bits a pass: every pass counts the next digit of the keys that still may be it, until all that are left stay.  The digits are those of a
// key's distance from the least one: weights have few exponents, and threads that count the same digit wait for one another.  Then each warp counts what
// stays of its tokens, and writes it where the counts in front of it end.  Sequences of more than 16384 tokens are shared by the CTAs of a cluster (x: rank
// in the cluster), which add their counts through distributed shared memory; of more than 131072, the keys are read from the pages again in every pass.
// Bound by latencies: table, weight and the passes' barriers follow one another, and a warp goes through its keys.  24 sequences of 1500 to 8192, 8 KV heads,
// one B200: with digits of the keys themselves 25 us, of distances 23.5, with 1024 threads in place of 512 20.8.
template <bool CLUSTER>
__global__ void __launch_bounds__(kE4SelectThreads, 2)
e4_select_kernel(const RbE4m3EvictArgs a RB_BOUNDS_PARAM) {
  pdl_wait();
  pdl_launch();
  extern __shared__ uint32_t e4_keys[];
  __shared__ uint32_t hist[2048], part[2], ends[2], digit[3];
  __shared__ uint32_t warp_n[2][kE4SelectWarps];
  __shared__ uint32_t warp_end[2][kE4SelectWarps];   // not warp_n: where all keys are equal, no barrier lies between its reads and the counts' writes
  const int ranks = CLUSTER ? gridDim.x : 1, rank = CLUSTER ? blockIdx.x : 0;
  const int h = blockIdx.y, b = blockIdx.z, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int bs = a.pages.block_size, G = a.pages.kv_heads, per_page = bs >> 4;
  const int n = static_cast<int>(max(0ll, min(static_cast<long long>(a.context_lens[b]), static_cast<long long>(a.max_blocks) * bs)));
  int* kept = a.kept + (static_cast<long long>(b) * G + h) * a.keep;
  if (h == 0 && rank == 0 && tid == 0) a.lens_out[b] = min(n, a.keep);
  if (n <= a.keep) {                                 // all CTAs of a cluster alike
    for (int j = rank * kE4SelectThreads + tid; j < a.keep; j += ranks * kE4SelectThreads) kept[j] = j < n ? j : -1;
    return;
  }
  const uint32_t take = a.keep - a.keep_first - a.recent;
  for (int j = rank * kE4SelectThreads + tid; j < a.keep_first; j += ranks * kE4SelectThreads) kept[j] = j;
  for (int j = rank * kE4SelectThreads + tid; j < a.recent; j += ranks * kE4SelectThreads) kept[a.keep - a.recent + j] = n - a.recent + j;
  if (take == 0) return;
  // this CTA's tokens among those that may go, `mine` from `lo` on, of which a warp has `span` one behind the other
  const int first = a.keep_first, count = n - a.recent - first, share = (count + ranks - 1) / ranks;
  const int lo = first + min(count, rank * share), mine = first + min(count, (rank + 1) * share) - lo;
  const int span = (mine + kE4SelectThreads - 1) / kE4SelectThreads * 32, w0 = warp * span, w1 = min(mine, w0 + span);
  const int* table = a.block_tables + static_cast<long long>(b) * a.max_blocks;
  auto page_of = [&](int t) { return table[per_page == 1 ? t >> 4 : t / bs]; };
  const float* weights = a.pages.weight + static_cast<long long>(h) * bs;
  const unsigned int blocks = static_cast<unsigned int>(a.pages.num_blocks);
  const long long per_block = static_cast<long long>(G) * bs;
  auto key_of = [&](int t, int page) {
    const bool there = static_cast<unsigned int>(page) < blocks;
    if (!there) RB_BOUNDS_HIT(104);
    const float w = weights[(there ? page : 0) * per_block + (per_page == 1 ? t & 15 : t % bs)];
    return there ? e4_key(w) : 0u;
  };
  const bool held = mine <= kE4SelectKeys;
  uint32_t least = 0xffffffffu, most = 0;            // keys
  if (held)
    for (int i0 = tid; i0 < mine; i0 += 4 * kE4SelectThreads) {         // four pages, then four weights: loads that do not wait for one another
      int page[4];
      uint32_t k[4];
#pragma unroll
      for (int x = 0; x < 4; ++x) page[x] = page_of(lo + min(i0 + x * kE4SelectThreads, mine - 1));
#pragma unroll
      for (int x = 0; x < 4; ++x) k[x] = key_of(lo + min(i0 + x * kE4SelectThreads, mine - 1), page[x]);
#pragma unroll
      for (int x = 0; x < 4; ++x)
        if (i0 + x * kE4SelectThreads < mine) e4_keys[i0 + x * kE4SelectThreads] = k[x];
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        least = min(least, k[x]);
        most = max(most, k[x]);
      }
    }
  // f(place, key) for this warp's tokens, 32 at a time; a lane without a token has place -1
  auto each = [&](auto f) {
    if (held) {
#pragma unroll 4
      for (int i = w0 + lane; i - lane < w1; i += 32) f(i < w1 ? lo + i : -1, i < w1 ? e4_keys[i] : 0u);
    } else {
#pragma unroll 4
      for (int i = w0 + lane; i - lane < w1; i += 32) f(i < w1 ? lo + i : -1, i < w1 ? key_of(lo + i, page_of(lo + i)) : 0u);
    }
  };
  if (!held)
    each([&](int t, uint32_t k) {
      if (t >= 0) {
        least = min(least, k);
        most = max(most, k);
      }
    });
  least = __reduce_min_sync(0xffffffffu, least);
  most = __reduce_max_sync(0xffffffffu, most);
  if (lane == 0) {
    warp_end[0][warp] = least;
    warp_end[1][warp] = most;
  }
  __syncthreads();
  least = __reduce_min_sync(0xffffffffu, warp_end[0][lane % kE4SelectWarps]);
  most = __reduce_max_sync(0xffffffffu, warp_end[1][lane % kE4SelectWarps]);
  if (CLUSTER) {
    if (tid == 0) {
      ends[0] = least;
      ends[1] = most;
    }
    cg::this_cluster().sync();
    for (int r = 1; r < ranks; ++r) {
      least = min(least, *cg::this_cluster().map_shared_rank(&ends[0], (rank + r) % ranks));
      most = max(most, *cg::this_cluster().map_shared_rank(&ends[1], (rank + r) % ranks));
    }
  }
  // bits from `shift` on of the distances from the least key: those above `prefix` stay, and `need` of those equal to it
  uint32_t prefix = 0, need = take;
  int shift = most > least ? 32 - __clz(most - least) : 0;
#pragma unroll 1
  while (shift > 0) {
    const int known = shift, width = min(shift, 11);
    shift -= width;
    constexpr int kBins = 2048 / kE4SelectThreads;   // of a thread
#pragma unroll
    for (int j = 0; j < kBins; ++j) hist[tid + j * kE4SelectThreads] = 0;
    __syncthreads();
    each([&](int t, uint32_t k) {
      const uint32_t d = k - least;
      if (t >= 0 && (d >> (known - 1) >> 1) == prefix) atomicAdd(&hist[(d >> shift) & ((1u << width) - 1)], 1u);
    });
    if (CLUSTER) cg::this_cluster().sync();
    else __syncthreads();
    uint32_t c[kBins], sum = 0;                      // digits 2047 - kBins * tid downwards
#pragma unroll
    for (int j = 0; j < kBins; ++j) {
      uint32_t* bin = &hist[2047 - tid * kBins - j];
      c[j] = *bin;
      if (CLUSTER)
        for (int r = 1; r < ranks; ++r) c[j] += *cg::this_cluster().map_shared_rank(bin, (rank + r) % ranks);
      sum += c[j];
    }
    uint32_t upto = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t v = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += v;
    }
    if (lane == 31) warp_n[0][warp] = upto;
    __syncthreads();
    uint32_t above = upto - sum + __reduce_add_sync(0xffffffffu, lane < warp ? warp_n[0][lane] : 0u);
    if (above < need && need <= above + sum) {       // one thread
#pragma unroll
      for (int j = 0; j < kBins; ++j) {
        if (above < need && need <= above + c[j]) {
          digit[0] = 2047 - tid * kBins - j;
          digit[1] = need - above;
          digit[2] = c[j];
        }
        above += c[j];
      }
    }
    if (CLUSTER) cg::this_cluster().sync();          // and nobody reads another's counts any more
    else __syncthreads();
    prefix = prefix << width | digit[0];
    need = digit[1];
    if (need == digit[2]) break;                     // all that are equal stay
  }
  // of the equal ones, the first `need` stay
  uint32_t above = 0, equal = 0;                     // of this warp
  each([&](int t, uint32_t k) {
    const uint32_t d = (k - least) >> shift;
    above += t >= 0 && d > prefix ? 1 : 0;
    equal += t >= 0 && d == prefix ? 1 : 0;
  });
  above = __reduce_add_sync(0xffffffffu, above);
  equal = __reduce_add_sync(0xffffffffu, equal);
  if (lane == 0) {
    warp_n[0][warp] = above;
    warp_n[1][warp] = equal;
  }
  __syncthreads();
  uint32_t before[2];                                // keys above and equal in the warps in front
#pragma unroll
  for (int x = 0; x < 2; ++x) {
    const uint32_t v = lane < kE4SelectWarps ? warp_n[x][lane] : 0u, all = __reduce_add_sync(0xffffffffu, v);
    before[x] = __reduce_add_sync(0xffffffffu, lane < warp ? v : 0u);
    if (CLUSTER && tid == 0) part[x] = all;
  }
  if (CLUSTER) {
    cg::this_cluster().sync();
    for (int r = 0; r < rank; ++r) {
      before[0] += *cg::this_cluster().map_shared_rank(&part[0], r);
      before[1] += *cg::this_cluster().map_shared_rank(&part[1], r);
    }
  }
  each([&](int t, uint32_t k) {
    const uint32_t d = (k - least) >> shift, gt = __ballot_sync(0xffffffffu, t >= 0 && d > prefix), eq = __ballot_sync(0xffffffffu, t >= 0 && d == prefix);
    const uint32_t in_front = (1u << lane) - 1;
    const uint32_t equals = before[1] + __popc(eq & in_front);           // equal ones in front of this token
    const uint32_t at = first + before[0] + __popc(gt & in_front) + min(equals, need);
    if (((gt >> lane) & 1 || ((eq >> lane) & 1 && equals < need)) && at < static_cast<uint32_t>(a.keep)) kept[at] = t;
    before[0] += __popc(gt);
    before[1] += __popc(eq);
  });
  if (CLUSTER) cg::this_cluster().sync();            // others may still read this CTA's counts
}

constexpr int kE4MoveThreads = 256, kE4MoveTokens = 64;

// Moves the kept tokens of a sequence and KV head.  A CTA takes whole pages, as many as have at most 64 tokens (or one that has more, in parts).
// INPLACE: the CTAs of a cluster take neighbouring runs of pages and go on together.  A token moves to a place in front of its own, or stays, so what
// one round writes lies in front of all that later rounds read; within a round all tokens are in registers before the first is written.  Pages of more
// than 64 tokens are taken by one CTA, where the same holds from part to part.  Otherwise the pages are of no other use and the grid has a CTA for
// each run of pages.
template <int D, bool INPLACE>
__global__ void __launch_bounds__(kE4MoveThreads)
e4_move_kernel(const RbE4m3EvictArgs a RB_BOUNDS_PARAM) {
  pdl_wait();
  pdl_launch();
  constexpr int kPieces = D / 16, kRows = kE4MoveThreads / kPieces, kPer = kE4MoveTokens / kRows;     // a thread has kPer pieces of keys and of values
  __shared__ long long row_sh[kE4MoveTokens];        // where a token comes from, in rows of D codes
  __shared__ int exp_sh[2][kE4MoveTokens], top_sh[2][kE4MoveTokens / 16], still_sh;
  const int h = blockIdx.y, b = blockIdx.z, tid = threadIdx.x;
  const int bs = a.pages.block_size, G = a.pages.kv_heads;
  const int n = a.lens_out[b];
  if (INPLACE && a.context_lens[b] <= a.keep) return;                  // a whole cluster
  const int* kept = a.kept + (static_cast<long long>(b) * G + h) * a.keep;
  const int* from = a.block_tables + static_cast<long long>(b) * a.max_blocks;
  const int held = static_cast<int>(max(0ll, min(static_cast<long long>(a.context_lens[b]), static_cast<long long>(a.max_blocks) * bs)));
  // The page that place t lies in.  A place that the sequence does not have counts as the first one, a page that is not there as page 0.
  auto page_of = [&](int& t) {
    if (t < 0 || t >= held) {
      RB_BOUNDS_HIT(104);
      t = 0;
    }
    const int page = from[t / bs];
    if (page >= 0 && page < a.pages.num_blocks) return page;
    RB_BOUNDS_HIT(104);
    return 0;
  };
  const int* to_tables = INPLACE ? a.block_tables : a.out_tables;
  const int to_blocks = INPLACE ? a.max_blocks : a.out_blocks;
  const int run = bs >= kE4MoveTokens ? bs : kE4MoveTokens / bs * bs;  // tokens of a CTA's run of pages
  for (int j0 = blockIdx.x * run; INPLACE ? j0 - static_cast<int>(blockIdx.x) * run < n : j0 < n; j0 += gridDim.x * run) {
    // exponents of the run's pages: the largest of their tokens'
    const int m = min(run, n - j0);                  // not positive: this CTA only keeps its cluster company
    int top_k = -128, top_v = -128;                  // of a page that is taken in parts
    for (int part = 0; part < run; part += kE4MoveTokens) {
      const int here = min(kE4MoveTokens, m - part);
      __syncthreads();
      if (tid < 2 * (kE4MoveTokens / 16)) (&top_sh[0][0])[tid] = -128;
      if (tid == 0) still_sh = 1;
      __syncthreads();
      float w = 0.f;
      if (tid < here) {
        const int j = j0 + part + tid;
        int t = kept[j];
        const long long tile = static_cast<long long>(page_of(t)) * G + h;
        const int ek = a.pages.k_exp[tile], ev = a.pages.v_exp[tile];
        row_sh[tid] = tile * bs + t % bs;
        exp_sh[0][tid] = ek;
        exp_sh[1][tid] = ev;
        w = a.pages.weight[tile * bs + t % bs];
        if (run <= kE4MoveTokens) {
          atomicMax(&top_sh[0][tid / bs], ek);
          atomicMax(&top_sh[1][tid / bs], ev);
        }
        if (t != j) still_sh = 0;
      }
      if (run > kE4MoveTokens && part == 0) {        // a page of many tokens: its exponents first
        for (int i = tid; i < m; i += kE4MoveThreads) {
          int t = kept[j0 + i];
          const long long tile = static_cast<long long>(page_of(t)) * G + h;
          top_k = max(top_k, static_cast<int>(a.pages.k_exp[tile]));
          top_v = max(top_v, static_cast<int>(a.pages.v_exp[tile]));
        }
        top_k = __reduce_max_sync(0xffffffffu, top_k);
        top_v = __reduce_max_sync(0xffffffffu, top_v);
        if ((tid & 31) == 0) {
          atomicMax(&top_sh[0][0], top_k);
          atomicMax(&top_sh[1][0], top_v);
        }
        __syncthreads();
        top_k = top_sh[0][0];
        top_v = top_sh[1][0];
      }
      __syncthreads();
      const bool moves = here > 0 && !(INPLACE && still_sh && run <= kE4MoveTokens);    // tokens that all keep their places stay as they are
      const int piece = tid % kPieces, r0 = tid / kPieces;
      uint4 u[2][kPer];
      if (moves) {
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          const uint8_t* src = reinterpret_cast<const uint8_t*>(x ? a.pages.v : a.pages.k);
#pragma unroll
          for (int i = 0; i < kPer; ++i) {
            const int r = r0 + i * kRows;
            if (r < here) u[x][i] = *reinterpret_cast<const uint4*>(src + row_sh[r] * D + piece * 16);
          }
        }
      }
      // everything of this round is in registers
      if (INPLACE && gridDim.x > 1) cg::this_cluster().sync();
      else if (INPLACE) __syncthreads();
      if (!moves) continue;
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        uint8_t* dst = reinterpret_cast<uint8_t*>(x ? a.pages.v : a.pages.k);
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
          const int r = r0 + i * kRows;
          if (r >= here) continue;
          const int j = j0 + part + r, pi = j / bs;
          const int page = pi < to_blocks ? to_tables[static_cast<long long>(b) * to_blocks + pi] : -1;
          if (page < 0 || page >= a.pages.num_blocks) {
            RB_BOUNDS_HIT(104);
            continue;
          }
          const int top = run > kE4MoveTokens ? (x ? top_v : top_k) : top_sh[x][r / bs];
          const int up = top - exp_sh[x][r];
          uint4 c = u[x][i];
          if (up > 0) c = make_uint4(e4_lower4(c.x, up), e4_lower4(c.y, up), e4_lower4(c.z, up), e4_lower4(c.w, up));
          const long long tile = static_cast<long long>(page) * G + h;
          *reinterpret_cast<uint4*>(dst + (tile * bs + j - pi * bs) * D + piece * 16) = c;
          // the page's exponent with its last token: tokens of a page that is taken in parts are read under the old one until then
          if (piece == 0 && (j - pi * bs == bs - 1 || j == n - 1)) (x ? a.pages.v_exp : a.pages.k_exp)[tile] = static_cast<signed char>(top);
        }
      }
      if (tid < here) {
        const int j = j0 + part + tid, pi = j / bs;
        const int page = pi < to_blocks ? to_tables[static_cast<long long>(b) * to_blocks + pi] : -1;
        if (page >= 0 && page < a.pages.num_blocks) a.pages.weight[(static_cast<long long>(page) * G + h) * bs + j - pi * bs] = w;
      }
    }
  }
}

}  // namespace rb

namespace {
template <int D>
cudaError_t move_tokens(const RbE4m3EvictArgs& a, cudaStream_t s) {
  const int bs = a.pages.block_size, run = bs >= rb::kE4MoveTokens ? bs : rb::kE4MoveTokens / bs * bs;
  if (a.out_tables)
    return rbhost::launch_pdl(rb::e4_move_kernel<D, false>, dim3((a.keep + run - 1) / run, a.pages.kv_heads, a.batch), dim3(rb::kE4MoveThreads), 0, s, 1,
                              a RB_BOUNDS_ARG);
  // as many CTAs for a sequence and head as the GPU has room for, four on an SM
  int cluster = 1;
  while (cluster < 8 && run <= rb::kE4MoveTokens && cluster * run < a.keep &&
         2ll * cluster * a.pages.kv_heads * a.batch <= 4ll * rbhost::device_sm_count())
    cluster *= 2;
  return rbhost::launch_pdl(rb::e4_move_kernel<D, true>, dim3(cluster, a.pages.kv_heads, a.batch), dim3(rb::kE4MoveThreads), 0, s, cluster, a RB_BOUNDS_ARG);
}
}  // namespace

RB_API int rb_e4m3_evict(const RbE4m3EvictArgs* args, void* stream_v) {
  const RbE4m3EvictArgs& a = *args;
  if (a.batch <= 0) return 0;
  if (const int bad = rbhost::e4_check(a.pages)) return bad;
  const long long tokens = static_cast<long long>(a.max_blocks) * a.pages.block_size;   // that a sequence can have
  if (!a.pages.weight || !a.block_tables || !a.context_lens || !a.kept || !a.lens_out || a.max_blocks <= 0 || (a.out_tables && a.out_blocks <= 0) || a.keep <= 0 ||
      a.recent < 0 || a.keep_first < 0 || static_cast<long long>(a.recent) + a.keep_first > a.keep || a.batch > 65535 || a.pages.kv_heads > 65535 ||
      tokens > 0x3fffffff || a.keep > 0x3fffffff)
    return -1;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream_v);
  int cluster = 1;                                   // as many CTAs for a sequence and head as hold its keys
  while (cluster < 8 && static_cast<long long>(cluster) * rb::kE4SelectKeys < tokens) cluster *= 2;
  const long long share = (tokens + cluster - 1) / cluster;
  const size_t smem = static_cast<size_t>(share < rb::kE4SelectKeys ? share : rb::kE4SelectKeys) * 4;
  static bool set[64] = {};
  const int dev = rbhost::device_slot();
  if (!set[dev]) {
    cudaError_t e = cudaFuncSetAttribute(rb::e4_select_kernel<false>, cudaFuncAttributeMaxDynamicSharedMemorySize, rb::kE4SelectKeys * 4);
    if (e == cudaSuccess) e = cudaFuncSetAttribute(rb::e4_select_kernel<true>, cudaFuncAttributeMaxDynamicSharedMemorySize, rb::kE4SelectKeys * 4);
    if (e != cudaSuccess) return static_cast<int>(e);
    set[dev] = true;
  }
  cudaError_t e = rbhost::launch_pdl(cluster > 1 ? rb::e4_select_kernel<true> : rb::e4_select_kernel<false>, dim3(cluster, a.pages.kv_heads, a.batch),
                                     dim3(rb::kE4SelectThreads), smem, s, cluster, a RB_BOUNDS_ARG);
  if (e == cudaSuccess) e = a.pages.head_dim == 64 ? move_tokens<64>(a, s) : move_tokens<128>(a, s);
  return static_cast<int>(e);
}
