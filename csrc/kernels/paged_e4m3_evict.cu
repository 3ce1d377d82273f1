// Eviction from a paged cache in e4m3: which tokens of a sequence stay, by their attention weight, and their move to the front.
#include "pdl.cuh"
#include "paged_e4m3.cuh"

namespace rb {

constexpr int kE4SelectThreads = 1024;

// order-preserving: larger weights have larger keys, -0 is 0, a NaN is largest
__device__ __forceinline__ uint32_t e4_key(float w) {
  if (!(w == w)) return 0xffffffffu;
  const uint32_t u = __float_as_uint(w + 0.f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// A CTA for a sequence and KV head: the `take`-th largest key of the tokens that may go, by radix selection in four passes of eight bits, then
// the places that stay, in order.
__global__ void __launch_bounds__(kE4SelectThreads)
e4_select_kernel(const RbE4m3EvictArgs a RB_BOUNDS_PARAM) {
  pdl_wait();
  pdl_launch();
  __shared__ uint32_t hist[256], warp_n[2][32];
  __shared__ uint32_t s_digit, s_need;
  const int h = blockIdx.x, b = blockIdx.y, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int bs = a.pages.block_size, G = a.pages.kv_heads;
  const int n = static_cast<int>(max(0ll, min(static_cast<long long>(a.context_lens[b]), static_cast<long long>(a.max_blocks) * bs)));
  int* kept = a.kept + (static_cast<long long>(b) * G + h) * a.keep;
  if (h == 0 && tid == 0) a.lens_out[b] = min(n, a.keep);
  if (n <= a.keep) {
    for (int j = tid; j < a.keep; j += kE4SelectThreads) kept[j] = j < n ? j : -1;
    return;
  }
  const int lo = a.keep_first, hi = n - a.recent;    // tokens that may go
  const uint32_t take = a.keep - a.keep_first - a.recent;
  auto key = [&](int t) {
    const int page = e4_page(a.block_tables, a.max_blocks, a.pages.num_blocks, b, t / bs);
    if (page < 0) {
      RB_BOUNDS_HIT(104);
      return 0u;
    }
    return e4_key(a.pages.weight[(static_cast<long long>(page) * G + h) * bs + t % bs]);
  };
  uint32_t prefix = 0, mask = 0, need = take;        // keys that begin with `prefix`; how many of them stay
  for (int shift = 24; shift >= 0 && need > 0; shift -= 8) {
    if (tid < 256) hist[tid] = 0;
    __syncthreads();
    for (int t = lo + tid; t < hi; t += kE4SelectThreads) {
      const uint32_t k = key(t);
      if ((k & mask) == prefix) atomicAdd(&hist[(k >> shift) & 255], 1u);
    }
    __syncthreads();
    if (tid == 0) {
      uint32_t above = 0;
      int d = 255;
      for (; d > 0 && above + hist[d] < need; --d) above += hist[d];
      s_digit = d;
      s_need = need - above;
    }
    __syncthreads();
    prefix |= s_digit << shift;
    mask |= 255u << shift;
    need = s_need;
  }
  // keys above `prefix` stay, and the first `need` of those equal to it
  uint32_t placed = a.keep_first, equal = 0;
  for (int j = tid; j < a.keep_first; j += kE4SelectThreads) kept[j] = j;
  for (int j = tid; j < a.recent; j += kE4SelectThreads) kept[a.keep - a.recent + j] = hi + j;
  if (take > 0)
    for (int t0 = lo; t0 < hi; t0 += kE4SelectThreads) {
      const int t = t0 + tid;
      const uint32_t k = t < hi ? key(t) : 0u;
      const bool is_equal = t < hi && k == prefix;
      const uint32_t eq = __ballot_sync(0xffffffffu, is_equal);
      if (lane == 0) warp_n[0][warp] = __popc(eq);
      __syncthreads();
      uint32_t before = equal + __popc(eq & ((1u << lane) - 1));
      for (int w = 0; w < 32; ++w) {
        if (w < warp) before += warp_n[0][w];
        equal += warp_n[0][w];
      }
      const bool stays = t < hi && (k > prefix || (is_equal && before < need));
      const uint32_t st = __ballot_sync(0xffffffffu, stays);
      if (lane == 0) warp_n[1][warp] = __popc(st);
      __syncthreads();
      uint32_t at = placed + __popc(st & ((1u << lane) - 1));
      for (int w = 0; w < 32; ++w) {
        if (w < warp) at += warp_n[1][w];
        placed += warp_n[1][w];
      }
      if (stays && at < static_cast<uint32_t>(a.keep)) kept[at] = t;
    }
}

// A CTA for a sequence and KV head, page after page: a token moves to a place in front of its own or to its own, so that what later pages take has not
// been written yet.
__global__ void __launch_bounds__(256)
e4_move_kernel(const RbE4m3EvictArgs a RB_BOUNDS_PARAM) {
  pdl_wait();
  pdl_launch();
  __shared__ int src_sh[256];                        // page of each token of a run of a page, and slot in it
  __shared__ short off_sh[256];
  __shared__ int exp_sh[2][256];
  __shared__ int top_sh[2];
  const int h = blockIdx.x, b = blockIdx.y, tid = threadIdx.x;
  const int bs = a.pages.block_size, G = a.pages.kv_heads, D = a.pages.head_dim;
  const int n = a.lens_out[b];
  const int* kept = a.kept + (static_cast<long long>(b) * G + h) * a.keep;
  if (!a.out_tables && static_cast<long long>(a.context_lens[b]) <= a.keep) return;
  const int* to_tables = a.out_tables ? a.out_tables : a.block_tables;
  const int to_blocks = a.out_tables ? a.out_blocks : a.max_blocks;
  for (int j0 = 0; j0 < n; j0 += bs) {
    const int m = min(bs, n - j0);
    const int to = e4_page(to_tables, to_blocks, a.pages.num_blocks, b, j0 / bs);
    __syncthreads();
    if (tid < 2) top_sh[tid] = -128;
    __syncthreads();
    for (int i = tid; i < m; i += 256) {
      const int t = kept[j0 + i];
      int page = e4_page(a.block_tables, a.max_blocks, a.pages.num_blocks, b, t / bs);
      if (page < 0) {
        RB_BOUNDS_HIT(104);
        page = 0;
      }
      const long long tile = static_cast<long long>(page) * G + h;
      atomicMax(&top_sh[0], static_cast<int>(a.pages.k_exp[tile]));
      atomicMax(&top_sh[1], static_cast<int>(a.pages.v_exp[tile]));
    }
    __syncthreads();
    const int top_k = top_sh[0], top_v = top_sh[1];
    const long long tile_to = static_cast<long long>(to < 0 ? 0 : to) * G + h;
    for (int i0 = 0; i0 < m; i0 += 16) {
      const int rows = min(16, m - i0);
      __syncthreads();
      float w = 0.f;
      if (tid < rows) {
        const int t = kept[j0 + i0 + tid];
        const int page = max(0, e4_page(a.block_tables, a.max_blocks, a.pages.num_blocks, b, t / bs));
        const long long tile = static_cast<long long>(page) * G + h;
        src_sh[tid] = page;
        off_sh[tid] = static_cast<short>(t % bs);
        exp_sh[0][tid] = a.pages.k_exp[tile];
        exp_sh[1][tid] = a.pages.v_exp[tile];
        if (a.pages.weight) w = a.pages.weight[tile * bs + t % bs];
      }
      __syncthreads();
      const int per = D / 16;                        // pieces of a row
      const int piece = tid % per, row = tid / per % 16, values = tid / (16 * per);
      uint4 u = make_uint4(0, 0, 0, 0);
      const bool mine = values < 2 && row < rows;
      if (mine) {
        const uint8_t* src = reinterpret_cast<const uint8_t*>(values ? a.pages.v : a.pages.k);
        u = *reinterpret_cast<const uint4*>(src + ((static_cast<long long>(src_sh[row]) * G + h) * bs + off_sh[row]) * D + piece * 16);
        const int up = (values ? top_v : top_k) - exp_sh[values][row];
        if (up > 0) u = make_uint4(e4_lower4(u.x, up), e4_lower4(u.y, up), e4_lower4(u.z, up), e4_lower4(u.w, up));
      }
      __syncthreads();
      if (to >= 0) {
        if (mine) {
          uint8_t* dst = reinterpret_cast<uint8_t*>(values ? a.pages.v : a.pages.k);
          *reinterpret_cast<uint4*>(dst + (tile_to * bs + i0 + row) * D + piece * 16) = u;
        }
        if (tid < rows && a.pages.weight) a.pages.weight[tile_to * bs + i0 + tid] = w;
      } else if (tid == 0) {
        RB_BOUNDS_HIT(104);
      }
    }
    __syncthreads();
    if (tid == 0 && to >= 0) {
      a.pages.k_exp[tile_to] = static_cast<signed char>(top_k);
      a.pages.v_exp[tile_to] = static_cast<signed char>(top_v);
    }
  }
}

}  // namespace rb

RB_API int rb_e4m3_evict(const RbE4m3EvictArgs* args, void* stream_v) {
  const RbE4m3EvictArgs& a = *args;
  if (a.batch <= 0) return 0;
  if (const int bad = rbhost::e4_check(a.pages)) return bad;
  if (!a.pages.weight || !a.block_tables || !a.context_lens || !a.kept || !a.lens_out || a.max_blocks <= 0 || (a.out_tables && a.out_blocks <= 0) || a.keep <= 0 ||
      a.recent < 0 || a.keep_first < 0 || static_cast<long long>(a.recent) + a.keep_first > a.keep || a.batch > 65535 || a.pages.block_size > 32768)
    return -1;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream_v);
  const dim3 grid(a.pages.kv_heads, a.batch);
  cudaError_t e = rbhost::launch_pdl(rb::e4_select_kernel, grid, dim3(rb::kE4SelectThreads), 0, s, 1, a RB_BOUNDS_ARG);
  if (e == cudaSuccess) e = rbhost::launch_pdl(rb::e4_move_kernel, grid, dim3(256), 0, s, 1, a RB_BOUNDS_ARG);
  return static_cast<int>(e);
}
