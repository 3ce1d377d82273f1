// Paged KV cache in e4m3: storing the keys and values of new tokens, and reading whole sequences back.
//
// Why a power of two for a tile: an e4m3 number has three bits behind its first whatever its size, so a scale only has to bring the tile's largest
// number under 448 and keep the small ones out of the subnormals; which of the scales within a factor of two does not matter for the others.  With a
// power of two the product with a code is exact in every type that has its range, and a tile whose exponent grows under a later token keeps its
// numbers as they were, but for those that become subnormal.  A scale that is not a power of two would round every code of the page again with every
// token that raises it.
#include "pdl.cuh"
#include "paged_e4m3.cuh"

namespace rb {

constexpr int kE4AppendHeads = 4;                    // of a CTA: a warp for the keys of each and one for its values

// A CTA takes the pages that begin, for this call, within `per_cta` rows, for four KV heads: those whose first new token is one of these rows.  A page's
// tokens may lie in the next CTA's rows too.
template <typename T, int D>
__global__ void __launch_bounds__(kE4AppendHeads * 64, sizeof(T) == 4 ? 2 : 4)
e4_append_kernel(const RbE4m3AppendArgs a, int per_cta RB_BOUNDS_PARAM) {
  pdl_wait();
  pdl_launch();
  const int lane = threadIdx.x & 31, values = threadIdx.x >> 5 & 1;    // even warps: keys, odd ones: values
  const int G = a.pages.kv_heads, bs = a.pages.block_size, h = blockIdx.y * kE4AppendHeads + (threadIdx.x >> 6);
  if (h >= G) return;
  const T* rows = reinterpret_cast<const T*>(values ? a.v_new : a.k_new);
  const long long ld = values ? a.ld_v : a.ld_k;
  uint8_t* codes = reinterpret_cast<uint8_t*>(values ? a.pages.v : a.pages.k);
  signed char* exps = values ? a.pages.v_exp : a.pages.k_exp;
  constexpr int LPR = D / 8, RPW = 32 / LPR;                           // lanes for a row, rows for a warp
  const int r_lane = lane / LPR, c_lane = (lane % LPR) * 8;
  const int end_all = a.row_starts ? min(a.row_starts[a.batch], a.rows) : a.rows, from = blockIdx.x * per_cta;
  const int stop = end_all - from < per_cta ? end_all : from + per_cta;
  for (int r = a.row_starts ? max(from, a.row_starts[0]) : from; r < stop;) {
    const int b = a.row_starts ? e4_sequence_of(a.row_starts, a.batch, r) : r;
    const int first = a.row_starts ? a.row_starts[b] : b, last = a.row_starts ? min(a.row_starts[b + 1], a.rows) : b + 1;
    const int pos = a.context_lens[b] - ((a.row_starts ? a.row_starts[b + 1] : b + 1) - r);
    if (pos < 0) {                                                     // more rows than the sequence has tokens
      r = max(r + 1, pos < r - last ? last : r - pos);
      continue;
    }
    const int i_page = pos / bs, off = pos - i_page * bs, n = min(bs - off, last - r), r0 = r;
    r += max(n, 1);                                  // starts that do not ascend end the loop too
    if (n <= 0) continue;
    if (off != 0 && r0 != first) continue;                             // the page's first new token is an earlier row
    const T* src = rows + static_cast<long long>(r0) * ld + static_cast<long long>(h) * D + c_lane;
    // up to 16 rows stay in registers between the search for their largest number and their rounding; of pages with more the rows are read again
    constexpr int kHeld = 16 / RPW;
    uint4 raw[kHeld][sizeof(T) / 2];
    uint32_t acc = 0;
    int page = -1;
    for (int i0 = 0; i0 < n; i0 += 16) {
#pragma unroll
      for (int k = 0; k < kHeld; ++k)
        if (i0 + k * RPW + r_lane < n) {
#pragma unroll
          for (int x = 0; x < static_cast<int>(sizeof(T) / 2); ++x) raw[k][x] = reinterpret_cast<const uint4*>(src + (i0 + k * RPW + r_lane) * ld)[x];
        }
      if (i0 == 0) {                                                   // looked up while the rows arrive
        page = e4_page(a.block_tables, a.max_blocks, a.pages.num_blocks, b, i_page);
        if (page < 0) {
          RB_BOUNDS_HIT(104);
          break;
        }
      }
#pragma unroll
      for (int k = 0; k < kHeld; ++k)
        if (i0 + k * RPW + r_lane < n) E4Row<T>::largest(raw[k], acc);
    }
    if (page < 0) continue;
    const long long tile = static_cast<long long>(page) * G + h;
    uint8_t* dst = codes + tile * bs * D;
    // Magnitudes are in the order of their bits: an instruction for a number or two, and only where one is not finite are they looked at one by one
    // (8192 rows of 8 heads of 128 in bf16 on one B200, looked at one by one 14.6 us, so 13.3).
    const uint32_t largest = __reduce_max_sync(0xffffffffu, E4Row<T>::one(acc));
    float most = E4Row<T>::value(largest);
    if (largest >= E4Row<T>::kNotFinite) {
      most = 0.f;
      for (int i = r_lane; i < n; i += RPW) {
        float x[8];
        E4Row<T>::load(src + i * ld, x);
#pragma unroll
        for (int j = 0; j < 8; ++j) most = fmaxf(most, e4_finite_abs(x[j]));
      }
      most = warp_max(most);
    }
    int e = e4_exponent(most);
    if (off > 0) {
      const int had = exps[tile];
      if (had >= e) e = had;
      else
        for (int i = lane * 16; i < off * D; i += 512) {               // the codes in front of the new ones
          uint4 u = *reinterpret_cast<const uint4*>(dst + i);
          u = make_uint4(e4_lower4(u.x, e - had), e4_lower4(u.y, e - had), e4_lower4(u.z, e - had), e4_lower4(u.w, e - had));
          *reinterpret_cast<uint4*>(dst + i) = u;
        }
    }
    const float down = e4_two(-e);
    for (int i0 = 0; i0 < n; i0 += 16) {
#pragma unroll
      for (int k = 0; k < kHeld; ++k) {
        const int i = i0 + k * RPW + r_lane;
        if (i >= n) continue;
        if (n > 16) {
#pragma unroll
          for (int x = 0; x < static_cast<int>(sizeof(T) / 2); ++x) raw[k][x] = reinterpret_cast<const uint4*>(src + i * ld)[x];
        }
        float x[8];
        E4Row<T>::of(raw[k], x);
        uint2 u;
        u.x = e4_pack2(x[0] * down, x[1] * down) | e4_pack2(x[2] * down, x[3] * down) << 16;
        u.y = e4_pack2(x[4] * down, x[5] * down) | e4_pack2(x[6] * down, x[7] * down) << 16;
        *reinterpret_cast<uint2*>(dst + (off + i) * D + c_lane) = u;
      }
    }
    __syncwarp();                                                      // every lane has the old exponent
    if (lane == 0) exps[tile] = static_cast<signed char>(e);
    if (!values && a.pages.weight)
      for (int i = lane; i < n; i += 32) a.pages.weight[tile * bs + off + i] = 0.f;
  }
}

constexpr int kE4ReadRows = 16;

// A CTA takes 16 rows.  A lane turns the codes of 16 bytes of its row's result, so that a warp writes 512 bytes without gaps; 16 such pieces of a warp are in
// flight.  Bound by its writes, two thirds of its bytes and more: a plain fill of memory reaches 3.9 TB/s on a B200 where a copy moves 6.4.
template <typename T, int D>
__global__ void __launch_bounds__(256)
e4_read_kernel(const RbE4m3ReadArgs a RB_BOUNDS_PARAM) {
  pdl_wait();
  pdl_launch();
  constexpr int kCodes = 16 / sizeof(T), LPR = D / kCodes, RPW = 32 / LPR;               // codes of a lane, lanes for a row, rows for a warp
  constexpr int kSteps = kE4ReadRows / RPW;          // pieces that make the rows' part of one head: 16, 8 or 4
  constexpr int kAhead = 8;
  __shared__ int page_sh[kE4ReadRows], off_sh[kE4ReadRows];              // page -1: the row has no position
  const int G = a.pages.kv_heads, bs = a.pages.block_size, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const long long r0 = static_cast<long long>(blockIdx.x) * kE4ReadRows;
  if (warp == 0) {
    const int end = min(a.rows, a.row_starts[a.batch]), b0 = e4_sequence_of(a.row_starts, a.batch, static_cast<int>(r0));
    const long long r = r0 + lane;
    int page = -1, off = 0;
    if (lane < kE4ReadRows && r < end && r >= a.row_starts[0]) {
      int b = b0;
      while (a.row_starts[b + 1] <= r) ++b;          // ends: r is in front of the last one
      const int i = static_cast<int>(r) - a.row_starts[b];
      if (i >= 0 && i < a.context_lens[b]) {           // starts that do not ascend may put a row in front of its sequence
        page = e4_page(a.block_tables, a.max_blocks, a.pages.num_blocks, b, i / bs);
        if (page < 0) RB_BOUNDS_HIT(104);
        off = i % bs;
      }
    }
    if (lane < kE4ReadRows) {
      page_sh[lane] = page;
      off_sh[lane] = off;
    }
  }
  __syncthreads();
  const int r_lane = lane / LPR, c_lane = lane % LPR * kCodes;
  // pieces of all heads' keys, then of their values, eight at a time
  constexpr int kHeads = kSteps < kAhead ? kAhead / kSteps : 1, kParts = kSteps > kAhead ? kSteps / kAhead : 1;
  const int units = (G + kHeads - 1) / kHeads * kParts;
  for (int unit = warp; unit < 2 * units; unit += 8) {
    const int values = unit >= units, in = values ? unit - units : unit, h0 = in / kParts * kHeads, step = in % kParts * kAhead;
    const uint8_t* codes = reinterpret_cast<const uint8_t*>(values ? a.pages.v : a.pages.k);
    const signed char* exps = values ? a.pages.v_exp : a.pages.k_exp;
    uint2 u[kAhead];
    int e[kAhead];
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      const int r = (step + k) % kSteps * RPW + r_lane, page = page_sh[r], h = h0 + k / kSteps;
      if (page < 0 || h >= G) continue;
      const long long tile = static_cast<long long>(page) * G + h;
      const uint8_t* src = codes + (tile * bs + off_sh[r]) * D + c_lane;
      e[k] = exps[tile];
      if (kCodes == 8) u[k] = *reinterpret_cast<const uint2*>(src);
      else u[k].x = *reinterpret_cast<const uint32_t*>(src);
    }
    T* out = reinterpret_cast<T*>(values ? a.v_out : a.k_out) + c_lane;
    const long long ld = values ? a.ld_v : a.ld_k;
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      const int r = (step + k) % kSteps * RPW + r_lane, h = h0 + k / kSteps;
      if (page_sh[r] < 0 || h >= G) continue;
      const float up = e4_two(e[k]);
      const uint32_t w[2] = {u[k].x, u[k].y};
      float x[8];
#pragma unroll
      for (int j = 0; j < kCodes / 2; ++j) {
        const float2 f = e4_float2(w[j >> 1] >> (16 * (j & 1)));
        x[2 * j] = f.x * up;
        x[2 * j + 1] = f.y * up;
      }
      T* to = out + (r0 + r) * ld + h * D;
      if (sizeof(T) == 4) *reinterpret_cast<float4*>(to) = make_float4(x[0], x[1], x[2], x[3]);
      else E4Row<T>::store(to, x);
    }
  }
}

}  // namespace rb

namespace {
template <typename T>
int append_by_dim(const RbE4m3AppendArgs& a, cudaStream_t s) {
  const int per_cta = a.row_starts ? a.pages.block_size : 1;
  const dim3 grid((a.rows + per_cta - 1) / per_cta, (a.pages.kv_heads + rb::kE4AppendHeads - 1) / rb::kE4AppendHeads);
  auto kern = a.pages.head_dim == 64 ? rb::e4_append_kernel<T, 64> : rb::e4_append_kernel<T, 128>;
  return static_cast<int>(rbhost::launch_pdl(kern, grid, dim3(rb::kE4AppendHeads * 64), 0, s, 1, a, per_cta RB_BOUNDS_ARG));
}
template <typename T>
int read_by_dim(const RbE4m3ReadArgs& a, cudaStream_t s) {
  auto kern = a.pages.head_dim == 64 ? rb::e4_read_kernel<T, 64> : rb::e4_read_kernel<T, 128>;
  const dim3 grid((a.rows + rb::kE4ReadRows - 1) / rb::kE4ReadRows);
  return static_cast<int>(rbhost::launch_pdl(kern, grid, dim3(256), 0, s, 1, a RB_BOUNDS_ARG));
}
template <typename A>
bool rows_fit(const A& a, const void* k, const void* v) {
  const int per16 = a.type == RB_E4M3_F32 ? 4 : 8;
  return !((reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v)) & 15) && a.ld_k % per16 == 0 && a.ld_v % per16 == 0;
}
}  // namespace

RB_API int rb_e4m3_append(const RbE4m3AppendArgs* args, void* stream_v) {
  const RbE4m3AppendArgs& a = *args;
  if (a.rows <= 0 || a.batch <= 0) return 0;
  if (const int bad = rbhost::e4_check(a.pages)) return bad;
  if (!a.k_new || !a.v_new || !a.block_tables || !a.context_lens || a.max_blocks <= 0 || a.pages.kv_heads > 65535 || (!a.row_starts && a.rows != a.batch))
    return -1;
  if (!rows_fit(a, a.k_new, a.v_new)) return -2;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream_v);
  switch (a.type) {
    case RB_E4M3_BF16: return append_by_dim<__nv_bfloat16>(a, s);
    case RB_E4M3_F16: return append_by_dim<__half>(a, s);
    case RB_E4M3_F32: return append_by_dim<float>(a, s);
  }
  return -1;
}

RB_API int rb_e4m3_read(const RbE4m3ReadArgs* args, void* stream_v) {
  const RbE4m3ReadArgs& a = *args;
  if (a.rows <= 0 || a.batch <= 0) return 0;
  if (const int bad = rbhost::e4_check(a.pages)) return bad;
  if (!a.k_out || !a.v_out || !a.block_tables || !a.context_lens || !a.row_starts || a.max_blocks <= 0) return -1;
  if (!rows_fit(a, a.k_out, a.v_out)) return -2;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream_v);
  switch (a.type) {
    case RB_E4M3_BF16: return read_by_dim<__nv_bfloat16>(a, s);
    case RB_E4M3_F16: return read_by_dim<__half>(a, s);
    case RB_E4M3_F32: return read_by_dim<float>(a, s);
  }
  return -1;
}
