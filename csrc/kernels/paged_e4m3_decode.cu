// Attention of single tokens over a paged cache in e4m3, with an optional sum of the attention weights of every cached token.
//
// With key j's score s_j (base 2: scale, log2 e and the keys' exponent included) and the exponent e_j of its value's tile, the output is
// sum_j 2^(s_j) 2^(e_j) c_j / sum_j 2^(s_j).  The maximum M that keeps the numbers in range is taken over s_j + e_j: the factors p_j = 2^(s_j + e_j - M)
// of the codes are then at most 2^15 whatever the tiles' exponents.  M lies 15 below the largest: an f16 ends at 2^16 and has all its bits down to 2^-14, so with
// factors up to 1 those below 2^-25 would be lost, of which a long context beside a token with nearly all the weight has many.  M is rounded up to a
// whole number, so that M - e_j and the factors that bring sums from one M to another are exact; with exponents of -100 a fractional M would cost the scores
// seven bits.
//
// The denominator has a maximum M' of its own, whole too: a factor p_j below 2^-126 is lost, which the numerator never misses, but the token behind it
// may have the largest score of all, with values that are small or zero beside others' large ones.  The tiles of a warp in a slice seldom have exponents
// far apart; if they are within 64 of the largest, E, the denominator is the sum of p_j 2^(E - e_j) under M' = M - E (a factor that is lost is then of a score
// 2^-61 below the largest, or less), otherwise of 2^(s_j - M') with a second exponential, where every lane has the largest of its own scores as M'.
#include <cooperative_groups.h>

#include <type_traits>

#include "pdl.cuh"
#include "paged_e4m3.cuh"

namespace rb {

namespace cg = cooperative_groups;

constexpr int kE4Room = 15;                          // factors of codes reach 2^15
constexpr int kE4Slice = 256;                        // tokens whose sums one CTA forms; the merge goes over them in order

__device__ __forceinline__ float e4_ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float e4_get(const __nv_bfloat16* p) { return __bfloat162float(*p); }
__device__ __forceinline__ float e4_get(const __half* p) { return __half2float(*p); }
__device__ __forceinline__ void e4_put(__nv_bfloat16* p, float v) { *p = __float2bfloat16(v); }
__device__ __forceinline__ void e4_put(__half* p, float v) { *p = __float2half(v); }
template <typename T>
__device__ __forceinline__ void e4_put4(T* p, const float4& x, float inv, const float2& size) {
  e4_put(p, x.x * inv * size.x * size.y);
  e4_put(p + 1, x.y * inv * size.x * size.y);
  e4_put(p + 2, x.z * inv * size.x * size.y);
  e4_put(p + 3, x.w * inv * size.x * size.y);
}

// Scratch: [batch, heads, slices, D + 4] fp32: maximum, denominator and its maximum, one unused, sums of a slice; then, where weights are summed, the scores
// [batch, KV heads, slices * 256, heads of a group] and what makes weights of them [batch, heads, 2].
__device__ __forceinline__ float* e4_partial(float* scratch, int heads, int slices, int D, int b, int h, int s) {
  return scratch + ((static_cast<long long>(b) * heads + h) * slices + s) * (D + 4);
}

__device__ __forceinline__ float2* e4_norm(const RbE4m3DecodeArgs& a, int slices, int b, int h) {
  const long long rows = static_cast<long long>(a.batch) * a.heads;
  return reinterpret_cast<float2*>(a.scratch + rows * slices * (a.pages.head_dim + 4 + kE4Slice)) + static_cast<long long>(b) * a.heads + h;
}
// The tokens of a sequence that its tables have room for.
__device__ __forceinline__ int e4_len(const RbE4m3DecodeArgs& a, int b) {
  const long long room = static_cast<long long>(a.max_blocks) * a.pages.block_size;
  return static_cast<int>(max(0ll, min(static_cast<long long>(a.context_lens[b]), room)));
}
__device__ __forceinline__ uint4 e4_lds128(uint32_t addr) {
  uint4 u;
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(u.x), "=r"(u.y), "=r"(u.z), "=r"(u.w) : "r"(addr));
  return u;
}
__device__ __forceinline__ uint2 e4_lds64(uint32_t addr) {
  uint2 u;
  asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(u.x), "=r"(u.y) : "r"(addr));
  return u;
}
__device__ __forceinline__ void e4_mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t e4_half2_of(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// A slice that a CTA works on, and how many follow in its run.
struct E4Place {
  int b, hk, s, left;
};

constexpr int kE4Warps = 4, kE4Stages = 4;           // a warp has the four tiles of a slice that are its own in flight

template <int D, int NH>
struct E4Layout {
  static constexpr int kTile = 16 * D;                                   // bytes of a tile's keys; its values follow
  static constexpr int kRing = kE4Warps * kE4Stages * 2 * kTile;
  // The warps' sums lie behind the ring, those of `kRound` heads at a time (of a cluster those of all heads): with 4 heads of 128 three CTAs fit on an SM.
  // 64 sequences of 4096, 4 KV heads for 32 heads of 128, one B200: 80.9 us with 8 at a time and two CTAs an SM, 74.9 so.
  static constexpr int kRound = NH == 1 && D == 128 ? 4 : 8;
  static int bytes(int heads) { return kRing + kE4Warps * heads * D * 4 + 1024; }
};

// Warp w of a CTA takes tiles w, w + 4, w + 8, w + 12 of 16 tokens of a slice; its sums and those of the other warps are added in the order of the
// warps, and a sequence's slices in order by the merge, so that a sequence has the same bits alone and beside others.
//
// S^T = K Q^T has the tokens as the 16 rows of m16n8k16 and the heads as its 8 columns (NH: 8 or 16 heads), O^T = V^T P^T the head dimensions as
// rows and the heads as columns, so that no row is left empty and a lane's factors are those of its own columns; P^T, rounded to f16, takes its place as
// the second operand by a transposition of 8 x 8 (movmatrix).  Codes become f16 exactly.  The contraction over head dimensions may take them in any
// order, so a lane reads 16 codes of a row at a time and these are its operands of four products; a swizzled tile gives every lane its 16 bytes without
// bank conflicts.  A query row is scaled to [1, 2) by a power of two first.  Rounding a factor p_j to f16 is off by at most 2^-11 of it, or by 2^-25 where it is
// below 2^-14 (2^-39 of the largest, which is 2^15 or, where M was rounded up, down to half of that).  2^-11 of an output is an eighth of what rounding it to bf16
// may take, 2^-8; an output in f16, which loses 2^-11 itself, would show it, and there what the rounding left of a factor is a second operand.
// HOW: kE4List: the slices of all sequences and KV heads, numbered one sequence after the other, are dealt in equal runs to CTAs that stay, and the next
// slice's tiles are copied while this one's are worked on.  Otherwise the grid is (slices, KV heads, sequences); kE4Cluster: the CTAs of a sequence and KV
// head are a cluster and merge their sums, and add the weights, through distributed shared memory.
enum { kE4Grid, kE4List, kE4Cluster };

// The factor that brings sums under the maximum m to the maximum `to` >= m.  Maxima are whole, so it is an exact power of two, and a sum of such sums does
// not depend on which maximum they are brought to on the way.  Zero where it would be below 2^-126 and where there is no maximum yet (-infinity).  A whole number that
// 1.5 * 2^23 is added to stands in the last bits of the sum: its exponent bits come without a conversion.
__device__ __forceinline__ float e4_factor(float m, float to) {
  return __int_as_float(__float_as_int(fmaxf(m - to, -127.f) + (12582912.f + 127.f)) << 23);
}

// A score from a sum of products of keys' codes and a scaled query, where it may leave the range of 32 bits.  The factor stays finite, so that a sum of zero is
// a score of zero; a score below the range is the least number, so that a tile of such scores has a maximum.
__device__ __forceinline__ float e4_far_score(float sum, float factor) {
  factor = factor > 3.4028235e38f ? 3.4028235e38f : factor < -3.4028235e38f ? -3.4028235e38f : factor;
  const float s = sum * factor;
  return s == -INFINITY ? -3.4028235e38f : s;
}

// What brings a sum under the maximum m, divided by a denominator under the maximum d, to its own size: 2^(m - d), in two steps that are in range.
__device__ __forceinline__ float2 e4_size(float m, float d) {
  const int e = static_cast<int>(fminf(fmaxf(m - d, -252.f), 252.f)), half = e >> 1;
  return make_float2(e4_two(half), e4_two(e - half));
}

// A weight is 2^(s - m) / den = 2^(s - (m + x)) / (den / 2^x), with the x that brings den / 2^x into [1, 2): (m + x, 2^x / den).
__device__ __forceinline__ float2 e4_norm_of(float m, float den) {
  const int x = static_cast<int>(__float_as_uint(den) >> 23) - 127;
  return make_float2(m + static_cast<float>(x), e4_two(x) / den);
}

template <typename T, int D, int NH, int HOW>
__global__ void __launch_bounds__(kE4Warps * 32, NH > 1 ? 2 : D == 64 ? 4 : 3)
e4_decode_kernel(const __grid_constant__ CUtensorMap k_map, const __grid_constant__ CUtensorMap v_map, const RbE4m3DecodeArgs a, int h0, int slices,
                 unsigned int* status RB_BOUNDS_PARAM) {
  pdl_wait();
  if (HOW != kE4List) pdl_launch();                  // CTAs that stay let the merge in at the end of their runs: 177 us at once, 159 then (64 of 4096 to 8192)
  constexpr bool LIST = HOW == kE4List, CLUSTER = HOW == kE4Cluster;
  using L = E4Layout<D, NH>;
  constexpr int KS = D / 16;                         // products of 16 in a score
  constexpr int MT = D / 16;                         // tiles of 16 output dimensions
  constexpr int BR = D / 8;                          // rows of 128 bytes in a tile
  constexpr int kNone = static_cast<int>(0x80000000);
  constexpr int PF = std::is_same<T, __half>::value ? 2 : 1;             // operands that a factor makes
  extern __shared__ uint8_t e4_raw[];
  __shared__ __align__(8) uint64_t bars[kE4Warps][kE4Stages];
  __shared__ float m_sh[kE4Warps][NH * 8], l_sh[kE4Warps][NH * 8], d_sh[kE4Warps][NH * 8];
  __shared__ float4 mld_sh[NH * 8];                  // maximum, denominator, its maximum
  __shared__ float2 norm_sh[NH * 8];
  __shared__ int abort_sh;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, gq = lane >> 2, tq = lane & 3;
  const uint32_t base = (smem_u32(e4_raw) + 1023u) & ~1023u;             // the swizzle goes by addresses
  const uint32_t ring = base + warp * (kE4Stages * 2 * L::kTile);
  float* merge = reinterpret_cast<float*>(e4_raw + (base - smem_u32(e4_raw)) + L::kRing);           // [warps][heads][D]
  float* scores_sh = nullptr;                        // CLUSTER, where weights are summed: [256][heads] behind it
  const int bs = a.pages.block_size, G = a.pages.kv_heads, group = a.heads / G;
  const int heads = min(NH * 8, group - h0);
  if (CLUSTER) scores_sh = merge + kE4Warps * heads * D;

  // ---- this CTA's run of slices
  E4Place at = {0, 0, 0, 1};
  if (!LIST) {
    at.b = blockIdx.z;
    at.hk = blockIdx.y;
    at.s = blockIdx.x;
    if (!CLUSTER && at.s * kE4Slice >= e4_len(a, at.b)) return;
  } else {
    int n = lane < a.batch ? (e4_len(a, lane) + kE4Slice - 1) / kE4Slice : 0, total = n;
    for (int i = lane + 32; i < a.batch; i += 32) total += (e4_len(a, i) + kE4Slice - 1) / kE4Slice;
    const unsigned int all = __reduce_add_sync(0xffffffffu, total) * static_cast<unsigned int>(G);      // the host bounds it
    const unsigned int share = all / gridDim.x, over = all - share * gridDim.x;
    at.left = share + (blockIdx.x < over ? 1 : 0);
    if (at.left == 0) {
      pdl_launch();
      return;
    }
    unsigned int skip = blockIdx.x * share + min(blockIdx.x, over);
    for (int b0 = 0;;) {
      unsigned int upto = n * G;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const unsigned int v = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += v;
      }
      const unsigned int behind = __ballot_sync(0xffffffffu, upto > skip);
      if (behind != 0u) {
        const int which = __ffs(behind) - 1;
        at.b = b0 + which;
        const int in = skip - __shfl_sync(0xffffffffu, upto - n * G, which), ns = __shfl_sync(0xffffffffu, n, which);
        at.hk = in / ns;
        at.s = in - at.hk * ns;
        break;
      }
      skip -= __shfl_sync(0xffffffffu, upto, 31);
      b0 += 32;
      if (b0 >= a.batch) return;                     // lengths that changed meanwhile
      n = b0 + lane < a.batch ? (e4_len(a, b0 + lane) + kE4Slice - 1) / kE4Slice : 0;
    }
  }

  if (threadIdx.x == 0) abort_sh = 0;
  if (lane == 0)
    for (int i = 0; i < kE4Stages; ++i) mbar_init(smem_u32(&bars[warp][i]), 1);
  fence_mbar_init();
  __syncthreads();

  // The page of this warp's tile `lane & 3` of a slice as the table says it, kNone where the sequence ends before the tile
  const int per_page = bs >> 4, tile_in = (lane & 3) * kE4Warps + warp;
  auto look_up = [&](const E4Place& p, int n) {
    const int t = p.s * (kE4Slice / 16) + tile_in;
    if (t * 16 >= n) return kNone;
    const int i = per_page == 1 ? t : t / per_page;
    return max(a.block_tables[static_cast<long long>(p.b) * a.max_blocks + i], -1);    // n is no more than the table has room for; never kNone
  };
  // the tile counted over a whole array (-1: none), and its page and head as the exponents are counted
  auto locate = [&](const E4Place& p, int page, int& tile, int& where) {
    tile = -1;
    if (page == kNone) return;
    if (page < 0 || page >= a.pages.num_blocks) {    // corrupt tables read block 0 instead of faulting
      RB_BOUNDS_HIT(104);
      page = 0;
    }
    where = page * G + p.hk;
    tile = per_page == 1 ? where : where * per_page + (p.s * (kE4Slice / 16) + tile_in) % per_page;
  };
  auto request = [&](int stage, int tile) {          // lane 0
    const uint32_t bar = smem_u32(&bars[warp][stage]), dst = ring + stage * 2 * L::kTile;
    mbar_arrive_expect_tx(bar, 2 * L::kTile);
    tma_load_2d(dst, &k_map, 0, tile * BR, bar);
    tma_load_2d(dst + L::kTile, &v_map, 0, tile * BR, bar);
  };
  auto advance = [&](E4Place& p, int& n) {           // the next slice of the run
    if (--p.left <= 0) {
      n = 0;
      return;
    }
    if (++p.s * kE4Slice < n) return;
    p.s = 0;
    if (++p.hk < G) return;
    p.hk = 0;
    do n = ++p.b < a.batch ? e4_len(a, p.b) : 0;
    while (n == 0 && p.b < a.batch);
    if (n == 0) p.left = 0;                          // lengths that changed meanwhile
  };
  // lanes 0 .. 3: exponents of the four tiles' keys, 4 .. 7 of their values
  auto exps_of = [&](int tile, int w) { return tile < 0 || lane >= 8 ? 0 : static_cast<int>((lane < 4 ? a.pages.k_exp : a.pages.v_exp)[w]); };

  int n_at = e4_len(a, at.b), tile_at, where = 0;
  locate(at, look_up(at, n_at), tile_at, where);
#pragma unroll
  for (int i = 0; i < kE4Stages; ++i) {
    const int t = __shfl_sync(0xffffffffu, tile_at, i);
    if (lane == 0 && t >= 0) request(i, t);
  }
  int exps = exps_of(tile_at, where);
  // Of a list, the next slice's tiles are known and their exponents on their way, and so are the pages of the one behind it: every load has a slice's
  // time to arrive.
  E4Place next = at, then = at;
  int n_next = n_at, n_then = n_at, tile_next = -1, exps_next = 0, page_then = 0;
  if (LIST) {
    advance(next, n_next);
    locate(next, look_up(next, n_next), tile_next, where);
    exps_next = exps_of(tile_next, where);
    then = next;
    n_then = n_next;
    advance(then, n_then);
    page_then = look_up(then, n_then);
  }

  const bool q_whole = !((reinterpret_cast<uintptr_t>(a.q) | static_cast<uintptr_t>(a.ld_q * 2)) & 15);
  uint32_t qf[KS][NH][2];                            // head r * 8 + gq, this lane's dimensions of it
  float q_up[NH][2];                                 // heads r * 8 + 2 tq and + 1: what a product with their rows is to be multiplied with
  int q_top = 0;                                     // the largest one's exponent
  uint32_t parity = 0;
  for (bool fresh = true;;) {
    if (fresh) {
      q_top = -127;
#pragma unroll
      for (int r = 0; r < NH; ++r) {
        const bool there = r * 8 + gq < heads;
        const T* src = reinterpret_cast<const T*>(a.q) + at.b * a.ld_q + (static_cast<long long>(at.hk) * group + h0 + r * 8 + gq) * D + tq * (D / 4);
        float x[D / 4], most = 0.f;
        if (there && q_whole) {
#pragma unroll
          for (int i = 0; i < D / 4; i += 8) {
            float y[8];
            E4Row<T>::load(src + i, y);
#pragma unroll
            for (int j = 0; j < 8; ++j) x[i + j] = y[j];
          }
        } else {
#pragma unroll
          for (int i = 0; i < D / 4; ++i) x[i] = there ? e4_get(src + i) : 0.f;
        }
#pragma unroll
        for (int i = 0; i < D / 4; ++i) most = fmaxf(most, fabsf(x[i]));
        most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 1));
        most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 2));
        const int e = min(max(static_cast<int>(__float_as_uint(most) >> 23) - 127, -126), 126);
        const float down = e4_two(-e), up = e4_two(e) * a.scale * 1.4426950408889634f;
        q_top = max(q_top, static_cast<int>(__float_as_uint(up) >> 23 & 255) - 127);
        q_up[r][0] = __shfl_sync(0xffffffffu, up, tq * 8);
        q_up[r][1] = __shfl_sync(0xffffffffu, up, tq * 8 + 4);
#pragma unroll
        for (int j = 0; j < KS; ++j) {
          qf[j][r][0] = e4_half2_of(x[4 * j] * down, x[4 * j + 1] * down);
          qf[j][r][1] = e4_half2_of(x[4 * j + 2] * down, x[4 * j + 3] * down);
        }
      }
      q_top = __reduce_max_sync(0xffffffffu, q_top);
    }
    // the exponents of this warp's values: the largest, and whether they are far apart
    const bool there = lane < 8 && at.s * kE4Slice + tile_in * 16 < n_at, values = there && lane >= 4;
    const int e_top = __reduce_max_sync(0xffffffffu, values ? exps : -128);
    const bool far = e_top - __reduce_min_sync(0xffffffffu, values ? exps : 127) > 64;
    // whether a score may leave the range: a sum is below 2 * 448 * 128 < 2^17, the query's factor below 2^(q_top + 1)
    const bool wide = __reduce_max_sync(0xffffffffu, there && lane < 4 ? exps : -128) + q_top + 18 > 127;
    float m[NH][2], l[NH][2], dm[NH][2], o[MT][NH][4];   // of heads r * 8 + 2 tq and + 1; l: this lane's tokens, dm (far): the largest score of them
#pragma unroll
    for (int r = 0; r < NH; ++r) {
      m[r][0] = m[r][1] = dm[r][0] = dm[r][1] = -INFINITY;
      l[r][0] = l[r][1] = 0.f;
#pragma unroll
      for (int i = 0; i < MT; ++i) o[i][r][0] = o[i][r][1] = o[i][r][2] = o[i][r][3] = 0.f;
    }
#pragma unroll 1
    for (int i = 0; i < kE4Stages; i += 2) {         // two tiles at a time, each in two chains of products
      int n_tok[2], coming[2], ev[2];                // tokens of a tile and behind it
      float up[2];
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        n_tok[u] = n_at - (at.s * kE4Slice + ((i + u) * kE4Warps + warp) * 16);
        coming[u] = __shfl_sync(0xffffffffu, tile_next, i + u);
        ev[u] = __shfl_sync(0xffffffffu, exps, 4 + i + u);
        up[u] = e4_two(__shfl_sync(0xffffffffu, exps, i + u));
      }
      if (n_tok[0] <= 0) {
        if (lane == 0) {
          if (coming[0] >= 0) request(i, coming[0]);
          if (coming[1] >= 0) request(i + 1, coming[1]);
        }
        continue;
      }
      float s[2][NH][4];                             // (token gq, heads 2 tq and + 1), (token gq + 8, the same)
      uint32_t vw[2][4][D / 32];                     // codes of tokens 2 tq, 2 tq + 1, 2 tq + 8, 2 tq + 9, dimensions gq * D / 8 ..
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        if (n_tok[u] > 0) {
          mbar_wait(smem_u32(&bars[warp][i + u]), (parity >> (i + u)) & 1, &abort_sh, status, 130);
          parity ^= 1u << (i + u);
        }
        const uint32_t kt = ring + (i + u) * 2 * L::kTile, vt = kt + L::kTile;
        uint32_t kw[2][D / 16];                      // codes of tokens gq and gq + 8, dimensions tq * D / 4 ..
        if (D == 128) {
#pragma unroll
          for (int t = 0; t < 2; ++t) {
#pragma unroll
            for (int p = 0; p < 2; ++p) {
              const uint4 x = e4_lds128(kt + (t * 8 + gq) * 128 + (((tq * 2 + p) ^ gq) << 4));
              kw[t][p * 4] = x.x; kw[t][p * 4 + 1] = x.y; kw[t][p * 4 + 2] = x.z; kw[t][p * 4 + 3] = x.w;
            }
          }
#pragma unroll
          for (int t = 0; t < 4; ++t) {
            const int row = tq * 2 + (t & 1) + (t >> 1) * 8;
            const uint4 x = e4_lds128(vt + row * 128 + ((gq ^ (row & 7)) << 4));
            vw[u][t][0] = x.x; vw[u][t][1] = x.y; vw[u][t][D / 32 - 2] = x.z; vw[u][t][D / 32 - 1] = x.w;
          }
        } else {                                     // two tokens in a row of 128 bytes
#pragma unroll
          for (int t = 0; t < 2; ++t) {
            const int tok = t * 8 + gq, row = tok >> 1;
            const uint4 x = e4_lds128(kt + row * 128 + ((((tok & 1) * 4 + tq) ^ row) << 4));
            kw[t][0] = x.x; kw[t][1] = x.y; kw[t][2] = x.z; kw[t][3] = x.w;
          }
#pragma unroll
          for (int t = 0; t < 4; ++t) {
            const int tok = tq * 2 + (t & 1) + (t >> 1) * 8, row = tok >> 1;
            const uint2 x = e4_lds64(vt + row * 128 + ((((tok & 1) * 4 + (gq >> 1)) ^ row) << 4) + (gq & 1) * 8);
            vw[u][t][0] = x.x; vw[u][t][1] = x.y;
          }
        }
        float odd[NH][4];
#pragma unroll
        for (int r = 0; r < NH; ++r) {
          s[u][r][0] = s[u][r][1] = s[u][r][2] = s[u][r][3] = 0.f;
          odd[r][0] = odd[r][1] = odd[r][2] = odd[r][3] = 0.f;
        }
#pragma unroll
        for (int j = 0; j < KS; ++j) {
          uint32_t a0, a1, a2, a3;
          e4_half4(kw[0][j], a0, a2);
          e4_half4(kw[1][j], a1, a3);
#pragma unroll
          for (int r = 0; r < NH; ++r) e4_mma(j & 1 ? odd[r] : s[u][r], a0, a1, a2, a3, qf[j][r][0], qf[j][r][1]);
        }
#pragma unroll
        for (int r = 0; r < NH; ++r) {
#pragma unroll
          for (int j = 0; j < 4; ++j) s[u][r][j] += odd[r][j];
        }
      }
      __syncwarp();                                  // the stages are free
      if (lane == 0) {
        if (coming[0] >= 0) request(i, coming[0]);
        if (coming[1] >= 0) request(i + 1, coming[1]);
      }
      uint32_t pf[2][NH][2][PF];
      float grow[NH][2];
      bool moved = false;
#pragma unroll
      for (int r = 0; r < NH; ++r) {
        if (wide) {
#pragma unroll
          for (int x = 0; x < 8; ++x) s[x >> 2][r][x & 3] = e4_far_score(s[x >> 2][r][x & 3], up[x >> 2] * q_up[r][x & 1]);
        } else {
#pragma unroll
          for (int x = 0; x < 8; ++x) s[x >> 2][r][x & 3] *= up[x >> 2] * q_up[r][x & 1];
        }
        float to[2] = {-INFINITY, -INFINITY};
#pragma unroll
        for (int u = 0; u < 2; ++u) {
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            if (n_tok[u] < 16 && gq + (j >> 1) * 8 >= n_tok[u]) s[u][r][j] = -INFINITY;
          }
          if (a.accumulate) {                        // [batch, KV heads, tokens, heads of a group]
            const int t = ((i + u) * kE4Warps + warp) * 16 + gq;
            float* scores = CLUSTER ? scores_sh + t * heads
                                    : a.scratch + static_cast<long long>(a.batch) * a.heads * slices * (D + 4) +
                                          ((static_cast<long long>(at.b) * G + at.hk) * slices * kE4Slice + at.s * kE4Slice + t) * group + h0;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const int h = r * 8 + tq * 2 + (j & 1);
              if (h < heads) scores[(j >> 1) * 8 * (CLUSTER ? heads : group) + h] = s[u][r][j];
            }
          }
#pragma unroll
          for (int j = 0; j < 2; ++j) to[j] = fmaxf(to[j], ceilf(fmaxf(s[u][r][j], s[u][r][2 + j])) + static_cast<float>(ev[u] - kE4Room));
        }
#pragma unroll
        for (int j = 0; j < 2; ++j) {
#pragma unroll
          for (int x = 4; x < 32; x <<= 1) to[j] = fmaxf(to[j], __shfl_xor_sync(0xffffffffu, to[j], x));
          to[j] = fmaxf(to[j], m[r][j]);
          grow[r][j] = e4_factor(m[r][j], to[j]);
          moved |= to[j] != m[r][j];
          m[r][j] = to[j];
        }
        if (far) {                                     // this lane's scores are its own
#pragma unroll
          for (int j = 0; j < 2; ++j) {
            const float top = fmaxf(dm[r][j], ceilf(fmaxf(fmaxf(s[0][r][j], s[0][r][2 + j]), fmaxf(s[1][r][j], s[1][r][2 + j]))));
            const float under = top == -INFINITY ? 0.f : top;            // no token yet
            l[r][j] *= e4_factor(dm[r][j], top);
            l[r][j] += e4_ex2(s[0][r][j] - under) + e4_ex2(s[0][r][2 + j] - under);
            l[r][j] += e4_ex2(s[1][r][j] - under) + e4_ex2(s[1][r][2 + j] - under);
            dm[r][j] = top;
          }
        } else {
          l[r][0] *= grow[r][0];
          l[r][1] *= grow[r][1];
        }
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const float e = static_cast<float>(ev[u]), down = far ? 0.f : e4_two(e_top - ev[u]);
          float p[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) p[j] = e4_ex2(s[u][r][j] - (to[j & 1] - e));
          l[r][0] = fmaf(p[0] + p[2], down, l[r][0]);
          l[r][1] = fmaf(p[1] + p[3], down, l[r][1]);
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            const uint32_t h2 = e4_half2_of(p[2 * c], p[2 * c + 1]);
            asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(pf[u][r][c][0]) : "r"(h2));
            if (PF > 1) {
              const float2 got = __half22float2(*reinterpret_cast<const __half2*>(&h2));
              const uint32_t rest = e4_half2_of(p[2 * c] - got.x, p[2 * c + 1] - got.y);
              asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(pf[u][r][c][PF - 1]) : "r"(rest));
            }
          }
        }
      }
      if (i > 0 && __any_sync(0xffffffffu, moved)) {
#pragma unroll
        for (int r = 0; r < NH; ++r) {
#pragma unroll
          for (int t = 0; t < MT; ++t) {
#pragma unroll
            for (int j = 0; j < 4; ++j) o[t][r][j] *= grow[r][j & 1];
          }
        }
      }
      // ---- O^T += V^T P^T
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        if (n_tok[u] < 16) {                         // what lies behind the last token may be anything, NaN too
#pragma unroll
          for (int t = 0; t < 4; ++t)
            if (tq * 2 + (t & 1) + (t >> 1) * 8 >= n_tok[u]) {
#pragma unroll
              for (int w = 0; w < D / 32; ++w) vw[u][t][w] = 0u;
            }
        }
#pragma unroll
        for (int w = 0; w < D / 32; ++w) {
          uint32_t a00, a01, a02, a03, a10, a11, a12, a13;
          e4_half4(__byte_perm(vw[u][0][w], vw[u][1][w], 0x5140), a00, a01);
          e4_half4(__byte_perm(vw[u][2][w], vw[u][3][w], 0x5140), a02, a03);
          e4_half4(__byte_perm(vw[u][0][w], vw[u][1][w], 0x7362), a10, a11);
          e4_half4(__byte_perm(vw[u][2][w], vw[u][3][w], 0x7362), a12, a13);
#pragma unroll
          for (int r = 0; r < NH; ++r) {
#pragma unroll
            for (int x = 0; x < PF; ++x) {
              e4_mma(o[2 * w][r], a00, a01, a02, a03, pf[u][r][0][x], pf[u][r][1][x]);
              e4_mma(o[2 * w + 1][r], a10, a11, a12, a13, pf[u][r][0][x], pf[u][r][1][x]);
            }
          }
        }
      }
    }
    // ---- the slice's sums: all warps' together, those of some heads after those of others
#pragma unroll
    for (int r = 0; r < NH; ++r) {
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        float top = m[r][j] - static_cast<float>(e_top);
        if (far) {
          top = dm[r][j];
#pragma unroll
          for (int x = 4; x < 32; x <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, x));
          l[r][j] *= e4_factor(dm[r][j], top);
        }
#pragma unroll
        for (int x = 4; x < 32; x <<= 1) l[r][j] += __shfl_xor_sync(0xffffffffu, l[r][j], x);
        if (gq == 0) {
          m_sh[warp][r * 8 + tq * 2 + j] = m[r][j];
          l_sh[warp][r * 8 + tq * 2 + j] = l[r][j];
          d_sh[warp][r * 8 + tq * 2 + j] = top;
        }
      }
    }
    const bool whole = !CLUSTER && n_at <= kE4Slice; // the sequence has no other slice
    constexpr int kRound = CLUSTER ? NH * 8 : L::kRound;
#pragma unroll 1
    for (int hb = 0; hb < heads; hb += kRound) {
      const int rows = min(kRound, heads - hb);        // of a warp in `merge`
      if (hb > 0) __syncthreads();
#pragma unroll
      for (int r = 0; r < NH; ++r) {
#pragma unroll
        for (int j = 0; j < 2; ++j) {                  // head r * 8 + 2 tq + j, dimensions gq * D / 8 .., 16 bytes at a time, swizzled by the head
          const int head = r * 8 + tq * 2 + j;
          if (head < hb || head >= hb + rows) continue;
          float* row = merge + (warp * rows + head - hb) * D;
#pragma unroll
          for (int t = 0; t < MT; t += 2)
            *reinterpret_cast<float4*>(row + (((gq * (D / 32) + t / 2) ^ tq) << 2)) = make_float4(o[t][r][j], o[t][r][2 + j], o[t + 1][r][j], o[t + 1][r][2 + j]);
        }
      }
      if (LIST && at.left <= 1) pdl_launch();
      __syncthreads();
      for (int i = threadIdx.x; i < rows * (D / 4); i += kE4Warps * 32) {
        const int head = hb + i / (D / 4), d = i % (D / 4);
        float top = m_sh[0][head], dtop = d_sh[0][head];
#pragma unroll
        for (int w = 1; w < kE4Warps; ++w) {
          top = fmaxf(top, m_sh[w][head]);
          dtop = fmaxf(dtop, d_sh[w][head]);
        }
        float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
        float den = 0.f;
#pragma unroll
        for (int w = 0; w < kE4Warps; ++w) {
          const float f = e4_factor(m_sh[w][head], top);
          den = fmaf(l_sh[w][head], e4_factor(d_sh[w][head], dtop), den);
          const float4 x = *reinterpret_cast<const float4*>(merge + (w * rows + head - hb) * D + ((d ^ (head >> 1 & 3)) << 2));
          sum.x = fmaf(x.x, f, sum.x);
          sum.y = fmaf(x.y, f, sum.y);
          sum.z = fmaf(x.z, f, sum.z);
          sum.w = fmaf(x.w, f, sum.w);
        }
        if (CLUSTER) {                                 // where this thread read the first warp's
          *reinterpret_cast<float4*>(merge + head * D + ((d ^ (head >> 1 & 3)) << 2)) = sum;
          if (d == 0) mld_sh[head] = make_float4(top, den, dtop, 0.f);
          continue;
        }
        const int h = at.hk * group + h0 + head;
        if (whole) {
          e4_put4(reinterpret_cast<T*>(a.out) + at.b * a.ld_o + static_cast<long long>(h) * D + d * 4, sum, 1.f / den, e4_size(top, dtop));
        }
        if (!whole || a.accumulate) {                  // the weights' denominators come from here too
          float* out = e4_partial(a.scratch, a.heads, slices, D, at.b, h, at.s);
          if (d == 0) *reinterpret_cast<float4*>(out) = make_float4(top, den, dtop, 0.f);
          *reinterpret_cast<float4*>(out + 4 + d * 4) = sum;
        }
      }
    }
    if (CLUSTER) {
      auto all = cg::this_cluster();
      const int ranks = gridDim.x, here = (n_at + kE4Slice - 1) / kE4Slice;              // slices that are there
      if (ranks > 1) all.sync();
      else __syncthreads();
      for (int i = threadIdx.x + blockIdx.x * (kE4Warps * 32); i < heads * (D / 4); i += ranks * (kE4Warps * 32)) {
        const int head = i / (D / 4), d = i % (D / 4), at_sh = head * D + ((d ^ (head >> 1 & 3)) << 2);
        float4 sum = make_float4(0.f, 0.f, 0.f, 0.f), x[8], mld[8];
        float top = -INFINITY, dtop = -INFINITY, den = 0.f;
#pragma unroll
        for (int k = 0; k < 8; ++k)
          if (k < here) {
            mld[k] = *all.map_shared_rank(&mld_sh[head], k);
            x[k] = *reinterpret_cast<const float4*>(all.map_shared_rank(merge + at_sh, k));
            top = fmaxf(top, mld[k].x);
            dtop = fmaxf(dtop, mld[k].z);
          }
#pragma unroll
        for (int k = 0; k < 8; ++k)
          if (k < here) {
            const float f = e4_factor(mld[k].x, top);
            sum.x = fmaf(x[k].x, f, sum.x);
            sum.y = fmaf(x[k].y, f, sum.y);
            sum.z = fmaf(x[k].z, f, sum.z);
            sum.w = fmaf(x[k].w, f, sum.w);
            den = fmaf(mld[k].y, e4_factor(mld[k].z, dtop), den);
          }
        const float inv = here > 0 ? 1.f / den : 0.f;                    // without tokens the sums are zero
        e4_put4(reinterpret_cast<T*>(a.out) + at.b * a.ld_o + (static_cast<long long>(at.hk) * group + h0 + head) * D + d * 4, sum, inv, e4_size(top, dtop));
      }
      if (a.accumulate) {
        if (static_cast<int>(threadIdx.x) < heads) {
          float4 mld[8];
          float top = -INFINITY, den = 0.f;
#pragma unroll
          for (int k = 0; k < 8; ++k)
            if (k < here) {
              mld[k] = *all.map_shared_rank(&mld_sh[threadIdx.x], k);
              top = fmaxf(top, mld[k].z);
            }
#pragma unroll
          for (int k = 0; k < 8; ++k)
            if (k < here) den = fmaf(mld[k].y, e4_factor(mld[k].z, top), den);
          norm_sh[threadIdx.x] = e4_norm_of(top, den);
        }
        __syncthreads();
        for (int t = threadIdx.x; t < min(kE4Slice, n_at - at.s * kE4Slice); t += kE4Warps * 32) {
          float w = 0.f;
          for (int h = 0; h < heads; ++h) w = fmaf(e4_ex2(scores_sh[t * heads + h] - norm_sh[h].x), norm_sh[h].y, w);
          const int token = at.s * kE4Slice + t;
          const int page = e4_page(a.block_tables, a.max_blocks, a.pages.num_blocks, at.b, token / bs);
          if (page >= 0) a.pages.weight[(static_cast<long long>(page) * G + at.hk) * bs + token % bs] += w;
        }
      }
      if (ranks > 1) all.sync();                     // others may still read this CTA's sums
    }
    if (!LIST || at.left <= 1) break;
    __syncthreads();
    fresh = next.b != at.b || next.hk != at.hk;
    at = next;
    n_at = n_next;
    exps = exps_next;
    next = then;
    n_next = n_then;
    if (abort_sh) {                                  // a copy did not arrive: no new ones
      next.left = then.left = 0;
      n_next = 0;
      page_then = kNone;
    }
    locate(next, page_then, tile_next, where);
    exps_next = exps_of(tile_next, where);
    advance(then, n_then);
    page_then = look_up(then, n_then);
  }
}

// Adds the slices of a sequence for one head: 16 chains of every 16th slice, in order (with more than 64 slices 64 chains), then the chains in order.
// COLS: 16-byte columns that a CTA takes, D / 4 of 128 threads or, MANY, where sequences may have more than 64 slices, 8 of 512 threads: one of 131072
// tokens takes 24 us with 128 threads and 16 chains, 6.4 so.  Grid: (heads, sequences, D / 4 / COLS).
template <typename T, int COLS, bool MANY>
__global__ void __launch_bounds__(MANY ? 512 : 128)
e4_merge_kernel(const RbE4m3DecodeArgs a, int slices) {
  pdl_wait();
  pdl_launch();
  constexpr int kChains = MANY ? 64 : 16, R = (MANY ? 512 : 128) / COLS, PER = kChains / R;
  __shared__ float4 sum_sh[kChains][COLS];
  __shared__ float4 mld_sh[kChains];                 // maximum, denominator, its maximum
  const int h = blockIdx.x, b = blockIdx.y, z = blockIdx.z, tid = threadIdx.x, D = a.pages.head_dim, c = tid % COLS, r = tid / COLS;
  T* out = reinterpret_cast<T*>(a.out) + b * a.ld_o + static_cast<long long>(h) * D + z * (COLS * 4);
  const int here = (e4_len(a, b) + kE4Slice - 1) / kE4Slice;
  if (here == 0) {
    if (tid < COLS * 4) e4_put(out + tid, 0.f);
    return;
  }
  if (here == 1 && !a.accumulate) return;            // already written
  const int chains = MANY && here <= 64 ? 16 : kChains;
  const float* first = e4_partial(a.scratch, a.heads, slices, D, b, h, 0);
  const long long pitch = D + 4;
  // Every sum beside its own maximum; a new maximum's factor is a power of two, so that the sums are those under the largest of all.  The maxima and
  // denominators of a chain, the same for all its columns, are looked after by one lane for each slice that is loaded together, and factors come from there.
  constexpr int kAhead = PER == 1 ? 8 : 1;           // slices of a chain that are loaded together
  constexpr int kHeads = PER * kAhead;
  static_assert(kHeads <= COLS, "a lane for every slice");
  const uint32_t group = COLS == 32 ? 0xffffffffu : ((1u << COLS) - 1) << (tid & 31 & ~(COLS - 1));
  const int ck = c / kAhead, ci = c % kAhead;
  float4 sum[PER];
  float m = -INFINITY, l = 0.f, dm = -INFINITY;      // of chain r + ck * R
#pragma unroll
  for (int k = 0; k < PER; ++k) sum[k] = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int s0 = r; s0 < here && (!MANY || r < chains); s0 += chains * kAhead) {
    float4 x[PER][kAhead], mld = make_float4(-INFINITY, 0.f, -INFINITY, 0.f);
    if (c < kHeads && s0 + ck * R + ci * chains < here) mld = *reinterpret_cast<const float4*>(first + (s0 + ck * R + ci * chains) * pitch);
#pragma unroll
    for (int k = 0; k < PER; ++k) {
#pragma unroll
      for (int i = 0; i < kAhead; ++i) {
        const int s = s0 + k * R + i * chains;
        x[k][i] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (s < here) x[k][i] = *reinterpret_cast<const float4*>(first + s * pitch + 4 + (z * COLS + c) * 4);
      }
    }
    float to = mld.x, dto = mld.z;
#pragma unroll
    for (int o = 1; o < kAhead; o <<= 1) {
      to = fmaxf(to, __shfl_xor_sync(group, to, o, COLS));
      dto = fmaxf(dto, __shfl_xor_sync(group, dto, o, COLS));
    }
    to = fmaxf(to, m);
    dto = fmaxf(dto, dm);
    const float f = e4_factor(m, to), g = e4_factor(mld.x, to), den = mld.y * e4_factor(mld.z, dto);
    l *= e4_factor(dm, dto);
    if (kAhead == 1) l += den;
    else
#pragma unroll
      for (int i = 0; i < kAhead; ++i) l += __shfl_sync(group, den, i, COLS);
    m = to;
    dm = dto;
#pragma unroll
    for (int k = 0; k < PER; ++k) {
      const float fk = __shfl_sync(group, f, k * kAhead, COLS);
      sum[k].x *= fk; sum[k].y *= fk; sum[k].z *= fk; sum[k].w *= fk;
#pragma unroll
      for (int i = 0; i < kAhead; ++i) {             // of a slice that is not there: zero
        const float gk = __shfl_sync(group, g, k * kAhead + i, COLS);
        sum[k].x = fmaf(x[k][i].x, gk, sum[k].x);
        sum[k].y = fmaf(x[k][i].y, gk, sum[k].y);
        sum[k].z = fmaf(x[k][i].z, gk, sum[k].z);
        sum[k].w = fmaf(x[k][i].w, gk, sum[k].w);
      }
    }
  }
#pragma unroll
  for (int k = 0; k < PER; ++k) sum_sh[r + k * R][c] = sum[k];
  if (c < kHeads && ci == 0) mld_sh[r + ck * R] = make_float4(m, l, dm, 0.f);
  __syncthreads();
  if (tid >= 32) return;
  // a lane forms the factors of its chains, so that no thread holds those of all
  constexpr int kMine = (kChains + 31) / 32;
  float4 mld[kMine];
  float f[kMine], lf[kMine], top = -INFINITY, dtop = -INFINITY, den = 0.f;
#pragma unroll
  for (int i = 0; i < kMine; ++i) {                  // -infinity where there is no such slice
    mld[i] = tid + 32 * i < kChains ? mld_sh[tid + 32 * i] : make_float4(-INFINITY, 0.f, -INFINITY, 0.f);
    top = fmaxf(top, mld[i].x);
    dtop = fmaxf(dtop, mld[i].z);
  }
  top = warp_max(top);
  dtop = warp_max(dtop);
#pragma unroll
  for (int i = 0; i < kMine; ++i) {
    f[i] = e4_factor(mld[i].x, top);
    lf[i] = mld[i].y * e4_factor(mld[i].z, dtop);
  }
  float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 16
  for (int k = 0; k < kChains; ++k) {
    const float fk = __shfl_sync(0xffffffffu, f[MANY ? k >> 5 : 0], k & 31), lk = __shfl_sync(0xffffffffu, lf[MANY ? k >> 5 : 0], k & 31);
    if (k < here && k < chains) {
      const float4 x = sum_sh[k][c];
      o.x = fmaf(x.x, fk, o.x);
      o.y = fmaf(x.y, fk, o.y);
      o.z = fmaf(x.z, fk, o.z);
      o.w = fmaf(x.w, fk, o.w);
      den += lk;
    }
  }
  if (here > 1 && tid < COLS) e4_put4(out + c * 4, o, 1.f / den, e4_size(top, dtop));
  if (a.accumulate && tid == 0 && z == 0) *e4_norm(a, slices, b, h) = e4_norm_of(dtop, den);
}

// Adds the attention weights of a slice to its tokens' sums, a thread a token.  (As a part of the merge, with denominators formed in every CTA, it was
// slower, 33 against 30 us for 24 sequences of 128 to 2560: the merge's registers leave room for fewer of its threads, and it waits for memory.)
__global__ void __launch_bounds__(kE4Slice)
e4_weight_kernel(const RbE4m3DecodeArgs a, int slices) {
  pdl_wait();
  pdl_launch();
  const int hk = blockIdx.y, b = blockIdx.z, bs = a.pages.block_size, G = a.pages.kv_heads, group = a.heads / G;
  const int t = blockIdx.x * kE4Slice + threadIdx.x;
  if (t >= e4_len(a, b)) return;
  const int page = e4_page(a.block_tables, a.max_blocks, a.pages.num_blocks, b, t / bs);
  if (page < 0) return;
  float* to = a.pages.weight + (static_cast<long long>(page) * G + hk) * bs + t % bs;
  const float* scores = a.scratch + static_cast<long long>(a.batch) * a.heads * slices * (a.pages.head_dim + 4) +
                        ((static_cast<long long>(b) * G + hk) * slices * kE4Slice + t) * group;
  const float2* norms = e4_norm(a, slices, b, hk * group);
  float w = 0.f;
  if (group % 4 == 0) {
    for (int h = 0; h < group; h += 4) {
      const float4 s = *reinterpret_cast<const float4*>(scores + h);
      w = fmaf(e4_ex2(s.x - norms[h].x), norms[h].y, w);
      w = fmaf(e4_ex2(s.y - norms[h + 1].x), norms[h + 1].y, w);
      w = fmaf(e4_ex2(s.z - norms[h + 2].x), norms[h + 2].y, w);
      w = fmaf(e4_ex2(s.w - norms[h + 3].x), norms[h + 3].y, w);
    }
  } else {
    for (int h = 0; h < group; ++h) w = fmaf(e4_ex2(scores[h] - norms[h].x), norms[h].y, w);
  }
  *to += w;
}

}  // namespace rb

namespace {
long long e4_slices(int max_blocks, int block_size) {
  return (static_cast<long long>(max_blocks) * block_size + rb::kE4Slice - 1) / rb::kE4Slice;
}
// Whether the CTAs of a sequence and KV head merge as a cluster: few slices, heads for one pass, and no more CTAs than fit on the GPU at a time (three on an
// SM).  It goes by what the tables have room for, which the host knows, not by the lengths: a captured step whose tables are as wide as the context plans for that.
// One B200, us from a captured graph, as a cluster / with a list or grid and its merge: one sequence of 300, 12 KV heads of 64 5.5 / 6.8; of 2047, 4 KV heads of
// 128, with weights 8.7 / 9.9 (as calls 11.1 / 17.1: two launches less); 48 of 16 to 1024, 8 KV heads of 64, 1536 CTAs, many without a token, 20.7 / 16.2.
bool in_clusters(int batch, int kv_heads, long long slices, int group) {
  return slices <= 8 && group <= 16 && batch * kv_heads * slices <= 3ll * rbhost::device_sm_count();
}
template <typename T, int D, int NH>
int decode_launch(const RbE4m3DecodeArgs& a, cudaStream_t stream) {
  using L = rb::E4Layout<D, NH>;
  const RbPagesE4m3& p = a.pages;
  const int slices = static_cast<int>(e4_slices(a.max_blocks, p.block_size));
  const uint64_t rows = static_cast<uint64_t>(p.num_blocks) * p.kv_heads * p.block_size * D / 128;
  if (rows > 0x7fffffffull) return -1;               // a copy's row is a 32-bit number
  int err = 0;
  const CUtensorMap* km = rbhost::get_tmap_2d(p.k, 1, 128, rows, 128, 128, D / 8, 1, &err);
  const CUtensorMap* vm = km ? rbhost::get_tmap_2d(p.v, 1, 128, rows, 128, 128, D / 8, 1, &err) : nullptr;
  unsigned int* status = rbhost::status_ptr();
  if (!vm || !status) return err ? err : -3;
  const int group = a.heads / p.kv_heads, most = group < NH * 8 ? group : NH * 8, smem = L::bytes(most < L::kRound ? most : L::kRound);
  static int per_sm[NH * 8 + 1][64] = {};            // CTAs of a list that fit on an SM, by the heads that a pass has
  const int dev = rbhost::device_slot();
  if (!per_sm[most][dev]) {
    const int bytes = L::bytes(NH * 8) + rb::kE4Slice * NH * 8 * 4;
    cudaError_t e = cudaFuncSetAttribute(rb::e4_decode_kernel<T, D, NH, rb::kE4List>, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e == cudaSuccess) e = cudaFuncSetAttribute(rb::e4_decode_kernel<T, D, NH, rb::kE4Grid>, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e == cudaSuccess) e = cudaFuncSetAttribute(rb::e4_decode_kernel<T, D, NH, rb::kE4Cluster>, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    int n = 0;
    if (e == cudaSuccess) e = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, rb::e4_decode_kernel<T, D, NH, rb::kE4List>, rb::kE4Warps * 32, smem);
    if (e != cudaSuccess) return static_cast<int>(e);
    per_sm[most][dev] = n > 0 ? n : 1;
  }
  const dim3 threads(rb::kE4Warps * 32), whole(slices, p.kv_heads, a.batch);
  if (in_clusters(a.batch, p.kv_heads, slices, group))
    return static_cast<int>(rbhost::launch_pdl(rb::e4_decode_kernel<T, D, NH, rb::kE4Cluster>, whole, threads,
                                               L::bytes(most) + (a.accumulate ? rb::kE4Slice * most * 4 : 0), stream, slices, *km, *vm, a, 0, slices, status RB_BOUNDS_ARG));
  const int some = per_sm[most][dev] * rbhost::device_sm_count();
  const bool list = static_cast<long long>(a.batch) * p.kv_heads * slices > some;
  auto kern = list ? rb::e4_decode_kernel<T, D, NH, rb::kE4List> : rb::e4_decode_kernel<T, D, NH, rb::kE4Grid>;
  cudaError_t e = cudaSuccess;
  for (int h0 = 0; h0 < group && e == cudaSuccess; h0 += NH * 8)        // wider groups take several passes
    e = rbhost::launch_pdl(kern, list ? dim3(some) : whole, threads, smem, stream, 1, *km, *vm, a, h0, slices, status RB_BOUNDS_ARG);
  if (e == cudaSuccess) {
    const bool many = slices > 64;
    e = rbhost::launch_pdl(many ? rb::e4_merge_kernel<T, 8, true> : rb::e4_merge_kernel<T, D / 4, false>, dim3(a.heads, a.batch, many ? D / 32 : 1),
                           dim3(many ? 512 : 128), 0, stream, 1, a, slices);
  }
  if (e == cudaSuccess && a.accumulate) e = rbhost::launch_pdl(rb::e4_weight_kernel, whole, dim3(rb::kE4Slice), 0, stream, 1, a, slices);
  return static_cast<int>(e);
}
template <typename T>
int decode_by_dim(const RbE4m3DecodeArgs& a, cudaStream_t s) {
  const bool narrow = a.heads / a.pages.kv_heads <= 8;
  if (a.pages.head_dim == 64) return narrow ? decode_launch<T, 64, 1>(a, s) : decode_launch<T, 64, 2>(a, s);
  return narrow ? decode_launch<T, 128, 1>(a, s) : decode_launch<T, 128, 2>(a, s);
}
}  // namespace

RB_API long long rb_e4m3_decode_scratch_floats(int batch, int heads, int kv_heads, int head_dim, int max_blocks, int block_size, int accumulate) {
  const long long slices = e4_slices(max_blocks, block_size), rows = static_cast<long long>(batch) * heads;
  if (in_clusters(batch, kv_heads, slices, heads / kv_heads)) return 0;
  return rows * slices * (head_dim + 4) + (accumulate ? rows * (slices * rb::kE4Slice + 2) : 0);
}

RB_API int rb_e4m3_decode(const RbE4m3DecodeArgs* args, void* stream_v) {
  const RbE4m3DecodeArgs& a = *args;
  if (a.batch <= 0) return 0;
  if (const int bad = rbhost::e4_check(a.pages)) return bad;
  if (!a.q || !a.out || !a.block_tables || !a.context_lens || a.max_blocks <= 0 || a.heads <= 0 || a.heads % a.pages.kv_heads ||
      (!a.scratch && !in_clusters(a.batch, a.pages.kv_heads, e4_slices(a.max_blocks, a.pages.block_size), a.heads / a.pages.kv_heads)) ||
      a.batch > 65535 || a.pages.kv_heads > 65535 || (a.accumulate && !a.pages.weight) || static_cast<long long>(a.max_blocks) * a.pages.block_size > 0x3fffffff ||
      static_cast<long long>(a.batch) * a.pages.kv_heads * e4_slices(a.max_blocks, a.pages.block_size) > 0x3fffffff)
    return -1;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream_v);
  switch (a.type) {
    case RB_E4M3_BF16: return decode_by_dim<__nv_bfloat16>(a, s);
    case RB_E4M3_F16: return decode_by_dim<__half>(a, s);
  }
  return -1;
}
