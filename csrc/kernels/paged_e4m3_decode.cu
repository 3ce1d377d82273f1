// Attention of single tokens over a paged cache in e4m3, with an optional sum of the attention weights of every cached token.
//
// With key j's score s_j (base 2: scale, log2 e and the keys' exponent included) and the exponent e_j of its value's tile, the output is
// sum_j 2^(s_j) 2^(e_j) c_j / sum_j 2^(s_j).  The maximum M that keeps the numbers in range is taken over s_j + e_j: the factors p_j = 2^(s_j + e_j - M)
// of the codes are then at most 1 whatever the tiles' exponents, and the denominator is summed in fp32 from p_j 2^(-e_j).  M is rounded up to a whole
// number, so that M - e_j and the factors that bring sums from one M to another are exact; with exponents of -100 a fractional M would cost the
// scores seven bits.
#include "pdl.cuh"
#include "paged_e4m3.cuh"

namespace rb {

constexpr int kE4Slice = 256;                        // tokens whose sums one CTA forms; the merge goes over them in order
constexpr int kE4Heads = 8;                          // query heads at a time

__device__ __forceinline__ float e4_ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float e4_get(const __nv_bfloat16* p) { return __bfloat162float(*p); }
__device__ __forceinline__ float e4_get(const __half* p) { return __half2float(*p); }
__device__ __forceinline__ void e4_put(__nv_bfloat16* p, float v) { *p = __float2bfloat16(v); }
__device__ __forceinline__ void e4_put(__half* p, float v) { *p = __float2half(v); }

// Scratch: [batch, heads, slices, D + 2] fp32: maximum, denominator, sums of a slice; then, where weights are summed, the scores
// [batch, heads, slices * 256] and the denominators as whole powers of two and factors [batch, heads, 2].
__device__ __forceinline__ float* e4_partial(float* scratch, int heads, int slices, int D, int b, int h, int s) {
  return scratch + ((static_cast<long long>(b) * heads + h) * slices + s) * (D + 2);
}

__device__ __forceinline__ float* e4_norm(float* scratch, int batch, int heads, int slices, int D, int b, int h) {
  const long long rows = static_cast<long long>(batch) * heads;
  return scratch + rows * slices * (D + 2 + kE4Slice) + (static_cast<long long>(b) * heads + h) * 2;
}

template <typename T, int D>
__global__ void __launch_bounds__(128)
e4_decode_kernel(const RbE4m3DecodeArgs a, int slices RB_BOUNDS_PARAM) {
  pdl_wait();
  pdl_launch();
  __shared__ float q_sh[kE4Heads][D];
  __shared__ float s_sh[kE4Heads][kE4Slice];
  __shared__ long long tile_sh[kE4Slice / 16];
  __shared__ float red[4];
  const int s = blockIdx.x, hk = blockIdx.y, b = blockIdx.z, tid = threadIdx.x;
  const int bs = a.pages.block_size, G = a.pages.kv_heads, group = a.heads / G;
  const int n = min(static_cast<long long>(a.context_lens[b]), static_cast<long long>(a.max_blocks) * bs) - static_cast<long long>(s) * kE4Slice;
  if (n <= 0) return;
  const int here = min(n, kE4Slice);
  if (tid < kE4Slice / 16) {
    const int t = s * kE4Slice + tid * 16;
    int page = tid * 16 < here ? e4_page(a.block_tables, a.max_blocks, a.pages.num_blocks, b, t / bs) : 0;
    if (page < 0) {                                  // corrupt tables read block 0 instead of faulting
      RB_BOUNDS_HIT(104);
      page = 0;
    }
    tile_sh[tid] = (static_cast<long long>(page) * G + hk) * bs + t % bs;          // token in the cache
  }
  __syncthreads();
  const uint8_t* K = reinterpret_cast<const uint8_t*>(a.pages.k);
  const uint8_t* V = reinterpret_cast<const uint8_t*>(a.pages.v);
  const float scale = a.scale * 1.4426950408889634f;
  for (int h0 = 0; h0 < group; h0 += kE4Heads) {
    const int heads = min(kE4Heads, group - h0), head = hk * group + h0;
    for (int i = tid; i < heads * D; i += 128)
      q_sh[i / D][i % D] = e4_get(reinterpret_cast<const T*>(a.q) + b * a.ld_q + static_cast<long long>(head) * D + i);
    __syncthreads();
    for (int t = tid; t < here; t += 128) {
      const long long at = tile_sh[t >> 4] + (t & 15);
      float acc[kE4Heads];
#pragma unroll
      for (int h = 0; h < kE4Heads; ++h) acc[h] = 0.f;
      for (int c = 0; c < D; c += 4) {
        const uint32_t u = *reinterpret_cast<const uint32_t*>(K + at * D + c);
        const float2 x = e4_float2(u), y = e4_float2(u >> 16);
#pragma unroll
        for (int h = 0; h < kE4Heads; ++h)
          acc[h] += q_sh[h][c] * x.x + q_sh[h][c + 1] * x.y + q_sh[h][c + 2] * y.x + q_sh[h][c + 3] * y.y;
      }
      const float up = e4_two(a.pages.k_exp[at / bs]) * scale;
#pragma unroll
      for (int h = 0; h < kE4Heads; ++h) s_sh[h][t] = acc[h] * up;
    }
    __syncthreads();
    for (int h = 0; h < heads; ++h) {
      float m = -INFINITY;
      for (int t = tid; t < here; t += 128) m = fmaxf(m, ceilf(s_sh[h][t]) + a.pages.v_exp[(tile_sh[t >> 4]) / bs]);
      m = warp_max(m);
      if ((tid & 31) == 0) red[tid >> 5] = m;
      __syncthreads();
      m = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
      __syncthreads();
      if (a.accumulate) {
        float* scores = a.scratch + static_cast<long long>(a.batch) * a.heads * slices * (D + 2) +
                        (static_cast<long long>(b) * a.heads + head + h) * slices * kE4Slice + s * kE4Slice;
        for (int t = tid; t < here; t += 128) scores[t] = s_sh[h][t];
      }
      float l = 0.f;
      for (int t = tid; t < here; t += 128) {
        const int e = a.pages.v_exp[(tile_sh[t >> 4]) / bs];
        const float p = e4_ex2(s_sh[h][t] - (m - e));
        l = fmaf(p, e4_two(-e), l);
        s_sh[h][t] = p;
      }
      l = warp_sum(l);
      if ((tid & 31) == 0) red[tid >> 5] = l;
      __syncthreads();
      float* out = e4_partial(a.scratch, a.heads, slices, D, b, head + h, s);
      if (tid == 0) {
        out[0] = m;
        out[1] = (red[0] + red[1]) + (red[2] + red[3]);
      }
      if (tid < D) {
        float o = 0.f;
        for (int t = 0; t < here; ++t) {
          const uint8_t* v = V + (tile_sh[t >> 4] + (t & 15)) * D + (tid & ~1);
          const float2 x = e4_float2(*reinterpret_cast<const uint16_t*>(v));
          o = fmaf(s_sh[h][t], tid & 1 ? x.y : x.x, o);
        }
        out[2 + tid] = o;
      }
      __syncthreads();
    }
  }
}

template <typename T>
__global__ void __launch_bounds__(128)
e4_merge_kernel(const RbE4m3DecodeArgs a, int slices) {
  pdl_wait();
  pdl_launch();
  const int h = blockIdx.x, b = blockIdx.y, tid = threadIdx.x, D = a.pages.head_dim;
  const long long len = min(static_cast<long long>(a.context_lens[b]), static_cast<long long>(a.max_blocks) * a.pages.block_size);
  const int here = len <= 0 ? 0 : static_cast<int>((len + kE4Slice - 1) / kE4Slice);
  float m = -INFINITY;
  for (int s = 0; s < here; ++s) m = fmaxf(m, e4_partial(a.scratch, a.heads, slices, D, b, h, s)[0]);
  float l = 0.f, o = 0.f;
  for (int s = 0; s < here; ++s) {
    const float* p = e4_partial(a.scratch, a.heads, slices, D, b, h, s);
    const float f = e4_ex2(p[0] - m);
    l = fmaf(p[1], f, l);
    if (tid < D) o = fmaf(p[2 + tid], f, o);
  }
  if (tid < D) e4_put(reinterpret_cast<T*>(a.out) + b * a.ld_o + static_cast<long long>(h) * D + tid, here ? o / l : 0.f);
  if (a.accumulate && tid == 0 && here) {
    // a weight is 2^(s - m) / l = 2^(s - (m + x)) / (l / 2^x), with the x that brings l / 2^x into [1, 2)
    const int x = static_cast<int>(__float_as_uint(l) >> 23) - 127;
    float* norm = e4_norm(a.scratch, a.batch, a.heads, slices, D, b, h);
    norm[0] = m + static_cast<float>(x);
    norm[1] = e4_two(x) / l;
  }
}

__global__ void __launch_bounds__(256)
e4_weight_kernel(const RbE4m3DecodeArgs a, int slices) {
  pdl_wait();
  pdl_launch();
  const int s = blockIdx.x, hk = blockIdx.y, b = blockIdx.z, D = a.pages.head_dim;
  const int bs = a.pages.block_size, G = a.pages.kv_heads, group = a.heads / G;
  const long long t = static_cast<long long>(s) * kE4Slice + threadIdx.x;
  if (t >= min(static_cast<long long>(a.context_lens[b]), static_cast<long long>(a.max_blocks) * bs)) return;
  const float* scores = a.scratch + static_cast<long long>(a.batch) * a.heads * slices * (D + 2);
  float w = 0.f;
  for (int h = 0; h < group; ++h) {
    const long long row = static_cast<long long>(b) * a.heads + hk * group + h;
    const float* norm = e4_norm(a.scratch, a.batch, a.heads, slices, D, b, hk * group + h);
    w = fmaf(e4_ex2(scores[row * slices * kE4Slice + t] - norm[0]), norm[1], w);
  }
  const int page = e4_page(a.block_tables, a.max_blocks, a.pages.num_blocks, b, static_cast<int>(t / bs));
  if (page >= 0) a.pages.weight[(static_cast<long long>(page) * G + hk) * bs + t % bs] += w;
}

}  // namespace rb

namespace {
long long e4_slices(int max_blocks, int block_size) {
  return (static_cast<long long>(max_blocks) * block_size + rb::kE4Slice - 1) / rb::kE4Slice;
}
template <typename T>
int decode_by_dim(const RbE4m3DecodeArgs& a, cudaStream_t s) {
  const int slices = static_cast<int>(e4_slices(a.max_blocks, a.pages.block_size));
  auto kern = a.pages.head_dim == 64 ? rb::e4_decode_kernel<T, 64> : rb::e4_decode_kernel<T, 128>;
  const dim3 grid(slices, a.pages.kv_heads, a.batch);
  cudaError_t e = rbhost::launch_pdl(kern, grid, dim3(128), 0, s, 1, a, slices RB_BOUNDS_ARG);
  if (e == cudaSuccess) e = rbhost::launch_pdl(rb::e4_merge_kernel<T>, dim3(a.heads, a.batch), dim3(128), 0, s, 1, a, slices);
  if (e == cudaSuccess && a.accumulate) e = rbhost::launch_pdl(rb::e4_weight_kernel, grid, dim3(256), 0, s, 1, a, slices);
  return static_cast<int>(e);
}
}  // namespace

RB_API long long rb_e4m3_decode_scratch_floats(int batch, int heads, int head_dim, int max_blocks, int block_size, int accumulate) {
  const long long slices = e4_slices(max_blocks, block_size), rows = static_cast<long long>(batch) * heads;
  return rows * slices * (head_dim + 2) + (accumulate ? rows * (slices * rb::kE4Slice + 2) : 0);
}

RB_API int rb_e4m3_decode(const RbE4m3DecodeArgs* args, void* stream_v) {
  const RbE4m3DecodeArgs& a = *args;
  if (a.batch <= 0) return 0;
  if (const int bad = rbhost::e4_check(a.pages)) return bad;
  if (!a.q || !a.out || !a.block_tables || !a.context_lens || !a.scratch || a.max_blocks <= 0 || a.heads <= 0 || a.heads % a.pages.kv_heads ||
      a.batch > 65535 || a.pages.kv_heads > 65535 || (a.accumulate && !a.pages.weight) || e4_slices(a.max_blocks, a.pages.block_size) > 0x7fffff)
    return -1;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream_v);
  switch (a.type) {
    case RB_E4M3_BF16: return decode_by_dim<__nv_bfloat16>(a, s);
    case RB_E4M3_F16: return decode_by_dim<__half>(a, s);
  }
  return -1;
}
