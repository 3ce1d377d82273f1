// Beam search's selection: log-softmax of every beam's logits, sums with the beams' scores, and the best continuations over beams and vocabulary, with
// no array of sums ever written.
//
// total(r, t) = s_r + x_rt - L_r, L_r = log sum_u exp x_ru.  Within a row the order of totals is the order of the logits, so a row's best `count`
// logits are found before L_r is known, in the same pass over the logits that sums the exponentials: the logits are read once.  A CTA holds a piece of a row in registers; it
// leaves the piece's maximum, the sum under it, and its best logits.  A second launch, a CTA for each group, joins the pieces' sums and orders
// the candidates of all its rows by s_r + x - L_r in 64 bits: two continuations of different beams are often closer than 32 bits of a sum can tell,
// and the one selected must not depend on how the sum was rounded.  Beams that have ended or have a score of minus infinity are not read.
//
// The best n of a set that lies in the registers of many threads: the n-th largest of the threads' own maxima is a lower bound of the n-th largest
// number (found by its bits, most significant first, with one count over the CTA per bit); numbers not below it, little more than n, go to a list, and a number's
// place is the count of those before it.  Where equal numbers overflow the list the best are taken one after the other.
#include "beam.h"

#include <cuda_fp16.h>
#include <float.h>

#include "pdl.cuh"
#include "rb_common.cuh"

namespace rb {

constexpr int kBsThreads = 256;
constexpr int kBsMostCount = 128;
constexpr int kBsMostBeams = 256;
constexpr int kBsList = 1024;                    // room for the numbers that are not below the bound

struct BsStat {
  float most, sum;                               // of a piece of a row: its maximum and the sum of exp(x - maximum)
};
struct BsCandidate {
  float x;
  int token;                                     // -1: none
};
struct BsParams {
  const void* logits;
  const float* scores;
  const unsigned char* ended;
  float* out_scores;
  long long* out_rows;
  long long* out_tokens;
  BsStat* stats;                                 // [rows, pieces]
  BsCandidate* found;                            // [rows, pieces, count]
  long long ld;
  int groups, beams, vocab, count, end_token, pieces, piece;
  int vec;                                       // elements of a load: 16 bytes, or one where rows do not begin on 16 bytes
};

__device__ __forceinline__ float bs_value(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float bs_value(__half v) { return __half2float(v); }
__device__ __forceinline__ float bs_value(float v) { return v; }
// NaN is minus infinity, plus infinity the largest number
__device__ __forceinline__ float bs_clean(float v) { return v != v ? -INFINITY : fminf(v, FLT_MAX); }
// Order of the numbers as order of whole numbers; minus infinity is the least, and no number gives 0.
__device__ __forceinline__ uint32_t bs_key(float v) {
  v += 0.f;                                      // -0 and 0 are equal
  const uint32_t u = __float_as_uint(v);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
constexpr uint32_t kBsLeast = 0x007fffffu;       // bs_key(-infinity)

__device__ __forceinline__ bool bs_live(const BsParams& p, int row) {
  const float s = bs_clean(p.scores[row]);
  return s != -INFINITY && !(p.ended && p.ended[row]);
}

// The n-th largest key of the CTA's threads (one key each), 1 <= n <= blockDim.x.  Every thread gets it.
__device__ __forceinline__ uint32_t bs_nth(uint32_t key, int n, int lowest_bit) {
  uint32_t at = 0;
  for (int bit = 31; bit >= lowest_bit; --bit) {
    const uint32_t with = at | 1u << bit;
    const int c = __syncthreads_count(key >= with);
    if (c >= n) at = with;
    if (c == n) break;                           // exactly the n largest are not below `with`
  }
  return at;
}

// ---- a piece of a row --------------------------------------------------------------------------------------------------------------------
// E: elements of a thread
template <typename T, int E>
__global__ void __launch_bounds__(kBsThreads)
beam_rows_kernel(const BsParams p) {
  pdl_wait();
  pdl_launch();
  const int row = blockIdx.x, piece = blockIdx.y;
  if (!bs_live(p, row)) return;
  constexpr int V = 16 / sizeof(T);              // elements of a wide load
  const T* x = static_cast<const T*>(p.logits) + static_cast<long long>(row) * p.ld;
  const int first = piece * p.piece, end = min(p.vocab, first + p.piece);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  // element e of a thread is number first + (e / V) * 256 V + tid * V + e % V
  float v[E];
#pragma unroll
  for (int j = 0; j < E / V; ++j) {
    const int at = first + (j * kBsThreads + tid) * V;
    if (p.vec > 1 && at + V <= end) {
      const uint4 u = __ldcs(reinterpret_cast<const uint4*>(x + at));
      const T* w = reinterpret_cast<const T*>(&u);
#pragma unroll
      for (int i = 0; i < V; ++i) v[j * V + i] = bs_clean(bs_value(w[i]));
    } else {
#pragma unroll
      for (int i = 0; i < V; ++i) v[j * V + i] = at + i < end ? bs_clean(bs_value(x[at + i])) : -INFINITY;
    }
  }
  float most = -INFINITY;
#pragma unroll
  for (int e = 0; e < E; ++e) most = fmaxf(most, v[e]);
  __shared__ float warp_most[kBsThreads / 32], warp_total[kBsThreads / 32];
  __shared__ int listed;
  __shared__ uint32_t list_key[kBsList];
  __shared__ int list_token[kBsList];
  const float wm = warp_max(most);
  if (lane == 0) warp_most[warp] = wm;
  if (tid == 0) listed = 0;
  __syncthreads();
  float top = warp_most[0];
#pragma unroll
  for (int w = 1; w < kBsThreads / 32; ++w) top = fmaxf(top, warp_most[w]);
  float sum = 0.f;
  if (top != -INFINITY)
#pragma unroll
    for (int e = 0; e < E; ++e) sum += __expf(v[e] - top);
  sum = warp_sum(sum);
  if (lane == 0) warp_total[warp] = sum;

  const long long place = static_cast<long long>(row) * p.pieces + piece;
  BsCandidate* found = p.found + place * p.count;
  const int n = p.count;
  // numbers of 16 bits have no lower bits in 32
  const uint32_t bound = max(bs_nth(bs_key(most), min(n, kBsThreads), sizeof(T) == 4 ? 0 : sizeof(T) == 2 ? 13 : 0), kBsLeast + 1);
  if (tid == 0) {
    float s = 0.f;
#pragma unroll
    for (int w = 0; w < kBsThreads / 32; ++w) s += warp_total[w];
    p.stats[place] = {top, s};
  }
  if (bs_key(most) >= bound) {
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const uint32_t k = bs_key(v[e]);
      if (k >= bound) {
        const int at = atomicAdd(&listed, 1);
        if (at < kBsList) {
          list_key[at] = k;
          list_token[at] = first + ((e / V) * kBsThreads + tid) * V + e % V;
        }
      }
    }
  }
  __syncthreads();
  const int m = listed;
  auto number = [](uint32_t k) { return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k); };
  if (m <= kBsList) {
    for (int i = tid; i < m; i += kBsThreads) {
      const uint32_t k = list_key[i];
      const int t = list_token[i];
      int before = 0;
      for (int j = 0; j < m; ++j) before += list_key[j] > k || (list_key[j] == k && list_token[j] < t) ? 1 : 0;
      if (before < n) found[before] = {number(k), t};
    }
    for (int i = m + tid; i < n; i += kBsThreads) found[i] = {0.f, -1};
    return;
  }
  // one after the other: the largest (key, lowest token) below the last
  __shared__ unsigned long long warp_best[kBsThreads / 32];
  unsigned long long last = ~0ull;
  for (int i = 0; i < n; ++i) {
    unsigned long long best = 0;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const int t = first + ((e / V) * kBsThreads + tid) * V + e % V;
      const uint32_t k = bs_key(v[e]);
      const unsigned long long c = static_cast<unsigned long long>(k) << 32 | (0xffffffffu - static_cast<uint32_t>(t));
      if (k > kBsLeast && c < last && c > best) best = c;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const unsigned long long other = __shfl_xor_sync(0xffffffffu, best, o);
      best = other > best ? other : best;
    }
    if (lane == 0) warp_best[warp] = best;
    __syncthreads();
    best = warp_best[0];
#pragma unroll
    for (int w = 1; w < kBsThreads / 32; ++w) best = warp_best[w] > best ? warp_best[w] : best;
    last = best;                                 // never 0: more than kBsList >= n numbers are above minus infinity
    if (tid == 0) found[i] = {number(static_cast<uint32_t>(best >> 32)), static_cast<int>(0xffffffffu - static_cast<uint32_t>(best))};
    __syncthreads();
  }
}

// ---- a group ---------------------------------------------------------------------------------------------------------------------------------
__device__ __forceinline__ unsigned long long bs_key64(double v) {
  v += 0.0;
  const unsigned long long u = static_cast<unsigned long long>(__double_as_longlong(v));
  return u >> 63 ? ~u : u | 0x8000000000000000ull;
}
__global__ void __launch_bounds__(kBsThreads)
beam_group_kernel(const BsParams p) {
  pdl_wait();
  pdl_launch();
  // of a row: its largest logit, and s_r - log sum exp(x - largest) (minus infinity: a row without continuations).  The largest is taken from a logit
  // before anything is added, so that logits of any size lose nothing.
  __shared__ double base[kBsMostBeams];
  __shared__ float row_most[kBsMostBeams];
  __shared__ int listed;
  __shared__ double list_total[kBsList];
  __shared__ int list_beam[kBsList], list_token[kBsList];
  __shared__ int chosen_token[kBsMostCount], chosen_beam[kBsMostCount];
  const int g = blockIdx.x, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int row0 = g * p.beams, per = p.pieces * p.count, total = p.beams * per + p.beams;
  const BsCandidate* found = p.found + static_cast<long long>(row0) * per;
  if (tid == 0) listed = 0;
  for (int r = warp; r < p.beams; r += kBsThreads / 32) {
    const float score = bs_clean(p.scores[row0 + r]);
    double b = -INFINITY;
    if (bs_live(p, row0 + r)) {
      const BsStat* st = p.stats + static_cast<long long>(row0 + r) * p.pieces;
      float most = -INFINITY;
      for (int i = lane; i < p.pieces; i += 32) most = fmaxf(most, st[i].most);
      most = warp_max(most);
      double sum = 0.0;
      if (most != -INFINITY)
        for (int i = lane; i < p.pieces; i += 32)
          if (st[i].most != -INFINITY) sum += static_cast<double>(st[i].sum) * exp(static_cast<double>(st[i].most) - most);
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
      if (most != -INFINITY) b = static_cast<double>(score) - log(sum);
      if (lane == 0) row_most[r] = most;
    }
    if (lane == 0) base[r] = b;
  }
  __syncthreads();
  // Candidate i: number i % per of row i / per, and behind them one for each ended row.
  auto candidate = [&](int i, double& t, int& token, int& beam) -> bool {
    if (i < p.beams * per) {
      beam = i / per;
      if (base[beam] == -INFINITY) return false;
      const BsCandidate c = found[i];
      token = c.token;
      t = base[beam] + (static_cast<double>(c.x) - row_most[beam]);
      return token >= 0;
    }
    beam = i - p.beams * per;
    token = p.end_token;
    t = static_cast<double>(bs_clean(p.scores[row0 + beam]));
    return p.ended && p.ended[row0 + beam] && t != -INFINITY;
  };
  const int n = p.count;
  uint32_t most = 0;
  for (int i = tid; i < total; i += kBsThreads) {
    double t;
    int token, beam;
    if (candidate(i, t, token, beam)) most = max(most, bs_key(fmaxf(static_cast<float>(t), -FLT_MAX)));
  }
  const uint32_t bound = max(bs_nth(most, min(n, kBsThreads), 0), kBsLeast + 1);
  if (most >= bound)
    for (int i = tid; i < total; i += kBsThreads) {
      double t;
      int token, beam;
      if (candidate(i, t, token, beam) && bs_key(fmaxf(static_cast<float>(t), -FLT_MAX)) >= bound) {
        const int at = atomicAdd(&listed, 1);
        if (at < kBsList) {
          list_total[at] = t;
          list_beam[at] = beam;
          list_token[at] = token;
        }
      }
    }
  __syncthreads();
  const int m = listed;
  int have;                                      // continuations that are not minus infinity, n at most
  auto put = [&](int i, double t, int beam, int token) {
    const long long o = static_cast<long long>(g) * n + i;
    p.out_scores[o] = static_cast<float>(t);
    p.out_rows[o] = row0 + beam;
    p.out_tokens[o] = token;
    chosen_beam[i] = beam;
    chosen_token[i] = token;
  };
  if (m <= kBsList) {
    for (int i = tid; i < m; i += kBsThreads) {
      const double t = list_total[i];
      const int beam = list_beam[i], token = list_token[i];
      int before = 0;
      for (int j = 0; j < m; ++j) {
        const double o = list_total[j];
        before += o > t || (o == t && (list_beam[j] < beam || (list_beam[j] == beam && list_token[j] < token))) ? 1 : 0;
      }
      if (before < n) put(before, t, beam, token);
    }
    have = min(m, n);
  } else {
    // one after the other: the largest (total, lowest row, lowest token) behind the last
    __shared__ unsigned long long warp_key[kBsThreads / 32], warp_order[kBsThreads / 32];
    unsigned long long last_key = ~0ull, last_order = 0;
    for (int i = 0; i < n; ++i) {
      unsigned long long key = 0, order = ~0ull;
      for (int c = tid; c < total; c += kBsThreads) {
        double t;
        int token, beam;
        if (!candidate(c, t, token, beam)) continue;
        const unsigned long long k = bs_key64(t), o = static_cast<unsigned long long>(beam) << 32 | static_cast<unsigned int>(token);
        const bool behind = k < last_key || (k == last_key && o > last_order);
        if (behind && (k > key || (k == key && o < order))) { key = k; order = o; }
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) {
        const unsigned long long k = __shfl_xor_sync(0xffffffffu, key, o), w = __shfl_xor_sync(0xffffffffu, order, o);
        if (k > key || (k == key && w < order)) { key = k; order = w; }
      }
      if (lane == 0) { warp_key[warp] = key; warp_order[warp] = order; }
      __syncthreads();
#pragma unroll
      for (int w = 0; w < kBsThreads / 32; ++w) {
        const unsigned long long k = warp_key[w], o = warp_order[w];
        if (w == 0 || k > key || (k == key && o < order)) { key = k; order = o; }
      }
      last_key = key;
      last_order = order;
      if (tid == 0) {
        const unsigned long long u = key >> 63 ? key & 0x7fffffffffffffffull : ~key;
        put(i, __longlong_as_double(static_cast<long long>(u)), static_cast<int>(order >> 32), static_cast<int>(order & 0xffffffffu));
      }
      __syncthreads();
    }
    have = n;
  }
  __syncthreads();
  // Fewer continuations than asked for: all of them have been chosen, and the first places of the group that are not among them have minus infinity.
  if (have < n && tid == 0) {
    int beam = 0, token = 0;
    for (int i = have; i < n; ++i) {
      for (bool taken = true; taken;) {
        taken = false;
        for (int j = 0; j < have; ++j) taken |= chosen_beam[j] == beam && chosen_token[j] == token;
        if (taken && ++token == p.vocab) { token = 0; ++beam; }
      }
      put(i, -INFINITY, beam, token);
      if (++token == p.vocab) { token = 0; ++beam; }
    }
  }
}

}  // namespace rb

namespace {
// Elements of a thread: 32 (8192 of a row for a CTA), fewer where that leaves SMs without a CTA: a piece is then loaded and searched in less time.
int elements(int groups, int beams, int vocab, int type) {
  const long long rows = static_cast<long long>(groups) * beams;
  const int least = type == 2 ? 4 : 8;
  int e = 32;
  while (e > least && rows * ((vocab + e * rb::kBsThreads - 1) / (e * rb::kBsThreads)) < 148) e /= 2;
  return e;
}
int pieces_of(int vocab, int e) { return (vocab + e * rb::kBsThreads - 1) / (e * rb::kBsThreads); }
}  // namespace

RB_API long long rb_beam_select_scratch_bytes(int groups, int beams, int vocab, int count, int type) {
  if (groups < 0 || beams < 1 || vocab < 1 || count < 1) return 0;
  const long long places = static_cast<long long>(groups) * beams * pieces_of(vocab, elements(groups, beams, vocab, type));
  return places * (sizeof(rb::BsStat) + count * sizeof(rb::BsCandidate)) + 16;
}

RB_API int rb_beam_select(const RbBeamSelectArgs* a, void* stream) {
  if (!a || a->groups < 0 || a->beams < 1 || a->beams > rb::kBsMostBeams || a->vocab < 1 || a->count < 1 || a->count > rb::kBsMostCount ||
      a->count > static_cast<long long>(a->beams) * a->vocab || a->type < 0 || a->type > 2 || a->ld < a->vocab)
    return -1;
  if (a->groups == 0) return 0;
  if (!a->logits || !a->scores || !a->out_scores || !a->out_rows || !a->out_tokens || !a->scratch) return -1;
  const long long rows = static_cast<long long>(a->groups) * a->beams;
  if (rows > 0x7fffffffll) return -2;
  if (a->ended && (a->end_token < 0 || a->end_token >= a->vocab)) return -3;
  const int size = a->type == 2 ? 4 : 2, e = elements(a->groups, a->beams, a->vocab, a->type);
  rb::BsParams p;
  p.logits = a->logits; p.scores = a->scores; p.ended = a->ended;
  p.out_scores = a->out_scores; p.out_rows = a->out_rows; p.out_tokens = a->out_tokens;
  p.ld = a->ld; p.groups = a->groups; p.beams = a->beams; p.vocab = a->vocab; p.count = a->count; p.end_token = a->end_token;
  p.pieces = pieces_of(a->vocab, e);
  p.piece = e * rb::kBsThreads;
  p.vec = (reinterpret_cast<unsigned long long>(a->logits) & 15) == 0 && (a->ld * size) % 16 == 0 ? 16 / size : 1;
  if (p.pieces > 65535 || static_cast<long long>(a->beams) * p.pieces * a->count + a->beams > 0x7fffffffll) return -2;
  p.stats = static_cast<rb::BsStat*>(a->scratch);
  p.found = reinterpret_cast<rb::BsCandidate*>(p.stats + rows * p.pieces);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const dim3 grid(static_cast<unsigned>(rows), p.pieces), block(rb::kBsThreads);
  auto go = [&](void (*k)(const rb::BsParams)) { return rbhost::launch_pdl(k, grid, block, 0, s, 1, p); };
  cudaError_t err;
  if (a->type == 2)
    err = e == 32 ? go(rb::beam_rows_kernel<float, 32>) : e == 16 ? go(rb::beam_rows_kernel<float, 16>)
          : e == 8 ? go(rb::beam_rows_kernel<float, 8>) : go(rb::beam_rows_kernel<float, 4>);
  else if (a->type == 1)
    err = e == 32 ? go(rb::beam_rows_kernel<__half, 32>) : e == 16 ? go(rb::beam_rows_kernel<__half, 16>) : go(rb::beam_rows_kernel<__half, 8>);
  else
    err = e == 32 ? go(rb::beam_rows_kernel<__nv_bfloat16, 32>) : e == 16 ? go(rb::beam_rows_kernel<__nv_bfloat16, 16>)
                                                                 : go(rb::beam_rows_kernel<__nv_bfloat16, 8>);
  if (err != cudaSuccess) return static_cast<int>(err);
  return static_cast<int>(rbhost::launch_pdl(rb::beam_group_kernel, dim3(a->groups), block, 0, s, 1, p));
}
