// Beam search's selection: log-softmax of every beam's logits, sums with the beams' scores, and the best continuations over beams and vocabulary, with
// no array of sums ever written.
//
// total(r, t) = s_r + x_rt - L_r, L_r = log sum_u exp x_ru.  Within a row the order of totals is the order of the logits, so a row's best `count`
// logits are found before L_r is known, in the same pass over the logits that sums the exponentials: the logits are read once.  A CTA goes through a piece of a row, tile by tile; it
// leaves the piece's maximum, the sum under it, and its best logits.  A second launch, a CTA for each group, joins the pieces' sums and orders
// the candidates of all its rows by s_r + x - L_r in 64 bits: two continuations of different beams are often closer than 32 bits of a sum can tell,
// and the one selected must not depend on how the sum was rounded.  Beams that have ended or have a score of minus infinity are not read.
//
// The best n of a set that lies with many threads: the n-th largest of the threads' own maxima is a lower bound of the n-th largest
// number (found by its bits, most significant first, with one count over the CTA per bit); numbers not below it, little more than n, go to a list, and a number's
// place is the count of those before it.
#include "beam.h"

#include <cuda_fp16.h>
#include <float.h>

#include <type_traits>

#include "pairs.cuh"
#include "pdl.cuh"
#include "warp_mma.cuh"

namespace rb {

constexpr int kBsThreads = 256;
constexpr float kBsLog2e = 1.4426950408889634f;
constexpr int kBsMostCount = 128;
constexpr int kBsMostBeams = 256;
constexpr int kBsList = 1024;                    // room for the numbers that are not below a bound

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
  bool wide;                                     // rows begin on 16 bytes
};

// Number i of words that hold numbers of type T one behind the other.
template <typename T>
__device__ __forceinline__ float bs_value(const uint32_t* w, int i);
template <>
__device__ __forceinline__ float bs_value<__nv_bfloat16>(const uint32_t* w, int i) { return __uint_as_float(i & 1 ? w[i / 2] & 0xffff0000u : w[i / 2] << 16); }
template <>
__device__ __forceinline__ float bs_value<__half>(const uint32_t* w, int i) {
  return __half2float(__ushort_as_half(static_cast<unsigned short>(i & 1 ? w[i / 2] >> 16 : w[i / 2])));
}
template <>
__device__ __forceinline__ float bs_value<float>(const uint32_t* w, int i) { return __uint_as_float(w[i]); }
// A word's worth of them from numbers at x that need not be aligned; minus infinity behind the last.
template <typename T>
__device__ __forceinline__ uint32_t bs_word(const T* x, int at, int end);
template <>
__device__ __forceinline__ uint32_t bs_word(const float* x, int at, int end) { return __float_as_uint(at < end ? x[at] : -INFINITY); }
template <typename T>
__device__ __forceinline__ uint32_t bs_word(const T* x, int at, int end) {
  constexpr uint32_t kLeast = std::is_same<T, __half>::value ? 0xfc00u : 0xff80u;
  const unsigned short* u = reinterpret_cast<const unsigned short*>(x);
  const uint32_t lo = at < end ? u[at] : kLeast, hi = at + 1 < end ? u[at + 1] : kLeast;
  return lo | hi << 16;
}
// The largest of W words of numbers; a NaN is none of them.
template <typename T, int W>
__device__ __forceinline__ float bs_most(const uint32_t* w) {
  if (sizeof(T) == 4) {
    float m = __uint_as_float(w[0]);
#pragma unroll
    for (int i = 1; i < W; ++i) m = fmaxf(m, __uint_as_float(w[i]));
    return fmaxf(m, -INFINITY);
  }
  using T2 = typename std::conditional<std::is_same<T, __half>::value, __half2, __nv_bfloat162>::type;
  T2 m = *reinterpret_cast<const T2*>(w);
#pragma unroll
  for (int i = 1; i < W; ++i) m = __hmax2(m, *reinterpret_cast<const T2*>(w + i));
  uint32_t u = *reinterpret_cast<const uint32_t*>(&m);
  return fmaxf(fmaxf(bs_value<typename std::conditional<sizeof(T) == 4, __half, T>::type>(&u, 0), bs_value<typename std::conditional<sizeof(T) == 4, __half, T>::type>(&u, 1)), -INFINITY);
}
// 16 bytes of numbers from x[at] on.
template <typename T>
__device__ __forceinline__ void bs_load(const T* x, int at, int end, bool wide, uint32_t* w) {
  constexpr int V = 16 / sizeof(T);
  if (wide && at + V <= end) {
    const uint4 u = __ldcs(reinterpret_cast<const uint4*>(x + at));
    w[0] = u.x; w[1] = u.y; w[2] = u.z; w[3] = u.w;
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = bs_word(x, at + i * (V / 4), end);
  }
}
// NaN is minus infinity, plus infinity the largest number
__device__ __forceinline__ float bs_clean(float v) { return v != v ? -INFINITY : fminf(v, FLT_MAX); }
// Order of the numbers as order of whole numbers; minus infinity is the least, and no number gives 0.
__device__ __forceinline__ uint32_t bs_key(float v) {
  v += 0.f;                                      // -0 and 0 are equal
  const uint32_t u = __float_as_uint(v);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float bs_number(uint32_t k) { return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k); }
constexpr uint32_t kBsLeast = 0x007fffffu;       // bs_key(-infinity)

__device__ __forceinline__ bool bs_live(const BsParams& p, int row) {
  const float s = bs_clean(p.scores[row]);
  return s != -INFINITY && !(p.ended && p.ended[row]);
}

// The n-th largest key of the CTA's threads (one key each), 1 <= n <= blockDim.x.  Every thread gets it.
__device__ __forceinline__ uint32_t bs_nth(uint32_t key, int n, int lowest_bit) {
  uint32_t at = 0;
#pragma unroll 1
  for (int bit = 31; bit >= lowest_bit; --bit) {
    const uint32_t with = at | 1u << bit;
    const int c = __syncthreads_count(key >= with);
    if (c >= n) at = with;
    if (c == n) break;                           // exactly the n largest are not below `with`
  }
  return at;
}

// ---- a piece of a row --------------------------------------------------------------------------------------------------------------------
// Numbers, each with a token, in no order; the better one is the larger word: the key above, the token's complement below.
template <int CAP>
struct BsList {
  alignas(16) unsigned long long item[CAP];
  int size;
};
__device__ __forceinline__ unsigned long long bs_item(uint32_t key, int token) {
  return static_cast<unsigned long long>(key) << 32 | (0xffffffffu - static_cast<uint32_t>(token));
}
__device__ __forceinline__ uint32_t bs_item_key(unsigned long long c) { return static_cast<uint32_t>(c >> 32); }
__device__ __forceinline__ int bs_item_token(unsigned long long c) { return static_cast<int>(0xffffffffu - static_cast<uint32_t>(c)); }
// Keeps the n best of the list's m numbers, in order.  All threads.  Items are counted two a load, eight at a time: one after the other a list of 64 took 3.6 us.
template <int CAP>
__device__ __forceinline__ void bs_keep(BsList<CAP>& l, int m, int n) {
  constexpr int kMine = (CAP + kBsThreads - 1) / kBsThreads;
  static_assert(CAP % 8 == 0, "whole rounds");
  if (threadIdx.x < 8 && m + static_cast<int>(threadIdx.x) < CAP) l.item[m + threadIdx.x] = 0ull;       // none is better than these
  __syncthreads();
  unsigned long long c[kMine];
  int at[kMine];
#pragma unroll
  for (int j = 0; j < kMine; ++j) {
    const int i = threadIdx.x + j * kBsThreads;
    at[j] = CAP;
    if (i < m) {
      c[j] = l.item[i];
      int before = 0;
#pragma unroll 1
      for (int o = 0; o < m; o += 8) {
        ulonglong2 w[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) w[k] = *reinterpret_cast<const ulonglong2*>(l.item + o + 2 * k);
#pragma unroll
        for (int k = 0; k < 4; ++k) before += (w[k].x > c[j] ? 1 : 0) + (w[k].y > c[j] ? 1 : 0);
      }
      at[j] = before;
    }
  }
  __syncthreads();
#pragma unroll
  for (int j = 0; j < kMine; ++j)
    if (at[j] < n) l.item[at[j]] = c[j];
  if (threadIdx.x == 0) l.size = min(m, n);
  __syncthreads();
}
// Puts the n best of the numbers i = 0 .. count - 1 into an empty list, however many are equal: the n-th largest key bit by bit, counting all numbers, then of those
// equal to it the highest token that is still taken, in the same way.  number(i, token) gives a number, -infinity for none.
template <typename F>
__device__ __forceinline__ void bs_search(BsList<kBsList>& l, int count, int n, F number) {
  auto counted = [&](auto f) {
    int c = 0;
    for (int i = threadIdx.x; i < count; i += kBsThreads) {
      int token;
      const uint32_t k = bs_key(number(i, token));
      c += f(k, token) ? 1 : 0;
    }
    __syncthreads();
    if (threadIdx.x == 0) l.size = 0;
    __syncthreads();
    if (c) atomicAdd(&l.size, c);
    __syncthreads();
    return l.size;
  };
  uint32_t nth = 0;
#pragma unroll 1
  for (int bit = 31; bit >= 0; --bit) {
    const uint32_t with = nth | 1u << bit;
    if (counted([&](uint32_t k, int) { return k >= with; }) >= n) nth = with;
  }
  const int room = n - counted([&](uint32_t k, int) { return k > nth; });
  int last = 0;                                  // tokens below it are fewer than the room
#pragma unroll 1
  for (int bit = 30; bit >= 0; --bit) {
    const int with = last | 1 << bit;
    if (counted([&](uint32_t k, int t) { return k == nth && t < with; }) < room) last = with;
  }
  __syncthreads();
  if (threadIdx.x == 0) l.size = 0;
  __syncthreads();
  for (int i = threadIdx.x; i < count; i += kBsThreads) {
    int token;
    const uint32_t k = bs_key(number(i, token));
    if (k > nth || (k == nth && token <= last)) {
      const int at = atomicAdd(&l.size, 1);
      l.item[at] = bs_item(k, token);
    }
  }
  __syncthreads();
}

// A ring of tiles in shared memory that bulk copies fill.
constexpr int kBsStages = 2;
constexpr int kBsApart = 4;                      // tiles between two looks at the noted chunks
constexpr int kBsChunks = 2 * kBsMostCount + 16 + kBsApart * kBsThreads;
__device__ __forceinline__ void bs_bulk(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
  mbar_arrive_expect_tx(bar, bytes);
  if (bytes)
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
                 ::"r"(dst), "l"(src), "r"(bytes), "r"(bar) : "memory");
}

// E: numbers of a thread and tile, neighbours, so that the order of (tile, thread) is the order of tokens.  A thread that meets a number not below the bound notes its whole
// chunk of E under the chunk's largest number: the n best numbers lie in the n chunks whose largest are the best (of equal ones the first), and which of a chunk's they are is
// looked up once, at the end.  So the pass over the logits is a maximum and an exponential per number, a barrier for four tiles and few chunks noted.
//
// 64 groups of 4 rows of 128256 numbers of 16 bits (65.7 MB): 29 us with the group's launch where the logits are in the L2, 36 with it flushed.  This kernel's part is 25 us and reads at
// 2.6 TB/s: 512 CTAs start (first tile, its bound) and end (lists) at the same times, with nothing in flight, and two stages are few in between.  When they were tried, against 32: three
// stages of the ring 39, twice the pieces 35, lists of numbers in place of chunks 46.
// BULK: tiles come through the ring; else a piece is one tile, or rows do not begin on 16 bytes.
template <typename T, int E, bool BULK>
__global__ void __launch_bounds__(kBsThreads, 4)
beam_rows_kernel(const BsParams p, unsigned int* status) {
  pdl_wait();
  pdl_launch();
  const int row = blockIdx.x, piece = blockIdx.y;
  if (!bs_live(p, row)) return;
  constexpr int V = 16 / sizeof(T), L = E / V, W = 4 * L;       // numbers of a wide load; loads and words of a thread and tile
  constexpr int kTile = E * kBsThreads;
  extern __shared__ __align__(128) uint8_t bs_tiles[];
  __shared__ BsList<kBsChunks> chunks;
  __shared__ BsList<kBsList> best;
  __shared__ float warp_most[kBsThreads / 32], warp_total[kBsThreads / 32];
  __shared__ uint64_t bars[2 * kBsStages];
  __shared__ int abort_flag;
  const T* x = static_cast<const T*>(p.logits) + static_cast<long long>(row) * p.ld;
  const int first = piece * p.piece, end = min(p.vocab, first + p.piece);
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, n = p.count;
  const uint32_t ring = smem_u32(bs_tiles), full = smem_u32(bars), empty = full + 8 * kBsStages;
  if (BULK && tid == 0) {
    for (int s = 0; s < kBsStages; ++s) {
      mbar_init(full + 8 * s, 1);
      mbar_init(empty + 8 * s, kBsThreads / 32);
    }
    abort_flag = 0;
    fence_mbar_init();
  }
  int seen = 0;                                  // tiles of the ring so far
  float most, sum;                               // this thread's maximum, and its sum of exp(x - maximum)
  uint32_t bound;
  uint32_t now[W];
  // Two passes where there are NaN or infinities: the first one's sum is NaN then, the second replaces them.
  auto pass = [&](auto replace) {
    constexpr bool kClean = decltype(replace)::value;
    auto value = [&](int e) { return kClean ? bs_clean(bs_value<T>(now, e)) : bs_value<T>(now, e); };
    // tile i of the piece into its place of the ring: whole 16 bytes, what is behind them is loaded where it is used
    auto request = [&](int i) {
      const int tile = first + i * kTile, s = (seen + i) % kBsStages;
      if (tile < end) bs_bulk(ring + s * kTile * static_cast<int>(sizeof(T)), x + tile, min(kTile, end - tile) / V * 16, full + 8 * s);
    };
    most = -INFINITY;
    sum = 0.f;
    bound = kBsLeast + 1;
    __syncthreads();
    if (tid == 0) {
      chunks.size = best.size = 0;
      if (BULK)
        for (int i = 0; i < kBsStages; ++i) request(i);
    }
    int i_tile = 0;
    for (int tile = first; tile < end; tile += kTile, ++i_tile) {
      const int mine = tile + tid * E;
      if (BULK) {
        const int at = seen + i_tile, s = at % kBsStages;
        if (tid == 0 && i_tile > 0 && tile + (kBsStages - 1) * kTile < end) {
          // the place of the tile in front is free once every warp has its numbers
          const int was = at - 1;
          mbar_wait(empty + 8 * (was % kBsStages), (was / kBsStages) & 1, &abort_flag, status, 63);
          request(i_tile - 1 + kBsStages);
        }
        mbar_wait(full + 8 * s, (at / kBsStages) & 1, &abort_flag, status, 62);
#pragma unroll
        for (int j = 0; j < L; ++j) {
          // neighbouring threads begin with different loads: no two of eight meet in a bank
          const int to = (j + (tid >> 1)) % L * V;
          if (mine + to + V <= end) {
            asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                         : "=r"(now[4 * j]), "=r"(now[4 * j + 1]), "=r"(now[4 * j + 2]), "=r"(now[4 * j + 3])
                         : "r"(ring + (s * kTile + tid * E + to) * static_cast<int>(sizeof(T)))
                         : "memory");
          } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) now[4 * j + i] = bs_word(x, mine + to + i * (V / 4), end);
          }
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(empty + 8 * s);
      } else {
#pragma unroll
        for (int j = 0; j < L; ++j) bs_load(x, mine + j * V, end, p.wide, now + 4 * j);
      }
      float top = -INFINITY;
      if (kClean) {
#pragma unroll
        for (int e = 0; e < E; ++e) top = fmaxf(top, value(e));
      } else {
        top = bs_most<T, W>(now);
      }
      const uint32_t key = bs_key(top);
      if (i_tile == 0) bound = max(bound, bs_nth(key, n, sizeof(T) == 4 ? 0 : 13));     // numbers of 16 bits have no lower bits in 32
      if (key >= bound) {
        const int at = atomicAdd(&chunks.size, 1);
        chunks.item[at] = bs_item(key, mine);
      }
      if (top > most) {
        sum *= wm_ex2((most - top) * kBsLog2e);
        most = top;
      }
      // exp(x - m) with the difference formed first: exact for the numbers that count
      const float from = most == -INFINITY ? 0.f : -most;
      const Pair from2 = pair_of(from, from), log2e = pair_of(kBsLog2e, kBsLog2e);
      Pair add[2] = {pair_of(0.f, 0.f), pair_of(0.f, 0.f)};
#pragma unroll
      for (int e = 0; e < E; e += 2) {
        const float2 y = floats(mul2(add2(pair_of(value(e), value(e + 1)), from2), log2e));
        add[e / 2 & 1] = add2(add[e / 2 & 1], pair_of(wm_ex2(y.x), wm_ex2(y.y)));
      }
      const float2 added = floats(add2(add[0], add[1]));
      sum += added.x + added.y;
      if (i_tile % kBsApart == kBsApart - 1 && tile + kTile < end) {
        __syncthreads();
        const int m = chunks.size;
        __syncthreads();
        if (m > 2 * n + 16) {                    // no more are left in front of the next tiles than the list has room for
          bs_keep(chunks, m, n);
          bound = max(bound, bs_item_key(chunks.item[n - 1]) + 1);             // later chunks lose against equal ones
        }
      }
    }
    seen += i_tile;
  };
  pass(std::false_type());
  const bool dirty = __syncthreads_or(sum != sum);
  if (dirty) {
    pass(std::true_type());
    __syncthreads();
  }

  // ---- the n best numbers of the noted chunks
  const bool one = !BULK && end - first <= kTile;
  if (one) {                                     // still in registers
    if (most != -INFINITY && bs_key(most) >= bound) {
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const float v = dirty ? bs_clean(bs_value<T>(now, e)) : bs_value<T>(now, e);
        if (bs_key(v) >= bound) {
          const int at = atomicAdd(&best.size, 1);
          if (at < kBsList) best.item[at] = bs_item(bs_key(v), first + tid * E + e);
        }
      }
    }
  } else {
    bs_keep(chunks, chunks.size, n);
    const int have = chunks.size;
    if (have == n) bound = bs_item_key(chunks.item[n - 1]);
    for (int i = tid; i < have * E; i += kBsThreads) {
      const int t = bs_item_token(chunks.item[i / E]) + i % E;
      if (t < end) {
        const uint32_t w = bs_word(x, t, end);
        const float v = bs_clean(bs_value<T>(&w, 0));
        if (bs_key(v) >= bound && v != -INFINITY) {
          const int at = atomicAdd(&best.size, 1);
          if (at < kBsList) best.item[at] = bs_item(bs_key(v), t);
        }
      }
    }
  }
  __syncthreads();
  int m = best.size;
  if (m > kBsList) {                             // many equal or neighbouring ones
    bs_search(best, one ? end - first : chunks.size * E, n, [&](int i, int& token) {
      token = one ? first + i : bs_item_token(chunks.item[i / E]) + i % E;
      const uint32_t w = bs_word(x, token, end);
      return bs_clean(bs_value<T>(&w, 0));
    });
    m = n;
  }
  bs_keep(best, m, n);

  const float wm = warp_max(most);
  const float ws = warp_sum(wm == -INFINITY ? 0.f : sum * wm_ex2((most - wm) * kBsLog2e));
  if (lane == 0) {
    warp_most[warp] = wm;
    warp_total[warp] = ws;
  }
  __syncthreads();
  const long long place = static_cast<long long>(row) * p.pieces + piece;
  if (tid == 0) {
    float top = warp_most[0], s = 0.f;
#pragma unroll
    for (int w = 1; w < kBsThreads / 32; ++w) top = fmaxf(top, warp_most[w]);
    if (top != -INFINITY)
#pragma unroll
      for (int w = 0; w < kBsThreads / 32; ++w) s += warp_total[w] * wm_ex2((warp_most[w] - top) * kBsLog2e);
    p.stats[place] = {top, s};
  }
  BsCandidate* found = p.found + place * n;
  for (int i = tid; i < n; i += kBsThreads) {
    if (i < m) found[i] = {bs_number(bs_item_key(best.item[i])), bs_item_token(best.item[i])};
    else found[i] = {0.f, -1};
  }
}

// ---- a group ---------------------------------------------------------------------------------------------------------------------------------
__device__ __forceinline__ unsigned long long bs_key64(double v) {
  v += 0.0;
  const unsigned long long u = static_cast<unsigned long long>(__double_as_longlong(v));
  return u >> 63 ? ~u : u | 0x8000000000000000ull;
}
// The pieces' candidates lie in order, so a thread has some of one list (or whole lists where there are more than threads) and knows their largest from the first.
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
  const int g = blockIdx.x, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, n = p.count;
  const int row0 = g * p.beams, lists = p.beams * p.pieces;
  const BsCandidate* found = p.found + static_cast<long long>(row0) * p.pieces * n;
  // lists of a thread: tid / share, and every kBsThreads / share-th behind it; items `from` .. `upto` - 1 of them
  const int share = max(1, kBsThreads / lists), step = kBsThreads / share, size = (n + share - 1) / share;
  const int from = tid % share * size, upto = min(n, from + size), list0 = tid < share * step ? tid / share : lists;
  BsCandidate head = {0.f, -1};                  // asked for before the rows' sums are formed
  if (list0 < lists && from < upto) head = found[static_cast<long long>(list0) * n + from];
  if (tid == 0) listed = 0;
  for (int r = warp; r < p.beams; r += kBsThreads / 32) {
    const float score = bs_clean(p.scores[row0 + r]);
    double b = -INFINITY;
    if (bs_live(p, row0 + r)) {
      const BsStat* st = p.stats + static_cast<long long>(row0 + r) * p.pieces;
      const BsStat mine = lane < p.pieces ? st[lane] : BsStat{-INFINITY, 0.f};
      float most = mine.most;
      for (int i = lane + 32; i < p.pieces; i += 32) most = fmaxf(most, st[i].most);
      most = warp_max(most);
      double sum = 0.0;
      if (most != -INFINITY) {
        if (mine.most != -INFINITY) sum = static_cast<double>(mine.sum) * exp(static_cast<double>(mine.most) - most);
        for (int i = lane + 32; i < p.pieces; i += 32)
          if (st[i].most != -INFINITY) sum += static_cast<double>(st[i].sum) * exp(static_cast<double>(st[i].most) - most);
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
      if (most != -INFINITY) b = static_cast<double>(score) - log(sum);
      if (lane == 0) row_most[r] = most;
    }
    if (lane == 0) base[r] = b;
  }
  __syncthreads();
  auto total_of = [&](int beam, float x) { return base[beam] + (static_cast<double>(x) - row_most[beam]); };
  auto rough = [](double t) { return bs_key(fmaxf(static_cast<float>(t), -FLT_MAX)); };       // keeps the order, but for what rounds to the same
  // a list's item, false behind the last: f(total, token, beam) until it returns false
  auto each = [&](auto f) {
    for (int i = list0; i < lists; i += step) {
      const int beam = i / p.pieces;
      if (base[beam] == -INFINITY) continue;
      for (int j = from; j < upto; ++j) {
        const BsCandidate c = i == list0 && j == from ? head : found[static_cast<long long>(i) * n + j];
        if (c.token < 0 || !f(total_of(beam, c.x), c.token, beam)) break;
      }
    }
    if (p.ended)
      for (int r = tid; r < p.beams; r += kBsThreads) {
        const float s = bs_clean(p.scores[row0 + r]);
        if (p.ended[row0 + r] && s != -INFINITY) f(static_cast<double>(s), p.end_token, r);
      }
  };
  uint32_t most = 0;
  each([&](double t, int, int) {
    most = max(most, rough(t));
    return false;                                // the rest of a list is smaller
  });
  const uint32_t bound = max(bs_nth(most, n, 0), kBsLeast + 1);
  if (most >= bound)
    each([&](double t, int token, int beam) {
      if (rough(t) < bound) return false;
      const int at = atomicAdd(&listed, 1);
      if (at < kBsList) {
        list_total[at] = t;
        list_beam[at] = beam;
        list_token[at] = token;
      }
      return true;
    });
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
#pragma unroll 8
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
      each([&](double t, int token, int beam) {
        const unsigned long long k = bs_key64(t), o = static_cast<unsigned long long>(beam) << 32 | static_cast<unsigned int>(token);
        const bool behind = k < last_key || (k == last_key && o > last_order);
        if (behind && (k > key || (k == key && o < order))) { key = k; order = o; }
        return true;
      });
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
struct Cut {
  int e, pieces, piece;                          // numbers of a thread and tile; pieces of a row, numbers of one
  bool bulk;
};
// Where there are at least two tiles of 8192 numbers (4096 in 32 bits) for each of an SM's four places, a CTA goes through several by bulk copies: only a piece's first
// tile has to be searched for a bound.  Else one tile for a CTA, smaller down to one load of a thread until there is a CTA for every SM.
Cut cut_of(int groups, int beams, int vocab, int type, bool wide) {
  const long long rows = static_cast<long long>(groups) * beams, places = 4ll * rbhost::device_sm_count();
  const int size = type == 2 ? 4 : 2, least = 16 / size;
  auto tiles = [&](int e) { return (vocab + e * rb::kBsThreads - 1) / (e * rb::kBsThreads); };
  Cut c;
  c.e = 64 / size;
  c.bulk = wide && rows * tiles(c.e) >= 2 * places;
  if (!c.bulk) {
    c.e /= 2;
    while (c.e > least && rows * tiles(c.e) < places / 4) c.e /= 2;
  }
  const int all = tiles(c.e);
  long long per = 1;                             // tiles of a piece
  if (c.bulk || rows * all > 8 * places) {
    const long long pieces = rows < places ? places / rows : 1;
    per = (all + pieces - 1) / pieces;
  }
  c.piece = static_cast<int>(per) * c.e * rb::kBsThreads;
  c.pieces = static_cast<int>((all + per - 1) / per);
  return c;
}
template <typename T, int E, bool BULK>
cudaError_t rows_kernel(const rb::BsParams& p, dim3 grid, cudaStream_t s) {
  const size_t smem = BULK ? rb::kBsStages * E * rb::kBsThreads * sizeof(T) : 0;
  static bool configured[64] = {false};
  const int dev = rbhost::device_slot();
  if (BULK && !configured[dev]) {
    const cudaError_t e = cudaFuncSetAttribute(rb::beam_rows_kernel<T, E, BULK>, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem));
    if (e != cudaSuccess) return e;
    configured[dev] = true;
  }
  return rbhost::launch_pdl(rb::beam_rows_kernel<T, E, BULK>, grid, dim3(rb::kBsThreads), smem, s, 1, p, rbhost::status_ptr());
}
template <typename T>
cudaError_t rows_of(const Cut& c, const rb::BsParams& p, dim3 grid, cudaStream_t s) {
  constexpr int kFull = 64 / sizeof(T);
  if (c.bulk) return rows_kernel<T, kFull, true>(p, grid, s);
  return c.e == kFull / 2 ? rows_kernel<T, kFull / 2, false>(p, grid, s) : rows_kernel<T, kFull / 4, false>(p, grid, s);
}
}  // namespace

static long long most_pieces(int groups, int beams, int vocab, int type) {
  const int a = cut_of(groups, beams, vocab, type, true).pieces, b = cut_of(groups, beams, vocab, type, false).pieces;
  return a > b ? a : b;
}
RB_API long long rb_beam_select_scratch_bytes(int groups, int beams, int vocab, int count, int type) {
  if (groups < 0 || beams < 1 || vocab < 1 || count < 1) return 0;
  const long long places = static_cast<long long>(groups) * beams * most_pieces(groups, beams, vocab, type);
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
  const int size = a->type == 2 ? 4 : 2;
  const bool wide = (reinterpret_cast<unsigned long long>(a->logits) & 15) == 0 && (a->ld * size) % 16 == 0;
  const Cut c = cut_of(a->groups, a->beams, a->vocab, a->type, wide);
  rb::BsParams p;
  p.logits = a->logits; p.scores = a->scores; p.ended = a->ended;
  p.out_scores = a->out_scores; p.out_rows = a->out_rows; p.out_tokens = a->out_tokens;
  p.ld = a->ld; p.groups = a->groups; p.beams = a->beams; p.vocab = a->vocab; p.count = a->count; p.end_token = a->end_token;
  p.pieces = c.pieces;
  p.piece = c.piece;
  p.wide = wide;
  if (p.pieces > 65535 || static_cast<long long>(a->beams) * p.pieces * a->count + a->beams > 0x7fffffffll) return -2;
  p.stats = static_cast<rb::BsStat*>(a->scratch);
  p.found = reinterpret_cast<rb::BsCandidate*>(p.stats + rows * p.pieces);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const dim3 grid(static_cast<unsigned>(rows), p.pieces);
  const cudaError_t err = a->type == 2 ? rows_of<float>(c, p, grid, s) : a->type == 1 ? rows_of<__half>(c, p, grid, s) : rows_of<__nv_bfloat16>(c, p, grid, s);
  if (err != cudaSuccess) return static_cast<int>(err);
  return static_cast<int>(rbhost::launch_pdl(rb::beam_group_kernel, dim3(a->groups), dim3(rb::kBsThreads), 0, s, 1, p));
}
