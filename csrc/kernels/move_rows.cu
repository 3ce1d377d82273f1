// Moves of rows inside tensors: blocks of a paged cache (or slots of recurrent state) to other blocks in all layers with one launch, and the states
// of a batch into the order of selected beams, in place.
//
// Both are bound by memory; neither computes anything.  The pairs of a copy and the tensors of either call are kernel parameters (at most 32 KB): no
// copy to the device goes ahead of the launch, and a captured graph keeps them.  A copy's CTA takes a piece of a row of at most 16 KB, each thread four loads
// of 16 bytes before its first store.
//
// In place, a row may be wanted by several others and be overwritten itself.  A thread owns one column, 16 bytes of every row of a group: it loads all of
// the column before it stores any of it, so that no other thread and no second buffer takes part, whatever the index says.  Rows that stay are
// neither read for themselves nor written.
//
// One B200: 256 blocks of 32 KB in the keys and values of 8 layers, 42.9 us, 6.26 TB/s of reads and writes (a plain copy: 6.57); 16 beams in groups of 4, keys and values of 4 layers
// of 12 heads over 1000 tokens, 47.7 us, 5.4 TB/s.  Small calls are their launch, 2.4 to 3.2 us.  Groups of more than 16 rows hold their columns in shared memory, a warp a CTA: the same
// caches, 2 layers, with groups of 32 rows 3.5 to 3.9 TB/s; one layer, groups of 64 2.1, of 256 (128 KB a warp, one on an SM) 0.43.
#include "move_rows.h"

#include <string.h>

#include <new>
#include <vector>

#include "pdl.cuh"
#include "rb_common.cuh"

namespace rb {

constexpr int kMvThreads = 256;
constexpr int kMvTensors = 32;                   // tensors of a launch
constexpr long long kMvPiece = 16384;            // bytes of a CTA at most

struct MvTensor {
  char* base;
  long long outer_stride, row_stride, seg_stride, seg_bytes;
  long long items_end;                           // CTAs up to and with this tensor
  long long piece;                               // bytes of a CTA (copy), columns of a row (reorder)
  int segs, pieces;                              // pieces of a segment
  int log_vec, outer;
};
template <int PAIRS>
struct MvCopyParams {
  MvTensor t[kMvTensors];
  int src[PAIRS], dst[PAIRS];
  int count, pairs;
};
struct MvReorderParams {
  MvTensor t[kMvTensors];
  const long long* index;
  int count, rows, group;
};

template <typename V>
__device__ __forceinline__ void mv_copy(char* to, const char* from, long long bytes) {
  const int n = static_cast<int>(bytes / sizeof(V));
  const V* f = reinterpret_cast<const V*>(from);
  V* d = reinterpret_cast<V*>(to);
  for (int i = threadIdx.x; i < n; i += 4 * kMvThreads) {
    V x[4];
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (i + j * kMvThreads < n) x[j] = f[i + j * kMvThreads];
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (i + j * kMvThreads < n) d[i + j * kMvThreads] = x[j];
  }
}

template <int PAIRS>
__global__ void __launch_bounds__(kMvThreads)
move_blocks_kernel(const __grid_constant__ MvCopyParams<PAIRS> p) {
  pdl_wait();
  pdl_launch();
  const long long item = blockIdx.x;
  int ti = 0;
  while (ti + 1 < p.count && item >= p.t[ti].items_end) ++ti;
  const MvTensor& t = p.t[ti];
  long long i = item - (ti ? p.t[ti - 1].items_end : 0);
  const int piece = static_cast<int>(i % t.pieces);
  i /= t.pieces;
  const int seg = static_cast<int>(i % t.segs);
  i /= t.segs;
  const int pair = static_cast<int>(i % p.pairs);
  const long long outer = i / p.pairs;
  char* at = t.base + outer * t.outer_stride + seg * t.seg_stride + piece * t.piece;
  const long long bytes = min(t.piece, t.seg_bytes - piece * t.piece);
  char* to = at + p.dst[pair] * t.row_stride;
  const char* from = at + p.src[pair] * t.row_stride;
  switch (t.log_vec) {
    case 4: mv_copy<uint4>(to, from, bytes); break;
    case 3: mv_copy<uint2>(to, from, bytes); break;
    case 2: mv_copy<uint32_t>(to, from, bytes); break;
    case 1: mv_copy<uint16_t>(to, from, bytes); break;
    default: mv_copy<uint8_t>(to, from, bytes); break;
  }
}

// One column of a group whose rows fit the registers of a thread.
template <typename V, int R>
__device__ __forceinline__ void mv_column(char* at, long long row_stride, const long long* index, int first, int n) {
  V x[R];
  uint32_t moves = 0;
#pragma unroll
  for (int i = 0; i < R; ++i) {
    if (i < n) {
      const long long s = index[first + i] - first;
      if (s >= 0 && s < n && s != i) {
        x[i] = *reinterpret_cast<const V*>(at + s * row_stride);
        moves |= 1u << i;
      }
    }
  }
#pragma unroll
  for (int i = 0; i < R; ++i)
    if (moves >> i & 1u) *reinterpret_cast<V*>(at + i * row_stride) = x[i];
}
// The same with the column in shared memory: places threadIdx.x + i * blockDim.x belong to this thread alone.
template <typename V>
__device__ __forceinline__ void mv_column_shared(char* at, long long row_stride, const long long* index, int first, int n, V* held) {
  for (int i = 0; i < n; ++i) {
    const long long s = index[first + i] - first;
    if (s >= 0 && s < n && s != i) held[i * blockDim.x + threadIdx.x] = *reinterpret_cast<const V*>(at + s * row_stride);
  }
  for (int i = 0; i < n; ++i) {
    const long long s = index[first + i] - first;
    if (s >= 0 && s < n && s != i) *reinterpret_cast<V*>(at + i * row_stride) = held[i * blockDim.x + threadIdx.x];
  }
}
template <typename V, int R>
__device__ __forceinline__ void mv_reorder(const MvTensor& t, const MvReorderParams& p, long long i, uint4* held) {
  // numbers within the tensor: columns fastest, then groups, then outer copies
  const int groups = p.rows / p.group;
  const long long blocks = t.pieces;                                   // CTAs for the columns of a row
  const long long column = i % blocks * blockDim.x + threadIdx.x;
  i /= blocks;
  const int g = static_cast<int>(i % groups);
  const long long outer = i / groups;
  if (column >= t.piece) return;
  const int per = static_cast<int>(t.seg_bytes / sizeof(V));
  const long long seg = column / per;
  char* at = t.base + outer * t.outer_stride + static_cast<long long>(g) * p.group * t.row_stride + seg * t.seg_stride +
             (column - seg * per) * static_cast<long long>(sizeof(V));
  if (R > 0) mv_column<V, R ? R : 1>(at, t.row_stride, p.index, g * p.group, p.group);
  else mv_column_shared<V>(at, t.row_stride, p.index, g * p.group, p.group, reinterpret_cast<V*>(held));
}

// R: rows of a group that fit (0: any number, in shared memory)
template <int R>
__global__ void __launch_bounds__(kMvThreads)
move_reorder_kernel(const __grid_constant__ MvReorderParams p) {
  extern __shared__ uint4 mv_held[];
  pdl_wait();
  pdl_launch();
  const long long item = blockIdx.x;
  int ti = 0;
  while (ti + 1 < p.count && item >= p.t[ti].items_end) ++ti;
  const MvTensor& t = p.t[ti];
  const long long i = item - (ti ? p.t[ti - 1].items_end : 0);
  switch (t.log_vec) {
    case 4: mv_reorder<uint4, R>(t, p, i, mv_held); break;
    case 3: mv_reorder<uint2, R>(t, p, i, mv_held); break;
    case 2: mv_reorder<uint32_t, R>(t, p, i, mv_held); break;
    case 1: mv_reorder<uint16_t, R>(t, p, i, mv_held); break;
    default: mv_reorder<uint8_t, R>(t, p, i, mv_held); break;
  }
}

}  // namespace rb

namespace {

constexpr int kSharedThreads = 32;               // of a CTA whose columns are in shared memory
constexpr int kMostGroup = 256;                  // 256 rows x 32 threads x 16 bytes: 128 KB

// The widest access that base, strides and pieces allow.
int log_vec(const RbMoveTensor& t) {
  unsigned long long bits = reinterpret_cast<unsigned long long>(t.base) | static_cast<unsigned long long>(t.seg_bytes) | static_cast<unsigned long long>(t.row_stride);
  if (t.outer > 1) bits |= static_cast<unsigned long long>(t.outer_stride);
  if (t.segs > 1) bits |= static_cast<unsigned long long>(t.seg_stride);
  for (int l = 4; l > 0; --l)
    if ((bits & ((1ull << l) - 1)) == 0) return l;
  return 0;
}

rb::MvTensor described(const RbMoveTensor& t) {
  rb::MvTensor d;
  memset(&d, 0, sizeof(d));
  d.base = static_cast<char*>(t.base);
  d.outer_stride = t.outer_stride; d.row_stride = t.row_stride; d.seg_stride = t.seg_stride; d.seg_bytes = t.seg_bytes;
  d.segs = t.segs; d.outer = t.outer;
  d.log_vec = log_vec(t);
  return d;
}

bool sound(const RbMoveTensor* t, int count) {
  if (count < 0 || (count > 0 && !t)) return false;
  for (int i = 0; i < count; ++i)
    if (!t[i].base || t[i].outer < 1 || t[i].segs < 1 || t[i].seg_bytes < 1) return false;
  return true;
}

// -2, -3, -4 as rb_move_blocks returns them, -5 without memory
int check_pairs(const int* src, const int* dst, int pairs, int num_rows) {
  for (int i = 0; i < pairs; ++i)
    if (src[i] < 0 || src[i] >= num_rows || dst[i] < 0 || dst[i] >= num_rows) return -2;
  if (pairs <= 16) {
    for (int i = 0; i < pairs; ++i)
      for (int j = 0; j < i; ++j)
        if (dst[i] == dst[j]) return -3;
    for (int i = 0; i < pairs; ++i)
      for (int j = 0; j < pairs; ++j)
        if (dst[i] == src[j]) return -4;
    return 0;
  }
  try {
    std::vector<unsigned char> is_dst(num_rows, 0);
    for (int i = 0; i < pairs; ++i) {
      if (is_dst[dst[i]]) return -3;
      is_dst[dst[i]] = 1;
    }
    for (int i = 0; i < pairs; ++i)
      if (is_dst[src[i]]) return -4;
  } catch (const std::bad_alloc&) {
    return -5;
  }
  return 0;
}

template <int PAIRS>
int launch_blocks(const RbMoveTensor* tensors, int count, const int* src, const int* dst, int pairs, cudaStream_t stream) {
  rb::MvCopyParams<PAIRS> p;
  p.count = count;
  p.pairs = pairs;
  memcpy(p.src, src, pairs * sizeof(int));
  memcpy(p.dst, dst, pairs * sizeof(int));
  long long items = 0;
  for (int i = 0; i < count; ++i) {
    rb::MvTensor d = described(tensors[i]);
    const long long most = (d.seg_bytes + rb::kMvPiece - 1) / rb::kMvPiece;
    d.piece = ((d.seg_bytes + most - 1) / most + 15) / 16 * 16;      // equal pieces, whole accesses
    const long long pieces = (d.seg_bytes + d.piece - 1) / d.piece;
    items += pieces * d.segs * d.outer * pairs;
    if (items > 0x7fffffffll) return -6;
    d.pieces = static_cast<int>(pieces);
    d.items_end = items;
    p.t[i] = d;
  }
  return static_cast<int>(rbhost::launch_pdl(rb::move_blocks_kernel<PAIRS>, dim3(static_cast<unsigned>(items)), dim3(rb::kMvThreads), 0, stream, 1, p));
}

}  // namespace

RB_API int rb_move_most_group() { return kMostGroup; }

RB_API int rb_move_blocks(const RbMoveTensor* tensors, int count, const int* src, const int* dst, int pairs, int num_rows, void* stream) {
  if (!sound(tensors, count) || pairs < 0 || (pairs > 0 && (!src || !dst))) return -1;
  const int bad = check_pairs(src, dst, pairs, num_rows);
  if (bad) return bad;
  constexpr int kMost = 3600;                    // 2 x 4 bytes each beside 32 tensors of 72: below the 32764 bytes of a kernel's parameters
  static_assert(sizeof(rb::MvCopyParams<kMost>) <= 32764, "kernel parameters");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  for (int p0 = 0; p0 < pairs; p0 += kMost)
    for (int t0 = 0; t0 < count; t0 += rb::kMvTensors) {
      const int n = pairs - p0 < kMost ? pairs - p0 : kMost, m = count - t0 < rb::kMvTensors ? count - t0 : rb::kMvTensors;
      const int e = n <= 32    ? launch_blocks<32>(tensors + t0, m, src + p0, dst + p0, n, s)
                    : n <= 512 ? launch_blocks<512>(tensors + t0, m, src + p0, dst + p0, n, s)
                               : launch_blocks<kMost>(tensors + t0, m, src + p0, dst + p0, n, s);
      if (e) return e;
    }
  return 0;
}

RB_API int rb_move_reorder(const RbMoveTensor* tensors, int count, const long long* index, int rows, int group, void* stream) {
  if (!sound(tensors, count) || rows < 0 || group < 1 || group > kMostGroup || rows % group || (rows > 0 && !index)) return -1;
  if (rows == 0) return 0;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const bool shared = group > 16;
  const int threads = shared ? kSharedThreads : rb::kMvThreads;
  for (int t0 = 0; t0 < count; t0 += rb::kMvTensors) {
    rb::MvReorderParams p;
    memset(&p, 0, sizeof(p));
    p.count = count - t0 < rb::kMvTensors ? count - t0 : rb::kMvTensors;
    p.index = index; p.rows = rows; p.group = group;
    long long items = 0;
    for (int i = 0; i < p.count; ++i) {
      rb::MvTensor d = described(tensors[t0 + i]);
      d.piece = (d.seg_bytes >> d.log_vec) * d.segs;                   // columns
      const long long blocks = (d.piece + threads - 1) / threads;
      items += blocks * (rows / group) * d.outer;
      if (items > 0x7fffffffll || blocks > 0x7fffffffll || (d.seg_bytes >> d.log_vec) > 0x7fffffffll) return -6;
      d.pieces = static_cast<int>(blocks);
      d.items_end = items;
      p.t[i] = d;
    }
    const dim3 grid(static_cast<unsigned>(items));
    cudaError_t e;
    if (shared) {
      const size_t smem = static_cast<size_t>(group) * threads * 16;
      static bool configured[64] = {false};
      const int dev = rbhost::device_slot();
      if (!configured[dev]) {
        e = cudaFuncSetAttribute(rb::move_reorder_kernel<0>, cudaFuncAttributeMaxDynamicSharedMemorySize, kMostGroup * kSharedThreads * 16);
        if (e != cudaSuccess) return static_cast<int>(e);
        configured[dev] = true;
      }
      e = rbhost::launch_pdl(rb::move_reorder_kernel<0>, grid, dim3(threads), smem, s, 1, p);
    } else if (group > 8) {
      e = rbhost::launch_pdl(rb::move_reorder_kernel<16>, grid, dim3(threads), 0, s, 1, p);
    } else {
      e = rbhost::launch_pdl(rb::move_reorder_kernel<8>, grid, dim3(threads), 0, s, 1, p);
    }
    if (e != cudaSuccess) return static_cast<int>(e);
  }
  return 0;
}
