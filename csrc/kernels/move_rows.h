// C interface of moves of rows inside tensors: blocks of a paged cache to other blocks, states of a batch into the order of selected beams
// (move_rows.cu).
//
// A tensor is `outer` copies, outer_stride bytes apart, of rows that are row_stride bytes apart; a row is `segs` pieces of seg_bytes, seg_stride
// bytes apart.  Rows of a tensor do not overlap, and no two tensors of a call share memory.
#pragma once
#ifdef __cplusplus
extern "C" {
#endif
typedef struct RbMoveTensor {
  void* base;
  long long outer_stride, row_stride, seg_stride, seg_bytes;
  int outer, segs;
} RbMoveTensor;

// Row dst[i] <- row src[i] for all i, in every tensor of `num_rows` rows.  src and dst are on the host and are read before the call returns.
// Returns -2 where a row is not in 0 .. num_rows - 1, -3 where a row is a destination twice, -4 where a destination is a source too, and
// then copies nothing.
int rb_move_blocks(const RbMoveTensor* tensors, int count, const int* src, const int* dst, int pairs, int num_rows, void* stream);

// Row i <- what row index[i] (on the device) was before the call, in every tensor of `rows` rows, which come in groups of `group` rows: an index outside
// its row's group leaves the row as it is.
int rb_move_reorder(const RbMoveTensor* tensors, int count, const long long* index, int rows, int group, void* stream);
// The largest group that rb_move_reorder takes.
int rb_move_most_group();
#ifdef __cplusplus
}
#endif
