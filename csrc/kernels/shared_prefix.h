// C interface of decode attention for sequences that share their first tokens (shared_prefix.cu).
//
// Sequences come in groups: group_of [batch] is every sequence's group, span_of [batch, 2] the first sequence of that group and of the next.  The first
// shared_lens[g] tokens of a group's sequences are the same and are read through the block table of its first one; what follows of the context_lens[b]
// tokens of sequence b through its own.  Of a group whose shortest sequence (those without tokens aside) has fewer tokens than shared_lens[g], only that many count
// as shared.  A sequence without tokens gets zeros.
// Lengths beyond a table's row end with it.
//
// q [batch, heads * head_dim] (pitch ld_q), out the same (ld_o); caches [num_blocks, block_size, kv_heads, head_dim], contiguous; type 0 bf16, 1 f16;
// head_dim 64 or 128; q, out and caches 16-byte aligned, pitches multiples of 8.
// scratch: rb_shared_prefix_scratch_bytes bytes, 16-byte aligned.
#pragma once
#ifdef __cplusplus
extern "C" {
#endif
typedef struct RbSharedPrefixArgs {
  const void* q;
  void* out;
  const void* k_cache;
  const void* v_cache;
  const int* block_tables;   // [batch, max_blocks]
  const int* context_lens;   // [batch]
  const int* shared_lens;    // [groups]
  const int* group_of;
  const int* span_of;        // 8-byte aligned
  void* scratch;
  long long ld_q, ld_o, num_blocks;
  int batch, groups, max_blocks, block_size, heads, kv_heads, head_dim, type, most_rows;   // most_rows: sequences of the largest group
  float scale;
} RbSharedPrefixArgs;
long long rb_shared_prefix_scratch_bytes(int batch, int groups, int heads, int kv_heads, int head_dim, int block_size, int most_rows);
int rb_shared_prefix(const RbSharedPrefixArgs* args, void* stream);
#ifdef __cplusplus
}
#endif
