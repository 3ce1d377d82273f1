// C interface of the paged KV cache in e4m3 (paged_e4m3.cu, paged_e4m3_decode.cu, paged_e4m3_evict.cu).
//
// A page holds block_size tokens of a sequence.  For every KV head it has a tile of codes [block_size, head_dim] for keys and one for
// values, and for each tile a power of two: the number that code c stands for is c * 2^exp, exp in [-100, 119].  block_size is a multiple
// of 16, at most 2^20, head_dim 64 or 128; a row of a block table has room for fewer than 2^30 tokens.  All arrays are contiguous and 16-byte aligned.
#pragma once
#ifdef __cplusplus
extern "C" {
#endif
typedef struct RbPagesE4m3 {
  void* k;                   // [num_blocks, kv_heads, block_size, head_dim] e4m3
  void* v;
  signed char* k_exp;        // [num_blocks, kv_heads]
  signed char* v_exp;
  float* weight;             // [num_blocks, kv_heads, block_size], or NULL: attention weight that each token has had so far
  long long num_blocks;
  int block_size, kv_heads, head_dim;
} RbPagesE4m3;

// Types of rows that are no codes.
enum RbE4m3Type { RB_E4M3_BF16 = 0, RB_E4M3_F16 = 1, RB_E4M3_F32 = 2 };

// Stores the keys and values of new tokens.  Rows row_starts[b] .. row_starts[b + 1] - 1 of k_new / v_new [rows, kv_heads * head_dim] are the last
// tokens of sequence b, which has context_lens[b] tokens with them; row_starts NULL: one row for each sequence.  A page whose first slot gets a
// token takes its exponents from this call's tokens; in any other page an exponent grows where it must and the codes in front of the new ones are
// rounded to it.  The new tokens' weights become 0.  Row pitches in elements; rows and pitches are multiples of 16 bytes.
typedef struct RbE4m3AppendArgs {
  RbPagesE4m3 pages;
  const void* k_new;
  const void* v_new;
  const int* block_tables;   // [batch, max_blocks]
  const int* context_lens;   // [batch]
  const int* row_starts;     // [batch + 1] or NULL
  long long ld_k, ld_v;
  int rows, batch, max_blocks, type;
} RbE4m3AppendArgs;
int rb_e4m3_append(const RbE4m3AppendArgs* args, void* stream);

// The numbers that the codes of whole sequences stand for: position i of sequence b goes to row row_starts[b] + i of k_out / v_out
// [rows, kv_heads * head_dim]; rows that no position has stay as they are.
typedef struct RbE4m3ReadArgs {
  RbPagesE4m3 pages;
  void* k_out;
  void* v_out;
  const int* block_tables;
  const int* context_lens;
  const int* row_starts;     // [batch + 1]
  long long ld_k, ld_v;
  int rows, batch, max_blocks, type;
} RbE4m3ReadArgs;
int rb_e4m3_read(const RbE4m3ReadArgs* args, void* stream);

// Attention of one token per sequence: q [batch, heads * head_dim], pitch ld_q, out the same with ld_o (bf16 or f16).  accumulate: every cached
// token's weight grows by its softmax weights, summed over the query heads of its KV head.  A sequence without tokens gets zeros.
// scratch: fp32 [rb_e4m3_decode_scratch_floats(...)], NULL where that is 0 (few and short sequences).
typedef struct RbE4m3DecodeArgs {
  RbPagesE4m3 pages;
  const void* q;
  void* out;
  const int* block_tables;
  const int* context_lens;
  float* scratch;
  long long ld_q, ld_o;
  int batch, max_blocks, heads, type, accumulate;
  float scale;
} RbE4m3DecodeArgs;
long long rb_e4m3_decode_scratch_floats(int batch, int heads, int kv_heads, int head_dim, int max_blocks, int block_size, int accumulate);
int rb_e4m3_decode(const RbE4m3DecodeArgs* args, void* stream);

// Sequences of more than `keep` tokens keep the first keep_first, the last `recent` and, of the others, those with the largest weights (of equal
// ones the earlier), in their order; they move to the front of the sequence's pages, or to the pages of out_tables, which then are not those of
// any sequence of block_tables.  kept [batch, kv_heads, keep]: where each came from, -1 behind the last; lens_out [batch].
typedef struct RbE4m3EvictArgs {
  RbPagesE4m3 pages;
  const int* block_tables;
  const int* context_lens;
  const int* out_tables;     // [batch, out_blocks], or NULL
  int* kept;
  int* lens_out;
  int batch, max_blocks, out_blocks, keep, recent, keep_first;
} RbE4m3EvictArgs;
int rb_e4m3_evict(const RbE4m3EvictArgs* args, void* stream);
#ifdef __cplusplus
}
#endif
