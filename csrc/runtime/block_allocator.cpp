// Paged-KV block allocator: a free list of fixed-size blocks and one block table per sequence, and for models with
// recurrent layers a free list of state slots of which every sequence holds one from its first reservation to its end.
// A block may be in several tables (rb_ba_fork): it counts its owners and is free again when the last one lets go of it.
// Semantics follow the reference's PagedCache (crates/nn/src/kv_cache.rs:382-432) with its defect removed: a
// second reservation for a sequence extends the table instead of overwriting it (kv_cache.rs:420-423).
#include <algorithm>
#include <mutex>
#include <unordered_map>
#include <vector>

#include "rb_runtime.h"

struct RbBlockAllocator {
  int num_blocks, block_size;
  std::vector<int32_t> free_list;                                // stack; lowest ids are handed out first
  std::vector<int32_t> owners;                                   // tables that each block is in
  int shared = 0;                                                // blocks with more than one
  std::unordered_map<int64_t, std::vector<int32_t>> tables;
  bool slotted = false;                                          // sequences also hold a state slot
  std::vector<int32_t> free_slots;
  std::unordered_map<int64_t, int32_t> slots;
  mutable std::mutex mu;

  int32_t take() {
    const int32_t b = free_list.back();
    free_list.pop_back();
    owners[b] = 1;
    return b;
  }
  void give(int32_t b) {
    const int left = --owners[b];
    if (left == 1) --shared;
    if (left == 0) free_list.push_back(b);
  }
};

extern "C" {

RbBlockAllocator* rb_ba_create(int num_blocks, int block_size) {
  if (num_blocks <= 0 || block_size <= 0) return nullptr;
  auto* a = new RbBlockAllocator;
  a->num_blocks = num_blocks;
  a->block_size = block_size;
  a->free_list.reserve(num_blocks);
  a->owners.assign(num_blocks, 0);
  for (int i = num_blocks - 1; i >= 0; --i) a->free_list.push_back(i);
  return a;
}
// Every sequence from now on also takes one of `num_slots` state slots; call it before the first reservation.
int rb_ba_set_state_slots(RbBlockAllocator* a, int num_slots) {
  std::lock_guard<std::mutex> l(a->mu);
  if (num_slots <= 0 || !a->tables.empty()) return -1;
  a->slotted = true;
  a->free_slots.clear();
  for (int i = num_slots - 1; i >= 0; --i) a->free_slots.push_back(i);
  return 0;
}
int rb_ba_state_slot(const RbBlockAllocator* a, int64_t seq_id) {
  std::lock_guard<std::mutex> l(a->mu);
  auto it = a->slots.find(seq_id);
  return it == a->slots.end() ? -1 : it->second;
}
int rb_ba_num_free_slots(const RbBlockAllocator* a) {
  std::lock_guard<std::mutex> l(a->mu);
  return (int)a->free_slots.size();
}
void rb_ba_destroy(RbBlockAllocator* a) { delete a; }
int rb_ba_num_free(const RbBlockAllocator* a) { std::lock_guard<std::mutex> l(a->mu); return (int)a->free_list.size(); }
int rb_ba_num_blocks(const RbBlockAllocator* a) { return a->num_blocks; }
int rb_ba_block_size(const RbBlockAllocator* a) { return a->block_size; }

static int blocks_for(const RbBlockAllocator* a, int tokens) { return (tokens + a->block_size - 1) / a->block_size; }

int rb_ba_can_reserve(const RbBlockAllocator* a, int64_t seq_id, int num_tokens) {
  std::lock_guard<std::mutex> l(a->mu);
  auto it = a->tables.find(seq_id);
  const int have = it == a->tables.end() ? 0 : (int)it->second.size();
  const int need = blocks_for(a, num_tokens) - have;
  if (a->slotted && it == a->tables.end() && a->free_slots.empty()) return 0;
  return need <= (int)a->free_list.size() ? 1 : 0;
}

int rb_ba_reserve(RbBlockAllocator* a, int64_t seq_id, int num_tokens) {
  if (num_tokens < 0) return -1;
  std::lock_guard<std::mutex> l(a->mu);
  auto it = a->tables.find(seq_id);
  const int have = it == a->tables.end() ? 0 : (int)it->second.size();
  const int need = blocks_for(a, num_tokens) - have;
  const bool fresh = it == a->tables.end();
  if (need > (int)a->free_list.size()) return -1;
  if (fresh && a->slotted) {
    if (a->free_slots.empty()) return -1;
    a->slots[seq_id] = a->free_slots.back();
    a->free_slots.pop_back();
  }
  if (need <= 0) {
    if (fresh) a->tables[seq_id];
    return 0;
  }
  auto& tab = a->tables[seq_id];
  for (int i = 0; i < need; ++i) tab.push_back(a->take());
  return need;
}

int rb_ba_free(RbBlockAllocator* a, int64_t seq_id) {
  std::lock_guard<std::mutex> l(a->mu);
  auto it = a->tables.find(seq_id);
  if (it == a->tables.end()) return 0;
  const int n = (int)it->second.size();
  for (auto rit = it->second.rbegin(); rit != it->second.rend(); ++rit) a->give(*rit);
  a->tables.erase(it);
  auto st = a->slots.find(seq_id);
  if (st != a->slots.end()) {
    a->free_slots.push_back(st->second);
    a->slots.erase(st);
  }
  return n;
}

// Gives back the blocks behind the first num_tokens tokens of a sequence, which keeps its other blocks and its state slot.  Returns their
// number, -1 for an unknown sequence.
int rb_ba_trim(RbBlockAllocator* a, int64_t seq_id, int num_tokens) {
  std::lock_guard<std::mutex> l(a->mu);
  auto it = a->tables.find(seq_id);
  if (it == a->tables.end() || num_tokens < 0) return -1;
  int n = 0;
  for (const size_t keep = blocks_for(a, num_tokens); it->second.size() > keep; ++n) {
    a->give(it->second.back());
    it->second.pop_back();
  }
  return n;
}

// Makes `child` a sequence that shares the parent's first num_tokens tokens: full blocks are in both tables, and for a block that these tokens end in the child takes one of its own.
// Returns 1 when the caller has to copy block *src to *dst, 0 when there is nothing to copy, -1 when the parent is unknown or has no blocks for so many tokens, or the child is there
// already, -2 when there is no free block or state slot (nothing changed).
int rb_ba_fork(RbBlockAllocator* a, int64_t parent, int64_t child, int num_tokens, int32_t* src, int32_t* dst) try {
  std::lock_guard<std::mutex> l(a->mu);
  auto it = a->tables.find(parent);
  if (it == a->tables.end() || num_tokens < 0 || blocks_for(a, num_tokens) > (int)it->second.size() || a->tables.count(child)) return -1;
  const int full = num_tokens / a->block_size;
  const bool partial = num_tokens % a->block_size != 0;
  if ((partial && a->free_list.empty()) || (a->slotted && a->free_slots.empty())) return -2;
  std::vector<int32_t> tab(it->second.begin(), it->second.begin() + full);
  const int32_t last = partial ? it->second[full] : -1;
  tab.reserve(full + 1);
  auto& at = a->tables[child];                                   // may move the parent's entry: not used from here on
  if (a->slotted) {
    a->slots[child] = a->free_slots.back();
    a->free_slots.pop_back();
  }
  for (int32_t b : tab)
    if (++a->owners[b] == 2) ++a->shared;
  if (partial) {
    *src = last;
    *dst = a->take();
    tab.push_back(*dst);
  }
  at.swap(tab);
  return partial ? 1 : 0;
} catch (...) {
  return -2;
}

int rb_ba_num_shared(const RbBlockAllocator* a) { std::lock_guard<std::mutex> l(a->mu); return a->shared; }

// Gives sequences blocks of their own in place of shared ones among those of tokens first[i] .. first[i] + count[i] - 1 of sequence ids[i], which are about to be written.  Returns how many
// pairs of blocks (src, dst, room for `max`) the caller has to copy, -1 for an unknown sequence or tokens without blocks, -2 without enough free blocks, room or memory (nothing changed
// in either case).  Of sequences that share a block with each other alone, the last one keeps it.
int rb_ba_own(RbBlockAllocator* a, const int64_t* ids, const int64_t* first, const int64_t* count, int n, int32_t* src, int32_t* dst, int max) try {
  std::lock_guard<std::mutex> l(a->mu);
  for (int i = 0; i < n; ++i) {
    auto it = a->tables.find(ids[i]);
    if (it == a->tables.end() || first[i] < 0 || count[i] < 0 || first[i] + count[i] > (int64_t)it->second.size() * a->block_size) return -1;
  }
  std::vector<int32_t*> changed;
  changed.reserve(std::min<size_t>(max < 0 ? 0 : max, a->free_list.size()));
  int k = 0;
  for (int i = 0; i < n; ++i) {
    if (count[i] == 0) continue;
    std::vector<int32_t>& tab = a->tables.find(ids[i])->second;
    for (int64_t j = first[i] / a->block_size; j <= (first[i] + count[i] - 1) / a->block_size; ++j) {
      int32_t& b = tab[j];
      if (a->owners[b] < 2) continue;
      if (k == max || a->free_list.empty()) {
        while (k-- > 0) {                                        // everything as it was, the order of the free list too
          a->owners[dst[k]] = 0;
          a->free_list.push_back(dst[k]);
          if (++a->owners[src[k]] == 2) ++a->shared;
          *changed[k] = src[k];
        }
        return -2;
      }
      src[k] = b;
      dst[k] = a->take();
      a->give(b);
      b = dst[k++];
      changed.push_back(&b);
    }
  }
  return k;
} catch (...) {
  return -2;
}

// Moves what is in use to the lowest blocks: tables, owners and the free list change at once, and the caller copies the blocks src[i] to dst[i] (room for num_blocks each).
// Returns the number of pairs, -1 without memory.
int rb_ba_compact(RbBlockAllocator* a, int32_t* src, int32_t* dst) try {
  std::lock_guard<std::mutex> l(a->mu);
  const int used = a->num_blocks - (int)a->free_list.size();
  std::vector<int32_t> to(a->num_blocks, -1), rest;
  rest.reserve(a->num_blocks);
  int n = 0, low = 0;
  for (int b = used; b < a->num_blocks; ++b) {
    if (!a->owners[b]) continue;
    while (a->owners[low]) ++low;
    src[n] = b;
    dst[n++] = low;
    to[b] = low;
    a->owners[low] = a->owners[b];
    a->owners[b] = 0;
  }
  for (int b = a->num_blocks - 1; b >= used; --b) rest.push_back(b);
  for (auto& t : a->tables)
    for (int32_t& b : t.second)
      if (to[b] >= 0) b = to[b];
  a->free_list.swap(rest);
  return n;
} catch (...) {
  return -1;
}

int rb_ba_table_len(const RbBlockAllocator* a, int64_t seq_id) {
  std::lock_guard<std::mutex> l(a->mu);
  auto it = a->tables.find(seq_id);
  return it == a->tables.end() ? -1 : (int)it->second.size();
}

int rb_ba_table(const RbBlockAllocator* a, int64_t seq_id, int32_t* out, int max_out) {
  std::lock_guard<std::mutex> l(a->mu);
  auto it = a->tables.find(seq_id);
  if (it == a->tables.end()) return -1;
  const int n = (int)it->second.size();
  for (int i = 0; i < n && i < max_out; ++i) out[i] = it->second[i];
  return n;
}

// Block tables of `n` sequences, one row of `width` entries each (zeros behind a table's end and for
// unknown sequences).  Returns 0, or -1 when a table is longer than that.
int rb_ba_tables(const RbBlockAllocator* a, const int64_t* seq_ids, int n, int width, int32_t* out) {
  std::lock_guard<std::mutex> l(a->mu);
  int rc = 0;
  for (int i = 0; i < n; ++i) {
    int32_t* row = out + (int64_t)i * width;
    int m = 0;
    auto it = a->tables.find(seq_ids[i]);
    if (it != a->tables.end()) {
      if ((int)it->second.size() > width) rc = -1;
      for (m = 0; m < width && m < (int)it->second.size(); ++m) row[m] = it->second[m];
    }
    for (; m < width; ++m) row[m] = 0;
  }
  return rc;
}

// Positions start .. start + n - 1 of a sequence and their cache slots.  Returns 0, or -1 when one of them has no block.
int rb_ba_slots(const RbBlockAllocator* a, int64_t seq_id, int64_t start, int64_t n, int64_t* pos, int64_t* slots) {
  std::lock_guard<std::mutex> l(a->mu);
  auto it = a->tables.find(seq_id);
  if (it == a->tables.end() || start < 0 || start + n > (int64_t)it->second.size() * a->block_size) return -1;
  for (int64_t i = 0; i < n; ++i) {
    const int64_t p = start + i;
    pos[i] = p;
    slots[i] = (int64_t)it->second[p / a->block_size] * a->block_size + p % a->block_size;
  }
  return 0;
}

int64_t rb_ba_slot(const RbBlockAllocator* a, int64_t seq_id, int token_index) {
  std::lock_guard<std::mutex> l(a->mu);
  auto it = a->tables.find(seq_id);
  if (it == a->tables.end() || token_index < 0) return -1;
  const int b = token_index / a->block_size;
  if (b >= (int)it->second.size()) return -1;
  return (int64_t)it->second[b] * a->block_size + token_index % a->block_size;
}

int rb_ba_num_sequences(const RbBlockAllocator* a) { std::lock_guard<std::mutex> l(a->mu); return (int)a->tables.size(); }

}  // extern "C"
