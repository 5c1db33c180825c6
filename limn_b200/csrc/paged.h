// What the kernels over a paged key and value cache share: the step as they take it, how a sequence's extents are read and checked
// on the device, and how a page is found.
#pragma once

#include <cuda_runtime.h>

#include "common.h"

namespace limn_b200 {
namespace paged {

// One side (K or V) of the cache: element (page, head, slot, 0) at base + page * page_stride + ..., in bytes.
struct Pages {
  unsigned char* base = nullptr;
  long long page = 0, head = 0, slot = 0;
};

// A pass of queries over paged keys.
struct Pass {
  const unsigned char* q = nullptr;
  unsigned char* out = nullptr;
  float* lse = nullptr;
  long long q_token = 0, q_head = 0, o_token = 0, o_head = 0;  // bytes
  Pages k, v;
  const int* table = nullptr;    // (batch, max_pages)
  const int* q_start = nullptr;  // (batch + 1)
  const int* kv_lens = nullptr;  // (batch)
  unsigned* errors = nullptr;
  const int* prefix_table = nullptr;
  int prefix_len = 0;
  int batch = 0, heads = 0, kv_heads = 0, group = 1;  // group: query heads to a key head
  int pieces = 0, pieces_v = 0;                       // groups of 8 columns of a row of Q and K, of V and O
  int page_size = 0, pages = 0, max_pages = 0, tokens = 0, max_t_q = 0;
  int causal = 0;
  float scale = 0.f;
};

// A sequence's extents: `first` token of `n`, `keys` in its pages. One that cannot be has n = 0 and is noted.
struct Extent {
  int first, n, keys;
};
__device__ __forceinline__ Extent extent_of(const int* q_start, const int* kv_lens, int b, int tokens, int max_t_q, int max_pages, int page_size, unsigned* errors) {
  const long long first = q_start[b], end = q_start[b + 1], keys = kv_lens[b];
  if (first < 0 || end < first || end > tokens || end - first > max_t_q || keys < 0 || keys > static_cast<long long>(max_pages) * page_size) {
    if (errors != nullptr) atomicOr(errors, LIMN_B200_PAGED_BAD_SEQUENCE);
    return Extent{0, 0, 0};
  }
  return Extent{static_cast<int>(first), static_cast<int>(end - first), static_cast<int>(keys)};
}

// The sequence whose tokens `token` is among: how many sequences end at or before it (batch: none of them goes on past it). A warp's
// 32-ary search over q_start[1..batch]; where the offsets do not rise the answer is some number up to batch.
__device__ __forceinline__ int sequence_of(const int* q_start, int batch, int token, int lane) {
  int low = 0, high = batch;  // the answer lies in [low, high]
  while (high > low) {
    const int span = (high - low + 31) / 32;
    const int probe = low + lane * span;
    const bool before = probe < high && q_start[probe + 1] <= token;
    const int many = __popc(__ballot_sync(0xffffffffu, before));
    if (many == 0) {
      high = low;
    } else {
      const int last = low + (many - 1) * span;  // this one ends at or before the token
      low = last + 1;
      high = min(last + span, high);
    }
  }
  return low;
}

// The page that `table` has at `at`, or -1 where it is none.
__device__ __forceinline__ int page_at(const int* table, int at, int pages, unsigned* errors) {
  const int page = table[at];
  if (page >= 0 && page < pages) return page;
  if (errors != nullptr) atomicOr(errors, LIMN_B200_PAGED_BAD_PAGE);
  return -1;
}

}  // namespace paged

// Checks of a step that every entry point makes, of its extents and strides and of its pointers; `name` is the op's.
int check_paged(const char* name, const limn_b200_paged* step);
int check_paged_pointers(const char* name, const limn_b200_paged* step);

}  // namespace limn_b200
