// What the kernels over a paged key and value cache share: the step as they take it, how a sequence's extents are read and checked
// on the device, how a page is found, how work is cut into equal shares, and where rows and parts of rows go.
#pragma once

#include <cuda_runtime.h>

#include "common.h"
#include "sm100_ptx.cuh"

namespace limn_b200 {
namespace paged {

constexpr float kLog2e = 1.4426950408889634f;

// One side (K or V) of the cache: element (page, head, slot, 0) at base + page * page_stride + ..., in bytes.
struct Pages {
  unsigned char* base = nullptr;
  long long page = 0, head = 0, slot = 0;
};

// One worker's share of the work may begin and end inside a problem. What it has of a problem that others share is a part: the sums
// O (unnormalised) and the statistics m (the score the weights are measured against, raw units) and l of its rows. A worker has
// room for two parts, 2 w: of a problem that began with a worker before, 2 w + 1: of one that begins here and goes on. The worker where
// a problem begins says in heads[w] which rows the parts are of and how many workers follow; 0 followers: nothing to join; kServesNone:
// nor has the pass anything for any row.
constexpr int kServesNone = -1;
struct Head {
  int followers;
  int first, n;   // the sequence's first token, and tokens
  int kv_head;
  int row0;       // the first row, rows being (token, head of the group)
  int tile_rows;  // rows of a tile: row r of a part is row row0 + r / 128 * tile_rows + r % 128, if r % 128 < tile_rows
};
struct Parts {
  double share = 0.0;      // 1 / workers
  float* o = nullptr;      // (2 workers, rows, width)
  float2* ml = nullptr;    // (2 workers, rows)
  Head* heads = nullptr;   // (workers)
  int workers = 0, rows = 0, width = 0;
  static size_t o_bytes(int workers, int rows, int width) { return static_cast<size_t>(2) * workers * rows * width * 4; }
  static size_t ml_bytes(int workers, int rows) { return static_cast<size_t>(2) * workers * rows * 8; }
  static size_t head_bytes(int workers) { return (static_cast<size_t>(workers) * sizeof(Head) + 255) / 256 * 256; }
  static size_t bytes(int workers, int rows, int width) { return o_bytes(workers, rows, width) + ml_bytes(workers, rows) + head_bytes(workers); }
  // A worker's share of `total`: shares of all workers cover it.
  __device__ __forceinline__ long long share_of(long long total) const { return static_cast<long long>(static_cast<double>(total) * share) + 1; }
  // Lays the parts out in `memory`, which has the bytes for them.
  void place(unsigned char* memory, int workers_, int rows_, int width_) {
    workers = workers_, rows = rows_, width = width_, share = 1.0 / workers_;
    o = reinterpret_cast<float*>(memory), memory += o_bytes(workers, rows, width);
    ml = reinterpret_cast<float2*>(memory), memory += ml_bytes(workers, rows);
    heads = reinterpret_cast<Head*>(memory);
  }
};

// Sums and statistics of every (token, head) row over some of its keys, in memory: what the pass over a shared prefix leaves and what the
// pass over the sequences' own keys does, for a last kernel to put together. Where a row's problem was shared by workers its sums are
// parts, and the statistics say so: kInParts in place of l, the worker where the problem begins as the bits of m, and in `part_row` the row there.
constexpr float kInParts = -1.f;  // (l is a sum of exponentials: never negative)
struct RowSums {
  float* o = nullptr;       // (tokens * heads, width), unnormalised
  float2* ml = nullptr;     // (tokens * heads)
  int* part_row = nullptr;  // (tokens * heads)
  static size_t bytes(size_t rows, int width) { return rows * (static_cast<size_t>(width) * 4 + 8) + (rows * 4 + 255) / 256 * 256; }
  void place(unsigned char* memory, size_t rows, int width) {
    o = reinterpret_cast<float*>(memory), memory += rows * width * 4;
    ml = reinterpret_cast<float2*>(memory), memory += rows * 8;
    part_row = reinterpret_cast<int*>(memory);
  }
};

// Quotients by a number that a launch knows: a product and a shift (exact for numerators from 0 to 2^31 - 1: the factor is 2^(31 + s) / d rounded
// up, with 2^s >= d, so its excess times the numerator stays below 2^(31 + s) / d).
struct Div {
  unsigned d = 1, factor = 1u << 31, shift = 31;
  Div() = default;
  explicit Div(int by) : d(static_cast<unsigned>(by)) {
    unsigned s = 0;
    while ((1ull << s) < d) ++s;
    shift = 31 + s, factor = static_cast<unsigned>(((1ull << shift) + d - 1) / d);
  }
  __host__ __device__ __forceinline__ int of(int n) const { return static_cast<int>((static_cast<unsigned long long>(static_cast<unsigned>(n)) * factor) >> shift); }
  __host__ __device__ __forceinline__ int rest(int n) const { return n - of(n) * static_cast<int>(d); }
};

// A pass of queries over paged keys.
struct Pass {
  const unsigned char* q = nullptr;
  unsigned char* out = nullptr;
  float* lse = nullptr;
  long long q_token = 0, q_head = 0, o_token = 0, o_head = 0;  // bytes
  Pages k, v;
  const int* table = nullptr;    // (batch, max_pages)
  const int* q_start = nullptr;  // (batch + 1); null: one sequence of all tokens
  const int* kv_lens = nullptr;  // (batch); null with q_start: `keys` of them
  unsigned* errors = nullptr;
  int keys = 0;
  // Keys that stand in front of every sequence's own: prefix_len of them in the pages that prefix_table names, counted as `front`, rounded up to whole units or
  // key tiles: a sequence's key f + j is key j of its own pages. Those between do not exist.
  const int* prefix_table = nullptr;
  int prefix_len = 0, front = 0;
  int batch = 0, heads = 0, kv_heads = 0, group = 1;  // group: query heads to a key head
  Div by_group, by_page;                              // quotients by it and by page_size
  int pieces = 0, pieces_v = 0;                       // groups of 8 columns of a row of Q and K, of V and O
  int page_size = 0, pages = 0, max_pages = 0, tokens = 0, max_t_q = 0;
  int causal = 0;
  float scale = 0.f;
  Parts parts;
  RowSums leave;  // where rows go instead of `out`, or null
  int blocks = 0;  // that make the pass, one to a multiprocessor
};

// A sequence's extents: `first` token of `n`, `keys` it has, those in front among them. One that cannot be has n = 0 and is noted; one whose offsets fall
// has first = kFalls besides: where any do, sequences that are possible each by itself could have tokens in common, so the pass serves none of them (every
// worker looks at all of them to find its share, and so at this).
constexpr int kFalls = -1;
struct Extent {
  int first, n, keys;
};
__device__ __forceinline__ Extent extent_of(const int* q_start, const int* kv_lens, int b, int tokens, int max_t_q, int max_pages, int page_size, unsigned* errors) {
  const long long first = q_start[b], end = q_start[b + 1], keys = kv_lens[b];
  const bool idle = first == end;  // it brings no token: its length, which may be of an earlier step, is of no concern
  if (first < 0 || end < first || end > tokens || end - first > max_t_q || (!idle && (keys < 0 || keys > static_cast<long long>(max_pages) * page_size))) {
    if (errors != nullptr) atomicOr(errors, LIMN_B200_PAGED_BAD_SEQUENCE);
    return Extent{end < first ? kFalls : 0, 0, 0};
  }
  if (idle) return Extent{static_cast<int>(first), 0, 0};
  return Extent{static_cast<int>(first), static_cast<int>(end - first), static_cast<int>(keys)};
}
__device__ __forceinline__ Extent extent_of(const Pass& p, int b) {
  if (p.q_start == nullptr) return Extent{0, p.tokens, p.keys};
  Extent e = extent_of(p.q_start, p.kv_lens, b, p.tokens, p.max_t_q, p.max_pages, p.page_size, p.errors);
  e.keys += p.front;
  return e;
}
// Of the keys on key's side of the end of the front: up to where they exist, the table's entry for one of them, and its slot.
__device__ __forceinline__ int side_end(const Pass& p, int key, int keys) { return key < p.front ? p.prefix_len : keys; }
__device__ __forceinline__ int entry_for(const Pass& p, int b, int key) {
  return key < p.front ? p.prefix_table[p.by_page.of(key)] : p.table[static_cast<long long>(b) * p.max_pages + p.by_page.of(key - p.front)];
}
__device__ __forceinline__ int slot_of(const Pass& p, int key) { return p.by_page.rest(key < p.front ? key : key - p.front); }

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

// `page` as the table has it, or -1 where it is none.
__device__ __forceinline__ int checked_page(int page, int pages, unsigned* errors) {
  if (page >= 0 && page < pages) return page;
  if (errors != nullptr) atomicOr(errors, LIMN_B200_PAGED_BAD_PAGE);
  return -1;
}

// Where row r of a sequence's (token, head of the group) rows has its result and its statistics.
struct RowPlace {
  long long row;      // token * heads + head
  unsigned char* out;
};
__device__ __forceinline__ RowPlace row_place(const Pass& p, int first, int kv_head, int r) {
  const int i = p.by_group.of(r), g = r - i * p.group;
  const long long token = first + i;
  const int head = kv_head * p.group + g;
  return RowPlace{token * p.heads + head, p.out + token * p.o_token + head * p.o_head};
}

// Two sides of a row put together: statistics (m, l) and (m_b, l_b) become those of both, `keep` and `add` what the sums of either count.
// (A side that has seen no key has m = -inf, l = 0 and counts 0; a NaN in l stays one.)
__device__ __forceinline__ void merge_stats(float& m, float& l, float m_b, float l_b, float sl2, float& keep, float& add) {
  const float top = fmaxf(m, m_b), base = top == -INFINITY ? 0.f : top;
  keep = ptx::exp2_approx((m - base) * sl2), add = ptx::exp2_approx((m_b - base) * sl2);
  m = top, l = l * keep + l_b * add;
}

// a / b of numbers below 2^52 whose quotient fits an int: by float64 and put right. (The compiler's 64-bit division is some 100 instructions.)
__device__ __forceinline__ int small_quotient(long long a, long long b) {
  long long q = static_cast<long long>(static_cast<double>(a) * (1.0 / static_cast<double>(b)));
  while (q * b > a) --q;
  while ((q + 1) * b <= a) ++q;
  return static_cast<int>(q);
}

// The place in ends[0..n), which rises, of the first that times `by` is above x.
__device__ __forceinline__ int first_above(const long long* ends, int n, int by, long long x) {
  int low = 0, high = n;
#pragma unroll 1
  while (low < high) {
    const int mid = (low + high) >> 1;
    if (ends[mid] * by <= x) low = mid + 1;
    else high = mid;
  }
  return low;
}

}  // namespace paged

// Checks of a step that every entry point makes, of its extents and strides and of its pointers; `name` is the op's.
int check_paged(const char* name, const limn_b200_paged* step);
int check_paged_pointers(const char* name, const limn_b200_paged* step);
// Whether the cache is memory that the current device's kernels can read, asked last of all.
int check_paged_device(const char* name, const limn_b200_paged* step);

constexpr long long kMaxKeys = 0x7fff0000LL;  // keys, positions and rows are counted in int, some key tiles past the last one included
constexpr int kPagedUnit = 16, kPagedTile = 128;  // keys that a prefix in front is rounded up to, by the kernel that makes the pass
// The kernels that make a pass, for few rows to a key head and for any number. Each lays its parts out in `workspace` and says so in pass.parts.
constexpr int kPagedFewRows = 16;  // max_t_q * group up to here
size_t paged_few_workspace(int rows, int width, int sms);
int paged_few_launch(paged::Pass& pass, bool fp16, int rows, unsigned char* workspace, cudaStream_t stream);
size_t paged_many_workspace(int width, int sms);
int paged_many_launch(paged::Pass& pass, bool fp16, unsigned char* workspace, cudaStream_t stream);
// Behind a pass: rows whose problems were shared, out of their parts (of the kernel for few rows, whose problems have few rows and many parts, or of the other one).
int paged_join_launch(const paged::Pass& pass, bool fp16, bool many_rows, cudaStream_t stream);
// Behind two passes that leave their rows' sums: the rows of both together, of up to so many heads (a block has four of one token, or one where rows are few).
constexpr int kPagedFinishHeads = 4 * 65535;
int paged_finish_launch(const paged::Pass& front, const paged::Pass& own, bool fp16, cudaStream_t stream);

}  // namespace limn_b200
