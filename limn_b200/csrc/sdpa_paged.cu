// Attention of a step's tokens over the pages of their sequences, and over a prefix that all of them share.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <cmath>

#include "paged.h"
#include "sm100_ptx.cuh"

namespace limn_b200 {
namespace {

using namespace paged;

// Which kernel a pass of at most `rows` rows to a (sequence, key head) takes, and the workspace it has to itself. Up to 16 rows a tile of mma.sync's
// holds them and the pass is bound by the keys' bytes; the other kernel's tiles are 128 rows. Few-rows kernel : the other, in us, keys of 128: 4 rows, 64 sequences of up to
// 8191 keys 181 : 202, 8 of 2000 keys 19 : 29; 16 rows 200 : 205 and 26 : 29. (17 rows and more only the other one has tiles for.)
size_t pass_workspace(long long rows, int width, int sms) {
  return rows <= kPagedFewRows ? paged_few_workspace(static_cast<int>(rows), width, sms) : paged_many_workspace(width, sms);
}
int launch_pass(Pass& pass, bool fp16, long long rows, unsigned char* workspace, cudaStream_t stream) {
  return rows <= kPagedFewRows ? paged_few_launch(pass, fp16, static_cast<int>(rows), workspace, stream) : paged_many_launch(pass, fp16, workspace, stream);
}

// A call behind a prefix either reads it once for the whole batch, in a pass of its own over all rows, whose sums are joined with those of the pass over the
// sequences' own keys; or it puts the prefix in front of every sequence's keys and makes one pass. The first reads and computes less. The second launches two
// kernels instead of three and leaves no sums in memory. Which is faster goes by what either costs beyond the other, as far as the host knows it:
//   apart: 6 us, and 16 bytes for each element of O, written and read at 3 TB/s;
//   in front, few rows to a key head: the prefix is read once more for every sequence, mostly out of L2, at 12 TB/s;
//   in front, more rows: a sequence's rows fill tiles of 128 less well than the batch's do; two such tiles by 128 keys of 128 columns take a multiprocessor 2.1 us.
// Measured, 32 heads over 8 key heads of 128, 100 to 800 keys of their own, apart : in front, in us: one token of 8 sequences behind 2048 keys 26.3 : 18.8, of 32
// behind 1024 33.7 : 31.7 and 2048 34.4 : 46.2, of 32 behind 8192 43.0 : 132, of 128 behind 128 73 : 54; up to 200 own keys, 8 to 16 tokens of 32 sequences behind 1024 43.4 : 45.7,
// behind 8192 82 : 145; 128 to 256 tokens of 32 sequences behind 1024 293 : 151, behind 8192 816 : 726. Over these and other heads (8 over 1, 28 over 4, 16 over 2 of 64), 106
// calls, the rule is never wrong by more than 3 us.
bool prefix_in_front(const limn_b200_paged* step, int prefix_len, int sms) {
  if (static_cast<long long>(step->max_pages) * step->page_size + prefix_len > kMaxKeys) return false;  // (positions in front and behind count in one int)
  const long long group = step->heads / step->kv_heads;
  const double apart = 6 + 16.0 * step->hd_v * step->tokens * step->heads / 3e6;
  if (step->max_t_q * group <= kPagedFewRows) {
    const double bytes = 2.0 * prefix_len * step->kv_heads * (step->hd + step->hd_v);
    return (step->batch - 1) * bytes / 12e6 <= apart;
  }
  const double rows = static_cast<double>(step->tokens) * group, width = std::max(step->hd, step->hd_v) > 64 ? 1 : 0.5;
  const double more = step->batch * std::ceil(rows / step->batch / 128) - std::ceil(rows / 128);  // tiles
  return more / 2 * step->kv_heads * std::ceil(prefix_len / 128.0) * width * 2.1 / sms <= apart;
}

// Shares of the work are counted in 64 bits, a warp's in 32 of them, 16 keys at a time: 2^43 keys that (tile, key head) pairs see is far below either.
bool countable(const limn_b200_paged* step, double keys) {
  const double group = step->heads / step->kv_heads;
  return step->kv_heads * (std::min(step->batch, step->tokens) + step->tokens * group / 64) * (keys + 256) <= 8.8e12;
}

// The workspace of a call: the parts of the pass over the own keys; behind a prefix also those of the pass over it, and the rows' sums
// over either, however long it is: a workspace that serves one prefix serves all.
struct Workspace {
  size_t own, front, sums;  // sums: of one pass
  size_t bytes() const { return own + front + 2 * sums; }
};
int workspace_of(const limn_b200_paged* step, int prefix_len, Workspace* w) {
  int sms = 0;
  if (int rc = sm_count(&sms)) return rc;
  const int width = step->hd <= 64 && step->hd_v <= 64 ? 64 : 128;
  const long long group = step->heads / step->kv_heads;
  const size_t rows = static_cast<size_t>(step->tokens) * step->heads;
  w->own = pass_workspace(step->max_t_q * group, width, sms);
  w->front = prefix_len > 0 ? pass_workspace(step->tokens * group, width, sms) : 0;
  w->sums = prefix_len > 0 ? (RowSums::bytes(rows, width) + 255) / 256 * 256 : 0;
  return LIMN_B200_OK;
}

int paged_pass(const char* name, const limn_b200_paged* step, const void* q, void* out, float* lse, const long long* strides, const int* prefix_table,
               int prefix_len, int causal, double scale, void* workspace, unsigned long long workspace_bytes, void* stream) {
  clear_error();
  reset_launches();
  if (int rc = check_paged(name, step)) return rc;
  if (int rc = check_paged_pointers(name, step)) return rc;
  if (!q || !out || !lse || !strides) return fail(LIMN_B200_BAD_ARGUMENT, "%s: a required pointer is null", name);
  if ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(out) | reinterpret_cast<uintptr_t>(workspace)) & 15u)
    return fail(LIMN_B200_BAD_ARGUMENT, "%s: an operand is not 16-byte aligned", name);
  if ((reinterpret_cast<uintptr_t>(lse) | reinterpret_cast<uintptr_t>(prefix_table)) & 3u)
    return fail(LIMN_B200_BAD_ARGUMENT, "%s: lse or the prefix's table is not 4-byte aligned", name);
  if (!countable(step, prefix_len)) return fail(LIMN_B200_UNSUPPORTED, "%s: %d sequences behind a prefix of %d keys are more work than a call counts", name, step->batch, prefix_len);
  for (int i = 0; i < 4; ++i)
    if (strides[i] < 0 || (strides[i] & 7)) return fail(LIMN_B200_BAD_ARGUMENT, "%s: strides must be non-negative multiples of 8 elements, got %lld", name, strides[i]);
  if (!(scale >= 1e-30 && scale <= 1e30)) return fail(LIMN_B200_UNSUPPORTED, "%s: the scale must be positive, from 1e-30 to 1e30", name);
  if (step->tokens == 0 || step->batch == 0) return LIMN_B200_OK;
  Workspace w;
  if (int rc = workspace_of(step, prefix_len, &w)) return rc;
  if (w.bytes() > 0 && (!workspace || workspace_bytes < w.bytes()))
    return fail(LIMN_B200_BAD_ARGUMENT, "%s: the workspace has %llu bytes, %llu are needed", name, workspace_bytes, static_cast<unsigned long long>(w.bytes()));
  if (int rc = check_paged_device(name, step)) return rc;
  Pass prm;
  prm.q = static_cast<const unsigned char*>(q), prm.out = static_cast<unsigned char*>(out), prm.lse = lse;
  prm.q_token = 2 * strides[0], prm.q_head = 2 * strides[1], prm.o_token = 2 * strides[2], prm.o_head = 2 * strides[3];
  prm.k = {static_cast<unsigned char*>(step->k_cache), 2 * step->k_strides[0], 2 * step->k_strides[1], 2 * step->k_strides[2]};
  prm.v = {static_cast<unsigned char*>(step->v_cache), 2 * step->v_strides[0], 2 * step->v_strides[1], 2 * step->v_strides[2]};
  prm.table = step->page_table, prm.q_start = step->q_start, prm.kv_lens = step->kv_lens, prm.errors = step->errors;
  prm.batch = step->batch, prm.heads = step->heads, prm.kv_heads = step->kv_heads, prm.group = step->heads / step->kv_heads;
  prm.pieces = step->hd / 8, prm.pieces_v = step->hd_v / 8;
  prm.page_size = step->page_size, prm.pages = step->pages, prm.max_pages = step->max_pages, prm.tokens = step->tokens, prm.max_t_q = step->max_t_q;
  prm.by_group = Div(prm.group), prm.by_page = Div(prm.page_size);
  prm.causal = causal != 0, prm.scale = static_cast<float>(scale);
  const bool fp16 = step->dtype == LIMN_B200_F16;
  const cudaStream_t on = static_cast<cudaStream_t>(stream);
  unsigned char* memory = static_cast<unsigned char*>(workspace);
  const long long rows = static_cast<long long>(step->max_t_q) * prm.group;
  if (int rc = sm_count(&prm.blocks)) return rc;
  const bool in_front = prefix_len > 0 && prefix_in_front(step, prefix_len, prm.blocks);
  if (in_front) {
    const int whole = rows <= kPagedFewRows ? kPagedUnit : kPagedTile;
    prm.prefix_table = prefix_table, prm.prefix_len = prefix_len, prm.front = (prefix_len + whole - 1) / whole * whole;
  }
  if (prefix_len == 0 || in_front) {
    if (int rc = launch_pass(prm, fp16, rows, memory, on)) return rc;
    return paged_join_launch(prm, fp16, rows > kPagedFewRows, on);
  }
  // every row over the prefix, as one sequence of all tokens that sees all of it (tokens that belong to no sequence too: nothing asks for those); every row
  // over its own keys; and the two together. Each kernel waits for the one in front of it before it reads memory: only that makes what was
  // written before the call, the step's new keys among it, visible to it.
  const int width = prm.pieces <= 8 && prm.pieces_v <= 8 ? 64 : 128;
  const size_t all_rows = static_cast<size_t>(step->tokens) * step->heads;
  Pass front = prm;
  front.table = prefix_table, front.q_start = nullptr, front.kv_lens = nullptr, front.keys = prefix_len, front.batch = 1, front.causal = 0;
  front.leave.place(memory + w.own + w.front, all_rows, width), prm.leave.place(memory + w.own + w.front + w.sums, all_rows, width);
  if (int rc = launch_pass(front, fp16, static_cast<long long>(step->tokens) * prm.group, memory + w.own, on)) return rc;
  if (int rc = launch_pass(prm, fp16, rows, memory, on)) return rc;
  return paged_finish_launch(front, prm, fp16, on);
}

}  // namespace

int check_paged(const char* name, const limn_b200_paged* s) {
  if (!s) return fail(LIMN_B200_BAD_ARGUMENT, "%s: null step", name);
  if (s->dtype < LIMN_B200_F32 || s->dtype > LIMN_B200_F64) return fail(LIMN_B200_BAD_ARGUMENT, "%s: unknown dtype code %d", name, s->dtype);
  if (s->batch < 0 || s->tokens < 0 || s->max_t_q <= 0 || s->heads <= 0 || s->kv_heads <= 0 || s->hd <= 0 || s->hd_v <= 0 || s->page_size <= 0 || s->pages <= 0 ||
      s->max_pages <= 0)
    return fail(LIMN_B200_BAD_ARGUMENT, "%s: extents must be positive, got batch=%d tokens=%d max_t_q=%d heads=%d kv_heads=%d hd=%d hd_v=%d page_size=%d pages=%d max_pages=%d",
                name, s->batch, s->tokens, s->max_t_q, s->heads, s->kv_heads, s->hd, s->hd_v, s->page_size, s->pages, s->max_pages);
  if (s->heads % s->kv_heads != 0) return fail(LIMN_B200_BAD_ARGUMENT, "%s: %d heads are no multiple of %d key heads", name, s->heads, s->kv_heads);
  if (s->first_position < 0) return fail(LIMN_B200_BAD_ARGUMENT, "%s: the first position is %d", name, s->first_position);
  if (s->dtype != LIMN_B200_F16 && s->dtype != LIMN_B200_BF16) return fail(LIMN_B200_UNSUPPORTED, "%s: a paged cache is served for f16/bf16", name);
  if (s->hd % 8 != 0 || s->hd > 128 || s->hd_v % 8 != 0 || s->hd_v > 128)
    return fail(LIMN_B200_UNSUPPORTED, "%s: a paged cache is served for hd and hd_v multiples of 8 up to 128, got %d and %d", name, s->hd, s->hd_v);
  if (s->page_size % 8 != 0) return fail(LIMN_B200_UNSUPPORTED, "%s: the page size must be a multiple of 8, got %d", name, s->page_size);
  if (s->heads / s->kv_heads > 128) return fail(LIMN_B200_UNSUPPORTED, "%s: %d query heads to a key head, at most 128 are served", name, s->heads / s->kv_heads);
  if (static_cast<long long>(s->tokens) * s->heads > kMaxKeys) return fail(LIMN_B200_UNSUPPORTED, "%s: %d tokens of %d heads do not fit 31 bits", name, s->tokens, s->heads);
  if (s->batch > kMaxKeys) return fail(LIMN_B200_UNSUPPORTED, "%s: %d sequences do not fit 31 bits", name, s->batch);
  if (static_cast<long long>(s->max_pages) * s->page_size > kMaxKeys - s->first_position)
    return fail(LIMN_B200_UNSUPPORTED, "%s: positions of %d pages of %d from %d on do not fit 31 bits", name, s->max_pages, s->page_size, s->first_position);
  if (!countable(s, static_cast<double>(s->max_pages) * s->page_size))
    return fail(LIMN_B200_UNSUPPORTED, "%s: %d sequences of up to %d pages of %d keys are more work than a call counts", name, s->batch, s->max_pages, s->page_size);
  for (int i = 0; i < 3; ++i)
    if (s->k_strides[i] < 0 || (s->k_strides[i] & 7) || s->v_strides[i] < 0 || (s->v_strides[i] & 7))
      return fail(LIMN_B200_BAD_ARGUMENT, "%s: cache strides must be non-negative multiples of 8 elements", name);
  return LIMN_B200_OK;
}

int check_paged_pointers(const char* name, const limn_b200_paged* s) {
  if (!s->k_cache || !s->v_cache || !s->page_table || !s->q_start || !s->kv_lens) return fail(LIMN_B200_BAD_ARGUMENT, "%s: a required pointer of the step is null", name);
  if ((reinterpret_cast<uintptr_t>(s->page_table) | reinterpret_cast<uintptr_t>(s->q_start) | reinterpret_cast<uintptr_t>(s->kv_lens) | reinterpret_cast<uintptr_t>(s->errors)) & 3u)
    return fail(LIMN_B200_BAD_ARGUMENT, "%s: the table, the offsets, the lengths or the word for errors is not 4-byte aligned", name);
  if ((reinterpret_cast<uintptr_t>(s->k_cache) | reinterpret_cast<uintptr_t>(s->v_cache)) & 15u) return fail(LIMN_B200_BAD_ARGUMENT, "%s: the cache is not 16-byte aligned", name);
  return LIMN_B200_OK;
}

int check_paged_device(const char* name, const limn_b200_paged* s) {
  int device = 0;
  cudaPointerAttributes of = {};
  LIMN_CUDA(cudaGetDevice(&device), "asking for the current device");
  LIMN_CUDA(cudaPointerGetAttributes(&of, s->k_cache), "asking where the cache is");  // (70 ns)
  if (of.type == cudaMemoryTypeUnregistered) return fail(LIMN_B200_BAD_ARGUMENT, "%s: the cache is not device memory", name);
  if (of.type == cudaMemoryTypeDevice && of.device != device)
    return fail(LIMN_B200_BAD_ARGUMENT, "%s: the cache is on device %d, the current one is %d", name, of.device, device);
  return LIMN_B200_OK;
}
}  // namespace limn_b200

using namespace limn_b200;

extern "C" {

int limn_b200_sdpa_paged_workspace(const limn_b200_paged* step, int prefix_len, unsigned long long* bytes) {
  clear_error();
  if (int rc = check_paged("sdpa_paged_workspace", step)) return rc;
  if (!bytes) return fail(LIMN_B200_BAD_ARGUMENT, "sdpa_paged_workspace: null result pointer");
  if (prefix_len < 0) return fail(LIMN_B200_BAD_ARGUMENT, "sdpa_paged_workspace: the prefix has %d keys", prefix_len);
  Workspace w;
  if (int rc = workspace_of(step, prefix_len, &w)) return rc;
  *bytes = w.bytes();
  return LIMN_B200_OK;
}

int limn_b200_sdpa_paged(const limn_b200_paged* step, const void* q, void* out, float* lse, const long long* strides, int causal, double scale, void* workspace,
                         unsigned long long workspace_bytes, void* stream) {
  return paged_pass("sdpa_paged", step, q, out, lse, strides, nullptr, 0, causal, scale, workspace, workspace_bytes, stream);
}

int limn_b200_sdpa_paged_prefix(const limn_b200_paged* step, const void* q, void* out, float* lse, const long long* strides, const int* prefix_table, int prefix_len,
                                int causal, double scale, void* workspace, unsigned long long workspace_bytes, void* stream) {
  clear_error();
  reset_launches();
  if (int rc = check_paged("sdpa_paged_prefix", step)) return rc;
  if (!prefix_table || prefix_len <= 0 || prefix_len > kMaxKeys)
    return fail(LIMN_B200_BAD_ARGUMENT, "sdpa_paged_prefix: a prefix of %d keys, or no table of its pages", prefix_len);
  if (step->heads > kPagedFinishHeads) return fail(LIMN_B200_UNSUPPORTED, "sdpa_paged_prefix: %d heads, at most %d are served behind a prefix", step->heads, kPagedFinishHeads);
  return paged_pass("sdpa_paged_prefix", step, q, out, lse, strides, prefix_table, prefix_len, causal, scale, workspace, workspace_bytes, stream);
}

}  // extern "C"
