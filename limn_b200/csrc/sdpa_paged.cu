// Attention of a step's tokens over the pages of their sequences, and over a prefix that all of them share.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "paged.h"
#include "sm100_ptx.cuh"

namespace limn_b200 {
namespace {

using namespace paged;

// One warp to a (token, head) row: four columns to a lane, keys one after the other.
template <bool kFp16>
__global__ void __launch_bounds__(128) sdpa_paged_row_kernel(const Pass prm) {
  ptx::grid_dependency_wait();
  const int lane = threadIdx.x & 31;
  const long long row = blockIdx.x * 4LL + (threadIdx.x >> 5);
  if (row >= static_cast<long long>(prm.tokens) * prm.heads) return;
  const int token = static_cast<int>(row / prm.heads), head = static_cast<int>(row - static_cast<long long>(token) * prm.heads), kv_head = head / prm.group;
  const int b = prm.q_start == nullptr ? 0 : sequence_of(prm.q_start, prm.batch, token, lane);
  if (b >= prm.batch) return;
  const Extent e = extent_of(prm, b);
  if (token < e.first || token - e.first >= e.n) return;
  const int own = prm.causal ? max(0, e.keys - e.n + (token - e.first) + 1) : e.keys;
  auto load4 = [&](const unsigned char* at, int pieces, float (&x)[4]) {
    x[0] = x[1] = x[2] = x[3] = 0.f;
    if (lane >= 2 * pieces) return;
    const uint2 w = *reinterpret_cast<const uint2*>(at + 8 * lane);
    if (kFp16) {
      const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&w.x)), c = __half22float2(*reinterpret_cast<const __half2*>(&w.y));
      x[0] = a.x, x[1] = a.y, x[2] = c.x, x[3] = c.y;
    } else {
      x[0] = __uint_as_float(w.x << 16), x[1] = __uint_as_float(w.x & 0xffff0000u), x[2] = __uint_as_float(w.y << 16), x[3] = __uint_as_float(w.y & 0xffff0000u);
    }
  };
  float q[4], acc[4] = {0.f, 0.f, 0.f, 0.f}, m = -INFINITY, l = 0.f;
  load4(prm.q + token * prm.q_token + head * prm.q_head, prm.pieces, q);
  const int* table = prm.table + static_cast<long long>(b) * prm.max_pages;
  for (int j = 0; j < own; ++j) {
    const int page = checked_page(table[j / prm.page_size], prm.pages, prm.errors), slot = j % prm.page_size;
    float s = NAN, v[4] = {0.f, 0.f, 0.f, 0.f};
    if (page >= 0) {
      float k[4];
      load4(prm.k.base + page * prm.k.page + kv_head * prm.k.head + slot * prm.k.slot, prm.pieces, k);
      load4(prm.v.base + page * prm.v.page + kv_head * prm.v.head + slot * prm.v.slot, prm.pieces_v, v);
      s = q[0] * k[0] + q[1] * k[1] + q[2] * k[2] + q[3] * k[3];
#pragma unroll
      for (int step = 16; step > 0; step >>= 1) s += __shfl_xor_sync(0xffffffffu, s, step);
    }
    const float top = fmaxf(m, s), base = top == -INFINITY ? 0.f : top, alpha = expf((m - base) * prm.scale), p = expf((s - base) * prm.scale);
    m = top, l = l * alpha + p;
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[i] = acc[i] * alpha + p * v[i];
  }
  const int width = prm.pieces <= 8 && prm.pieces_v <= 8 ? 64 : 128;
  if (prm.leave.o != nullptr) {
    if (4 * lane < width) *reinterpret_cast<float4*>(prm.leave.o + row * width + 4 * lane) = make_float4(acc[0], acc[1], acc[2], acc[3]);
    if (lane == 0) prm.leave.ml[row] = make_float2(m, l);
    return;
  }
  if (prm.join.o != nullptr) {
    const float2 ml = prm.join.ml[row];
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    if (4 * lane < width) o = *reinterpret_cast<const float4*>(prm.join.o + row * width + 4 * lane);
    const float top = fmaxf(m, ml.x), base = top == -INFINITY ? 0.f : top, keep = expf((m - base) * prm.scale), add = expf((ml.x - base) * prm.scale);
    m = top, l = l * keep + ml.y * add;
    acc[0] = acc[0] * keep + o.x * add, acc[1] = acc[1] * keep + o.y * add, acc[2] = acc[2] * keep + o.z * add, acc[3] = acc[3] * keep + o.w * add;
  }
  if (lane < 2 * prm.pieces_v) {
    const float a = acc[0] / l, c = acc[1] / l, d = acc[2] / l, f = acc[3] / l;
    *reinterpret_cast<uint2*>(prm.out + token * prm.o_token + head * prm.o_head + 8 * lane) =
        kFp16 ? make_uint2(ptx::pack_f16(a, c), ptx::pack_f16(d, f)) : make_uint2(ptx::pack_bf16(a, c), ptx::pack_bf16(d, f));
  }
  if (lane == 0) prm.lse[row] = m * prm.scale + logf(l);
}

int launch_rows(const Pass& prm, bool fp16, cudaStream_t stream) {
  const long long blocks = (static_cast<long long>(prm.tokens) * prm.heads + 3) / 4;
  if (blocks > 0x7fffffffLL) return fail(LIMN_B200_UNSUPPORTED, "sdpa_paged: %d tokens of %d heads need more blocks than one grid holds", prm.tokens, prm.heads);
  auto kernel = fp16 ? sdpa_paged_row_kernel<true> : sdpa_paged_row_kernel<false>;
  LIMN_CUDA(launch_overlapped(kernel, dim3(static_cast<unsigned>(blocks)), dim3(128), 0, stream, prm), "launching the paged sdpa kernel");
  note_launches(1);
  return LIMN_B200_OK;
}

// Which kernel a pass of at most `rows` rows to a (sequence, key head) takes, and the workspace it has to itself.
size_t pass_workspace(long long rows, int width, int sms) { return rows <= kPagedFewRows ? paged_few_workspace(static_cast<int>(rows), width, sms) : 0; }
int launch_pass(const Pass& pass, bool fp16, long long rows, void* workspace, cudaStream_t stream) {
  return rows <= kPagedFewRows ? paged_few_launch(pass, fp16, static_cast<int>(rows), workspace, stream) : launch_rows(pass, fp16, stream);
}

// The workspace of a call: the parts of whichever pass has more, and behind them the rows' sums over the prefix.
struct Workspace {
  size_t parts, sums, stats;
  size_t bytes() const { return parts + sums + stats; }
};
int workspace_of(const limn_b200_paged* step, int prefix_len, Workspace* w) {
  int sms = 0;
  if (int rc = sm_count(&sms)) return rc;
  const int width = step->hd <= 64 && step->hd_v <= 64 ? 64 : 128;
  const long long group = step->heads / step->kv_heads;
  const size_t own = pass_workspace(step->max_t_q * group, width, sms), front = prefix_len > 0 ? pass_workspace(step->tokens * group, width, sms) : 0;
  w->parts = ((own > front ? own : front) + 255) / 256 * 256;
  const size_t rows = static_cast<size_t>(step->tokens) * step->heads;
  w->sums = prefix_len > 0 ? rows * width * 4 : 0, w->stats = prefix_len > 0 ? rows * 8 : 0;
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
  for (int i = 0; i < 4; ++i)
    if (strides[i] < 0 || (strides[i] & 7)) return fail(LIMN_B200_BAD_ARGUMENT, "%s: strides must be non-negative multiples of 8 elements, got %lld", name, strides[i]);
  if (!(scale > 0.0) || scale > 1e30) return fail(LIMN_B200_UNSUPPORTED, "%s: the scale must be positive and finite", name);
  if (step->tokens == 0 || step->batch == 0) return LIMN_B200_OK;
  Workspace w;
  if (int rc = workspace_of(step, prefix_len, &w)) return rc;
  if (w.bytes() > 0 && (!workspace || workspace_bytes < w.bytes()))
    return fail(LIMN_B200_BAD_ARGUMENT, "%s: the workspace has %llu bytes, %llu are needed", name, workspace_bytes, static_cast<unsigned long long>(w.bytes()));
  Pass prm;
  prm.q = static_cast<const unsigned char*>(q), prm.out = static_cast<unsigned char*>(out), prm.lse = lse;
  prm.q_token = 2 * strides[0], prm.q_head = 2 * strides[1], prm.o_token = 2 * strides[2], prm.o_head = 2 * strides[3];
  prm.k = {static_cast<unsigned char*>(step->k_cache), 2 * step->k_strides[0], 2 * step->k_strides[1], 2 * step->k_strides[2]};
  prm.v = {static_cast<unsigned char*>(step->v_cache), 2 * step->v_strides[0], 2 * step->v_strides[1], 2 * step->v_strides[2]};
  prm.table = step->page_table, prm.q_start = step->q_start, prm.kv_lens = step->kv_lens, prm.errors = step->errors;
  prm.batch = step->batch, prm.heads = step->heads, prm.kv_heads = step->kv_heads, prm.group = step->heads / step->kv_heads;
  prm.pieces = step->hd / 8, prm.pieces_v = step->hd_v / 8;
  prm.page_size = step->page_size, prm.pages = step->pages, prm.max_pages = step->max_pages, prm.tokens = step->tokens, prm.max_t_q = step->max_t_q;
  prm.causal = causal != 0, prm.scale = static_cast<float>(scale);
  const bool fp16 = step->dtype == LIMN_B200_F16;
  const cudaStream_t on = static_cast<cudaStream_t>(stream);
  if (prefix_len > 0) {
    // every row over the prefix, as one sequence of all tokens that sees all of it; tokens that belong to no sequence get sums
    // too, which nothing reads
    Pass front = prm;
    front.table = prefix_table, front.q_start = nullptr, front.kv_lens = nullptr, front.keys = prefix_len, front.batch = 1, front.causal = 0;
    front.leave.o = reinterpret_cast<float*>(static_cast<unsigned char*>(workspace) + w.parts);
    front.leave.ml = reinterpret_cast<float2*>(static_cast<unsigned char*>(workspace) + w.parts + w.sums);
    if (int rc = launch_pass(front, fp16, static_cast<long long>(step->tokens) * prm.group, workspace, on)) return rc;
    prm.join = front.leave;
  }
  return launch_pass(prm, fp16, static_cast<long long>(step->max_t_q) * prm.group, workspace, on);
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
  if (static_cast<long long>(s->max_pages) * s->page_size > 0x7fffffffLL - s->first_position)
    return fail(LIMN_B200_UNSUPPORTED, "%s: positions of %d pages of %d from %d on do not fit 31 bits", name, s->max_pages, s->page_size, s->first_position);
  for (int i = 0; i < 3; ++i)
    if (s->k_strides[i] < 0 || (s->k_strides[i] & 7) || s->v_strides[i] < 0 || (s->v_strides[i] & 7))
      return fail(LIMN_B200_BAD_ARGUMENT, "%s: cache strides must be non-negative multiples of 8 elements", name);
  return LIMN_B200_OK;
}

int check_paged_pointers(const char* name, const limn_b200_paged* s) {
  if (!s->k_cache || !s->v_cache || !s->page_table || !s->q_start || !s->kv_lens) return fail(LIMN_B200_BAD_ARGUMENT, "%s: a required pointer of the step is null", name);
  if ((reinterpret_cast<uintptr_t>(s->k_cache) | reinterpret_cast<uintptr_t>(s->v_cache)) & 15u) return fail(LIMN_B200_BAD_ARGUMENT, "%s: the cache is not 16-byte aligned", name);
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
  if (!prefix_table || prefix_len <= 0) return fail(LIMN_B200_BAD_ARGUMENT, "sdpa_paged_prefix: a prefix of %d keys, or no table of its pages", prefix_len);
  return paged_pass("sdpa_paged_prefix", step, q, out, lse, strides, prefix_table, prefix_len, causal, scale, workspace, workspace_bytes, stream);
}

}  // extern "C"
