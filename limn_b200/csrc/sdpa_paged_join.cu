// What workers of a paged pass left of problems that they shared, put together; and the rows of two passes, over a prefix and over a
// sequence's own keys. Sums of up to 148 parts, 512 bytes a row and part at most: bound by the latency of the loads, which are made four
// at a time. The order is fixed, so two runs give the same bits. What a join adds to a call, the launch and what the
// pass in front of it leaves in memory for it included: 2.4 us of a batch of few rows, 9 us of 148 x 256 rows of 128 columns (38 MB of parts).
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "paged_rows.cuh"

namespace limn_b200 {
namespace {

using namespace paged;

constexpr int kJoinWarps = 4;  // (small blocks find room beside a pass that is ending: 0.5 to 1 % of a call against 8)
constexpr int kUnroll = 4;
constexpr int kEach = 2;       // (one row 1 % slower, and four, which take 100 registers, 2 %)

// The parts of a problem that begins with worker `w`, `by` of them at a time beginning with part `from`: part 0 is the head's, part i the i-th follower's.
template <int D>
__device__ __forceinline__ void add_parts(Sums& sums, const Parts& parts, int w, int followers, int r, int column, int from, int by, float sl2) {
  auto part = [&](int i) { return (i == 0 ? 2LL * w + 1 : 2LL * (w + i)) * parts.rows + r; };
#pragma unroll 1
  for (int i0 = from; i0 <= followers; i0 += kUnroll * by) {
    float2 ml[kUnroll];
    float4 o[kUnroll];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const int i = i0 + u * by;
      ml[u] = make_float2(-INFINITY, 0.f), o[u] = make_float4(0.f, 0.f, 0.f, 0.f);
      if (i <= followers) ml[u] = parts.ml[part(i)], o[u] = *reinterpret_cast<const float4*>(parts.o + part(i) * D + column);
    }
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) sums.add(ml[u].x, ml[u].y, o[u], sl2);
  }
}

// The sides of a warp that has several parts at once, in lane order, into the first.
template <int D>
__device__ __forceinline__ void add_sides(Sums& sums, float sl2) {
  __syncwarp();
#pragma unroll
  for (int d = D / 4; d < 32; d <<= 1) {
    const float4 o = make_float4(__shfl_down_sync(0xffffffffu, sums.acc.x, d), __shfl_down_sync(0xffffffffu, sums.acc.y, d), __shfl_down_sync(0xffffffffu, sums.acc.z, d),
                                 __shfl_down_sync(0xffffffffu, sums.acc.w, d));
    const float m = __shfl_down_sync(0xffffffffu, sums.m, d), l = __shfl_down_sync(0xffffffffu, sums.l, d);
    sums.add(m, l, o, sl2);
  }
}

// A row of one problem: the warps of a block share its parts.
template <int D, bool kFp16>
__global__ void __launch_bounds__(kJoinWarps * 32) sdpa_paged_join_kernel(const Pass prm, const unsigned*) {
  constexpr int kLanes = D / 4;          // lanes to a row
  constexpr int kAtOnce = 32 / kLanes;   // parts a warp takes side by side
  __shared__ float4 all_sums[kJoinWarps][32];
  __shared__ float2 all_stats[kJoinWarps];
  ptx::grid_dependency_wait();
  ptx::grid_launch_dependents();
  const Head head = prm.parts.heads[blockIdx.x];
  if (head.followers <= 0) return;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int r = blockIdx.y, column = (lane % kLanes) * 4, side = lane / kLanes;
  const float sl2 = prm.scale * kLog2e;
  const int row = head.row0 + r;  // (few rows: one tile)
  if (r >= head.tile_rows || row >= head.n * prm.group) return;  // (the whole block)
  Sums sums;
  add_parts<D>(sums, prm.parts, blockIdx.x, head.followers, r, column, warp * kAtOnce + side, kJoinWarps * kAtOnce, sl2);
  add_sides<D>(sums, sl2);
  all_sums[warp][lane] = sums.acc;
  if (lane == 0) all_stats[warp] = make_float2(sums.m, sums.l);
  __syncthreads();
  if (warp > 0) return;
#pragma unroll 1
  for (int i = 1; i < kJoinWarps; ++i) sums.add(all_stats[i].x, all_stats[i].y, all_sums[i][lane], sl2);
  if (side == 0) store4<D, kFp16>(prm, row_place(prm, head.first, head.kv_head, row), column, sums.acc, sums.m, sums.l);
}

// Many rows of one problem, which few workers share: D / 4 lanes to a row, kEach rows one behind the other whose parts are asked for together. None where a
// kernel has given up: a worker of the pass may then not have left the parts that another has announced. (The pass of few rows waits for nothing.)
template <int D, bool kFp16>
__global__ void __launch_bounds__(kJoinWarps * 32) sdpa_paged_join_rows_kernel(const Pass prm, const unsigned* status) {
  constexpr int kLanes = D / 4, kAtOnce = 32 / kLanes, kParts = 2;
  ptx::grid_dependency_wait();
  ptx::grid_launch_dependents();
  const Head head = prm.parts.heads[blockIdx.x];
  if (head.followers <= 0 || *reinterpret_cast<const volatile unsigned*>(status) != ptx::kStatusOk) return;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int column = (lane % kLanes) * 4, r0 = (blockIdx.y * kJoinWarps + warp) * kEach * kAtOnce + lane / kLanes;
  const float sl2 = prm.scale * kLog2e;
  auto row_at = [&](int r) { return head.row0 + r / 128 * head.tile_rows + r % 128; };
  Sums sums[kEach];
  bool there[kEach];
#pragma unroll
  for (int u = 0; u < kEach; ++u) {
    const int r = r0 + u * kAtOnce;
    there[u] = r % 128 < head.tile_rows && row_at(r) < head.n * prm.group;
  }
#pragma unroll 1
  for (int i0 = 0; i0 <= head.followers; i0 += kParts) {
    float2 ml[kEach][kParts];
    float4 o[kEach][kParts];
#pragma unroll
    for (int u = 0; u < kEach; ++u)
#pragma unroll
      for (int v = 0; v < kParts; ++v) {
        const int i = i0 + v;
        const long long part = (i == 0 ? 2LL * blockIdx.x + 1 : 2LL * (blockIdx.x + i)) * prm.parts.rows + r0 + u * kAtOnce;
        ml[u][v] = make_float2(-INFINITY, 0.f), o[u][v] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (there[u] && i <= head.followers) ml[u][v] = prm.parts.ml[part], o[u][v] = *reinterpret_cast<const float4*>(prm.parts.o + part * D + column);
      }
#pragma unroll
    for (int u = 0; u < kEach; ++u)
#pragma unroll
      for (int v = 0; v < kParts; ++v) sums[u].add(ml[u][v].x, ml[u][v].y, o[u][v], sl2);
  }
#pragma unroll
  for (int u = 0; u < kEach; ++u)
    if (there[u]) store4<D, kFp16>(prm, row_place(prm, head.first, head.kv_head, row_at(r0 + u * kAtOnce)), column, sums[u].acc, sums[u].m, sums[u].l);
}

// A (token, head) row to kSplit warps: what both passes left of it, of a sequence that is one. Rows of tokens that belong to none are left alone; all of
// them where a kernel has given up, since a pass may then not have left what is read here.
template <int D, bool kFp16, int kSplit>
__global__ void __launch_bounds__(kJoinWarps * 32) sdpa_paged_finish_kernel(const Pass front, const Pass own, const unsigned* status) {
  constexpr int kRows = kJoinWarps / kSplit, kLanes = D / 4, kAtOnce = 32 / kLanes;
  __shared__ float4 all_sums[kJoinWarps][32];
  __shared__ float2 all_stats[kJoinWarps];
  ptx::grid_dependency_wait();
  ptx::grid_launch_dependents();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, split = warp % kSplit;
  const int token = blockIdx.x, head = min(static_cast<int>(blockIdx.y) * kRows + warp / kSplit, own.heads - 1);  // (the last block's spare warps repeat a row)
  const int column = (lane % kLanes) * 4, side = lane / kLanes;
  const float sl2 = own.scale * kLog2e;
  const long long row = static_cast<long long>(token) * own.heads + head;
  // (all asked for before whose token it is is known: the memory is there for every row)
  const bool served = own.parts.heads[0].followers != kServesNone;
  const float2 front_ml = front.leave.ml[row], own_ml = own.leave.ml[row];
  const float4 front_o = *reinterpret_cast<const float4*>(front.leave.o + row * D + column), own_o = *reinterpret_cast<const float4*>(own.leave.o + row * D + column);
  if (__syncthreads_or(threadIdx.x == 0 && *reinterpret_cast<const volatile unsigned*>(status) != ptx::kStatusOk)) return;
  const int b = sequence_of(own.q_start, own.batch, token, lane);
  if (!served || b >= own.batch) return;  // (as is all of the block)
  const Extent e = extent_of(own, b);
  if (token < e.first || token - e.first >= e.n) return;
  Sums sums;
  auto add = [&](const Pass& pass, const float2& ml, const float4& o) {
    if (ml.y == kInParts) {
      // (a pass that stood down, or gave up, may have left anything: no number from memory is followed out of the workspace)
      const int w = __float_as_int(ml.x), r = pass.leave.part_row[row];
      if (w < 0 || w >= pass.parts.workers || r < 0 || r >= pass.parts.rows) return;
      add_parts<D>(sums, pass.parts, w, min(pass.parts.heads[w].followers, pass.parts.workers - 1 - w), r, column, split * kAtOnce + side, kSplit * kAtOnce, sl2);
    } else if (side == 0 && split == 0) {
      sums.add(ml.x, ml.y, o, sl2);
    }
  };
  add(front, front_ml, front_o);
  add(own, own_ml, own_o);
  add_sides<D>(sums, sl2);
  if (kSplit > 1) {
    all_sums[warp][lane] = sums.acc;
    if (lane == 0) all_stats[warp] = make_float2(sums.m, sums.l);
    __syncthreads();
    if (split > 0) return;
#pragma unroll
    for (int i = 1; i < kSplit; ++i) sums.add(all_stats[warp + i].x, all_stats[warp + i].y, all_sums[warp + i][lane], sl2);
  }
  if (side == 0) store4<D, kFp16>(own, RowPlace{row, own.out + token * own.o_token + head * own.o_head}, column, sums.acc, sums.m, sums.l);
}

template <int D, bool kFp16>
int launch_join(const Pass& pass, bool many_rows, cudaStream_t stream) {
  constexpr int kRows = kJoinWarps * kEach * (128 / D);  // rows to a block of the kernel for many
  const unsigned blocks = static_cast<unsigned>(many_rows ? pass.parts.rows / kRows : pass.parts.rows);
  unsigned* status = nullptr;
  if (int rc = status_word(&status)) return rc;
  auto kernel = many_rows ? sdpa_paged_join_rows_kernel<D, kFp16> : sdpa_paged_join_kernel<D, kFp16>;
  LIMN_CUDA(launch_overlapped(kernel, dim3(static_cast<unsigned>(pass.parts.workers), blocks), dim3(kJoinWarps * 32), 0, stream, pass, status), "launching the kernel that joins parts");
  note_launches(1);
  return LIMN_B200_OK;
}

template <int D, bool kFp16, int kSplit>
int launch_finish_s(const Pass& front, const Pass& own, cudaStream_t stream) {
  unsigned* status = nullptr;
  if (int rc = status_word(&status)) return rc;
  constexpr int kRows = kJoinWarps / kSplit;
  static_assert(kSplit > 1 || kRows * 65535 >= kPagedFinishHeads);
  const dim3 grid(static_cast<unsigned>(own.tokens), static_cast<unsigned>((own.heads + kRows - 1) / kRows));
  LIMN_CUDA(launch_overlapped(sdpa_paged_finish_kernel<D, kFp16, kSplit>, grid, dim3(kJoinWarps * 32), 0, stream, front, own, status), "launching the kernel that joins a prefix");
  note_launches(1);
  return LIMN_B200_OK;
}

// Few rows have many parts each, and wait for them; many rows have few. Behind 8192 keys, four warps to a row : one, in us: 512 rows 33.5 : 39.5 (behind 20000), 2048
// 52.5 : 53.5, 4096 77.7 : 72.3, 8192 125 : 112.
template <int D, bool kFp16>
int launch_finish(const Pass& front, const Pass& own, cudaStream_t stream) {
  if (static_cast<long long>(own.tokens) * own.heads <= 2048) return launch_finish_s<D, kFp16, 4>(front, own, stream);
  return launch_finish_s<D, kFp16, 1>(front, own, stream);
}

}  // namespace

int paged_join_launch(const Pass& pass, bool fp16, bool many_rows, cudaStream_t stream) {
  if (pass.parts.width == 64) return fp16 ? launch_join<64, true>(pass, many_rows, stream) : launch_join<64, false>(pass, many_rows, stream);
  return fp16 ? launch_join<128, true>(pass, many_rows, stream) : launch_join<128, false>(pass, many_rows, stream);
}

int paged_finish_launch(const Pass& front, const Pass& own, bool fp16, cudaStream_t stream) {
  if (own.parts.width == 64) return fp16 ? launch_finish<64, true>(front, own, stream) : launch_finish<64, false>(front, own, stream);
  return fp16 ? launch_finish<128, true>(front, own, stream) : launch_finish<128, false>(front, own, stream);
}

}  // namespace limn_b200
