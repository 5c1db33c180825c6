// Rows of a paged pass on their way out, four columns to a lane.
#pragma once

#include "paged.h"
#include "sm100_ptx.cuh"

namespace limn_b200 {
namespace paged {

template <int D, bool kFp16>
__device__ __forceinline__ void store4(const Pass& prm, const RowPlace& place, int column, const float4& acc, float m, float l) {
  const float inv = 1.f / l;  // (no key: 0 * inf = NaN)
  if (column < prm.pieces_v * 8)
    *reinterpret_cast<uint2*>(place.out + 2 * column) = kFp16 ? make_uint2(ptx::pack_f16(acc.x * inv, acc.y * inv), ptx::pack_f16(acc.z * inv, acc.w * inv))
                                                              : make_uint2(ptx::pack_bf16(acc.x * inv, acc.y * inv), ptx::pack_bf16(acc.z * inv, acc.w * inv));
  if (column == 0) prm.lse[place.row] = m * prm.scale + logf(l);
}

// To the result, or to where the pass leaves its rows' sums.
template <int D, bool kFp16>
__device__ __forceinline__ void finish4(const Pass& prm, const RowPlace& place, int column, const float4& acc, float m, float l) {
  if (prm.leave.o == nullptr) return store4<D, kFp16>(prm, place, column, acc, m, l);
  *reinterpret_cast<float4*>(prm.leave.o + place.row * D + column) = acc;
  if (column == 0) prm.leave.ml[place.row] = make_float2(m, l);
}

// The row's sums are parts of this worker's and of those behind it, there as row `part_row`.
__device__ __forceinline__ void leave_in_parts(const Pass& prm, long long row, int part_row) {
  prm.leave.ml[row] = make_float2(__int_as_float(static_cast<int>(blockIdx.x)), kInParts);
  prm.leave.part_row[row] = part_row;
}

// A row's sums as they come together: a side that has seen no key adds nothing, and what its sums hold is of no concern.
struct Sums {
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  float m = -INFINITY, l = 0.f;
  __device__ __forceinline__ void add(float m_b, float l_b, const float4& o_b, float sl2) {
    if (m_b == -INFINITY && l_b == 0.f) return;
    float keep, more;
    merge_stats(m, l, m_b, l_b, sl2, keep, more);
    acc = make_float4(acc.x * keep + o_b.x * more, acc.y * keep + o_b.y * more, acc.z * keep + o_b.z * more, acc.w * keep + o_b.w * more);
  }
};

}  // namespace paged
}  // namespace limn_b200
