// New keys and values into their pages, turned to their positions on the way, and the queries turned beside them.
//
// A token's row of H + Hk + Hk heads is read once and written once; that traffic is the floor. A CTA has one token: one warp finds
// the token's sequence (its offset among q_start, 32 probes at a time), its slot and its page; the first threads make the
// token's cosines and sines, which all of its heads share, and leave them in shared memory; then every thread keeps to one column unit
// and walks the heads. A unit is what turns together: 16 bytes of a row and the 16 bytes half the rotated width further on (halves),
// or 16 bytes that hold their own pairs (neighbours), 8 bytes where a half is no multiple of 16 bytes.
//
// The angle p * f is taken as a number of turns in float64 and only its fraction goes to float32: at position 10^6 a float32
// product would be off by 0.06 radians, this is off by 2 pi 2^-25. The turn is float32, rounded once to 16 bits.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "paged.h"
#include "sm100_ptx.cuh"

namespace limn_b200 {
namespace {

using namespace paged;

constexpr int kThreads = 256;
constexpr int kMaxPairs = 64;
constexpr double kTurn = 6.283185307179586476925286766559;

struct AppendParams {
  const unsigned char *q, *k, *v;
  unsigned char* q_out;
  long long q_token, q_head, o_token, o_head, k_token, k_head, v_token, v_head;  // bytes
  Pages k_pages, v_pages;
  const double* frequencies;
  const int *table, *q_start, *kv_lens;
  unsigned* errors;
  int batch, heads, kv_heads;  // heads: 0 without queries
  int width, width_v;          // columns
  int page_size, pages, max_pages, tokens, max_t_q, first_position;
  Div by_page;
  int rotated;                 // columns
};

template <int E>
struct Unit {  // E 16-bit elements
  uint32_t w[E / 2];
};
template <int E>
__device__ __forceinline__ Unit<E> load_unit(const unsigned char* at) {
  Unit<E> u;
  if constexpr (E == 8) {
    const uint4 x = *reinterpret_cast<const uint4*>(at);
    u.w[0] = x.x, u.w[1] = x.y, u.w[2] = x.z, u.w[3] = x.w;
  } else {
    const uint2 x = *reinterpret_cast<const uint2*>(at);
    u.w[0] = x.x, u.w[1] = x.y;
  }
  return u;
}
template <int E>
__device__ __forceinline__ void store_unit(unsigned char* at, const Unit<E>& u) {
  if constexpr (E == 8) *reinterpret_cast<uint4*>(at) = make_uint4(u.w[0], u.w[1], u.w[2], u.w[3]);
  else *reinterpret_cast<uint2*>(at) = make_uint2(u.w[0], u.w[1]);
}
template <bool kFp16>
__device__ __forceinline__ float2 widen(uint32_t w) {
  if (kFp16) return __half22float2(*reinterpret_cast<const __half2*>(&w));
  return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}
template <bool kFp16>
__device__ __forceinline__ uint32_t narrow(float lo, float hi) {
  return kFp16 ? ptx::pack_f16(lo, hi) : ptx::pack_bf16(lo, hi);
}

// Units of a row: the turning ones first, then the others.
template <bool kFp16, int E, bool kNeighbours>
__device__ __forceinline__ void turn_rows(const unsigned char* from, long long from_head, unsigned char* to, long long to_head, int rows, int width,
                                          int rotated, const float2* turns) {
  const int turning = kNeighbours ? rotated / E : rotated / 2 / E;
  const int units = turning + (width - rotated) / E;
  const int step = kThreads / units;  // (width <= 128 and E >= 4: at most 32 units)
  const int row0 = threadIdx.x / units, unit = threadIdx.x - row0 * units;
  if (row0 >= step) return;
  const int column = unit < turning ? unit * E : rotated + (unit - turning) * E;
  from += 2 * column, to += 2 * column;
  if (unit >= turning) {
#pragma unroll 2
    for (int r = row0; r < rows; r += step) store_unit<E>(to + r * to_head, load_unit<E>(from + r * from_head));
    return;
  }
  if constexpr (kNeighbours) {
    float2 t[E / 2];
#pragma unroll
    for (int i = 0; i < E / 2; ++i) t[i] = turns[unit * (E / 2) + i];
#pragma unroll 2
    for (int r = row0; r < rows; r += step) {
      Unit<E> u = load_unit<E>(from + r * from_head);
#pragma unroll
      for (int i = 0; i < E / 2; ++i) {
        const float2 x = widen<kFp16>(u.w[i]);
        u.w[i] = narrow<kFp16>(x.x * t[i].x - x.y * t[i].y, x.x * t[i].y + x.y * t[i].x);
      }
      store_unit<E>(to + r * to_head, u);
    }
  } else {
    float2 t[E];
#pragma unroll
    for (int i = 0; i < E; ++i) t[i] = turns[unit * E + i];
    const int half = rotated;  // bytes from a column to its partner: rotated / 2 elements
#pragma unroll 2
    for (int r = row0; r < rows; r += step) {
      Unit<E> a = load_unit<E>(from + r * from_head), b = load_unit<E>(from + r * from_head + half);
#pragma unroll
      for (int i = 0; i < E / 2; ++i) {
        const float2 x = widen<kFp16>(a.w[i]), y = widen<kFp16>(b.w[i]);
        a.w[i] = narrow<kFp16>(x.x * t[2 * i].x - y.x * t[2 * i].y, x.y * t[2 * i + 1].x - y.y * t[2 * i + 1].y);
        b.w[i] = narrow<kFp16>(x.x * t[2 * i].y + y.x * t[2 * i].x, x.y * t[2 * i + 1].y + y.y * t[2 * i + 1].x);
      }
      store_unit<E>(to + r * to_head, a);
      store_unit<E>(to + r * to_head + half, b);
    }
  }
}

template <bool kFp16, int E, bool kNeighbours>
__global__ void __launch_bounds__(kThreads) kv_append_kernel(const AppendParams prm) {
  __shared__ float2 turns[kMaxPairs];
  __shared__ int found_page, found_slot;
  const int token = blockIdx.x, lane = threadIdx.x & 31;
  ptx::grid_dependency_wait();
  ptx::grid_launch_dependents();
  if (threadIdx.x < 32) {
    const int low = sequence_of(prm.q_start, prm.batch, token, lane);
    int page = -1, slot = 0;
    if (low < prm.batch) {
      const Extent e = extent_of(prm.q_start, prm.kv_lens, low, prm.tokens, prm.max_t_q, prm.max_pages, prm.page_size, prm.errors);
      if (token >= e.first && token - e.first < e.n) {  // (not so where the offsets are out of order)
        slot = e.keys - e.n + (token - e.first);
        if (e.keys < e.n) {  // more tokens than keys: there is no slot for the first of them
          if (lane == 0 && prm.errors != nullptr) atomicOr(prm.errors, LIMN_B200_PAGED_BAD_SEQUENCE);
        } else {
          page = checked_page(prm.table[static_cast<long long>(low) * prm.max_pages + prm.by_page.of(slot)], prm.pages, prm.errors);
        }
      }
    }
    if (lane == 0) found_page = page, found_slot = slot;
  }
  __syncthreads();
  const int page = found_page, slot = found_slot;
  if (page < 0) return;
  if (threadIdx.x < prm.rotated / 2) {
    const double round = (static_cast<double>(prm.first_position) + slot) * (prm.frequencies[threadIdx.x] * (1.0 / kTurn));
    float s, c;
    sincospif(2.f * static_cast<float>(round - rint(round)), &s, &c);
    turns[threadIdx.x] = make_float2(c, s);
  }
  __syncthreads();
  const int in_page = prm.by_page.rest(slot);
  const long long at = token;
  turn_rows<kFp16, E, kNeighbours>(prm.k + at * prm.k_token, prm.k_head, prm.k_pages.base + page * prm.k_pages.page + in_page * prm.k_pages.slot, prm.k_pages.head,
                                   prm.kv_heads, prm.width, prm.rotated, turns);
  turn_rows<kFp16, 8, true>(prm.v + at * prm.v_token, prm.v_head, prm.v_pages.base + page * prm.v_pages.page + in_page * prm.v_pages.slot, prm.v_pages.head,
                            prm.kv_heads, prm.width_v, 0, turns);
  if (prm.heads > 0)
    turn_rows<kFp16, E, kNeighbours>(prm.q + at * prm.q_token, prm.q_head, prm.q_out + at * prm.o_token, prm.o_head, prm.heads, prm.width, prm.rotated, turns);
}

template <bool kFp16>
int launch_append(const AppendParams& prm, int pairing, cudaStream_t stream) {
  auto kernel = pairing == LIMN_B200_NEIGHBOURS ? kv_append_kernel<kFp16, 8, true> : (prm.rotated % 16 == 0 ? kv_append_kernel<kFp16, 8, false> : kv_append_kernel<kFp16, 4, false>);
  LIMN_CUDA(launch_overlapped(kernel, dim3(static_cast<unsigned>(prm.tokens)), dim3(kThreads), 0, stream, prm), "launching the append kernel");
  note_launches(1);
  return LIMN_B200_OK;
}

}  // namespace
}  // namespace limn_b200

using namespace limn_b200;

extern "C" int limn_b200_kv_append(const limn_b200_paged* step, const void* q, const void* k, const void* v, void* q_out, const long long* strides,
                                   const double* frequencies, int rotated, int pairing, void* stream) {
  clear_error();
  reset_launches();
  if (int rc = check_paged("kv_append", step)) return rc;
  if (int rc = check_paged_pointers("kv_append", step)) return rc;
  if (!k || !v || !strides || (q == nullptr) != (q_out == nullptr)) return fail(LIMN_B200_BAD_ARGUMENT, "kv_append: a required pointer is null");
  if (rotated < 0 || rotated > step->hd || rotated % 8 != 0) return fail(LIMN_B200_BAD_ARGUMENT, "kv_append: rotated columns must be a multiple of 8 from 0 to hd, got %d", rotated);
  if (rotated > 0 && !frequencies) return fail(LIMN_B200_BAD_ARGUMENT, "kv_append: rotated columns without frequencies");
  if (pairing != LIMN_B200_HALVES && pairing != LIMN_B200_NEIGHBOURS) return fail(LIMN_B200_BAD_ARGUMENT, "kv_append: unknown pairing code %d", pairing);
  if ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(q_out) | reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v)) & 15u)
    return fail(LIMN_B200_BAD_ARGUMENT, "kv_append: an operand is not 16-byte aligned");
  for (int i = q ? 0 : 4; i < 8; ++i)
    if (strides[i] < 0 || (strides[i] & 7)) return fail(LIMN_B200_BAD_ARGUMENT, "kv_append: strides must be non-negative multiples of 8 elements, got %lld", strides[i]);
  if (step->tokens == 0 || step->batch == 0) return LIMN_B200_OK;
  AppendParams prm = {};
  prm.k = static_cast<const unsigned char*>(k), prm.v = static_cast<const unsigned char*>(v);
  if (q) {
    prm.q = static_cast<const unsigned char*>(q), prm.q_out = static_cast<unsigned char*>(q_out);
    prm.q_token = 2 * strides[0], prm.q_head = 2 * strides[1], prm.o_token = 2 * strides[2], prm.o_head = 2 * strides[3];
    prm.heads = step->heads;
  }
  prm.k_token = 2 * strides[4], prm.k_head = 2 * strides[5], prm.v_token = 2 * strides[6], prm.v_head = 2 * strides[7];
  prm.k_pages = {static_cast<unsigned char*>(step->k_cache), 2 * step->k_strides[0], 2 * step->k_strides[1], 2 * step->k_strides[2]};
  prm.v_pages = {static_cast<unsigned char*>(step->v_cache), 2 * step->v_strides[0], 2 * step->v_strides[1], 2 * step->v_strides[2]};
  prm.frequencies = frequencies;
  prm.table = step->page_table, prm.q_start = step->q_start, prm.kv_lens = step->kv_lens, prm.errors = step->errors;
  prm.batch = step->batch, prm.kv_heads = step->kv_heads, prm.width = step->hd, prm.width_v = step->hd_v;
  prm.page_size = step->page_size, prm.pages = step->pages, prm.max_pages = step->max_pages;
  prm.tokens = step->tokens, prm.max_t_q = step->max_t_q, prm.first_position = step->first_position;
  prm.rotated = rotated, prm.by_page = Div(step->page_size);
  return step->dtype == LIMN_B200_F16 ? launch_append<true>(prm, pairing, static_cast<cudaStream_t>(stream)) : launch_append<false>(prm, pairing, static_cast<cudaStream_t>(stream));
}
