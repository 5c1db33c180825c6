// New keys and values into their pages, turned to their positions on the way, and the queries turned beside them.
//
// A token's H + Hk + Hk rows are read once and written once; that traffic is the floor. One to eight warps have a token, each on its own:
// it finds the token's sequence (its offset among q_start, 32 probes at a time), its slot and its page, makes the token's cosines and
// sines, two to a lane, which all of its heads share, and then every lane keeps to one column unit and walks the heads, four rows in
// flight. A unit is what turns together: 16 bytes of a row and the 16 bytes half the rotated width further on (halves),
// or 16 bytes that hold their own pairs (neighbours), 8 bytes where a half is no multiple of 16 bytes.
//
// The angle p * f is taken as a number of turns in float64 and only its fraction goes to float32: at position 10^6 a float32
// product would be off by 0.06 radians, this is off by 2 pi 2^-25. The turn is float32, rounded once to 16 bits.
//
// Measured: 24 600 tokens of 32 + 8 + 8 rows of 128 (605 MB) 95 us, 6.3 TB/s, 97 % of a plain copy's rate; without the host 600 tokens of 36 rows of 80 5.0 us and one token 4.1 us,
// of which some 3 us are the launch and the chain of dependent loads: offsets, length, table, rows.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "paged.h"
#include "sm100_ptx.cuh"

namespace limn_b200 {
namespace {

using namespace paged;

constexpr int kWarps = 8;
constexpr int kThreads = kWarps * 32;
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
  Div by_page, by_units, by_units_v;  // units of a row of q and k, of v
  int warps_log;                      // 2^this warps to a token
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

// A lane's unit of rows row0, row0 + step, ...: the turning units of a row come first, then the others.
template <bool kFp16, int E, bool kNeighbours>
__device__ __forceinline__ void turn_rows(const unsigned char* from, long long from_head, unsigned char* to, long long to_head, int row0, int step, int rows, int unit, int turning,
                                          int rotated, const float2* turns) {
  constexpr int kAtOnce = 4;
  const int column = unit < turning ? unit * E : rotated + (unit - turning) * E;
  from += row0 * from_head + 2 * column, to += row0 * to_head + 2 * column;
  from_head *= step, to_head *= step;
  const int many = row0 < rows ? (rows - row0 + step - 1) / step : 0;
  const bool turns_here = unit < turning;
  const int half = kNeighbours || !turns_here ? 0 : rotated;  // bytes from a column to its partner: rotated / 2 elements
  float2 t[kNeighbours ? E / 2 : E];
#pragma unroll
  for (int i = 0; i < (kNeighbours ? E / 2 : E); ++i) t[i] = turns_here ? turns[unit * (kNeighbours ? E / 2 : E) + i] : make_float2(1.f, 0.f);
  for (int done = 0; done < many; done += kAtOnce) {
    Unit<E> a[kAtOnce], b[kAtOnce];
#pragma unroll
    for (int u = 0; u < kAtOnce; ++u) {
      if (done + u >= many) break;
      a[u] = load_unit<E>(from + u * from_head);
      if (!kNeighbours && turns_here) b[u] = load_unit<E>(from + u * from_head + half);
    }
#pragma unroll
    for (int u = 0; u < kAtOnce; ++u) {
      if (done + u >= many) break;
      if (turns_here) {
#pragma unroll
        for (int i = 0; i < E / 2; ++i) {
          const float2 x = widen<kFp16>(a[u].w[i]);
          if constexpr (kNeighbours) {
            a[u].w[i] = narrow<kFp16>(x.x * t[i].x - x.y * t[i].y, x.x * t[i].y + x.y * t[i].x);
          } else {
            const float2 y = widen<kFp16>(b[u].w[i]);
            a[u].w[i] = narrow<kFp16>(x.x * t[2 * i].x - y.x * t[2 * i].y, x.y * t[2 * i + 1].x - y.y * t[2 * i + 1].y);
            b[u].w[i] = narrow<kFp16>(x.x * t[2 * i].y + y.x * t[2 * i].x, x.y * t[2 * i + 1].y + y.y * t[2 * i + 1].x);
          }
        }
        if (!kNeighbours) store_unit<E>(to + u * to_head + half, b[u]);
      }
      store_unit<E>(to + u * to_head, a[u]);
    }
    from += kAtOnce * from_head, to += kAtOnce * to_head;
  }
}

template <bool kFp16, int E, bool kNeighbours>
__global__ void __launch_bounds__(kThreads) kv_append_kernel(const AppendParams prm) {
  __shared__ float2 turns_of[kWarps][kMaxPairs];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const long long id = static_cast<long long>(blockIdx.x) * kWarps + warp;
  const int token = static_cast<int>(id >> prm.warps_log), share = static_cast<int>(id & ((1 << prm.warps_log) - 1)), shares = 1 << prm.warps_log;
  ptx::grid_dependency_wait();
  ptx::grid_launch_dependents();
  if (token >= prm.tokens) return;
  double frequency[2];  // (asked for before what the sequence's place hangs on)
#pragma unroll
  for (int i = 0; i < 2; ++i) frequency[i] = i * 32 + lane < prm.rotated / 2 ? prm.frequencies[i * 32 + lane] * (1.0 / kTurn) : 0.0;
  const int b = sequence_of(prm.q_start, prm.batch, token, lane);
  if (b >= prm.batch) return;
  const Extent e = extent_of(prm.q_start, prm.kv_lens, b, prm.tokens, prm.max_t_q, prm.max_pages, prm.page_size, prm.errors);
  if (token < e.first || token - e.first >= e.n) return;  // (so where the offsets are out of order)
  if (e.keys < e.n) {  // more tokens than keys: there is no slot for the first of them
    if (lane == 0 && prm.errors != nullptr) atomicOr(prm.errors, LIMN_B200_PAGED_BAD_SEQUENCE);
    return;
  }
  const int slot = e.keys - e.n + (token - e.first), at_page = prm.by_page.of(slot);
  const int page = checked_page(prm.table[static_cast<long long>(b) * prm.max_pages + at_page], prm.pages, prm.errors);
  if (page < 0) return;
  float2* turns = turns_of[warp];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int pair = i * 32 + lane;
    if (pair >= prm.rotated / 2) break;
    const double round = (static_cast<double>(prm.first_position) + slot) * frequency[i];
    float s, c;
    sincospif(2.f * static_cast<float>(round - rint(round)), &s, &c);
    turns[pair] = make_float2(c, s);
  }
  __syncwarp();
  const long long in_page = slot - at_page * prm.page_size, at = token;
  {
    const int units = prm.by_units.d, rows_at_once = 32 / units, row0 = prm.by_units.of(lane), unit = lane - row0 * units;
    const int turning = kNeighbours ? prm.rotated / E : prm.rotated / 2 / E;
    if (row0 < rows_at_once) {
      const int first = share * rows_at_once + row0, step = shares * rows_at_once;
      if (prm.heads > 0)
        turn_rows<kFp16, E, kNeighbours>(prm.q + at * prm.q_token, prm.q_head, prm.q_out + at * prm.o_token, prm.o_head, first, step, prm.heads, unit, turning, prm.rotated, turns);
      turn_rows<kFp16, E, kNeighbours>(prm.k + at * prm.k_token, prm.k_head, prm.k_pages.base + page * prm.k_pages.page + in_page * prm.k_pages.slot, prm.k_pages.head, first, step,
                                       prm.kv_heads, unit, turning, prm.rotated, turns);
    }
  }
  {
    const int units = prm.by_units_v.d, rows_at_once = 32 / units, row0 = prm.by_units_v.of(lane), unit = lane - row0 * units;
    if (row0 < rows_at_once)
      turn_rows<kFp16, 8, true>(prm.v + at * prm.v_token, prm.v_head, prm.v_pages.base + page * prm.v_pages.page + in_page * prm.v_pages.slot, prm.v_pages.head,
                                share * rows_at_once + row0, shares * rows_at_once, prm.kv_heads, unit, 0, 0, turns);
  }
}

template <bool kFp16>
int launch_append(AppendParams& prm, int pairing, cudaStream_t stream) {
  const bool neighbours = pairing == LIMN_B200_NEIGHBOURS;
  const int unit = neighbours || prm.rotated % 16 == 0 ? 8 : 4;
  prm.by_units = Div(neighbours ? prm.width / 8 : (prm.width - prm.rotated / 2) / unit), prm.by_units_v = Div(prm.width_v / 8);
  auto kernel = neighbours ? kv_append_kernel<kFp16, 8, true> : (unit == 8 ? kv_append_kernel<kFp16, 8, false> : kv_append_kernel<kFp16, 4, false>);
  int sms = 0;
  if (int rc = sm_count(&sms)) return rc;
  // Eight warps to a token, fewer from where the grid has eight warps to a multiprocessor without. Few tokens wait for a token's rows one after the other, many gain
  // nothing from more warps that each look up the token's place. One : up to eight : eight for all, in us, 32 heads over 8 key heads of 128: 64 tokens 6.3 : 4.7 :
  // 4.7, 600 6.7 : 6.7 : 9.4, 5000 28.8 : 28.8 : 66; by up to 32 warps to a multiprocessor 1000 tokens took 9.9 where this takes 6.6.
  prm.warps_log = 3;
  while (prm.warps_log > 0 && (static_cast<long long>(prm.tokens) << prm.warps_log) > 8LL * sms) --prm.warps_log;
  const long long blocks = ((static_cast<long long>(prm.tokens) << prm.warps_log) + kWarps - 1) / kWarps;
  LIMN_CUDA(launch_overlapped(kernel, dim3(static_cast<unsigned>(blocks)), dim3(kThreads), 0, stream, prm), "launching the append kernel");
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
  if (reinterpret_cast<uintptr_t>(frequencies) & 7u) return fail(LIMN_B200_BAD_ARGUMENT, "kv_append: the frequencies are not 8-byte aligned");
  if (pairing != LIMN_B200_HALVES && pairing != LIMN_B200_NEIGHBOURS) return fail(LIMN_B200_BAD_ARGUMENT, "kv_append: unknown pairing code %d", pairing);
  if ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(q_out) | reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(v)) & 15u)
    return fail(LIMN_B200_BAD_ARGUMENT, "kv_append: an operand is not 16-byte aligned");
  for (int i = q ? 0 : 4; i < 8; ++i)
    if (strides[i] < 0 || (strides[i] & 7)) return fail(LIMN_B200_BAD_ARGUMENT, "kv_append: strides must be non-negative multiples of 8 elements, got %lld", strides[i]);
  if (step->tokens == 0 || step->batch == 0) return LIMN_B200_OK;
  if (int rc = check_paged_device("kv_append", step)) return rc;
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
