// Attention over paged keys for any number of query rows to a key head, on the tensor cores: prompts and pieces of prompts behind what
// is cached, batches in which some sequences bring one token and others thousands, and all rows of a batch over the prefix they share.
//
// The rows of a sequence and key head are its (token, head of the group) pairs, token by token, so that grouped heads share a tile and
// with it the keys they read. A tile is as many whole tokens as 128 rows hold (one box of a tensor map: group heads x tokens), an item
// is two consecutive tiles and the key tiles of 128 they see, fetched page by page:
//   S_t = Q_t K_j^T          tcgen05.mma, both operands K-major in shared memory, S_t in tensor memory
//   P_t = exp2(S_t - m_t)    128 softmax threads per tile, one row each; P_t overwrites S_t as 16-bit
//   O_t += P_t V_j           tcgen05.mma, A = P_t from tensor memory, B = V_j (MN-major) from shared memory
// An item with one tile has it in both places, the even key tiles to the first and the odd ones to the second, and the epilogue puts the
// two together.
//
// Lengths are known on the device only, and they differ. So the work is cut there, into equal shares of (item, key) cost, one share to a
// CTA and one CTA to an SM: a share is the rest of an item, whole items, and the beginning of one. Whole items go to the result; what a
// CTA has of an item that others share goes into its parts (paged.h), which a kernel behind this one joins. The cost of an item is the number of keys its last
// token sees, half of it where one tile has both places, and a constant; its sum over a sequence has a closed form, and so has the share a CTA begins
// with: nothing is planned on the host or by a kernel in front.
//
// Past a sequence's end a tile holds what its last page has there, or what the stage held before: the scores are replaced, and the rows of V
// are zeroed before the product that reads them, since 0 * NaN would reach every row. (Boxes outside the cache, which TMA fills with zeros,
// would do too: pages that are none are fetched so.)
//
// P is rounded to the operands' type, which the product that reads it from tensor memory asks for: half a step of each weight; their sum l is taken before.
//
// Measured, calls with their join one after the other, 32 heads over 8 of 128, bf16: a prompt of 8192 tokens 524 us, 1050 TFLOP/s, 75 % of the measured sustained matrix rate
// (1612 MHz under the power cap; 450 us on a GPU that has rested): softmax and tensor pipe in turn (the tensor pipe is active 59 % of the time). Eight pieces of 1 to 1000 tokens
// behind up to 7000 keys 257 us, 818 TFLOP/s (1552 MHz; 220 rested): 12 us until the first scores of a launch, items that their rows fill in part, parts. 16 questions
// of 20 to 150 tokens, 32 heads over 4, behind 4113 keys 122 us, 778 TFLOP/s.
// What is compared further down was timed as calls in a graph, without the host, on a GPU that had rested (1965 MHz).
//
// Warp roles (12 warps): 0-3 softmax and epilogue of tile 0, 4-7 of tile 1, 8 TMA producer, 9 MMA issuer and tensor-memory owner; 10 and 11 have gone home.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "paged_rows.cuh"
#include "tensor_map.h"

namespace limn_b200 {
namespace {

using namespace ptx;
using namespace paged;

constexpr int kTile = kPagedTile;  // rows of a tile, keys of a key tile
static_assert(kTile == 128);
constexpr int kThreads = 384;
// A launch gets 168 registers a thread, here three groups of four warps; the softmax threads hold a row of 128 scores and take 40 more each from the third group, whose
// last two warps have nothing to do. Without that (10 warps, 148 bytes of them spilled) an 8192-token prompt takes 467 us, with it 448, with 184 for the softmax 465; at head
// dim 64 pieces of prompts 190, 175 and 184.
constexpr int kSoftmaxRegs = 208, kOtherRegs = 88;
static_assert(2 * 128 * kSoftmaxRegs + 128 * kOtherRegs <= kThreads * 168);
// What a step of an item with one tile costs, in keys. It computes as much as a step with two, a key tile of 128 each, but loads two key tiles to that one's one, which
// no copy further ahead hides: by 176 the eight pieces above took 219 us, by 128 (the arithmetic alone) 274, by 240 222 (with the registers below 3 us less). Pages of 8 make the producer issue twice
// the boxes, and that bounds it: 224 takes 222 us where 176 takes 243.
__device__ __forceinline__ int paged_single_step(int chunk_log) { return chunk_log == 3 ? 224 : 176; }
constexpr int kProducerWarp = 8;
constexpr int kMmaWarp = 9;
constexpr uint32_t kTmemCols = 512;
constexpr float kRescaleSlack = 8.f;
// A weight's exponent is s * scale - m * scale in log2 units, one multiply-add a score, and m * scale is rounded: by 2^-15 at 2^10, which is no more than the score's
// own float32 error there. Beyond, m is taken off the scores first (a weight against a maximum of 2^31 would not be a number otherwise). The
// vote for it is 1 % of the 8192-token prompt, taken for each tile or only where a maximum has moved.
constexpr float kFar = 1024.f;
constexpr int kItem = 256;     // what an item costs besides its keys, in keys: Q, the first scores, the way out
constexpr int kLeast = 256;    // cost of the smallest share: about that of the smallest item, and of no step more, so that a share inside an item has one at least

// kPacked: how a tile of K or V lies in shared memory at head dim 128. Column block after column block (64 columns of all 128 rows each), a box
// of TMA fetches 64 columns of a run of keys; packed, the two column blocks of 8 rows lie side by side, and a box fetches all columns of the
// run. A box costs the producer about 100 clocks to issue, whatever it holds, and a key tile of pages of 16 is 32 boxes or 16: the eight pieces above 235 us and 220, with pages
// of 8 286 and 219, with pages of 64 no difference.
template <int D, bool kPacked>
struct Layout {
  static constexpr int kTileBytes = kTile * D * 2;
  static constexpr int kAtomBytes = kTile * 128;                     // Q: from one column block to the next
  static constexpr int kKVAtom = kPacked ? 1024 : kAtomBytes;        // K and V: from one column block to the next
  static constexpr int kKVGroup = kPacked ? 1024 * (D / 64) : 1024;  // and from 8 rows to the next 8
  static_assert(!kPacked || D == 128);
  static constexpr int kStages = 2;
  static constexpr int kQOff = 0;
  static constexpr int kKOff = kQOff + 2 * kTileBytes;
  static constexpr int kVOff = kKOff + kStages * kTileBytes;
  static constexpr int kBarOff = kVOff + kStages * kTileBytes;
  static constexpr int kBytes = kBarOff + 512 + 1024;
  static constexpr int kSCol = 0;    // S_t at kSCol + 128 t (P_t overlays its first 64)
  static constexpr int kOCol = 256;  // O_t at kOCol + D t
};
struct Bars {
  static constexpr int kS = 2;                   // stages
  static constexpr int q_full = 0;               // + t
  static constexpr int k_full = 2;               // + stage
  static constexpr int k_empty = k_full + kS;
  static constexpr int v_full = k_empty + kS;
  static constexpr int v_empty = v_full + kS;
  static constexpr int s_full = v_empty + kS;    // + t
  static constexpr int p_full = s_full + 2;      // + t
  static constexpr int o_full = p_full + 2;      // + t
  static constexpr int p_half = o_full + 2;      // + t: the first 64 keys' worth of P_t is in place (and O_t rescaled)
  static constexpr int q_empty = p_half + 2;     // + t: the last S_t of the segment has been computed
  static constexpr int o_free = q_empty + 2;     // + t: the epilogue has read O_t
  static constexpr int work_full = o_free + 2;   // + slot
  static constexpr int work_empty = work_full + 2;
  static constexpr int merge_full = work_empty + 2;  // tile 1's part of every row is complete (both places one tile)
  static constexpr int count = merge_full + 1;
};

// What a CTA does of one item, as the producer hands it to the others.
struct Segment {
  int valid;
  int b, first, n, keys, kv_head;
  int row0;        // first row of tile 0
  int first_tile;  // first key tile
  int loads;       // key tiles it streams
  int count[2];    // of them, those that the tile in each place goes through
  int both;        // one tile in both places
  int begun;       // it begins with the item's first key tile
  int whole;       // and ends with its last
};

__device__ __forceinline__ int tiles_of(int keys) { return (keys + kTile - 1) >> 7; }

// ---- the cost of items, in keys (int holds an item's: 2^31 keys would be 2^35 bytes of a head). A sequence has `pairs` items per key head, pair j of tokens [j span, (j + 1) span) ----
struct Costs {
  int pairs, span, half, seen_first;  // span: tokens of a pair; half: of a tile; seen_first: keys that are there before the first token
  int keys, n, causal, single_step, least;  // least: keys that a token sees at the least, those in front; one, masked, where there are none
  Div by_span;
  __device__ __forceinline__ Costs(const Extent& e, const Div& by_span_, const Pass& p, int chunk_log)
      : pairs(by_span_.of(e.n + static_cast<int>(by_span_.d) - 1)), span(by_span_.d), half(by_span_.d / 2), seen_first(e.keys - e.n), keys(e.keys), n(e.n), causal(p.causal), single_step(paged_single_step(chunk_log)), least(max(1, p.front)), by_span(by_span_) {}
  // keys that the first `tokens` tokens see at most
  __device__ __forceinline__ int seen(int tokens) const { return max(least, causal ? seen_first + min(tokens, n) : keys); }
  __device__ __forceinline__ bool single(int j) const { return n - j * span <= half; }
  __device__ __forceinline__ int of(int j) const { return kItem + (single(j) ? static_cast<int>((static_cast<long long>(seen((j + 1) * span)) * single_step) >> 8) + 1 : seen((j + 1) * span)); }
  // sum over the pairs in front of j (all of them two whole tiles)
  __device__ __forceinline__ long long before(long long j) const {
    if (!causal) return j * (kItem + max(least, keys));
    const long long none = seen_first >= least ? 0 : min(j, static_cast<long long>(by_span.of(least - 1 - seen_first)));  // pairs whose last token sees the least
    return j * kItem + none * least + (j - none) * seen_first + span * (j * (j + 1) / 2 - none * (none + 1) / 2);
  }
  __device__ __forceinline__ long long all() const { return pairs == 0 ? 0 : before(pairs - 1) + of(pairs - 1); }
  // steps of key tiles (pairs of key tiles for a single tile) of pair j
  __device__ __forceinline__ int steps(int j) const {
    const int tiles = tiles_of(seen((j + 1) * span));
    return single(j) ? (tiles + 1) >> 1 : tiles;
  }
  __device__ __forceinline__ int step_cost(int j) const { return single(j) ? single_step : kTile; }
  // the step nearest to `cost` into pair j; what lies in front of the keys counts as the first one's beginning
  __device__ __forceinline__ int step_at(int j, long long cost) const {
    const int into = max(0, static_cast<int>(cost) - kItem + step_cost(j) / 2);
    return min(steps(j), single(j) ? into / single_step : into >> 7);
  }
};

struct Place {
  int b, kv_head, j, step;
  Extent e;
  long long into;  // cost from the item's beginning
};

struct Maps {
  CUtensorMap q, k, v;
  // packed maps have the key head in the dimension of column blocks (heads side by side: k_side) or in that of pages
  int k_side, v_side;
};

template <int D, bool kFp16, bool kPacked>
__global__ void __launch_bounds__(kThreads, 1) sdpa_paged_many_kernel(const __grid_constant__ Maps maps, const Pass prm, const Div by_span, const int chunk_log, unsigned* status) {
  using L = Layout<D, kPacked>;
  using B = Bars;
  extern __shared__ unsigned char smem_unaligned[];
  __shared__ uint32_t tmem_slot;
  __shared__ uint32_t abort_flag;
  __shared__ Segment ring[2];
  __shared__ float merge_m[kTile], merge_l[kTile];

  const uint32_t base = (smem_addr(smem_unaligned) + 1023u) & ~1023u;
  const uint32_t bars = base + L::kBarOff;
  auto bar = [&](int i) { return bars + 8u * i; };
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0);
  const int lane = threadIdx.x & 31;
  const int tile_tokens = by_span.d / 2, tile_rows = tile_tokens * prm.group;  // an item's two tiles have by_span.d tokens
  const int chunk = 1 << chunk_log;

  if (threadIdx.x == kProducerWarp * 32) {
    for (int i = 0; i < B::count; ++i) {
      unsigned arrivals = 1u;
      if ((i >= B::p_full && i < B::p_full + 2) || (i >= B::p_half && i < B::p_half + 2) || (i >= B::o_free && i < B::o_free + 2) || i == B::merge_full)
        arrivals = 128u;                                               // every thread of a softmax group
      if (i >= B::work_empty && i < B::work_empty + 2) arrivals = 9u;  // the MMA warp and the eight softmax warps
      mbar_init(bar(i), arrivals);
    }
    mbar_init_fence();
    tma_prefetch_descriptor(&maps.q);
    tma_prefetch_descriptor(&maps.k);
    tma_prefetch_descriptor(&maps.v);
  }
  // up to here nothing has touched global memory; and where all tokens are one sequence of a known length, the shares need none either
  const bool known = prm.q_start == nullptr;
  if (!known) grid_dependency_wait();
  // ---- where this CTA's share begins and ends: the producer's business ----
  long long total = 0, share = 0, from = 0, to = 0;
  Place p = {};  // in the warp's halves
  auto share_out = [&](long long all) {
    total = all * prm.kv_heads, share = max(static_cast<long long>(kLeast), prm.parts.share_of(total));
    from = blockIdx.x * share, to = from + share;
    return lane < 16 ? from : min(to, total - 1);
  };
  // `rest` into the sequence p.b, which costs `all` a key head
  auto place_in = [&](long long rest, long long all) {
    const Costs costs(p.e, by_span, prm, chunk_log);
    p.kv_head = small_quotient(rest, all);
    rest -= p.kv_head * all;
    int low = 0, high = costs.pairs - 1;  // the last pair that begins at or before `rest`
#pragma unroll 1
    while (low < high) {
      const int mid = (low + high + 1) / 2;
      if (costs.before(mid) <= rest) low = mid;
      else high = mid - 1;
    }
    p.j = low;
    p.into = rest - costs.before(low);
    p.step = costs.step_at(low, p.into);
    __syncwarp();
  };
  bool falls = false;  // q_start does, somewhere: nothing is served (the producer knows)
  if (prm.batch <= 32) {
    // a lane has a sequence, and the producer adds them up for itself: without barriers or reading an extent again (two prompts of 542 tokens at most 20.3 us, by the block 21.2)
    if (warp == kProducerWarp) {
      const Extent e = lane < prm.batch ? extent_of(prm, lane) : Extent{0, 0, 0};
      falls = __any_sync(0xffffffffu, e.first == kFalls);
      const long long all = Costs(e, by_span, prm, chunk_log).all();
      long long upto = all;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const long long other = __shfl_up_sync(0xffffffffu, upto, d);
        if (lane >= d) upto += other;
      }
      const long long x = share_out(falls ? 0 : __shfl_sync(0xffffffffu, upto, 31));
      if (from < total) {
        const int begins = __popc(__ballot_sync(0xffffffffu, upto * prm.kv_heads <= from)), ends = __popc(__ballot_sync(0xffffffffu, upto * prm.kv_heads <= min(to, total - 1)));
        p.b = lane < 16 ? begins : ends;
        p.e = Extent{__shfl_sync(0xffffffffu, e.first, p.b), __shfl_sync(0xffffffffu, e.n, p.b), __shfl_sync(0xffffffffu, e.keys, p.b)};
        const long long of_it = __shfl_sync(0xffffffffu, all, p.b);
        place_in(x - (__shfl_sync(0xffffffffu, upto, p.b) - of_it) * prm.kv_heads, of_it);
      }
    }
  } else {
    // every thread adds up its run of sequences, the block adds up the threads
    const int run = (prm.batch + kThreads - 1) / kThreads;
    long long mine = 0;
    bool mine_falls = false;
#pragma unroll 1
    for (int i = 0; i < run; ++i) {
      const int b = threadIdx.x * run + i;
      if (b >= prm.batch) break;
      const Extent e = extent_of(prm, b);
      mine += Costs(e, by_span, prm, chunk_log).all(), mine_falls |= e.first == kFalls;
    }
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const long long other = __shfl_up_sync(0xffffffffu, mine, d);
      if (lane >= d) mine += other;
    }
    __shared__ long long share_end[kThreads];
    __shared__ long long warp_sum[kThreads / 32];
    if (lane == 31) warp_sum[warp] = mine;
    falls = __syncthreads_or(mine_falls);
#pragma unroll 1
    for (int w = 0; w < warp; ++w) mine += warp_sum[w];
    share_end[threadIdx.x] = mine;
    __syncthreads();
    const long long x = share_out(falls ? 0 : share_end[kThreads - 1]);
    if (warp == kProducerWarp && from < total) {
      const int before = first_above(share_end, kThreads, prm.kv_heads, x);
      long long rest = x - (before == 0 ? 0 : share_end[before - 1] * prm.kv_heads), all;
      p.b = before * run - 1;
      do {
        ++p.b;
        p.e = extent_of(prm, p.b);
        all = Costs(p.e, by_span, prm, chunk_log).all();
        if (rest < all * prm.kv_heads) break;
        rest -= all * prm.kv_heads;
      } while (p.b + 1 < prm.batch);
      place_in(rest, all);
    }
  }
  if (known) grid_dependency_wait();
  grid_launch_dependents();
  if (threadIdx.x == 0) {
    abort_flag = *reinterpret_cast<volatile unsigned*>(status) != kStatusOk;  // an earlier kernel gave up: this one stands down
    prm.parts.heads[blockIdx.x].followers = 0;                                // (also then: nothing is joined)
  }
  if (warp == kMmaWarp) {
    tmem_alloc(smem_addr(&tmem_slot), kTmemCols);
    tmem_relinquish();
  }
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem = __shfl_sync(0xffffffffu, tmem_slot, 0);
  bool ok = !abort_flag;

  auto wait = [&](int i, uint32_t parity, unsigned tag) { return __all_sync(0xffffffffu, mbar_wait(bar(i), parity, status, tag)); };
  auto next_segment = [&](unsigned n_item, Segment& s) {
    const unsigned slot = n_item & 1u;
    if (!wait(B::work_full + slot, (n_item >> 1) & 1u, 0x0400u | slot)) return false;
    const volatile int* from = reinterpret_cast<const volatile int*>(&ring[slot]);
    int* to = reinterpret_cast<int*>(&s);
#pragma unroll
    for (int i = 0; i < static_cast<int>(sizeof(Segment) / sizeof(int)); ++i) to[i] = from[i];
    __syncwarp();
    if (lane == 0) mbar_arrive(bar(B::work_empty + slot));
    return true;
  };

  if (warp >= kProducerWarp) {
    registers_down<kOtherRegs>();
    if (warp == kProducerWarp) {
      // ================= the share, and TMA =================
      if (falls && lane == 0) prm.parts.heads[blockIdx.x].followers = kServesNone;
      const bool any = ok && from < total;
      auto of_half = [&](int from_lane) {
        auto word = [&](int x) { return __shfl_sync(0xffffffffu, x, from_lane); };
        return Place{word(p.b), word(p.kv_head), word(p.j), word(p.step), Extent{word(p.e.first), word(p.e.n), word(p.e.keys)}, __shfl_sync(0xffffffffu, p.into, from_lane)};
      };
      Place at = of_half(0), end = of_half(16);
      if (to >= total) end.b = prm.batch, end.kv_head = end.j = 0;  // nothing ends it
      unsigned n_item = 0, q_uses[2] = {0u, 0u}, step = 0;
      bool more = any;
      // a lane fetches one box of a key tile: `chunk` keys of one page, 64 columns
      const int chunks = kTile >> chunk_log;
      const int my_chunk = lane & (chunks - 1), my_atom = (lane << chunk_log) / kTile;
      constexpr int kBoxAtoms = kPacked ? 1 : D / 64;  // boxes to a chunk
      while (more && ok) {
        const Costs costs(at.e, by_span, prm, chunk_log);
        const bool last = at.b == end.b && at.kv_head == end.kv_head && at.j == end.j;
        const int steps = costs.steps(at.j), until = last ? end.step : steps;
        if (until > at.step) {
          Segment s;
          const bool single = costs.single(at.j);
          const int tiles = tiles_of(costs.seen((at.j + 1) * costs.span));  // key tiles of the item
          s.valid = 1, s.b = at.b, s.first = at.e.first, s.n = at.e.n, s.keys = at.e.keys, s.kv_head = at.kv_head;
          s.row0 = at.j * 2 * tile_rows;
          s.begun = at.step == 0, s.whole = at.step == 0 && until == steps;
          if (single) {
            s.first_tile = 2 * at.step;
            s.loads = min(2 * until, tiles) - s.first_tile;
            s.both = s.loads > 1;
            s.count[1] = s.loads / 2, s.count[0] = s.loads - s.count[1];
          } else {
            s.first_tile = at.step;
            const int tiles_0 = tiles_of(costs.seen(at.j * costs.span + costs.half));
            s.count[0] = max(0, min(until, tiles_0) - at.step);
            s.count[1] = until - at.step;
            s.loads = s.count[1], s.both = 0;
          }
          const unsigned slot = n_item & 1u;
          ok = wait(B::work_empty + slot, ((n_item >> 1) & 1u) ^ 1u, 0x0120u | slot);
          if (!ok) break;
          if (lane == 0) {
            ring[slot] = s;
            mbar_arrive(bar(B::work_full + slot));
          }
          __syncwarp();
          ++n_item;
#pragma unroll
          for (int t = 0; t < 2; ++t) {
            if (s.count[t] == 0) continue;
            ok = wait(B::q_empty + t, (q_uses[t] & 1u) ^ 1u, 0x0130u | t);
            if (!ok) break;
            ++q_uses[t];
            if (lane == 0) {
              mbar_expect_tx(bar(B::q_full + t), static_cast<uint32_t>(tile_rows) * D * 2);
              const int token = s.first + (2 * at.j + (s.both ? 0 : t)) * tile_tokens;
#pragma unroll
              for (int a = 0; a < D / 64; ++a) tma_load_5d(base + L::kQOff + t * L::kTileBytes + a * L::kAtomBytes, &maps.q, bar(B::q_full + t), a * 64, s.kv_head * prm.group, token, 0, 0);
            }
            __syncwarp();
          }
          if (!ok) break;
          // the page of this lane's box of key tile `tile`; one that is none is a coordinate outside the cache, whose box TMA fills with zeros
          auto entry = [&](int tile) {
            const int key = tile * kTile + my_chunk * chunk;
            return key < side_end(prm, key, s.keys) ? entry_for(prm, s.b, key) : 0;
          };
          int page_next[2] = {entry(s.first_tile), entry(s.first_tile + 1)};  // two tiles ahead
#pragma unroll 1
          for (int j = 0; j < s.loads && ok; ++j, ++step) {
            const int tile = s.first_tile + j, key = tile * kTile + my_chunk * chunk;
            const int end = side_end(prm, key, s.keys);  // (the same for the whole tile)
            const bool fetch = key < end && my_atom < kBoxAtoms;
            const int page = fetch ? checked_page(page_next[0], prm.pages, prm.errors) : 0;
            const int boxes = min(chunks, max(0, (end - tile * kTile + chunk - 1) >> chunk_log));  // those that have keys
            const uint32_t bytes = static_cast<uint32_t>(boxes * chunk) * (D * 2);
            page_next[0] = page_next[1], page_next[1] = entry(tile + 2);
            const int in_page = slot_of(prm, key);
            const int stage = step % B::kS;
            const uint32_t wrap = (step / B::kS) & 1;
            ok = wait(B::k_empty + stage, wrap ^ 1u, 0x0100u | stage);
            if (!ok) break;
            if (lane == 0) mbar_expect_tx(bar(B::k_full + stage), bytes);
            __syncwarp();
            const uint32_t box = stage * L::kTileBytes + my_atom * L::kAtomBytes + my_chunk * (chunk / 8) * L::kKVGroup;
            auto load = [&](uint32_t to, const CUtensorMap& map, int side, uint32_t full) {
              if constexpr (kPacked) tma_load_5d(to, &map, full, 0, 0, side ? s.kv_head * (D / 64) : 0, in_page >> 3, side ? page : page * prm.kv_heads + s.kv_head);
              else tma_load_5d(to, &map, full, my_atom * 64, in_page, s.kv_head, page, 0);
            };
            if (fetch) load(base + L::kKOff + box, maps.k, maps.k_side, bar(B::k_full + stage));
            __syncwarp();
            ok = wait(B::v_empty + stage, wrap ^ 1u, 0x0110u | stage);
            if (!ok) break;
            if (lane == 0) mbar_expect_tx(bar(B::v_full + stage), bytes);
            __syncwarp();
            if (fetch) load(base + L::kVOff + box, maps.v, maps.v_side, bar(B::v_full + stage));
            __syncwarp();
          }
          if (s.begun && !s.whole && lane == 0) {
            // workers behind this one whose share begins inside the item, before the middle of its last step
            const long long begins = to - end.into, limit = min(static_cast<long long>(costs.of(at.j)), kItem + steps * static_cast<long long>(costs.step_cost(at.j)) - costs.step_cost(at.j) / 2);
            prm.parts.heads[blockIdx.x] = Head{small_quotient(begins + limit - 1, share) - static_cast<int>(blockIdx.x), s.first, s.n, s.kv_head, s.row0, tile_rows};
          }
        }
        // the next item
        if (last) break;
        at.step = 0;
        if (++at.j < costs.pairs) continue;
        at.j = 0;
        if (++at.kv_head < prm.kv_heads) continue;
        at.kv_head = 0;
        do {
          if (++at.b >= prm.batch) {
            more = false;
            break;
          }
          at.e = extent_of(prm, at.b);
        } while (at.e.n == 0);
      }
      const unsigned slot = n_item & 1u;
      if (ok) ok = wait(B::work_empty + slot, ((n_item >> 1) & 1u) ^ 1u, 0x0121u | slot);
      if (ok && lane == 0) {
        ring[slot].valid = 0;
        mbar_arrive(bar(B::work_full + slot));
      }
    } else if (warp == kMmaWarp) {
      // ================= MMA issuer =================
      constexpr uint32_t idesc_s = mma_idesc(kTile, kTile, kFp16, false, false);
      constexpr uint32_t idesc_pv = mma_idesc(kTile, D, kFp16, false, true);
      auto issue_s = [&](int t, int stage) {
        const uint32_t q_lo = desc_lo(base + L::kQOff + t * L::kTileBytes, 0);
        const uint32_t k_lo = desc_lo(base + L::kKOff + stage * L::kTileBytes, 0);
        const uint32_t c = tmem + L::kSCol + t * 128;
        mma_ss_lo<false, desc_hi(L::kKVGroup)>(c, q_lo, k_lo, idesc_s);
#pragma unroll
        for (int kk = 1; kk < D / 16; ++kk) {  // (offsets in 16-byte units)
          mma_ss_lo<true, desc_hi(L::kKVGroup)>(c, q_lo + (kk / 4) * (L::kAtomBytes >> 4) + (kk % 4) * 2, k_lo + (kk / 4) * (L::kKVAtom >> 4) + (kk % 4) * 2, idesc_s);
        }
      };
      auto issue_pv = [&](int t, int stage, int part, bool first) {
        const uint32_t v_lo = desc_lo(base + L::kVOff + stage * L::kTileBytes, L::kKVAtom);
        const uint32_t c = tmem + L::kOCol + t * D;
        const uint32_t a = tmem + L::kSCol + t * 128;
#pragma unroll
        for (int kk = 4 * part; kk < 4 * part + 4; ++kk) mma_ts_lo<desc_hi(L::kKVGroup)>(c, a + kk * 8, v_lo + kk * (2 * L::kKVGroup >> 4), idesc_pv, (kk > 0 || !first) ? 1u : 0u);
      };
      // rows from `from` on of the V tile in `stage` become zeros: slots of a sequence's last page that it has not filled, and what was there before
      auto clear_rows = [&](int stage, int from) {
#pragma unroll 1
        for (int i = from * (D / 8) + lane; i < kTile * (D / 8); i += 32) {
          const int row = i / (D / 8), piece = i % (D / 8);
          st_shared_v4(base + L::kVOff + stage * L::kTileBytes + (row / 8) * L::kKVGroup + (piece / 8) * L::kKVAtom + (row % 8) * 128 + (piece % 8) * 16, 0u, 0u, 0u, 0u);
        }
        fence_async_shared();
        __syncwarp();
      };
      unsigned q_uses[2] = {0u, 0u};  // segments finished in which the tile in place t had key tiles
      unsigned tiles[2] = {0u, 0u};   // key tiles it has been through, over all segments
      unsigned step = 0;
      for (unsigned n_item = 0; ok; ++n_item) {
        Segment s;
        ok = next_segment(n_item, s);
        if (!ok || !s.valid) break;
        const bool both = s.both != 0;
        auto at = [&](int t, int j) { return step + (both ? 2 * j + t : j); };
        unsigned cleared = 0;  // + 1 of the load whose rows past the sequence's end have been cleared
#pragma unroll
        for (int t = 0; t < 2; ++t)
          if (s.count[t] > 0 && ok) ok = wait(B::q_full + t, q_uses[t] & 1u, 0x0200u | t);
        if (!ok) break;
#pragma unroll
        for (int t = 0; t < 2; ++t)
          if (s.count[t] > 0 && ok) {
            const unsigned first = at(t, 0);
            const int stage = first % B::kS;
            ok = wait(B::k_full + stage, (first / B::kS) & 1, 0x0210u);
            if (!ok) break;
            tc_fence_after_sync();
            // (the S_t region is free: MMAs run in issue order, and the last one issued for this tile consumed the P_t there)
            if (elect_one()) {
              issue_s(t, stage);
              mma_commit(bar(B::s_full + t));
              if (s.count[t] == 1) mma_commit(bar(B::q_empty + t));
              if (both) mma_commit(bar(B::k_empty + stage));
            }
            __syncwarp();
          }
        if (!ok) break;
        if (!both && elect_one()) mma_commit(bar(B::k_empty + step % B::kS));
        __syncwarp();
        const int rounds = max(s.count[0], s.count[1]);
#pragma unroll 1
        for (int j = 0; j < rounds && ok; ++j) {
          bool issued_next = false;
#pragma unroll
          for (int t = 0; t < 2; ++t) {
            if (!ok || j >= s.count[t]) continue;
            const unsigned here = at(t, j), then = at(t, j + 1);
            const int stage = here % B::kS, next = then % B::kS;
            ok = wait(B::v_full + stage, (here / B::kS) & 1, 0x0220u | stage);
            if (!ok) break;
            const int tile_at = (s.first_tile + static_cast<int>(here - step)) * kTile;
            const int left = side_end(prm, tile_at, s.keys) - tile_at;  // keys of the tile that there are
            if (left < kTile && cleared != here + 1) {
              clear_rows(stage, max(0, left));
              cleared = here + 1;
            }
            const uint32_t phase = tiles[t] & 1u;
            ok = wait(B::p_half + t, phase, 0x0260u | t);
            if (!ok) break;
            // the segment's first product overwrites O_t: the epilogue before must have read it
            if (j == 0) ok = wait(B::o_free + t, (q_uses[t] & 1u) ^ 1u, 0x0270u | t);
            if (!ok) break;
            tc_fence_after_sync();
            if (elect_one()) issue_pv(t, stage, 0, j == 0);
            __syncwarp();
            ok = wait(B::p_full + t, phase, 0x0230u | t);
            if (!ok) break;
            tc_fence_after_sync();
            const bool last = j + 1 >= s.count[t];
            if (elect_one()) {
              issue_pv(t, stage, 1, j == 0);
              if (last) mma_commit(bar(B::o_full + t));
              if (both) mma_commit(bar(B::v_empty + stage));
            }
            __syncwarp();
            ++tiles[t];
            if (!last) {
              // the scores can only follow the product that consumed the P_t lying over them
              ok = wait(B::k_full + next, (then / B::kS) & 1, 0x0240u | next);
              if (!ok) break;
              tc_fence_after_sync();
              if (elect_one()) {
                issue_s(t, next);
                mma_commit(bar(B::s_full + t));
                if (j + 2 == s.count[t]) mma_commit(bar(B::q_empty + t));
                if (both) mma_commit(bar(B::k_empty + next));
              }
              __syncwarp();
              issued_next = true;
            }
          }
          if (!ok) break;
          if (!both && elect_one()) {
            mma_commit(bar(B::v_empty + (step + j) % B::kS));
            if (issued_next) mma_commit(bar(B::k_empty + (step + j + 1) % B::kS));
          }
          __syncwarp();
        }
        step += s.loads;
#pragma unroll
        for (int t = 0; t < 2; ++t)
          if (s.count[t] > 0) ++q_uses[t];
      }
    }
  } else {
    registers_up<kSoftmaxRegs>();
    // ================= softmax + epilogue, one thread per row =================
    const int t = warp >> 2;
    const int row_in_tile = threadIdx.x & 127;
    const uint32_t lane_base = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const uint32_t t_s = tmem + lane_base + L::kSCol + t * 128;
    const uint32_t t_o = tmem + lane_base + L::kOCol + t * D;
    const float sl2 = prm.scale * kLog2e;
    const uint64_t sl2_2 = f2_pack(sl2, sl2);
    const int chunks = kTile >> chunk_log;
    unsigned tiles = 0;   // key tiles this group has been through, over all segments
    unsigned o_uses = 0;  // segments it has finished with key tiles
    unsigned merges = 0;
    for (unsigned n_item = 0; ok; ++n_item) {
      Segment s;
      ok = next_segment(n_item, s);
      if (!ok || !s.valid) break;
      const bool both = s.both != 0;
      const int n = t ? s.count[1] : s.count[0];
      const int top_row = s.row0 + (both ? 0 : t) * tile_rows;       // the tile's first row
      const int row = top_row + row_in_tile;
      const bool there = row_in_tile < tile_rows && row < s.n * prm.group;
      const long long part = (2LL * blockIdx.x + (s.begun ? 1 : 0)) * (2 * kTile) + t * kTile + row_in_tile;
      if (n == 0) {
        // nothing of this share for the tile's rows (its keys end before): a part without keys, if they have one
        if (!s.whole && there) prm.parts.ml[part] = make_float2(-INFINITY, 0.f);
        if (!s.whole && there && s.begun && prm.leave.o != nullptr) leave_in_parts(prm, row_place(prm, s.first, s.kv_head, row).row, t * kTile + row_in_tile);
        continue;
      }
      const int seen_first = s.keys - s.n;
      const int sees = prm.causal ? max(prm.front, min(s.keys, seen_first + prm.by_group.of(row) + 1)) : s.keys;            // keys [0, sees)
      const int sees_least = prm.causal ? max(prm.front, min(s.keys, seen_first + prm.by_group.of(top_row) + 1)) : s.keys;  // the tile's first token
      auto key0 = [&](int j) { return (s.first_tile + (both ? 2 * j + t : j)) * kTile; };
      // pages are looked at once more here, a key tile ahead
      auto entry = [&](int j) {
        const int key = key0(j) + lane * chunk;
        return lane < chunks && key < side_end(prm, key, s.keys) ? entry_for(prm, s.b, key) : 0;
      };
      int entry_next = entry(0);
      float m = -INFINITY, l = 0.f;
#pragma unroll 1
      for (int j = 0; j < n; ++j, ++tiles) {
        const unsigned none = __ballot_sync(0xffffffffu, entry_next < 0 || entry_next >= prm.pages);
        if (j + 1 < n) entry_next = entry(j + 1);
        ok = wait(B::s_full + t, tiles & 1u, 0x0300u | t);
        if (!ok) break;
        tc_fence_after_sync();
        uint32_t x[4][32];
#pragma unroll
        for (int c = 0; c < 4; ++c) tmem_ld32(t_s + 32 * c, x[c]);
        tmem_ld_wait();
        const int kv0 = key0(j);
        // a row that sees a key of a page that is none: l, and with it all of the row, is NaN from here on
        const bool in_front = kv0 < prm.front;
        const int limit = (in_front ? prm.prefix_len : sees) - kv0;
        if (none != 0u && (__ffs(none) - 1) * chunk < limit) l = NAN;
        if (kv0 + kTile > (in_front ? prm.prefix_len : sees_least)) {
#pragma unroll
          for (int c = 0; c < 4; ++c)
#pragma unroll
            for (int i = 0; i < 32; ++i)
              if (c * 32 + i >= limit) x[c][i] = 0xff800000u;  // -inf
        }
        float mx4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int c = 0; c < 4; ++c)
#pragma unroll
          for (int i = 0; i < 32; i += 2) mx4[(i >> 1) & 3] = max3(mx4[(i >> 1) & 3], __uint_as_float(x[c][i]), __uint_as_float(x[c][i + 1]));
        const float mx = fmaxf(fmaxf(mx4[0], mx4[1]), fmaxf(mx4[2], mx4[3]));
        const bool moves = (mx - m) * sl2 > kRescaleSlack;  // true at the first score above -inf, where m is -inf
        float alpha = 1.f;
        if (moves) {
          alpha = exp2_approx((m - mx) * sl2);
          m = mx;
        }
        float shift = m == -INFINITY ? 0.f : -m * sl2;
        const bool far = fabsf(shift) > kFar;
        if (__any_sync(0xffffffffu, far)) {
          const float against = far ? m : 0.f;
#pragma unroll
          for (int c = 0; c < 4; ++c)
#pragma unroll
            for (int i = 0; i < 32; ++i) x[c][i] = __float_as_uint(__uint_as_float(x[c][i]) - against);
          shift = far ? 0.f : shift;
        }
        const uint64_t shift2 = f2_pack(shift, shift);
        uint64_t sum2[2] = {0ull, 0ull};
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          if (h == 1) {
            // O_t was last written by the product of tile j - 1, which s_full also covers
            if (j > 0 && __any_sync(0xffffffffu, moves)) {
#pragma unroll 1
              for (int c = 0; c < D / 32; ++c) {
                uint32_t o[32];
                tmem_ld32(t_o + 32 * c, o);
                tmem_ld_wait();
#pragma unroll
                for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * alpha);
                tmem_st32(t_o + 32 * c, o);
              }
            }
          }
          uint32_t packed[32];
#pragma unroll
          for (int cc = 0; cc < 2; ++cc) {
            const int c = 2 * h + cc;
#pragma unroll
            for (int i = 0; i < 32; i += 2) {
              const uint64_t x2 = f2_fma(f2_pack_bits(x[c][i], x[c][i + 1]), sl2_2, shift2);
              float p0, p1;
              if (D == 64 && ((i >> 1) & 7) < 2) {  // (as in the dense forward: some of the exponentials on the FMA pipe; at head dim 128 an eighth of them costs 2.5 %)
                exp2_poly2<5>(x2, p0, p1);
              } else {
                f2_unpack(x2, p0, p1);
                p0 = exp2_approx(p0);
                p1 = exp2_approx(p1);
              }
              sum2[(i >> 1) & 1] = f2_add(sum2[(i >> 1) & 1], f2_pack(p0, p1));
              packed[cc * 16 + (i >> 1)] = kFp16 ? pack_f16(p0, p1) : pack_bf16(p0, p1);
            }
            if (h == 1 && cc == 0) {
              // the first half's store was issued a chunk of exponentials ago; hand it over
              tmem_st_wait();
              tc_fence_before_sync();
              mbar_arrive(bar(B::p_half + t));
            }
          }
          tmem_st32(t_s + 32 * h, packed);
        }
        float sum_a, sum_b, sum_c, sum_d;
        f2_unpack(sum2[0], sum_a, sum_b);
        f2_unpack(sum2[1], sum_c, sum_d);
        l = l * alpha + ((sum_a + sum_b) + (sum_c + sum_d));
        tmem_st_wait();
        tc_fence_before_sync();
        mbar_arrive(bar(B::p_full + t));
      }
      if (!ok) break;
      ok = wait(B::o_full + t, o_uses & 1u, 0x0310u | t);
      if (!ok) break;
      tc_fence_after_sync();
      ++o_uses;
      float keep = 1.f, from_1 = 0.f;  // what this place's sums and the other one's count (one tile in both)
      if (both) {
        if (t == 1) {
          merge_m[row_in_tile] = m, merge_l[row_in_tile] = l;
          tc_fence_before_sync();
          mbar_arrive(bar(B::merge_full));
          continue;
        }
        ok = wait(B::merge_full, merges & 1u, 0x0340u);
        if (!ok) break;
        ++merges;
        tc_fence_after_sync();
        const float m_1 = *const_cast<volatile float*>(&merge_m[row_in_tile]), l_1 = *const_cast<volatile float*>(&merge_l[row_in_tile]);
        merge_stats(m, l, m_1, l_1, sl2, keep, from_1);
      }
      // kTogether times 32 columns of the row. (All 64 of a head: 191 us where 32 at a time take 194; 64 of 128, with more code than 32: no gain)
      constexpr int kTogether = D == 64 ? 2 : 1;
      auto take = [&](int col, uint32_t (&o)[kTogether][32]) {
#pragma unroll
        for (int k = 0; k < kTogether; ++k) tmem_ld32(t_o + col + 32 * k, o[k]);
        if (both) {
          uint32_t o_1[kTogether][32];
#pragma unroll
          for (int k = 0; k < kTogether; ++k) tmem_ld32(t_o + D + col + 32 * k, o_1[k]);
          tmem_ld_wait();
#pragma unroll
          for (int k = 0; k < kTogether; ++k)
#pragma unroll
            for (int i = 0; i < 32; ++i) o[k][i] = __float_as_uint(__uint_as_float(o[k][i]) * keep + __uint_as_float(o_1[k][i]) * from_1);
        } else {
          tmem_ld_wait();
        }
      };
      const RowPlace place = row_place(prm, s.first, s.kv_head, there ? row : 0);
      if (s.whole && prm.leave.o == nullptr) {
        const float inv = 1.f / l;
        // Of wide heads, neighbouring rows' pieces are exchanged before they are stored, so that an instruction writes 64 bytes of each row it touches (the 8192-token prompt 451
        // us, without 470); at head dim 64 every thread writes its own row, which is one line (eight prompts of 37 to 774 tokens, 64 heads 72 us, with the exchange 75).
        constexpr bool kExchange = D == 128;
        unsigned char* to_row[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const unsigned long long mine_at = there ? reinterpret_cast<unsigned long long>(place.out) : 0ull;
          const unsigned long long at = kExchange ? __shfl_sync(0xffffffffu, mine_at, (lane & ~3) + i) : mine_at;
          to_row[i] = at == 0ull ? nullptr : reinterpret_cast<unsigned char*>(at) + 16 * (kExchange ? lane & 3 : i);
        }
#pragma unroll 1
        for (int c0 = 0; c0 < D / 32; c0 += kTogether) {
          uint32_t o[kTogether][32];
          take(32 * c0, o);
#pragma unroll
          for (int k = 0; k < kTogether; ++k) {
            const int c = c0 + k;
            uint32_t w[4][4];
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              const float a = __uint_as_float(o[k][2 * i]) * inv, b = __uint_as_float(o[k][2 * i + 1]) * inv;
              w[i / 4][i % 4] = kFp16 ? pack_f16(a, b) : pack_bf16(a, b);
            }
            if (kExchange) swap_rows_for_pieces<4>(w);
#pragma unroll
            for (int i = 0; i < 4; ++i)
              if (to_row[i] != nullptr && 4 * c + (kExchange ? lane & 3 : i) < prm.pieces_v) *reinterpret_cast<uint4*>(to_row[i] + 64 * c) = make_uint4(w[i][0], w[i][1], w[i][2], w[i][3]);
          }
        }
        if (there) prm.lse[place.row] = m * prm.scale + logf(l);
      } else {
        // to the parts, whose rows follow one another, neighbouring rows' pieces are exchanged first, so that an instruction writes 64
        // bytes of each row it touches; rows that there are not go along. To the rows' sums every thread writes its own row
        float* to = s.whole ? prm.leave.o + place.row * D : prm.parts.o + (part - lane + (lane & ~3)) * D + 4 * (lane & 3);
#pragma unroll 1
        for (int c0 = 0; c0 < D / 32; c0 += kTogether) {
          uint32_t o[kTogether][32];
          take(32 * c0, o);
          if (s.whole) {
            if (there) {
#pragma unroll
              for (int i = 0; i < 32 * kTogether; i += 4) *reinterpret_cast<uint4*>(to + 32 * c0 + i) = make_uint4(o[i / 32][i % 32], o[i / 32][i % 32 + 1], o[i / 32][i % 32 + 2], o[i / 32][i % 32 + 3]);
            }
          } else {
#pragma unroll
            for (int half = 0; half < 2 * kTogether; ++half) {
              uint32_t w[4][4];
#pragma unroll
              for (int i = 0; i < 16; ++i) w[i / 4][i % 4] = o[half / 2][16 * (half % 2) + i];
              swap_rows_for_pieces<4>(w);
#pragma unroll
              for (int i = 0; i < 4; ++i) *reinterpret_cast<uint4*>(to + i * D + 32 * c0 + 16 * half) = make_uint4(w[i][0], w[i][1], w[i][2], w[i][3]);
            }
          }
        }
        if (there) *(s.whole ? prm.leave.ml + place.row : prm.parts.ml + part) = make_float2(m, l);
        if (there && !s.whole && s.begun && prm.leave.o != nullptr) leave_in_parts(prm, place.row, t * kTile + row_in_tile);
      }
      // O_t is in registers or stored: the next segment's first product may overwrite it
      tc_fence_before_sync();
      mbar_arrive(bar(B::o_free + t));
      if (both) mbar_arrive(bar(B::o_free + 1));
    }
  }

  // ---- teardown ----
  tc_fence_before_sync();
  __syncthreads();
  if (warp == kMmaWarp) {
    if (abort_flag || *reinterpret_cast<volatile unsigned*>(status) != kStatusOk) {
      // a wait gave up somewhere: give copies and MMAs still in flight time to land before the memory they target is released
      for (int i = 0; i < 2000; ++i) __nanosleep(1000);
    }
    tc_fence_after_sync();
    tmem_free(tmem, kTmemCols);
  }
}

unsigned long long u(long long x) { return static_cast<unsigned long long>(x); }

// Boxes of `chunk` keys of one page and key head: 64 columns each.
BoxShape pages_map(const Pass& p, const Pages& side, int pieces, int chunk) {
  return BoxShape{{u(pieces) * 8, u(p.page_size), u(p.kv_heads), u(p.pages), 1}, {side.slot, side.head, side.page, side.page}, {64, static_cast<unsigned>(chunk), 1, 1, 1}};
}
// Or all 128 columns, the two column blocks of 8 keys side by side. Five dimensions hold (column, key of 8, column block, 8 keys, page) and leave
// none for the head, so it has to continue the column blocks (heads side by side in a token) or the pages (heads of a page one after the other).
bool packs(const Pass& p, const Pages& side, int pieces) {
  if (pieces != 16) return false;
  if (p.kv_heads == 1 || side.head == 256) return true;
  return side.page == p.kv_heads * side.head && static_cast<long long>(p.pages) * p.kv_heads <= 0x7fffffffLL;
}
BoxShape packed_map(const Pass& p, const Pages& side, int chunk, int* heads_side_by_side) {
  const bool beside = p.kv_heads == 1 || side.head == 256;
  *heads_side_by_side = beside;
  return BoxShape{{64, 8, beside ? 2 * u(p.kv_heads) : 2, u(p.page_size) / 8, beside ? u(p.pages) : u(p.pages) * u(p.kv_heads)},
                  {side.slot, 128, 8 * side.slot, beside ? side.page : side.head},
                  {64, 8, 2, static_cast<unsigned>(chunk) / 8, 1}};
}

template <int D, bool kFp16, bool kPacked>
int launch_many(const Pass& pass, unsigned* status, cudaStream_t stream) {
  using L = Layout<D, kPacked>;
  int chunk = pass.page_size;  // the largest run of keys that neither a page nor a key tile cuts: the common divisor of both, a power of two
  for (int rest = kTile % chunk; rest != 0;) {
    const int r = chunk % rest;
    chunk = rest, rest = r;
  }
  int chunk_log = 3;
  while (1 << chunk_log < chunk) ++chunk_log;
  const int tile_tokens = kTile / pass.group;
  Maps maps = {};
  const BoxShape q = {{u(pass.pieces) * 8, u(pass.heads), u(pass.tokens), 1, 1},
                      {pass.q_head, pass.q_token, pass.q_token, pass.q_token},
                      {64, static_cast<unsigned>(pass.group), static_cast<unsigned>(tile_tokens), 1, 1}};
  if (int rc = make_box_map("sdpa_paged", &maps.q, pass.q, kFp16, q)) return rc;
  if (int rc = make_box_map("sdpa_paged", &maps.k, pass.k.base, kFp16, kPacked ? packed_map(pass, pass.k, chunk, &maps.k_side) : pages_map(pass, pass.k, pass.pieces, chunk))) return rc;
  if (int rc = make_box_map("sdpa_paged", &maps.v, pass.v.base, kFp16, kPacked ? packed_map(pass, pass.v, chunk, &maps.v_side) : pages_map(pass, pass.v, pass.pieces_v, chunk))) return rc;
  auto kernel = sdpa_paged_many_kernel<D, kFp16, kPacked>;
  static bool sized[64] = {};
  int device = 0;
  LIMN_CUDA(cudaGetDevice(&device), "asking for the current device");
  if (device >= 0 && device < 64 && !sized[device]) {
    LIMN_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, L::kBytes), "sizing shared memory for the paged sdpa kernel");
    sized[device] = true;
  }
  LIMN_CUDA(launch_overlapped(kernel, dim3(static_cast<unsigned>(pass.parts.workers)), dim3(kThreads), L::kBytes, stream, maps, pass, Div(2 * tile_tokens), chunk_log, status),
            "launching the paged sdpa kernel");
  note_launches(1);
  return LIMN_B200_OK;
}

template <int D, bool kPacked>
int launch_many_d(const Pass& pass, bool fp16, unsigned* status, cudaStream_t stream) {
  return fp16 ? launch_many<D, true, kPacked>(pass, status, stream) : launch_many<D, false, kPacked>(pass, status, stream);
}

}  // namespace

size_t paged_many_workspace(int width, int sms) { return Parts::bytes(sms, 2 * kTile, width); }

int paged_many_launch(Pass& pass, bool fp16, unsigned char* workspace, cudaStream_t stream) {
  unsigned* status = nullptr;
  if (int rc = status_word(&status)) return rc;
  const int width = pass.pieces <= 8 && pass.pieces_v <= 8 ? 64 : 128;
  pass.parts.place(workspace, pass.blocks, 2 * kTile, width);
  if (width == 64) return launch_many_d<64, false>(pass, fp16, status, stream);
  if (packs(pass, pass.k, pass.pieces) && packs(pass, pass.v, pass.pieces_v)) return launch_many_d<128, true>(pass, fp16, status, stream);
  return launch_many_d<128, false>(pass, fp16, status, stream);
}

}  // namespace limn_b200
