// Attention over paged keys for few query rows to a key head (a new token, or a few, times the query heads that share the key head: up
// to 16): generation from a cache. K and V are read once, and that is the time it takes; the arithmetic has to stay out of the way.
//
// Work is cut into equal shares, whatever the sequences' lengths: the unit is 16 keys of one (sequence, key head), every warp of the
// grid takes the same number of consecutive units. A warp works alone: it copies its units' rows into its own ring in shared memory with
// 16-byte asynchronous copies, so that bytes are in flight all the time and nothing waits for other warps. What it has of a problem that
// its neighbours share it leaves in memory; at the end the block puts its warps' parts together, and a problem that reaches into other
// blocks is joined by a kernel behind this one (paged.h).
//
// Per unit, with mma.sync m16n8k16 and the keys as M so that 8 query rows are enough for a tile:
//   S^T (16 keys x rows) = K Q^T            A = K by ldmatrix, B = Q, in registers
//   P^T = exp2(S^T - m) as 16-bit           the accumulator's layout turned into B's by movmatrix
//   O^T (columns x rows) += V^T P^T         A = V by ldmatrix.trans
// Tensor-memory MMAs have nothing to add here: their 128 rows would hold 1 to 16, and the tensor pipe is idle most of the time.
// m moves only when a row's maximum has outgrown it by 8 in log2 units (weights then reach 2^8, which 16 bits hold), as in
// the tensor-core forward. The weights are rounded to the operands' type because the matrix instructions take both operands in one; it is half a step of each, while their sum
// l is taken before and is free of it.
//
// Measured, a call with its join among others: 64 sequences of 500 to 8191 keys, 32 heads over 8 of 128 (1.12 GB) 184 us, 6.1 TB/s, 93 % of a plain copy's rate (sustained, at the
// 1762 MHz that the power cap leaves); two of 131 000 keys (0.95 GB) 153 us, 6.2 TB/s; 24 of 3000 keys and 1 to 5 tokens, 12 heads of 80 (139 MB) 37 us, 3.8 TB/s: the copies'
// 16-byte pieces fill 10 lanes of 16 and the beginning weighs; one of 2000 keys, 8 heads of 64 (4 MB) 8.7 us on the device, nearly all of it beginnings: code fetched
// for the first time, some 50 clocks a line, and four loads that hang on one another before the first key arrives.
// What is compared further down was timed as calls in a graph, without the host, on a GPU that had rested (1965 MHz).
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>

#include "paged_rows.cuh"
#include "sm100_ptx.cuh"

namespace limn_b200 {
namespace {

using namespace paged;

// Warps of a block, which have its registers and its shared memory to themselves: 8, or 12 for narrow rows. A unit of those is fewer bytes and no less work, which more warps hide;
// but they make smaller shares, more of them to a problem, and of rows that lie token by token they read less in order. 8 : 12, in us, keys of 64 columns: two sequences of
// 131 000 keys, head by head, 91 : 81; 24 of 30 000 200 : 177; 64 of up to 8191, token by token, 110 : 114, of 32 columns 111 : 90; eight of 2000 12.0 : 12.8; one 8.9 : 10.
constexpr int kMostWarps = 12;
int most_warps(int width, int rows) { return width == 64 && rows <= 8 ? kMostWarps : 8; }
int warps_for(const Pass& p, int width, int rows) {
  const double keys = static_cast<double>(std::min(p.batch, p.tokens)) * p.kv_heads * (p.kv_lens != nullptr ? static_cast<double>(p.max_pages) * p.page_size + p.front : p.keys);
  const bool in_order = p.k.slot == 16 * p.pieces && p.v.slot == 16 * p.pieces_v;
  return keys >= 1 << 18 && (in_order || p.pieces + p.pieces_v <= 8) ? most_warps(width, rows) : 8;
}
constexpr int kUnit = kPagedUnit;  // keys
static_assert(kUnit == 16);
constexpr int kBegin = 4;  // units that a problem costs besides its keys: its queries, its page table, its way out
constexpr float kSlack = 8.f;

__device__ __forceinline__ void ldmatrix4(uint32_t (&r)[4], uint32_t at) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
}
__device__ __forceinline__ void ldmatrix4_trans(uint32_t (&r)[4], uint32_t at) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
}
__device__ __forceinline__ uint32_t transposed(uint32_t x) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
  return r;
}
template <bool kFp16>
__device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if (kFp16)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// 16 bytes global -> shared; `there` false: zeros, and `from` is not read
__device__ __forceinline__ void copy16(uint32_t to, const unsigned char* from, bool there) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(there ? 16 : 0) : "memory");
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copies_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

// D: columns the kernel computes with, of which a row has `pieces` groups of 8; the others are zeros in shared memory from the start (computing with 96
// columns instead, for rows that have no more: 8 % slower at 80, the lanes' copies and rows of memory no longer matching). The 16-byte
// pieces of a row are exchanged so that the eight rows of a matrix that ldmatrix reads fall on distinct banks and a copied row fills whole lines (rows
// 16 bytes further apart than they are long instead: 10 % slower).
template <int D, int W>
struct Ring {
  static constexpr int kSide = kUnit * D * 2;  // K or V of a unit
  static constexpr int kStages = D == 128 ? 3 : 48 / W;
  static constexpr int kWarpBytes = kStages * 2 * kSide;
  static constexpr int kBytes = W * kWarpBytes;  // 192 KB
  __device__ static __forceinline__ uint32_t place(int row, int piece) { return row * (D * 2) + ((piece ^ (row & 7)) << 4); }
};

// Where a warp is in the work: unit `unit` of `units` of problem (b, kv_head), `cost` into its share. What a problem costs besides its keys
// lies in front of its first unit, which belongs to whoever has that place.
struct Cursor {
  int b, kv_head, unit, units, cost;
  Extent e;
};
__device__ __forceinline__ int units_of(const Extent& e) { return e.n == 0 ? 0 : max(1, (e.keys + kUnit - 1) / kUnit); }
__device__ __forceinline__ int cost_of(const Extent& e) { return e.n == 0 ? 0 : kBegin + units_of(e); }
__device__ __forceinline__ void next_problem(const Pass& prm, Cursor& c) {
  c.unit = 0, c.cost += kBegin;
  if (++c.kv_head < prm.kv_heads) return;
  c.kv_head = 0, c.units = 0;
  while (c.units == 0 && ++c.b < prm.batch) c.e = extent_of(prm, c.b), c.units = units_of(c.e);
}

// What a warp has of problems that its neighbours share, for the block to put together.
struct Shared {
  int enters, through;      // part 2 w is there; and its problem goes on behind this warp
  int begins;               // part 2 w + 1 is there: a problem begins here and goes on
  int first[2], n[2], kv_head[2];  // of either
  long long end;            // the unit behind the beginning problem's last
};

template <int D, bool kFp16, int NT, int kWarps>
__global__ void __launch_bounds__(kWarps * 32, 1) sdpa_paged_few_kernel(const Pass prm, const Parts by_warp) {
  using R = Ring<D, kWarps>;
  constexpr int kThreads = kWarps * 32;
  extern __shared__ __align__(128) unsigned char ring[];
  __shared__ Shared shared[kWarps];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const float sl2 = prm.scale * kLog2e;
  const bool known = prm.q_start == nullptr;  // one sequence of a known length: the shares need no memory
  if (!known) ptx::grid_dependency_wait();

  // ---- the shares ----
  const int worker = blockIdx.x * kWarps + warp;
  if (lane == 0) shared[warp].enters = shared[warp].begins = 0;
  Cursor at = {};
  long long share, from, to;
  int span;
  auto share_out = [&](long long total) {
    share = by_warp.share_of(total);
    from = min(total, worker * share), to = min(total, from + share);
    span = static_cast<int>(to - from);
  };
  auto begin_at = [&](long long rest, int cost) {
    at.kv_head = small_quotient(rest, cost);
    const int into = static_cast<int>(rest - static_cast<long long>(at.kv_head) * cost);
    at.unit = max(0, into - kBegin), at.cost = max(0, kBegin - into);
  };
  bool falls;  // q_start does, somewhere: nothing is served
  if (prm.batch <= 32) {
    // a lane has a sequence, and every warp adds them up for itself, without barriers or reading an extent again: eight sequences of 2000 keys 13.6 us, by the block 14.6. (Up to 128,
    // four to a lane: 0 to 0.4 us slower than this up to 32, and no faster than the block beyond)
    const Extent e = lane < prm.batch ? extent_of(prm, lane) : Extent{0, 0, 0};
    falls = __any_sync(0xffffffffu, e.first == kFalls);
    long long upto = cost_of(e);
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const long long other = __shfl_up_sync(0xffffffffu, upto, d);
      if (lane >= d) upto += other;
    }
    share_out(falls ? 0 : __shfl_sync(0xffffffffu, upto, 31) * prm.kv_heads);
    if (span > 0) {
      at.b = __popc(__ballot_sync(0xffffffffu, upto * prm.kv_heads <= from));  // (below 32: `from` is below the total)
      at.e = Extent{__shfl_sync(0xffffffffu, e.first, at.b), __shfl_sync(0xffffffffu, e.n, at.b), __shfl_sync(0xffffffffu, e.keys, at.b)};
      at.units = units_of(at.e);
      const int cost = cost_of(at.e);
      begin_at(from - (__shfl_sync(0xffffffffu, upto, at.b) - cost) * prm.kv_heads, cost);
    }
  } else {
    // every thread adds up its run of sequences, the block adds up the threads
    const int run = (prm.batch + kThreads - 1) / kThreads;
    long long mine = 0;
    bool mine_falls = false;
    for (int i = 0; i < run; ++i) {
      const int b = threadIdx.x * run + i;
      if (b >= prm.batch) break;
      const Extent e = extent_of(prm, b);
      mine += cost_of(e), mine_falls |= e.first == kFalls;
    }
    long long upto = mine;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const long long other = __shfl_up_sync(0xffffffffu, upto, d);
      if (lane >= d) upto += other;
    }
    __shared__ long long share_end[kThreads];  // cost of the sequences up to and with a thread's, per key head
    __shared__ long long warp_sum[kWarps];
    if (lane == 31) warp_sum[warp] = upto;
    falls = __syncthreads_or(mine_falls);
    for (int w = 0; w < warp; ++w) upto += warp_sum[w];
    share_end[threadIdx.x] = upto;
    __syncthreads();
    share_out(falls ? 0 : share_end[kThreads - 1] * prm.kv_heads);
    if (span > 0) {
      const int before = first_above(share_end, kThreads, prm.kv_heads, from);  // the run of sequences that `from` falls into
      long long rest = from - (before == 0 ? 0 : share_end[before - 1] * prm.kv_heads);
      at.b = before * run - 1;
      int cost;
      do {
        ++at.b;
        at.e = extent_of(prm, at.b);
        at.units = units_of(at.e), cost = cost_of(at.e);
        if (rest < static_cast<long long>(cost) * prm.kv_heads) break;
        rest -= static_cast<long long>(cost) * prm.kv_heads;
      } while (at.b + 1 < prm.batch);
      begin_at(rest, cost);
    }
  }

  if (known) ptx::grid_dependency_wait();
  ptx::grid_launch_dependents();
  if (threadIdx.x == 0) prm.parts.heads[blockIdx.x].followers = falls ? kServesNone : 0;

  // ---- copies: run ahead of the arithmetic with a cursor of their own ----
  Cursor ahead = at;
  int loaded = 0;
  const uint32_t mine = ptx::smem_addr(ring) + warp * R::kWarpBytes;
  // a lane's copies of the 8 rows of a half unit: where from (beyond the first row's first byte) and where to
  constexpr int kPieces = D / 8, kCopies = kPieces / 4;
  long long k_off[kCopies], v_off[kCopies];
  uint32_t to_off[kCopies];
  bool k_there[kCopies], v_there[kCopies];
  int row_of[kCopies];
#pragma unroll
  for (int j = 0; j < kCopies; ++j) {
    const int r = (j * 32 + lane) / kPieces, piece = (j * 32 + lane) % kPieces;
    row_of[j] = r, to_off[j] = R::place(r, piece);
    k_off[j] = r * prm.k.slot + piece * 16, v_off[j] = r * prm.v.slot + piece * 16;
    k_there[j] = piece < prm.pieces, v_there[j] = piece < prm.pieces_v;
  }
  if (prm.pieces < kPieces || prm.pieces_v < kPieces) {
    for (int i = lane; i < R::kStages * 2 * kUnit * kPieces; i += 32) {
      const int side_row = i / kPieces, piece = i % kPieces;
      if (piece >= ((side_row / kUnit) & 1 ? prm.pieces_v : prm.pieces)) ptx::st_shared_v4(mine + side_row / kUnit * R::kSide + R::place(side_row % kUnit, piece), 0u, 0u, 0u, 0u);
    }
  }
  // A lane keeps the page of one of 32 groups of 8 keys (no page ends inside one), 16 units, and the table's entry for the 16 units behind.
  int block = -1, page = -1, entry_next = -1;
  unsigned none = 0;  // two bits for each place of the ring: which 8 of its unit's keys have a page that is none
  auto entry_of = [&](const Cursor& c, int blk) {
    const int key = (blk * 32 + lane) * 8;
    return key < side_end(prm, key, c.e.keys) ? entry_for(prm, c.b, key) : 0;
  };
  auto issue = [&]() {
    if (ahead.cost < span) {
      const int blk = ahead.unit / 16;
      if (blk != block) {
        const int raw = block >= 0 && blk == block + 1 ? entry_next : entry_of(ahead, blk);
        block = blk;
        entry_next = entry_of(ahead, blk + 1);
        const int key = (blk * 32 + lane) * 8;
        page = key < side_end(prm, key, ahead.e.keys) ? checked_page(raw, prm.pages, prm.errors) : -1;
      }
      const int place_at = loaded % R::kStages;
      const uint32_t k_to = mine + place_at * 2 * R::kSide, v_to = k_to + R::kSide;
      none &= ~(3u << (2 * place_at));
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        const int key0 = ahead.unit * kUnit + half * 8;
        const int p = __shfl_sync(0xffffffffu, page, (key0 / 8) & 31);
        const int slot = slot_of(prm, key0), end = side_end(prm, key0, ahead.e.keys);
        const long long in_page = max(p, 0);
        if (p < 0 && key0 < end) none |= 1u << (2 * place_at + half);
        const unsigned char* k_from = prm.k.base + in_page * prm.k.page + ahead.kv_head * prm.k.head + slot * prm.k.slot;
        const unsigned char* v_from = prm.v.base + in_page * prm.v.page + ahead.kv_head * prm.v.head + slot * prm.v.slot;
        const int rows_there = p >= 0 ? end - key0 : 0;  // (the others are zeros, and what they would be is not read)
#pragma unroll
        for (int j = 0; j < kCopies; ++j) {
          const bool there = row_of[j] < rows_there;
          const uint32_t to = to_off[j] + half * 8 * (D * 2);  // (the second 8 rows lie as the first)
          if (k_there[j]) copy16(k_to + to, k_from + k_off[j], there);
          if (v_there[j]) copy16(v_to + to, v_from + v_off[j], there);
        }
      }
      ++loaded, ++ahead.cost;
      if (++ahead.unit == ahead.units && ahead.cost + kBegin < span) next_problem(prm, ahead), block = -1;
    }
    copies_commit();
  };
  // ---- arithmetic ----
  const int kq = lane >> 2, cq = lane & 3;  // in a fragment: row (key or column of O), and pair of query rows
  uint32_t q[NT][D / 16][2];
  float o[NT][D / 16][4];
  float m[NT][2], l[NT][2];
  int limit[NT][2], least_limit = 0;
  bool begun = at.unit == 0;
  auto begin = [&] {
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int r = nt * 8 + kq;
      const int i = prm.by_group.of(r), g = r - i * prm.group;
      const unsigned char* row = prm.q + (static_cast<long long>(at.e.first) + i) * prm.q_token + (at.kv_head * prm.group + g) * prm.q_head;
      const bool there = i < at.e.n;
#pragma unroll
      for (int kk = 0; kk < D / 16; ++kk)
#pragma unroll
        for (int j = 0; j < 2; ++j)
          q[nt][kk][j] = there && kk * 2 + j < prm.pieces ? *reinterpret_cast<const uint32_t*>(row + (kk * 16 + j * 8 + cq * 2) * 2) : 0u;
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const int token = prm.by_group.of(nt * 8 + cq * 2 + c);
        limit[nt][c] = prm.causal ? max(prm.front, min(at.e.keys, at.e.keys - at.e.n + token + 1)) : at.e.keys;
        m[nt][c] = -INFINITY, l[nt][c] = 0.f;
      }
#pragma unroll
      for (int mt = 0; mt < D / 16; ++mt)
#pragma unroll
        for (int c = 0; c < 4; ++c) o[nt][mt][c] = 0.f;
    }
    least_limit = prm.causal ? at.e.keys - at.e.n + 1 : at.e.keys;
  };
  bool fresh = true;  //  a problem, or the share, begins
  // (the first turns only issue copies; one loop for all, since code that a launch runs once is fetched once, at some 50 clocks a line)
  // Long shares of rows that lie one behind the other (pages head by head) come faster with one unit on the way than with two: two sequences of 131 000 keys 148 us : 154, 64 of up to
  // 8191 177 : 182. Token by token it is the other way round (150 : 145 and 180 : 177), so it is for short shares (64 of 500 keys, 25 units a warp, 26.8 : 26.1) and narrower
  // rows, whose copies are not all that a unit takes (96 columns 152 : 138).
  const bool one_ahead = D == 128 && span >= 64 && prm.k.slot == 2 * D && prm.v.slot == 2 * D && prm.pieces == D / 8 && prm.pieces_v == D / 8;
#pragma unroll 1
  for (int step = (one_ahead ? 2 : 1) - R::kStages; at.cost < span; ++step) {
    if (fresh) begin(), fresh = false;
    if (step >= 0) {
      if (one_ahead) copies_wait<R::kStages - 3>();
      else copies_wait<R::kStages - 2>();
      __syncwarp();
    }
    issue();
    if (step < 0) {
      if (ahead.cost >= span) {  // no more to copy: the places left stay empty (the turns that would say so one by one are 0.4 us of a call of few keys)
        for (; step < -1; ++step) copies_commit();
      }
      continue;
    }
    const int place_at = step % R::kStages;
    const uint32_t k_at = mine + place_at * 2 * R::kSide, v_at = k_at + R::kSide;
    float s[NT][4];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int c = 0; c < 4; ++c) s[nt][c] = 0.f;
#pragma unroll
    for (int kk = 0; kk < D / 16; ++kk) {
      // A: 16 keys x 16 columns; lanes 0-15 name the keys' first 8 columns' pieces, 16-31 the second's
      uint32_t a[4];
      const int r = lane & 15, pc = kk * 2 + (lane >> 4);
      ldmatrix4(a, k_at + R::place(r, pc));
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) mma<kFp16>(s[nt], a, q[nt][kk][0], q[nt][kk][1]);
    }
    const int key = at.unit * kUnit + kq;
    if (at.unit * kUnit + kUnit > least_limit) {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int c = 0; c < 4; ++c)
          if (key + (c >> 1) * 8 >= limit[nt][c & 1]) s[nt][c] = -INFINITY;
    }
    if (at.unit * kUnit < prm.front && at.unit * kUnit + kUnit > prm.prefix_len) {  // the last keys of the front do not exist
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int c = 0; c < 4; ++c)
          if (key + (c >> 1) * 8 >= prm.prefix_len) s[nt][c] = -INFINITY;
    }
    const unsigned none_here = (none >> (2 * place_at)) & 3u;
    if (none_here != 0u) {  // a row that sees a key of a page that is none: l is NaN from here on
      const int seen_from = at.unit * kUnit + (none_here & 1u ? 0 : 8);
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int c = 0; c < 2; ++c)
          if (seen_from < limit[nt][c]) l[nt][c] = NAN;
    }
    uint32_t p[NT][2];
    bool moved = false;
    float alpha[NT][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        float top = fmaxf(s[nt][c], s[nt][c + 2]);
#pragma unroll
        for (int d = 4; d < 32; d <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
        alpha[nt][c] = 1.f;
        if ((top - m[nt][c]) * sl2 > kSlack) {  // (true at the first score above -inf, where m is -inf)
          alpha[nt][c] = ptx::exp2_approx((m[nt][c] - top) * sl2);
          m[nt][c] = top, moved = true;
        }
        // (the difference first: a rounded m * sl2 would be in every weight, 2^-24 of it in log2 units, whatever the scores' size)
        const float against = m[nt][c] == -INFINITY ? 0.f : m[nt][c];
        s[nt][c] = ptx::exp2_approx((s[nt][c] - against) * sl2);
        s[nt][c + 2] = ptx::exp2_approx((s[nt][c + 2] - against) * sl2);
        l[nt][c] = fmaf(l[nt][c], alpha[nt][c], s[nt][c] + s[nt][c + 2]);
      }
      p[nt][0] = transposed(kFp16 ? ptx::pack_f16(s[nt][0], s[nt][1]) : ptx::pack_bf16(s[nt][0], s[nt][1]));
      p[nt][1] = transposed(kFp16 ? ptx::pack_f16(s[nt][2], s[nt][3]) : ptx::pack_bf16(s[nt][2], s[nt][3]));
    }
    if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int mt = 0; mt < D / 16; ++mt)
#pragma unroll
          for (int c = 0; c < 4; ++c) o[nt][mt][c] *= alpha[nt][c & 1];
    }
#pragma unroll
    for (int mt = 0; mt < D / 16; ++mt) {
      // A: 16 columns x 16 keys out of rows of keys: (keys 0-7, columns 0-7), (keys 0-7, columns 8-15), (keys 8-15, ...)
      uint32_t a[4];
      const int r = (lane & 7) + ((lane >> 4) << 3), pc = mt * 2 + ((lane >> 3) & 1);
      ldmatrix4_trans(a, v_at + R::place(r, pc));
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) mma<kFp16>(o[nt][mt], a, p[nt][0], p[nt][1]);
    }
    ++at.unit, ++at.cost;
    const bool ends = at.unit == at.units;
    if (!ends && at.cost < span) continue;

    // ---- the problem, or this warp's part of it, is done ----
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int c = 0; c < 2; ++c)
#pragma unroll
        for (int d = 4; d < 32; d <<= 1) l[nt][c] += __shfl_xor_sync(0xffffffffu, l[nt][c], d);
    const bool whole = begun && ends;
    const long long part = (2LL * worker + (begun ? 1 : 0)) * (NT * 8);
    const int rows = at.e.n * prm.group;
    if (!whole || prm.leave.o != nullptr) {
      // sums and statistics as they are: to the warp's part, or where the pass leaves them
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          const int r = nt * 8 + cq * 2 + c;
          if (r >= rows) continue;
          const long long row = whole ? row_place(prm, at.e.first, at.kv_head, r).row : part + r;
          float* to_o = (whole ? prm.leave.o : by_warp.o) + row * D + kq;
#pragma unroll
          for (int mt = 0; mt < D / 16; ++mt) to_o[mt * 16] = o[nt][mt][c], to_o[mt * 16 + 8] = o[nt][mt][c + 2];
          if (kq == 0) (whole ? prm.leave.ml : by_warp.ml)[row] = make_float2(m[nt][c], l[nt][c]);
        }
    } else {
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        const float inv[2] = {1.f / l[nt][0], 1.f / l[nt][1]};  // (no key: 0 * inf = NaN)
        const int r = nt * 8 + kq;  // the row whose columns this lane has once they are turned round
        const RowPlace place = row_place(prm, at.e.first, at.kv_head, r);
#pragma unroll
        for (int mt = 0; mt < D / 16; ++mt)
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            const float a = o[nt][mt][2 * half] * inv[0], b = o[nt][mt][2 * half + 1] * inv[1];
            const uint32_t pair = transposed(kFp16 ? ptx::pack_f16(a, b) : ptx::pack_bf16(a, b));
            if (r < rows && mt * 2 + half < prm.pieces_v) *reinterpret_cast<uint32_t*>(place.out + 2 * (mt * 16 + half * 8 + cq * 2)) = pair;
          }
#pragma unroll
        for (int c = 0; c < 2; ++c)
          if (kq == 0 && nt * 8 + cq * 2 + c < rows) prm.lse[row_place(prm, at.e.first, at.kv_head, nt * 8 + cq * 2 + c).row] = m[nt][c] * prm.scale + logf(l[nt][c]);
      }
    }
    if (!whole && lane == 0) {
      Shared& mine_shared = shared[warp];
      const int which = begun ? 1 : 0;
      mine_shared.first[which] = at.e.first, mine_shared.n[which] = at.e.n, mine_shared.kv_head[which] = at.kv_head;
      if (begun) mine_shared.begins = 1, mine_shared.end = to + at.units - at.unit;
      else mine_shared.enters = 1, mine_shared.through = !ends;
    }
    if (!ends || at.cost + kBegin >= span) break;
    next_problem(prm, at);
    begun = fresh = true;
  }

  // ---- the block's parts: chain 0 enters from the block before, chain 1 + w begins with warp w ----
  __syncthreads();
  constexpr int kLanes = D / 4, kAtOnce = 32 / kLanes;  // lanes to a row of sums, rows a warp has at once
  int turn = 0;
#pragma unroll 1
  for (int chain = 0; chain <= kWarps; ++chain) {
    const Shared& at_head = shared[chain == 0 ? 0 : chain - 1];
    if (!(chain == 0 ? at_head.enters : at_head.begins)) continue;
    int members = 0;  // warps chain, chain + 1, ... that it enters
    bool open = true;
    while (open && chain + members < kWarps) open = shared[chain + members].through != 0, ++members;
    const int which = chain == 0 ? 0 : 1;
    const int first = at_head.first[which], n = at_head.n[which], kv_head = at_head.kv_head[which], rows = n * prm.group;
    const int warp0 = blockIdx.x * kWarps + chain;  // the first worker it enters
    if (chain > 0 && open && threadIdx.x == 0) {
      const int last = small_quotient(at_head.end - 1, share) / kWarps;  // the block that has the problem's last unit
      prm.parts.heads[blockIdx.x] = Head{last - static_cast<int>(blockIdx.x), first, n, kv_head, 0, kPagedFewRows};
    }
#pragma unroll 1
    for (int r0 = 0; r0 < rows; r0 += kAtOnce) {
      if (turn++ % kWarps != warp) continue;
      const int r = r0 + lane / kLanes, column = (lane % kLanes) * 4;
      if (r >= rows) continue;
      Sums sums;
      // four parts at a time: the beginning's own first (chain > 0), then those of the warps it enters
#pragma unroll 1
      for (int i0 = -which; i0 < members; i0 += 4) {
        float2 ml[4];
        float4 o[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          const int member = i0 + u;
          const long long part = (member < 0 ? 2LL * (warp0 - 1) + 1 : 2LL * (warp0 + member)) * (NT * 8) + r;
          ml[u] = make_float2(-INFINITY, 0.f), o[u] = make_float4(0.f, 0.f, 0.f, 0.f);
          if (member < members) ml[u] = by_warp.ml[part], o[u] = *reinterpret_cast<const float4*>(by_warp.o + part * D + column);
        }
#pragma unroll
        for (int u = 0; u < 4; ++u) sums.add(ml[u].x, ml[u].y, o[u], sl2);
      }
      if (chain > 0 && !open) {
        finish4<D, kFp16>(prm, row_place(prm, first, kv_head, r), column, sums.acc, sums.m, sums.l);
      } else {
        const long long part = (2LL * blockIdx.x + which) * (NT * 8) + r;
        *reinterpret_cast<float4*>(prm.parts.o + part * D + column) = sums.acc;
        if (column == 0) {
          prm.parts.ml[part] = make_float2(sums.m, sums.l);
          if (chain > 0 && prm.leave.o != nullptr) leave_in_parts(prm, row_place(prm, first, kv_head, r).row, r);
        }
      }
    }
  }
}

template <int D, bool kFp16, int NT, int kWarps>
int launch_few(const Pass& pass, const Parts& by_warp, cudaStream_t stream) {
  auto kernel = sdpa_paged_few_kernel<D, kFp16, NT, kWarps>;
  static bool sized[64] = {};
  int device = 0;
  LIMN_CUDA(cudaGetDevice(&device), "asking for the current device");
  if (device >= 0 && device < 64 && !sized[device]) {
    LIMN_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, Ring<D, kWarps>::kBytes), "sizing shared memory for the paged sdpa kernel");
    sized[device] = true;
  }
  LIMN_CUDA(launch_overlapped(kernel, dim3(static_cast<unsigned>(pass.parts.workers)), dim3(kWarps * 32), Ring<D, kWarps>::kBytes, stream, pass, by_warp), "launching the paged sdpa kernel");
  note_launches(1);
  return LIMN_B200_OK;
}

template <int D>
int launch_few_d(const Pass& pass, const Parts& by_warp, bool fp16, int rows, int warps, cudaStream_t stream) {
  if constexpr (D == 64) {
    if (warps == kMostWarps) return fp16 ? launch_few<D, true, 1, kMostWarps>(pass, by_warp, stream) : launch_few<D, false, 1, kMostWarps>(pass, by_warp, stream);
  }
  if (rows <= 8) return fp16 ? launch_few<D, true, 1, 8>(pass, by_warp, stream) : launch_few<D, false, 1, 8>(pass, by_warp, stream);
  return fp16 ? launch_few<D, true, 2, 8>(pass, by_warp, stream) : launch_few<D, false, 2, 8>(pass, by_warp, stream);
}

int few_tile(int rows) { return rows <= 8 ? 8 : kPagedFewRows; }

}  // namespace

size_t paged_few_workspace(int rows, int width, int sms) { return Parts::bytes(sms, few_tile(rows), width) + Parts::bytes(sms * most_warps(width, rows), few_tile(rows), width); }

int paged_few_launch(Pass& pass, bool fp16, int rows, unsigned char* workspace, cudaStream_t stream) {
  Parts by_warp;
  const int width = pass.pieces <= 8 && pass.pieces_v <= 8 ? 64 : 128, warps = warps_for(pass, width, rows);
  pass.parts.place(workspace, pass.blocks, few_tile(rows), width);
  by_warp.place(workspace + Parts::bytes(pass.blocks, few_tile(rows), width), pass.blocks * warps, few_tile(rows), width);
  if (width == 64) return launch_few_d<64>(pass, by_warp, fp16, rows, warps, stream);
  return launch_few_d<128>(pass, by_warp, fp16, rows, warps, stream);
}

}  // namespace limn_b200
