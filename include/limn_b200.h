/* limn_b200: fused scaled-dot-product attention for NVIDIA B200 (sm_100a), C ABI.
 *
 * These are the entry points a host binds in place of the three CUSTOM kernels limn's cuda
 * device compiles with NVRTC (limn/backend_cuda.py:352-361 builds them from the emitters at
 * limn/cuda_emit.py:921-1083). Every tensor is dense row-major with its leading dims
 * flattened into `bh` independent problems, exactly as the reference's block decoding does
 * (limn/cuda_emit.py:765-775, :853-862). All pointers are device pointers unless a function
 * says otherwise; nothing here allocates per call, synchronises, or keeps a pointer after
 * it returns. Kernels are enqueued on `stream` (NULL = the legacy default stream, which is
 * where limn launches: limn/backend_cuda.py:413).
 *
 * Every function returns 0 on success and a non-zero code otherwise; the message for the
 * calling thread's last failure is limn_b200_last_error(). The host binding turns that
 * into the RuntimeError the reference raises from check() (limn/backend_cuda.py:154-162).
 */
#ifndef LIMN_B200_H
#define LIMN_B200_H

#ifdef __cplusplus
extern "C" {
#endif

/* Storage dtypes of q, k, v, dO and the outputs (limn/ops.py:24-27). The row statistics
 * L and delta are float32 for F32/F16/BF16 and float64 for F64 (limn/ops.py:53-62). */
enum limn_b200_dtype {
  LIMN_B200_F32 = 0,
  LIMN_B200_F16 = 1,
  LIMN_B200_BF16 = 2,
  LIMN_B200_F64 = 3
};

enum limn_b200_status {
  LIMN_B200_OK = 0,
  LIMN_B200_BAD_ARGUMENT = 1,   /* null pointer, non-positive extent, causal with t_q != t_k, unknown dtype */
  LIMN_B200_UNSUPPORTED = 2,    /* extents beyond what any kernel here serves */
  LIMN_B200_CUDA_ERROR = 3,     /* a CUDA runtime/driver call failed; the message names it */
  LIMN_B200_DEVICE_TIMEOUT = 4  /* a kernel gave up on a bounded wait; see limn_b200_device_status */
};

/* Which kernel family served (or would serve) a problem. */
enum limn_b200_path {
  LIMN_B200_PATH_GENERAL = 0,  /* everything else, any float dtype, any hd/hd_v: SIMT kernels, except that float32 with hd and hd_v up
                                  to 128 and sides of 16 rows and more runs on the tensor cores where that is faster, at float32
                                  accuracy (this query does not tell the two apart) */
  LIMN_B200_PATH_TCGEN05 = 1,  /* TMA + tcgen05 kernels: f16/bf16, hd and hd_v multiples of 8 up to 128 (run as 64 or 128), any t_q/t_k, with or without key mask */
  LIMN_B200_PATH_DECODE = 2    /* forward only, no causal mask (the step of a kv cache), hd and hd_v multiples of 8 up to 128,
                                  rows on 16-byte boundaries: t_q <= 4 in f16/bf16 (dense or strided), t_q < 16 in float32 (dense). One CTA
                                  or cluster streams a problem's keys and values once, bound by HBM, no tensor cores */
};

/* "sdpa": replaces emit_sdpa (limn/cuda_emit.py:921-965); oracle limn/sdpa.py:91-137.
 *   q (bh, t_q, hd), k (bh, t_k, hd), v (bh, t_k, hd_v), key_mask (bh, t_k) in the same dtype
 *   or NULL (0 hides a key), out (bh, t_q, hd_v) in the same dtype, lse (bh, t_q) float32
 *   (float64 for F64). A query row with no visible key gets NaN and lse = -inf. */
int limn_b200_sdpa_fwd(const void* q, const void* k, const void* v, const void* key_mask,
                       void* out, void* lse,
                       int dtype, long long bh, int t_q, int t_k, int hd, int hd_v,
                       int causal, double scale, void* stream);

/* "sdpa_bwd_q": replaces emit_sdpa_bwd_q (limn/cuda_emit.py:968-1005); oracle limn/sdpa.py:140-170.
 *   dout (bh, t_q, hd_v); lse and delta (bh, t_q) in the statistics dtype; dq (bh, t_q, hd). */
int limn_b200_sdpa_bwd_q(const void* q, const void* k, const void* v, const void* dout,
                         const void* lse, const void* delta, const void* key_mask,
                         void* dq,
                         int dtype, long long bh, int t_q, int t_k, int hd, int hd_v,
                         int causal, double scale, void* stream);

/* "sdpa_bwd_q" with the row dot folded in: the same dQ as limn_b200_sdpa_delta followed by limn_b200_sdpa_bwd_q,
 * one launch and one pass over O and dO fewer where that is the faster way (short sequences); for dense operands
 * with more than 512 keys the call runs the row-dot kernel and the dQ kernel itself, which is faster there. Either
 * way one call. Replaces the pair limn's frontend schedules between the forward and
 * the backward ops (the reduce of limn/tensor.py:705-706 and emit_sdpa_bwd_q, limn/cuda_emit.py:968-1005).
 *   out is the forward's O (bh, t_q, hd_v), an input here; delta (bh, t_q) in the statistics dtype is an OUTPUT:
 *   every CTA computes the statistic of the query rows it owns from their rows of O and dO and leaves it there for
 *   limn_b200_sdpa_bwd_kv, which needs it for every query it streams and therefore has to run after this call. */
int limn_b200_sdpa_bwd_q_fused(const void* q, const void* k, const void* v, const void* out, const void* dout,
                               const void* lse, const void* key_mask,
                               void* dq, void* delta,
                               int dtype, long long bh, int t_q, int t_k, int hd, int hd_v,
                               int causal, double scale, void* stream);

/* "sdpa_bwd_kv": replaces emit_sdpa_bwd_kv (limn/cuda_emit.py:1008-1083); oracle limn/sdpa.py:173-203.
 *   dk (bh, t_k, hd), dv (bh, t_k, hd_v). Rows of a hidden key are written as exact zeros. */
int limn_b200_sdpa_bwd_kv(const void* q, const void* k, const void* v, const void* dout,
                          const void* lse, const void* delta, const void* key_mask,
                          void* dk, void* dv,
                          int dtype, long long bh, int t_q, int t_k, int hd, int hd_v,
                          int causal, double scale, void* stream);

/* dQ for hosts that must not allocate. No counterpart in the reference: limn's frontend always
 * brings delta in a buffer of its own (limn/tensor.py:705-707) and its cuda device allocates freely.
 *   Same result as limn_b200_sdpa_delta followed by limn_b200_sdpa_bwd_q, but delta and the kernels'
 *   status word live in a fixed array inside the library image instead of in memory somebody has to
 *   allocate: a host whose own pool holds all device memory, or code that runs where CUDA allocation
 *   calls are not allowed, passes only inputs and outputs. `out` is the forward's O (bh, t_q, hd_v);
 *   `status_out` is an optional device word that receives the kernels' status (0 = no wait gave up).
 *   Limits: bh * t_q <= LIMN_B200_STATIC_MAX_ROWS, else LIMN_B200_UNSUPPORTED and nothing is launched.
 *   All calls on a device share the array: calls that can overlap on the GPU race and must be
 *   serialised by the caller. The first call on a device looks the array's address up (and, with CUDA's lazy
 *   module loading, is when the driver places the array and the kernels on that GPU): make it before any
 *   stream capture on that device and while the device still has ~10 MiB free, or set CUDA_MODULE_LOADING=EAGER.
 *   Every argument check happens before anything is enqueued: a refused call launches nothing and leaves the
 *   array untouched. */
#define LIMN_B200_STATIC_MAX_ROWS (1LL << 20)
int limn_b200_sdpa_bwd_q_static(const void* q, const void* k, const void* v, const void* out,
                                const void* dout, const void* lse, const void* key_mask,
                                void* dq, unsigned int* status_out,
                                int dtype, long long bh, int t_q, int t_k, int hd, int hd_v,
                                int causal, double scale, void* stream);

/* delta = sum_d dout * out per query row, in the statistics dtype: the row dot the frontend
 * computes between the forward and the two backward ops (limn/tensor.py:705-706). Offered so
 * a host that drives the three ops directly need not bring its own reduce kernel. */
int limn_b200_sdpa_delta(const void* out, const void* dout, void* delta,
                         int dtype, long long rows, int hd_v, void* stream);

/* ---- operands as the model holds them: (batch, t, heads, hd) ----
 * limn's frontend permutes (batch, t, heads, hd) activations to (batch, heads, t, hd) and wraps each operand in
 * CONTIGUOUS before the CUSTOM node (limn/tensor.py:561-562; the gradient of that permute copies again on the way
 * back, limn/tensor.py:736-746), so every attention call is surrounded by full-tensor copies. These entry points
 * read and write the token-major layout in place through the tensor maps' strides, so a frontend that skips the
 * permute can skip the copies too. They have no counterpart in the reference.
 *   layout LIMN_B200_BHTD: q, k, v, dout, out, dq, dk, dv are (batch, heads, t, hd) dense: the same as the entry
 *     points above with bh = batch * heads.
 *   layout LIMN_B200_BTHD: they are (batch, t, heads, hd) dense.
 *   Either way lse and delta are (batch * heads, t_q) and key_mask (batch * heads, t_k), as above.
 *   LIMN_B200_BTHD is served for f16/bf16 with hd and hd_v multiples of 8 up to 128 (the tensor-core kernels); anything else
 *   returns LIMN_B200_UNSUPPORTED and launches nothing. */
enum limn_b200_layout {
  LIMN_B200_BHTD = 0,
  LIMN_B200_BTHD = 1
};
int limn_b200_sdpa_fwd_layout(const void* q, const void* k, const void* v, const void* key_mask,
                              void* out, void* lse,
                              int layout, int dtype, int batch, int heads, int t_q, int t_k, int hd, int hd_v,
                              int causal, double scale, void* stream);
int limn_b200_sdpa_bwd_q_layout(const void* q, const void* k, const void* v, const void* dout,
                                const void* lse, const void* delta, const void* key_mask,
                                void* dq,
                                int layout, int dtype, int batch, int heads, int t_q, int t_k, int hd, int hd_v,
                                int causal, double scale, void* stream);
int limn_b200_sdpa_bwd_q_fused_layout(const void* q, const void* k, const void* v, const void* out, const void* dout,
                                      const void* lse, const void* key_mask,
                                      void* dq, void* delta,
                                      int layout, int dtype, int batch, int heads, int t_q, int t_k, int hd, int hd_v,
                                      int causal, double scale, void* stream);
int limn_b200_sdpa_bwd_kv_layout(const void* q, const void* k, const void* v, const void* dout,
                                 const void* lse, const void* delta, const void* key_mask,
                                 void* dk, void* dv,
                                 int layout, int dtype, int batch, int heads, int t_q, int t_k, int hd, int hd_v,
                                 int causal, double scale, void* stream);
int limn_b200_sdpa_delta_layout(const void* out, const void* dout, void* delta,
                                int layout, int dtype, int batch, int heads, int t_q, int hd_v, void* stream);

/* ---- operands with strides of their own ----
 * q, k and v of an attention layer are usually slices of one projection's output, (batch, t, 3, heads, hd), and the
 * layer's result is wanted as (batch, t, heads * hd): no single layout describes both. These entry points take one
 * (batch, head, row) stride triple per operand, in elements (columns are contiguous; every stride a multiple of 8,
 * every pointer 16-byte aligned and already offset to the operand's first element), so a frontend can hand over its
 * views as they are instead of copying them (limn/tensor.py:561-562, :736-746 make those copies). lse and delta stay
 * (batch * heads, t_q), key_mask (batch * heads, t_k). No counterpart in the reference. f16/bf16 with hd and hd_v
 * multiples of 8 up to 128 only; anything else returns LIMN_B200_UNSUPPORTED and launches nothing.
 *   limn_b200_sdpa_fwd_strided:          strides of q, k, v, out                 (4 triples)
 *   limn_b200_sdpa_bwd_q_fused_strided:  strides of q, k, v, out, dout, dq        (6 triples); delta is written
 *   limn_b200_sdpa_bwd_kv_strided:       strides of q, k, v, dout, dk, dv         (6 triples) */
int limn_b200_sdpa_fwd_strided(const void* q, const void* k, const void* v, const void* key_mask,
                               void* out, void* lse, const long long* strides,
                               int dtype, int batch, int heads, int t_q, int t_k, int hd, int hd_v,
                               int causal, double scale, void* stream);
int limn_b200_sdpa_bwd_q_fused_strided(const void* q, const void* k, const void* v, const void* out, const void* dout,
                                       const void* lse, const void* key_mask,
                                       void* dq, void* delta, const long long* strides,
                                       int dtype, int batch, int heads, int t_q, int t_k, int hd, int hd_v,
                                       int causal, double scale, void* stream);
int limn_b200_sdpa_bwd_kv_strided(const void* q, const void* k, const void* v, const void* dout,
                                  const void* lse, const void* delta, const void* key_mask,
                                  void* dk, void* dv, const long long* strides,
                                  int dtype, int batch, int heads, int t_q, int t_k, int hd, int hd_v,
                                  int causal, double scale, void* stream);

/* ---- a paged key and value cache: append with rotary positions, attention over the pages, a shared prefix ----
 * The step of a server that generates for many sequences at once. Keys and values lie in pages of page_size tokens; a
 * sequence has a row of page numbers, its page table, and slot j of the sequence is slot j % page_size of page
 * table[j / page_size]. The step's tokens are packed: sequence b has tokens q_start[b] to q_start[b + 1], and they are the
 * last ones of its kv_lens[b] keys: token i of n is at slot kv_lens[b] - n + i. Table, offsets and lengths are read on the device
 * by each call, so a captured call follows what they hold when it is replayed. No counterpart in the reference,
 * which has no cache (its decode shape is t_q < t_k of dense tensors, tests/test_attention.py:385-396).
 *   f16/bf16, hd and hd_v multiples of 8 up to 128, heads a multiple of kv_heads (query head h reads key head
 *   h / (heads / kv_heads)) and at most 128 to a key head, page_size a multiple of 8; strides in elements, multiples of 8, columns
 *   contiguous, bases 16-byte aligned, every other array as its type is. Positions, tokens * heads and max_pages * page_size fit 31 bits. Anything
 *   else is refused and nothing is launched, a cache in host memory or on another device than the current one too.
 * What only the device knows is checked there. A sequence whose offsets or length are impossible (q_start falling, beyond
 * `tokens` or more than max_t_q apart; kv_lens negative or beyond max_pages * page_size, unless the sequence brings no token) is left out: nothing of it is appended
 * and no row of its result is written. Where q_start falls anywhere, no row of any sequence's result is written, and other sequences' tokens may not be appended. One that brings more tokens than it has
 * keys has no slots for the first of them: none of it is appended, and those tokens see no key. A page number outside [0, pages) is never followed: a new token that belongs there is
 * not appended, and a query row that sees a key there gets NaN (O and L). Either is noted in *errors (LIMN_B200_PAGED_BAD_*
 * bits are or-ed in; the caller clears the word). Tokens from q_start[batch] on, empty slots of pages, and pages that no table
 * names are neither read for a result nor written. */
#define LIMN_B200_PAGED_BAD_PAGE 1u
#define LIMN_B200_PAGED_BAD_SEQUENCE 2u
typedef struct limn_b200_paged {
  void* k_cache;              /* element (page, head, slot, column): base + page * k_strides[0] + head * k_strides[1] + slot * k_strides[2] + column */
  void* v_cache;
  const int* page_table;      /* (batch, max_pages), dense */
  const int* q_start;         /* (batch + 1) */
  const int* kv_lens;         /* (batch): keys in the sequence's pages, the step's tokens among them */
  unsigned int* errors;       /* device word, or NULL */
  long long k_strides[3];     /* page, head, slot */
  long long v_strides[3];
  int dtype;                  /* LIMN_B200_F16 or LIMN_B200_BF16 */
  int batch, heads, kv_heads, hd, hd_v;
  int page_size, pages, max_pages;
  int tokens;                 /* rows that q, k, v and the results have */
  int max_t_q;                /* a sequence brings at most this many tokens */
  int first_position;         /* position (for the rotation) of a sequence's slot 0: the length of a prefix that lies elsewhere */
} limn_b200_paged;

/* Which columns turn together: j and j + rotated / 2, or 2 j and 2 j + 1. */
enum limn_b200_pairing {
  LIMN_B200_HALVES = 0,
  LIMN_B200_NEIGHBOURS = 1
};

/* Put the step's keys and values into their slots, turned to their positions, and turn the queries beside them.
 *   q (tokens, heads, hd) -> q_out, or both NULL; k (tokens, kv_heads, hd), v (tokens, kv_heads, hd_v) into the cache.
 *   strides: (token, head) pairs of q, q_out, k, v (4 pairs; those of absent operands are not read). q_out may be q, with its strides.
 *   The first `rotated` columns of a row (a multiple of 8, 0 to hd) turn: pair j of a token at position p = first_position + slot
 *   by the angle p * frequencies[j], (x, y) -> (x cos - y sin, x sin + y cos); frequencies is a device array of rotated / 2
 *   doubles (NULL where rotated is 0). The angle is reduced in float64, the turn is float32, rounded once. Of a token that is not appended
 *   the row of q_out is not written either.
 *   Two new tokens of the batch must not share a slot. */
int limn_b200_kv_append(const limn_b200_paged* step, const void* q, const void* k, const void* v, void* q_out,
                        const long long* strides, const double* frequencies, int rotated, int pairing, void* stream);

/* Attention of the step's tokens over their sequences' pages (what limn_b200_kv_append has put there included).
 *   q (tokens, heads, hd), out (tokens, heads, hd_v), lse (tokens, heads) float32, dense; strides: (token, head) pairs of q, out.
 *   out and lse overlap no operand. scale is from 1e-30 to 1e30. The same call gives the same bits; a row's last bits may depend on what else is in the batch.
 *   causal: token i sees the keys up to its own; otherwise all of its sequence's. A row that sees no key gets NaN and
 *   lse = -inf. Keys and values that a row does not see but another row of its sequence in this step does count as 0 * v in its sum, as
 *   everywhere in 16 bits here: an infinity among them gives NaN. Empty slots may hold anything.
 *   A row's weights are rounded to the operands' type before they multiply v, half a step each (float16 holds none below 2^-25 of the largest); scores and sums are float32, as the
 *   matrix instructions make them, and the weights' sum is of the unrounded ones. Against 64 bits out is off by 1.2 to 1.4 times what 32 bits throughout would be off by, which is
 *   out's own rounding. Keys that each weigh less than 2^-23 of what the row has gathered count in lse and may be lost from out: a hundred thousand of them 0.2 % of it.
 *   workspace: device memory of limn_b200_sdpa_paged_workspace bytes, 16-byte aligned, contents of no concern before
 *   and after the call; calls that can overlap on the GPU need one each. */
int limn_b200_sdpa_paged(const limn_b200_paged* step, const void* q, void* out, float* lse, const long long* strides,
                         int causal, double scale, void* workspace, unsigned long long workspace_bytes, void* stream);

/* The same for a batch whose sequences all continue one prefix: every row sees the prefix_len keys of the pages prefix_table
 * names (device array, ceil(prefix_len / page_size) entries) and behind them its sequence's own as above. Where that costs less
 * the prefix is read once for the whole batch, in a pass of its own, else in front of every sequence's keys; a result's bits depend on which. Keys in a sequence's own pages are counted from the prefix's end: kv_lens, q_start and page_table do not
 * include it, first_position does. At most 262140 heads. */
int limn_b200_sdpa_paged_prefix(const limn_b200_paged* step, const void* q, void* out, float* lse, const long long* strides,
                                const int* prefix_table, int prefix_len, int causal, double scale,
                                void* workspace, unsigned long long workspace_bytes, void* stream);

/* Bytes of workspace a call for this step needs on the current device, whatever the device arrays hold; prefix_len 0 for
 * limn_b200_sdpa_paged, any other for a prefix of any length. Pointers in *step are not looked at. */
int limn_b200_sdpa_paged_workspace(const limn_b200_paged* step, int prefix_len, unsigned long long* bytes);

/* Which path the dispatcher picks for a problem (a limn_b200_path value), or -1 with an
 * error message if the arguments are invalid. Launches nothing. */
int limn_b200_sdpa_path(int dtype, long long bh, int t_q, int t_k, int hd, int hd_v,
                        int causal, int has_mask, double scale);

/* How many kernels the last successful limn_b200_sdpa_* call on this thread enqueued. */
int limn_b200_last_launch_count(void);

/* Message for the calling thread's most recent failure ("" if none). Stands where the
 * driver's error string stands in limn/backend_cuda.py:154-162. */
const char* limn_b200_last_error(void);

/* Library version, major * 10000 + minor * 100 + patch. */
int limn_b200_version(void);

/* Kernels that wait (on TMA or tensor-core completion) give up after a bounded time and
 * record a code in a per-device status word instead of hanging; kernels of that kind launched on that
 * device afterwards return within some milliseconds, writing nothing, until the word has been read
 * (the float64, CUDA-core, decode and row-dot kernels wait for nothing and run; so do limn_b200_kv_append and, for at most 16 query
 * rows to a key head, limn_b200_sdpa_paged). This synchronises the
 * current device, reads its word into *status and clears it. Returns LIMN_B200_OK with *status == 0
 * when no kernel gave up, LIMN_B200_DEVICE_TIMEOUT with *status = 0x5741rrbb (role rr, barrier bb)
 * when one did. The reference reports a failed kernel from its batch barrier
 * (limn/backend_cuda.py:349 through check(), :154-162); limn_b200.install() makes finish() call this. */
int limn_b200_device_status(unsigned int* status);

/* Diagnostic, no counterpart in the reference: one warp waits on a barrier nobody arrives at, with the
 * production kernels' bounded wait but a budget of `budget_ticks` clock ticks (at most 1e8), so that the wait
 * runs out, the status word of the current device receives 0x57417e57 and the kernel returns normally.
 * `gave_up` is an optional device word that receives 1 (the wait ran out) or 0. It lets a test walk the
 * give-up path (status code, later launches standing down, counters left clean, read-and-clear) without
 * making any production kernel misbehave and without hanging or faulting anything. */
int limn_b200_wait_probe(long long budget_ticks, unsigned int* gave_up, void* stream);

/* ---- the gather of (batch, head) shards over NCCL, for sharded hosts without a communication library of their own ----
 * No counterpart in the reference, which is single-GPU (limn/backend_cuda.py:283 takes device 0). The problems of a
 * batch are independent: rank r of N computes problems [r BH/N, (r+1) BH/N) with the entry points above and no
 * communication, and the outputs are then gathered into one tensor on every GPU. One process per GPU, one
 * communicator per process; NCCL (libnccl.so.2, or the file LIMN_B200_NCCL_LIBRARY names) is loaded when the first of
 * these is called, so a single-GPU host never needs it. Failures come back as status codes with a message, never as
 * an abort: LIMN_B200_UNSUPPORTED when NCCL cannot be loaded, LIMN_B200_BAD_ARGUMENT for a misuse,
 * LIMN_B200_CUDA_ERROR with NCCL's own error string otherwise.
 *   limn_b200_nccl_unique_id: rank 0 fills LIMN_B200_NCCL_ID_BYTES bytes (host memory); the host carries them to the
 *     other ranks by whatever means it has (a file, a socket, its launcher).
 *   limn_b200_nccl_init: every rank, with its own device current, the same id and world size.
 *   limn_b200_nccl_all_gather: recv (world * bytes_per_rank bytes) receives every rank's send (bytes_per_rank bytes) in
 *     rank order, enqueued on `stream`; send may be the rank's own slice of recv.
 *   limn_b200_nccl_destroy: releases the communicator. */
#define LIMN_B200_NCCL_ID_BYTES 128
int limn_b200_nccl_unique_id(void* id_out);
int limn_b200_nccl_init(int rank, int world, const void* id);
int limn_b200_nccl_all_gather(const void* send, void* recv, unsigned long long bytes_per_rank, void* stream);
int limn_b200_nccl_destroy(void);

/* ---- plumbing for hosts without a CUDA binding of their own (tests, benchmark) ----
 * limn itself allocates and copies through the driver API (limn/backend_cuda.py:297-326)
 * and never calls these. */
int limn_b200_device_count(int* count);
int limn_b200_set_device(int ordinal);
int limn_b200_mem_alloc(void** device_ptr, unsigned long long nbytes);
int limn_b200_mem_free(void* device_ptr);
int limn_b200_mem_set(void* device_ptr, int byte, unsigned long long nbytes, void* stream);
int limn_b200_host_alloc(void** pinned_ptr, unsigned long long nbytes);
int limn_b200_host_free(void* pinned_ptr);
int limn_b200_copy_h2d(void* device_dst, const void* host_src, unsigned long long nbytes, void* stream);
int limn_b200_copy_d2h(void* host_dst, const void* device_src, unsigned long long nbytes, void* stream);
int limn_b200_copy_d2d(void* device_dst, const void* device_src, unsigned long long nbytes, void* stream);
int limn_b200_stream_create(void** stream);
int limn_b200_stream_destroy(void* stream);
int limn_b200_stream_wait_event(void* stream, void* event);
int limn_b200_stream_sync(void* stream);
int limn_b200_device_sync(void);
int limn_b200_event_create(void** event);
int limn_b200_event_destroy(void* event);
int limn_b200_event_record(void* event, void* stream);
int limn_b200_event_elapsed_ms(void* start, void* stop, float* ms);

#ifdef __cplusplus
}
#endif
#endif /* LIMN_B200_H */
