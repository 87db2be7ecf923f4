/*
 * flashlite_attn.h -- C ABI of the MI355X (gfx950) FlashAttention-2 forward
 * engine.  Plain pointers and sizes only: no torch, no HIP types.  The
 * stream is passed as an opaque `void*` holding a `hipStream_t` (NULL = the
 * legacy default stream).
 *
 * Reference surface replaced (thebigblender/FlashLite):
 *   - the host entry of `flash_attn_wmma.forward_flash2`,
 *     csrc/kernel_flash2.cu:732-839 (declared csrc/includes/flash_attn.h:117-124,
 *     bound at csrc/flash_attn.cpp:18-28);
 *   - the host entry of `flash_attn_wmma.forward_naive`,
 *     csrc/kernel_naive.cu:242-323 (declared csrc/includes/flash_attn.h:100-106,
 *     bound at csrc/flash_attn.cpp:7-16).
 * The torch-side checks (device, contiguity, dtype, rank, shapes, `out=`) stay
 * in the binding (flashlite_amd/csrc/flash_attn.cpp) with the reference's
 * messages; the checks below are the ones a raw-pointer caller needs.
 *
 * Layout: q, o are fp16 [batch, heads, seq_q, head_dim] and k, v fp16
 * [batch, heads, seq_k, head_dim], contiguous (fl_attn_fwd_f16_ex takes
 * strides).
 * The library allocates nothing, never synchronises, keeps no mutable global
 * state (beyond, per GPU, the cached address of the scratch array of
 * fl_attn_fwd_f16_splitkv_noalloc) and may be called from several host
 * threads at once.  Launches are
 * asynchronous on `stream`; results are visible after the stream reaches
 * them.  `o` may alias `q` (each work-group reads its own query rows before
 * it writes them); it must not alias `k` or `v`.
 */
#ifndef FLASHLITE_ATTN_H
#define FLASHLITE_ATTN_H

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* Status codes returned by every entry point. */
enum fl_status {
  FL_OK = 0,
  FL_ERR_INVALID_ARGUMENT = 1, /* NULL pointer, negative size, non-finite scale */
  FL_ERR_UNSUPPORTED = 2,      /* head_dim != 64 (flash2; 64 or 128 for the _ex entries),
                                  strides or sizes past limits */
  FL_ERR_MISALIGNED = 3,       /* flash2 needs 16-byte aligned q/k/v/o */
  FL_ERR_LAUNCH = 4,           /* the HIP launch itself failed */
  FL_ERR_BAD_CONFIG = 5        /* forced tile configuration out of range */
};

typedef struct fl_attn_params {
  const void* q;      /* fp16 [B, H, N, D]; N = seq_q */
  const void* k;      /* fp16 [B, H, N_k, D] */
  const void* v;      /* fp16 [B, H, N_k, D] */
  void* o;            /* fp16 [B, H, N, D], written for rows < N */
  int64_t batch;      /* B */
  int64_t heads;      /* H */
  int64_t seq_q;      /* N (query rows) */
  int64_t seq_k;      /* N_k key/value rows (k, v are [B, H, N_k, D]); may differ from N */
  int64_t head_dim;   /* D */
  double sm_scale;    /* 0.0 means 1/sqrt(D) (kernel_flash2.cu:769-771) */
  int32_t causal;     /* non-zero: key j visible to query i iff j <= i + N_k - N (bottom-right
                         aligned; top-left when N_k == N); a row with no visible key gets 0 */
} fl_attn_params;

/*
 * FlashAttention-2 forward, fp16 in/out, fp32 accumulation, D == 64.
 * Replaces flash_attn_forward_flash2's validation tail, scale handling,
 * adaptive dispatcher and launch (csrc/kernel_flash2.cu:756-757, 769-772,
 * 786-837).  The tile configuration comes from the built-in dispatcher.
 */
int fl_attn_fwd_f16(const fl_attn_params* p, void* stream);

/*
 * Same as fl_attn_fwd_f16 with the tile configuration forced (`config` in
 * [0, fl_attn_num_configs()), or -1 for the dispatcher's choice).  Replaces
 * the reference's two hard-wired launch branches (Br=64 / Br=128,
 * csrc/kernel_flash2.cu:789-835); used by sweeps and by tests that check
 * every configuration against the oracle.  Configuration 5
 * (br256_kv256_w8_stream) takes N_k <= 256 only and configuration 6
 * (br32_kv512_w4_quarters) N_k <= 512 only; they return FL_ERR_BAD_CONFIG
 * otherwise.
 */
int fl_attn_fwd_f16_cfg(const fl_attn_params* p, int32_t config, void* stream);

/*
 * Strided layouts and the log-sum-exp output.  `base` carries the pointers,
 * sizes, scale and mask exactly as for fl_attn_fwd_f16 (its layout comment
 * aside); the strides below replace the contiguous [B, H, N, D] layout.
 * Each stride triple is {batch, head, row} in elements; head_dim is unit
 * stride.  A [B, N, H, D] tensor (the layout of the `flash_attn` package,
 * which the reference's benchmark builds by transposing,
 * benchmarks/benchmark_throughput.py:110-112) has strides
 * {N*H*D, D, H*D}.  Strides are non-negative multiples of 8 elements, row
 * strides in [64, 2^30); K and V rows must lie within 2^31 bytes of their
 * head's first row.  Output rows must not overlap each other or q, k, v
 * (o == q with equal strides is allowed, as for fl_attn_fwd_f16).
 *
 * lse: optional fp32 [B, H, N] (contiguous), written with each query row's
 * ln(sum_j exp(sm_scale * q.k_j)) over its visible keys, -inf for a row
 * with no visible key; NULL to skip.
 *
 * head_dim is 64 or 128.  At both, Q enters the MFMA unscaled and the fp32
 * scores are scaled by sm_scale*log2(e), as in the reference
 * (csrc/kernel_flash2.cu:188-195).  At 64, `config` is as for
 * fl_attn_fwd_f16_cfg;
 * at 128 it is -1 or one of the two slot-scheduled configurations
 * (3 "br256_bc64_w8_slot", 4 "br128_bc64_w4_slot"; same work-group shapes,
 * 32-key tiles), FL_ERR_BAD_CONFIG otherwise.
 *
 * No counterpart in the reference, which accepts only contiguous
 * [B, H, N, 64] tensors (csrc/kernel_flash2.cu:741-757) and returns no
 * log-sum-exp.
 */
typedef struct fl_attn_params_ex {
  fl_attn_params base;
  int64_t q_stride[3];
  int64_t k_stride[3];
  int64_t v_stride[3];
  int64_t o_stride[3];
  float* lse;
} fl_attn_params_ex;

int fl_attn_fwd_f16_ex(const fl_attn_params_ex* p, int32_t config, void* stream);

/*
 * bf16 q, k, v and o (same layouts, strides, lse and head_dims as
 * fl_attn_fwd_f16_ex; `config` -1 or, at head_dim 64, any configuration but
 * the pipelined 0 and 1, at head_dim 128 3 or 4).  Q enters the MFMA
 * unscaled and the fp32 scores are scaled by sm_scale*log2(e); P is rounded
 * to bf16 before the PV product and the row sums are fp32.
 *
 * No counterpart in the reference, which accepts fp16 only
 * (csrc/kernel_flash2.cu:745-747).
 */
int fl_attn_fwd_bf16_ex(const fl_attn_params_ex* p, int32_t config, void* stream);

/*
 * The dispatcher's choice for either element type (FL_DTYPE_*) and head_dim
 * (64 or 128), with split-KV where it pays: as fl_attn_fwd_f16_ex /
 * fl_attn_fwd_bf16_ex with config -1, but a problem with few query rows over
 * many keys cuts its key range into chunks whose partial results go to
 * `workspace` and are merged by a second kernel on the same stream.
 * fl_attn_workspace_bytes returns the bytes such a call uses (0: one pass,
 * -1: `p` is rejected).  With less (or a NULL workspace) the call runs one
 * pass.  The workspace is 16-byte aligned device memory owned by the caller;
 * calls that may overlap must not share one.
 *
 * No counterpart in the reference.
 */
#define FL_DTYPE_F16 0
#define FL_DTYPE_BF16 1
int64_t fl_attn_workspace_bytes(const fl_attn_params_ex* p, int32_t dtype);
int fl_attn_fwd_ws(const fl_attn_params_ex* p, int32_t dtype, void* workspace,
                   int64_t workspace_bytes, void* stream);

/*
 * Split-KV forward ("flash-decoding"), fp16 at head_dim 64, for few query
 * rows over many keys:
 * the key range of every (batch, head) is cut into chunks processed by
 * separate work-groups, whose partial results (unnormalised O, stabiliser,
 * row sum) go to `workspace`; a second kernel on the same stream merges
 * them into O (and lse).  Same parameters, layouts and results as
 * fl_attn_fwd_f16_ex up to fp32 rounding.
 *
 * num_splits > 0 asks for that many chunks (at most the number of 64-key
 * tiles, and 256); num_splits <= 0 lets the library choose, which may be
 * "no split": then the one-pass kernel runs and no workspace is needed.
 * fl_attn_splitkv_workspace_bytes returns the bytes a call with the same
 * `p` and `num_splits` needs (0 when it will not split, -1 if `p` is
 * rejected).  The workspace is 16-byte aligned device memory owned by the
 * caller; calls that may overlap must not share one.
 *
 * No counterpart in the reference (one work-group per 64/128 query rows,
 * csrc/kernel_flash2.cu:786-835, which leaves a decode step with N = 1 on a
 * handful of CUs); its README advertises `out=` for serving/decode loops
 * (README.md:119-126).
 */
int64_t fl_attn_splitkv_workspace_bytes(const fl_attn_params_ex* p, int32_t num_splits);
int fl_attn_fwd_f16_splitkv(const fl_attn_params_ex* p, int32_t num_splits, void* workspace,
                            int64_t workspace_bytes, void* stream);

/*
 * fl_attn_fwd_f16_splitkv without a workspace argument and without any
 * allocation: the partial results go to a scratch array of
 * FL_ATTN_SCRATCH_BYTES (8 MiB) that the library holds in device memory on
 * every GPU it runs on, until the process ends.  Same parameters and
 * results as fl_attn_fwd_f16_splitkv, bit for bit, for the same chunk
 * count.  num_splits > 0 is taken as asked; a count whose partials exceed
 * the limit returns FL_ERR_UNSUPPORTED and launches nothing.
 * num_splits <= 0 lets the library choose as for fl_attn_fwd_f16_splitkv,
 * lowered to the most chunks whose partials fit the limit, or to one pass
 * (no scratch) when fewer than two fit: the library's own choice never
 * fails for lack of scratch.  fl_attn_splitkv_noalloc_bytes returns the
 * scratch bytes a call with the same `p` and `num_splits` uses (0 for one
 * pass, -1 if `p` is rejected; above FL_ATTN_SCRATCH_BYTES only for a
 * requested count that will be refused).  Launches on the
 * current device, into `stream`, which must belong to it.  Every call on a
 * GPU shares that GPU's array (each call writes every partial it reads, so
 * nothing has to start at zero): calls that may overlap on one GPU -- other
 * streams, other host threads -- race and must be serialised by the caller.
 *
 * No counterpart in the reference.  For callers that cannot allocate device
 * memory: code under HIP graph capture, tight serving loops, harnesses that
 * forbid hipMalloc.
 */
#define FL_ATTN_SCRATCH_BYTES (8 << 20)
int fl_attn_fwd_f16_splitkv_noalloc(const fl_attn_params_ex* p, int32_t num_splits, void* stream);
int64_t fl_attn_splitkv_noalloc_bytes(const fl_attn_params_ex* p, int32_t num_splits);

/*
 * Serving over a paged cache: the blocks and slots of each step's tokens, the
 * ancestors of drafted tokens, rotary positions with the cache's writes, and
 * attention for drafted tokens (or one token) over the cache.  No counterpart
 * in the reference.
 *
 * The cache is blocks of block_size rows of every key/value head: k_cache and
 * v_cache are [num_blocks, kv_heads, block_size, head_dim] views with strides
 * {block, head, row} in elements (a cache stored [blocks, block_size, heads,
 * dim] passes as its transpose).  Token t of request b lies in row
 * t % block_size of block block_tables[b][t / block_size]; its slot is
 * block * block_size + row.  A cache that is not paged is one block a request.
 * Rows that a call writes must not overlap: a written view's strides nest, each
 * at least what the smaller ones span (views of dense memory do).
 */

/*
 * Blocks, slots and positions of a step's new tokens, on the GPU from the
 * requests' lengths.
 *
 * lengths[b] tokens are in the cache, counts[b] come (0 .. width; more are
 * taken as width); counts[b] < 0: the request has ended and gives its blocks
 * back.  held[b] blocks of row b of block_tables are its own.  The free blocks
 * are a ring: free_state = {head, count}, the count entries of free_blocks
 * from head on (modulo pool).  A request that needs more blocks than it holds
 * (ceil((lengths + counts) / block_size)) takes them from the ring's head, in
 * the order of the requests; blocks of ended requests are put behind the
 * ring's last, in order, and are free from the next call on (what a full ring
 * has no room for is dropped).
 *
 * Outputs: block_tables (entries of the blocks taken), held_out and
 * free_state_out (each its input, or apart from it), positions [batch, width] =
 * lengths[b] + i, slots [batch, width], both -1 where there is no token (i >=
 * counts[b], a request not served, a negative table entry), and info [batch,
 * 4]: {0 served, 1 not enough free blocks, 2 the table row is too short;
 * blocks held before; blocks taken, or minus those put back; the ring's index
 * of the first of them}.  A request that is not served keeps what it has; one
 * with nothing to take is always served.  Values out of range are brought into
 * it, never followed (a held count past the row, a count of free blocks past
 * the ring: clamped; a head past it: modulo pool).  info is 16-byte aligned;
 * batch is at most 65535.
 */
typedef struct fl_cache_plan_params {
  const int32_t* lengths;
  const int32_t* counts;
  int32_t* block_tables; /* rows of max_blocks entries, table_stride apart */
  const int32_t* held;
  int32_t* held_out;
  int32_t* free_blocks;
  const int32_t* free_state;
  int32_t* free_state_out;
  int32_t* positions;
  int64_t* slots;
  int32_t* info;
  int64_t batch;
  int64_t width;
  int64_t block_size;
  int64_t max_blocks;
  int64_t table_stride;
  int64_t pool;
} fl_cache_plan_params;

int fl_attn_cache_plan(const fl_cache_plan_params* p, void* stream);

/*
 * Ancestors and positions of drafted tokens.  parents[b][i] is the draft that
 * draft i follows, an earlier one; any other value means that it follows the
 * request's last token.  mask[b][i] gets the bits of i and its ancestors, in
 * ceil(drafts / 64) words (bit j % 64 of word j / 64 for draft j), positions
 * lengths[b] + the number of ancestors.  Drafts from counts[b] on (counts may
 * be NULL: all are there) get an empty mask and position -1.  At most
 * FL_ATTN_MAX_DRAFTS drafts a request.
 */
#define FL_ATTN_MAX_DRAFTS 512
typedef struct fl_tree_plan_params {
  const int32_t* parents; /* rows parent_stride apart */
  const int32_t* lengths;
  const int32_t* counts;
  int64_t* mask;
  int32_t* positions;
  int64_t batch;
  int64_t drafts;
  int64_t parent_stride;
} fl_tree_plan_params;

int fl_attn_tree_plan(const fl_tree_plan_params* p, void* stream);

/*
 * Rotary positions: the pairs of the first 2 * pairs columns of every q and k
 * row turn by the angle position * freqs[j] (freqs: radians a position,
 * 64-bit; the angle is reduced in 64 bits, so far positions stay exact), and
 * are multiplied by `scale`; the other columns are copied.  Pair j is columns
 * {j, j + pairs}, or {2j, 2j + 1} with interleaved.  With transpose the angle
 * is negated: the gradient of the same call.  q, k, q_out and k_out are
 * [batch, heads or kv_heads, rows, head_dim] views with strides {batch, head,
 * row} in elements; outputs may be their inputs (no other overlap).  k may be
 * NULL (no k), and q where heads is 0.
 * positions are int32 (or int64: position_bits 64) [batch, rows], strides
 * {batch, row}.  head_dim 64 or 128; dtype FL_DTYPE_F16, FL_DTYPE_BF16 or (not
 * with a cache) FL_DTYPE_F32.
 *
 * fl_attn_rotary_cache does the same for a step's tokens and stores them:
 * rotated k and v go to row slots[b][i] of the caches, rotated q to q_out
 * (k_out is not used).  A token whose slot is negative or past num_blocks *
 * block_size is passed over: its q_out row and the cache stay as they were.
 * Two tokens must not have the same slot.
 */
#define FL_DTYPE_F32 2
typedef struct fl_rotary_params {
  const void* q;
  const void* k;
  void* q_out;
  void* k_out;
  int64_t q_stride[3];
  int64_t k_stride[3];
  int64_t q_out_stride[3];
  int64_t k_out_stride[3];
  const void* positions;
  int64_t position_stride[2];
  int32_t position_bits;
  int32_t dtype;
  const double* freqs;
  int64_t pairs;
  int64_t batch;
  int64_t heads;
  int64_t kv_heads;
  int64_t rows;
  int64_t head_dim;
  double scale;
  int32_t interleaved;
  int32_t transpose;
} fl_rotary_params;

typedef struct fl_cache_store {
  const void* v;
  int64_t v_stride[3];
  void* k_cache;
  void* v_cache;
  int64_t k_cache_stride[3];
  int64_t v_cache_stride[3];
  int64_t num_blocks;
  int64_t block_size;
  const int64_t* slots;
  int64_t slot_stride[2];
} fl_cache_store;

int fl_attn_rotary(const fl_rotary_params* p, void* stream);
int fl_attn_rotary_cache(const fl_rotary_params* p, const fl_cache_store* c, void* stream);

/*
 * Norms of q and k for each head with the rotary positions in the same pass:
 * y = R(x r w), r = 1 / sqrt(mean(x x) + eps) over a head's row, w its weight
 * plus weight_offset, R the rotation above with its scale; products and sums
 * in 32 bits, rounded once (mean(x x) + eps below 2^-126 counts as 0).  q_weight
 * and k_weight are [head_dim], fp32 or of the rows' dtype (weight_dtype); NULL:
 * that tensor is only rotated.
 *
 * Positions may have several axes (time, height and width of a picture's
 * patches): with axes, int32 [pairs], pair j turns by the token's position on
 * axis axes[j] (brought into 0 .. num_axes - 1), and positions are [num_axes,
 * batch, rows], axis_stride elements apart.  axes NULL: one position a token.
 *
 * fl_attn_norm_rotary_cache stores the rows of a step's tokens as
 * fl_attn_rotary_cache does.
 *
 * fl_attn_norm_rotary_bwd takes the gradients of the outputs as q and k of `p`
 * and writes those of the inputs to its q_out and k_out (which may be the
 * gradients' own memory): with g = R' dy, dx = r (g w - x r r mean(g w x)), and
 * dq_weight, dk_weight = sum over batch, heads and rows of g x r, fp32
 * [head_dim] (each NULL: not wanted).  d->q and d->k are the forward pass'
 * inputs, not read where the weight is NULL.  The same inputs give the same
 * bits.  The workspace (fl_attn_norm_rotary_workspace_bytes) is 16-byte aligned
 * device memory that needs no initial values; calls that may overlap must not
 * share one.  `transpose` is not looked at.
 */
typedef struct fl_norm_params {
  const void* q_weight;
  const void* k_weight;
  int32_t weight_dtype;
  double eps;
  double weight_offset;
  const int32_t* axes;
  int64_t num_axes;
  int64_t axis_stride;
} fl_norm_params;

typedef struct fl_norm_grads {
  const void* q;
  const void* k;
  int64_t q_stride[3];
  int64_t k_stride[3];
  float* dq_weight;
  float* dk_weight;
} fl_norm_grads;

int fl_attn_norm_rotary(const fl_rotary_params* p, const fl_norm_params* n, void* stream);
int fl_attn_norm_rotary_cache(const fl_rotary_params* p, const fl_norm_params* n,
                              const fl_cache_store* c, void* stream);
int64_t fl_attn_norm_rotary_workspace_bytes(const fl_rotary_params* p);
int fl_attn_norm_rotary_bwd(const fl_rotary_params* p, const fl_norm_params* n,
                            const fl_norm_grads* d, void* workspace, int64_t workspace_bytes,
                            void* stream);

/*
 * Attention of drafted tokens over a paged cache (fp16 or bf16, head_dim 64 or
 * 128).  Request b has lengths[b] tokens and counts[b] drafts (counts may be
 * NULL: `drafts` of them), whose keys and values are in the cache behind them,
 * draft j as token lengths[b] + j.  Draft i sees every token, and draft j
 * where bit j of its mask is set (mask [batch, drafts, ceil(drafts / 64)]
 * words, batches mask_stride words apart, 0 for one mask for all; without a
 * mask the drafts are a chain, draft i sees drafts 0 .. i: a decode step at
 * drafts = 1, a prompt's chunk beyond).  q and o are [batch, heads, drafts,
 * head_dim] views with strides {batch, head, row}; heads is a multiple of
 * kv_heads, head h reads key/value head h / (heads / kv_heads).
 *
 * A row that sees nothing is 0 (its log-sum-exp -inf); rows of drafts from
 * counts[b] on are left as they were, o and lse alike.  A key whose block
 * table entry is not in [0, num_blocks) is seen by nobody.  What a row does
 * not see does not reach it, NaN and infinities in k_cache and v_cache
 * included.  max_blocks * block_size is below 2^31 - 65536.  lengths are clamped to the table's rows (max_blocks *
 * block_size), with the drafts behind them.  lse: optional fp32 [batch, heads,
 * drafts] (contiguous).  Block and row strides of the caches are below 2^31
 * elements.
 *
 * Few query rows over many keys are split over the CUs; partial results go to
 * `workspace` (fl_attn_tree_workspace_bytes, from the sizes and whether heads
 * or rows are closer together in k_cache; 0: none
 * is used, -1: `p` is rejected) and a second kernel merges them.  With less
 * (or NULL) the call runs without.  The workspace is 16-byte aligned device
 * memory that needs no initial values; calls that may overlap must not share
 * one.
 */
typedef struct fl_tree_params {
  const void* q;
  const void* k_cache;
  const void* v_cache;
  void* o;
  float* lse;
  int64_t q_stride[3];
  int64_t o_stride[3];
  int64_t k_stride[3]; /* {block, head, row} */
  int64_t v_stride[3];
  const int32_t* block_tables; /* rows of max_blocks entries, table_stride apart */
  int64_t table_stride;
  const int32_t* lengths;
  const int32_t* counts;
  const int64_t* mask;
  int64_t mask_stride;
  int64_t batch;
  int64_t heads;
  int64_t kv_heads;
  int64_t drafts;
  int64_t head_dim;
  int64_t num_blocks;
  int64_t block_size;
  int64_t max_blocks;
  double sm_scale; /* 0.0 means 1/sqrt(head_dim) */
  int32_t dtype;
} fl_tree_params;

int64_t fl_attn_tree_workspace_bytes(const fl_tree_params* p);
int fl_attn_tree_fwd(const fl_tree_params* p, void* workspace, int64_t workspace_bytes,
                     void* stream);

/*
 * Attention over packed sequences and its gradient (fp16 or bf16, head_dim 64
 * or 128).  Sequence i has rows starts[i] .. starts[i + 1] - 1 of q and o and
 * key_starts[i] .. key_starts[i + 1] - 1 of k and v (key_starts NULL: the same
 * as starts, with key_rows == rows), and attends to its own keys only; either
 * may be empty.  starts have sequences + 1 entries, which do not fall and lie in
 * [0, rows]; others are brought into range, never followed.  q and o are [heads,
 * rows, head_dim] and k and v [kv_heads, key_rows, head_dim] views with strides
 * {head, row} in elements (heads in front of or behind the rows, also views of
 * one projection); heads is a multiple of kv_heads, head h reads key/value head
 * h / (heads / kv_heads).  With causal, query i of nq sees key j of nk iff
 * j <= i + nk - nq.  lse: optional (forward) fp32 [heads, rows], contiguous.
 *
 * A row that sees nothing is 0 (its log-sum-exp -inf); rows of no sequence are
 * neither read nor written.  What a row does not see does not reach it, NaN and
 * infinities included, in the gradients too.
 *
 * fl_attn_packed_bwd takes the forward pass' o and lse and the gradient dout
 * of o, and writes dq, dk and dv (of shared key heads: the sum over their
 * query heads): with p = exp(s - lse) and s = sm_scale q.k, dv = p' dout,
 * ds = p (dout v' - dout . o), dq = sm_scale ds k, dk = sm_scale ds' q.  The
 * same inputs give the same bits.  p and ds are rounded to the element type for
 * their products, whose sums are fp32.  dq, dk and dv must not overlap the
 * inputs or each other; o may be q in the forward pass.  The workspace
 * (fl_attn_packed_bwd_workspace_bytes, from the sizes; -1: `p` is rejected) is
 * 16-byte aligned device memory that needs no initial values; calls that may
 * overlap must not share one.
 *
 * sm_scale is at least 1e-30 in size.  Row strides are below 2^24 elements,
 * those of q, k, v and o at least head_dim; rows and key_rows are at most 2^30,
 * sequences 2^24, and all rows of k and of v, and 128 more, lie within 2^31 bytes
 * of a head's first.
 */
typedef struct fl_packed_params {
  const void* q;
  const void* k;
  const void* v;
  void* o;
  float* lse;
  int64_t q_stride[2];
  int64_t k_stride[2];
  int64_t v_stride[2];
  int64_t o_stride[2];
  const int32_t* starts;
  const int32_t* key_starts;
  int64_t sequences;
  int64_t rows;
  int64_t key_rows;
  int64_t heads;
  int64_t kv_heads;
  int64_t head_dim;
  double sm_scale; /* 0.0 means 1/sqrt(head_dim) */
  int32_t causal;
  int32_t dtype;
} fl_packed_params;

typedef struct fl_packed_grads {
  const void* dout;
  void* dq;
  void* dk;
  void* dv;
  int64_t dout_stride[2];
  int64_t dq_stride[2];
  int64_t dk_stride[2];
  int64_t dv_stride[2];
} fl_packed_grads;

int fl_attn_packed_fwd(const fl_packed_params* p, void* stream);
int64_t fl_attn_packed_bwd_workspace_bytes(const fl_packed_params* p);
int fl_attn_packed_bwd(const fl_packed_params* p, const fl_packed_grads* d, void* workspace,
                       int64_t workspace_bytes, void* stream);

/*
 * Un-fused baseline: one work-group per query row, scores staged in LDS.
 * Any head_dim >= 1; seq limited by LDS (about 40k keys at D=64).
 * Replaces flash_attn_forward_naive's scale handling and launch
 * (csrc/kernel_naive.cu:278-320), without the reference's shared-memory
 * write-after-read race between its two block reductions (:66 vs :81-83).
 */
int fl_attn_naive_f16(const fl_attn_params* p, void* stream);

/* Detail message of the last non-OK status on the calling thread. */
const char* fl_attn_last_error(void);

/* Dispatcher introspection (no counterpart in the reference, whose dispatch
 * rule is the fixed `seq_len >= 2048` test at csrc/kernel_flash2.cu:789). */
int fl_attn_num_configs(void);
const char* fl_attn_config_name(int32_t config);
/* The id of the configuration named `name` (as fl_attn_config_name returns
 * it), or -1 if no configuration has that name.  Ids can change between
 * versions of the library; names do not, so a caller that forces a
 * configuration should look its id up by name. */
int fl_attn_config_id(const char* name);
/* Returns the public table's choice for `p`, or -1 if `p` is rejected (the
 * reason is in fl_attn_last_error()).  This is the table's rule, whose answers
 * are kept; what a call launches is fl_attn_launch_name's answer. */
int fl_attn_select_config(const fl_attn_params* p);
/* The name of the kernel that the dispatcher launches for `p` in one pass
 * (fl_attn_fwd_f16 and the *_ex entry points with config -1; dtype FL_DTYPE_*):
 * a configuration's name, or "br32_rows", the 32-row groups, which are
 * internal to the library and cannot be forced.  NULL if `p` is rejected; ""
 * if there is no row to compute and nothing is launched. */
const char* fl_attn_launch_name(const fl_attn_params_ex* p, int32_t dtype);

#ifdef __cplusplus
}
#endif

#endif /* FLASHLITE_ATTN_H */
