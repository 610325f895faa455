/*
 * streaming_attention.h -- C ABI of the B200 (sm_100a) streaming Taylor-moment
 * + block-coreset causal attention library (libsa_b200.so).
 *
 * Every entry point takes raw pointers and sizes, enqueues its work on the
 * given CUDA stream (a cudaStream_t passed as void*, NULL = legacy default
 * stream) of the current device, and returns an int status (SA_OK == 0,
 * negative on error).  Nothing throws across this boundary.  After an error,
 * sa_last_error() returns a message for the calling thread.
 *
 * Tensor layouts (all contiguous, row-major, fp32 unless noted):
 *   q, k  [bh, n, d]      v, out  [bh, n, dv]
 *   bh = B*H sequences ("heads"); each is processed independently.
 *
 * Coreset draw tables (host-generated, copied to the device; see
 * streaming_attention_b200/draws.py).  nc = completed blocks per head =
 * (n - 1) / block_size, m = (block_size + 1) / 2 reps per completed block:
 *   dirs  [bh, nc, d]              fp32, unit projection direction per block
 *   coins [bh, nc, block_size/2]   fp32 uniform draws in [0,1) per pair
 *   perms [bh, nc, m]              int32 block-local indices (random
 *                                  compressor, and sorted_pair when
 *                                  block_size <= 2)
 *
 * Reference interfaces replaced (PositiveLoss/streaming-attention):
 *   sa_fast_attention      fast_article_causal_attention
 *                          (fast_article_attention.py:634-719) and its
 *                          per-sequence body (:522-631)
 *   sa_compress_blocks     _build_completed_block_reps (:364-434) +
 *                          _compress_one_completed_block (:312-361)
 *   sa_low_moments         low_degree_taylor_causal_sums (:262-285) and the
 *                          moment sketch (streaming_taylor_coreset_attention.py:229-296)
 *   sa_residual_combine    _block_coreset_residual_tail (:467-514),
 *                          _full_residual_tail (:437-464) and the final
 *                          num / clamp(den, eps) (:596-598)
 *   sa_feature_count       num_taylor_features (:137-148) /
 *                          SymmetricTaylorFeatureMap.total_features
 *                          (streaming_taylor_coreset_attention.py:180-182)
 */
#ifndef STREAMING_ATTENTION_H_
#define STREAMING_ATTENTION_H_

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* status codes */
#define SA_OK 0
#define SA_ERR_INVALID_ARG (-1)   /* bad shape / size / pointer; ValueError */
#define SA_ERR_UNSUPPORTED (-2)   /* degree or dims beyond the kernels; NotImplementedError */
#define SA_ERR_CUDA (-3)          /* CUDA launch or runtime error; RuntimeError */
#define SA_ERR_TIMEOUT (-4)       /* a bounded device-side wait gave up */
#define SA_ERR_WORKSPACE (-5)     /* workspace smaller than sa_*_workspace_size */
#define SA_ERR_DEVICE_CHECK (-6)  /* a device-side index check failed (libsa_b200_checks.so only) */

/* compressor kinds (fast_article_attention.py:326, :332, :383) */
#define SA_COMPRESSOR_NONE 0
#define SA_COMPRESSOR_SORTED_PAIR 1
#define SA_COMPRESSOR_RANDOM 2

/* largest supported Taylor degree and feature count */
#define SA_MAX_DEGREE 3
#define SA_MAX_DIM 256
#define SA_MAX_VALUE_DIM 256

/* Library version, e.g. 100 for 0.1.0. */
int sa_version(void);

/* Message of the last error on this thread ("" if none). */
const char* sa_last_error(void);

/* Feature count sum_{l<=degree} C(dim+l-1, l). */
int sa_feature_count(int dim, int degree, int64_t* count);

/* Number of completed blocks that a later query reads: (n-1)/block_size
 * (fast_article_attention.py:403-407).  *reps_per_block = (block_size+1)/2,
 * or block_size for compressor none. */
int sa_block_counts(int64_t n, int block_size, int compressor, int64_t* completed_blocks,
                    int64_t* reps_per_block);

/* C1: compress every completed block of every head.
 * Outputs: rep_idx [bh, nc*m] int32 (global token index within the head, the
 * bit-exact selection), rep_k [bh, nc*m, d], rep_v [bh, nc*m, dv],
 * rep_w [bh, nc*m].  Any of rep_k / rep_v / rep_w may be NULL. */
int sa_compress_blocks(const float* k, const float* v, int64_t bh, int64_t n, int d, int dv,
                       int block_size, int compressor, const float* dirs, const float* coins,
                       const int32_t* perms, int32_t* rep_idx, float* rep_k, float* rep_v,
                       float* rep_w, void* stream);

/* Low-degree Taylor term of every query, with the moment state taken over the
 * completed blocks before the query's own block:
 *   low[i, :dv] = sum_{j < bstart(i)} P_t(scale q_i.k_j) v_j,
 *   low[i, dv]  = sum_{j < bstart(i)} P_t(scale q_i.k_j),
 * where bstart(i) = (i / block_size) * block_size.  low is [bh, n, dv+1].
 * When the tensor-core kernel applies (dv <= 64) it needs a caller workspace
 * of sa_low_moments_workspace_size bytes (256-byte aligned); otherwise the
 * workspace may be NULL. */
int sa_low_moments_workspace_size(int64_t bh, int64_t n, int d, int dv, int degree, int block_size,
                                  size_t* bytes);
int sa_low_moments(const float* q, const float* k, const float* v, int64_t bh, int64_t n, int d,
                   int dv, int degree, int block_size, float scale, float* low, void* workspace,
                   size_t workspace_bytes, void* stream);

/* Residual over the completed-block reps + exact current block, added to the
 * low term, then out = num / max(den, eps).  rep_k/rep_v/rep_w are the
 * outputs of sa_compress_blocks ([bh, nc*m, *]); for compressor none they are
 * ignored (every earlier key is a rep of weight 1).  For d <= 64 and
 * dv <= 128 the tensor-core kernel runs and needs a caller workspace of
 * sa_residual_combine_workspace_size bytes (256-byte aligned); otherwise the
 * workspace may be NULL. */
int sa_residual_combine_workspace_size(int64_t bh, int64_t n, int d, int dv, int block_size,
                                       int compressor, size_t* bytes);
int sa_residual_combine(const float* q, const float* k, const float* v, const float* rep_k,
                        const float* rep_v, const float* rep_w, const float* low, int64_t bh,
                        int64_t n, int d, int dv, int degree, int block_size, int compressor,
                        float scale, float eps, float* out, void* workspace,
                        size_t workspace_bytes, void* stream);

/* Bytes of device workspace sa_fast_attention needs. */
int sa_fast_attention_workspace_size(int64_t bh, int64_t n, int d, int dv, int degree,
                                     int block_size, int compressor, size_t* bytes);

/* The whole forward of fast_article_causal_attention for bh sequences.
 * rep_idx (nullable) receives the coreset selection [bh, nc*m].  workspace is
 * caller-owned device memory of at least sa_fast_attention_workspace_size
 * bytes, 256-byte aligned.  The call is ordered on `stream` like one kernel:
 * with a compressor and the tensor-core kernels, its moment scan runs on a
 * second stream of the device's highest priority (made, with two events, at
 * the first such call per host thread and caller stream -- at most 16 per
 * thread -- and kept until the process ends) that forks from and joins back
 * into `stream`; under graph capture, while stage events are set, or with
 * sa_set_moment_fork(0), everything runs on `stream` itself. */
int sa_fast_attention(const float* q, const float* k, const float* v, int64_t bh, int64_t n, int d,
                      int dv, int degree, int block_size, float scale, int compressor,
                      const float* dirs, const float* coins, const int32_t* perms, float eps,
                      float* out, int32_t* rep_idx, void* workspace, size_t workspace_bytes,
                      void* stream);

/* ---- run-time controls and status (no counterpart in the reference) -------
 * The reference runs eagerly on one device and has neither device-side waits
 * nor a status word; these entry points belong to this library's own runtime. */

/* The launch status word that sa_fast_attention, sa_low_moments,
 * sa_residual_combine, sa_article_segment_mean, sa_flash_causal_attention and
 * the shard calls keep in the first 4 bytes of their workspace: synchronises
 * `stream`, then returns SA_OK when no bounded device-side wait of the last
 * call on that workspace gave up, else SA_ERR_TIMEOUT (sa_last_error() names
 * the kernel's wait code), or SA_ERR_DEVICE_CHECK in a checks build. */
int sa_workspace_status(const void* workspace, void* stream);

/* Whether sa_fast_attention may fork its moment scan onto a second stream
 * (see sa_fast_attention), for the calling host thread: 1 (the default) lets
 * it, 0 runs every stage in order on the caller's stream.  Callers that
 * already overlap several forwards on streams of their own (this library's
 * host-tensor path does, for its chunks) gain nothing from the fork: a later
 * forward's moment scan, at the higher priority, then delays the earlier
 * forward's residual.  sa_moment_fork_enabled returns the current setting. */
int sa_set_moment_fork(int enable);
int sa_moment_fork_enabled(void);

/* 1 in libsa_b200_checks.so, the build with device-side index checks
 * (-DSA_DEVICE_CHECKS: a check that fails records its code, 900..999, in the
 * status word and the offending index 8 bytes after it, and skips the access;
 * sa_workspace_status then returns SA_ERR_DEVICE_CHECK), 0 in libsa_b200.so. */
int sa_device_checks_enabled(void);

/* How long one bounded device-side wait of the tensor-core kernels may take
 * before its CTA gives up, drains what it issued, records SA_ERR_TIMEOUT's
 * cause in the status word and leaves (the process-wide default, 0, means
 * 2 s).  Applies to launches made after the call, from any thread. */
int sa_set_wait_limit_ns(uint64_t limit_ns);

/* Measurement hook for the calling host thread: while `count` > 0,
 * sa_fast_attention records events[i] (cudaEvent_t handles, created by the
 * caller) on its stream at stage boundaries: 0 start, 1 after the k / v
 * operand splits, 2 after the compressor (and the split of its reps), 3 after
 * the moment scan, 4 after the residual (the end); the stages then run one
 * after another on that stream.  count = 0 turns it off. */
int sa_set_stage_events(void* const* events, int count);

/* ---- streaming (decode) state: ArticleStreamingAttention -------------------
 * The reference keeps, per attention stream, a Taylor moment sketch and a
 * merge-and-reduce coreset (streaming_taylor_coreset_attention.py:229-616).
 * Here that state lives in caller-owned device buffers: num [F, dv] and den [F]
 * (fp32, F = sa_feature_count(d, degree)), a pending block of raw keys /
 * values, and the level items (keys [m, d], values [m, dv], weights [m]).
 * The caller keeps the level structure and draws the compressor's random
 * numbers (as the streaming class in streaming_attention_b200/streaming.py does). */

/* Replaces TaylorMomentSketch.update (streaming_taylor_coreset_attention.py:262-279):
 * num[f, :] += (weight * phi_k(key)[f]) * value, den[f] += weight * phi_k(key)[f],
 * product then add, each rounded to fp32, as the reference does. */
int sa_stream_update(const float* key, const float* value, int d, int dv, int degree, float weight,
                     float* num_state, float* den_state, void* stream);

/* Replaces MergeReduceCoreset._compress (streaming_taylor_coreset_attention.py:414-470)
 * for one block of n >= 2 weighted items: sorted_pair (direction [d], coins
 * [n/2]; n <= 2 uses perm) or random (perm [ceil(n/2)] of the first draws of
 * randperm(n)).  Writes ceil(n/2) items; outputs must not overlap inputs. */
int sa_stream_compress(const float* keys, const float* values, const float* weights, int64_t n, int d,
                       int dv, int compressor, const float* direction, const float* coins,
                       const int32_t* perm, float* out_keys, float* out_values, float* out_weights,
                       void* stream);

/* Bytes of device workspace sa_stream_query needs. */
int sa_stream_query_workspace_size(int d, int dv, int degree, size_t* bytes);

/* Replaces ArticleStreamingAttention.query (streaming_taylor_coreset_attention.py:572-606):
 * out [dv] = (phi_q(scale q).[num, den] + sum over the pending block (weight 1)
 * and the level items of w (exp(x) - P_t(x)) [v, 1]) / max(den, eps), with
 * x = scale * (k . q).  dens (nullable) receives {den, low den, tail den}. */
int sa_stream_query(const float* query, int d, int dv, int degree, float scale, const float* num_state,
                    const float* den_state, const float* buf_keys, const float* buf_values, int64_t n_buf,
                    const float* lvl_keys, const float* lvl_values, const float* lvl_weights,
                    int64_t n_lvl, float eps, float* out, float* dens, void* workspace,
                    size_t workspace_bytes, void* stream);

/* ---- one shard of a long sequence split along N over GPUs ------------------
 * The reference has no multi-GPU path; these split one forward of
 * fast_article_causal_attention (fast_article_attention.py:634-719) over P
 * ranks that each hold a contiguous token range of every sequence (a whole
 * number of blocks).  Rank r: sa_shard_begin (local compression with the
 * global block ids, local moment scan, its moment state T_r), then the caller
 * all-gathers the states and reps, then sa_shard_end (exclusive prefix of the
 * earlier states, their contribution to the shard's queries, the residual
 * over the reps of every earlier block).  Needs the tensor-core kernels. */

/* Floats of one shard's moment state (the unit of the all-gather). */
int sa_shard_state_floats(int64_t bh, int d, int dv, int degree, int64_t* floats);

/* Bytes of workspace for both calls of a shard of n tokens whose residual reads
 * rep_rows reps per sequence (the reps of the blocks before the shard's last). */
int sa_shard_workspace_size(int64_t bh, int64_t n, int d, int dv, int degree, int block_size,
                            int64_t rep_rows, size_t* bytes);

/* Local part.  dirs/coins/perms hold the draws of the shard's n_compress
 * blocks (global blocks c_off .. c_off+n_compress-1 of the sequence);
 * rep_k/rep_v/rep_w [bh, n_compress*m, *] receive the raw reps, rep_idx
 * (nullable) their global token indices; state_out receives T_r. */
int sa_shard_begin(const float* q, const float* k, const float* v, int64_t bh, int64_t n, int d, int dv,
                   int degree, int block_size, float scale, int compressor, const float* dirs,
                   const float* coins, const int32_t* perms, int64_t n_compress, int64_t c_off,
                   float* state_out, float* rep_k, float* rep_v, float* rep_w, int32_t* rep_idx,
                   void* workspace, size_t workspace_bytes, void* stream);

/* Global part, after the exchange.  states_before: the n_before states of the
 * earlier shards, contiguous in shard order; rep_k/rep_v/rep_w [bh, rep_rows,
 * *]: the reps of global blocks 0.. in order (for compressor none: every
 * earlier token, weight 1).  Same workspace as sa_shard_begin. */
int sa_shard_end(const float* q, const float* k, const float* v, int64_t bh, int64_t n, int d, int dv,
                 int degree, int block_size, float scale, int compressor, float eps,
                 const float* states_before, int n_before, int64_t c_off, const float* rep_k,
                 const float* rep_v, const float* rep_w, int64_t rep_rows, float* out, void* workspace,
                 size_t workspace_bytes, void* stream);

/* Bytes of the library's built-in device scratch (per GPU). */
#define SA_STATIC_SCRATCH_BYTES (64u * 1024u * 1024u)

/* sa_fast_attention for callers that cannot allocate device memory.  It has
 * no counterpart in the reference; it exists for callers such as programs
 * whose device memory belongs entirely to another allocator, serving loops
 * that forbid cudaMalloc after start-up, or plain-C callers with no device
 * allocator.  Same arguments and result as sa_fast_attention, minus the
 * workspace: the scratch is a SA_STATIC_SCRATCH_BYTES array built into the
 * library, held by every GPU that loads it until the process exits.  Problems
 * whose sa_fast_attention_workspace_size exceeds it are rejected with
 * SA_ERR_INVALID_ARG.  The first call on each device loads the library's
 * device code there (make it before any stream capture); every call looks up
 * the array's address anew, so a device reset that moves it is harmless.  All
 * calls share the array: calls that overlap on the GPU race, so order them.
 * Allocates nothing. */
int sa_fast_attention_static_scratch(const float* q, const float* k, const float* v, int64_t bh,
                                     int64_t n, int d, int dv, int degree, int block_size,
                                     float scale, int compressor, const float* dirs,
                                     const float* coins, const int32_t* perms, float eps,
                                     float* out, int32_t* rep_idx, void* stream);

/* ---- the segment-mean variant (deterministic reps) -------------------------
 * Replaces triton_article_causal_attention (triton_article_attention.py:448-578)
 * and its kernel _article_direct_kernel (:266-370): the same low-degree
 * moments and exact current-block residual as sa_fast_attention, but each
 * completed block is represented by the means of its block_size/compress_stride
 * runs of compress_stride adjacent tokens, each of weight compress_stride, and
 * the exp of a score is taken of min(score, 80) (:331-333, :359).  degree 0, 1
 * or 2 (else SA_ERR_UNSUPPORTED); block_size % compress_stride != 0 is
 * SA_ERR_INVALID_ARG.  d <= 128 and dv <= 128.  key_dtype / value_dtype say
 * how the reference's reps were stored (the dtypes of its k and v, SA_REP_*):
 * the key and value means are rounded to them. */
#define SA_REP_FLOAT32 0
#define SA_REP_FLOAT16 1
#define SA_REP_BFLOAT16 2

/* Replaces build_segment_mean_coreset (triton_article_attention.py:190-245):
 * rep_k [bh, R, d], rep_v [bh, R, dv], R = (n-1)/block_size *
 * (block_size/compress_stride) (0 rows when n <= block_size). */
int sa_segment_mean_reps(const float* k, const float* v, int64_t bh, int64_t n, int d, int dv,
                         int block_size, int compress_stride, int key_dtype, int value_dtype,
                         float* rep_k, float* rep_v, void* stream);

/* Bytes of device workspace sa_article_segment_mean needs. */
int sa_article_segment_mean_workspace_size(int64_t bh, int64_t n, int d, int dv, int degree,
                                           int block_size, int compress_stride, size_t* bytes);

/* The whole forward of the segment-mean variant for bh sequences. */
int sa_article_segment_mean(const float* q, const float* k, const float* v, int64_t bh, int64_t n,
                            int d, int dv, int degree, int block_size, int compress_stride,
                            float scale, int key_dtype, int value_dtype, float eps, float* out,
                            void* workspace,
                            size_t workspace_bytes, void* stream);

/* ---- exact causal softmax attention ----------------------------------------
 * Replaces triton_flash_causal_attention (triton_article_attention.py:580-637)
 * and its kernel _flash_causal_kernel (:372-435): out = softmax(scale q k^T,
 * causal) v with the running-maximum (online) softmax and
 * out = acc / max(l, 1e-20).  d <= 128, dv <= 256 (else SA_ERR_INVALID_ARG).
 * Tensor cores (3xTF32) for d <= 64 and dv <= 128 with a workspace of
 * sa_flash_causal_attention_workspace_size bytes (256-byte aligned); CUDA
 * cores otherwise (workspace size 0, may be NULL). */
int sa_flash_causal_attention_workspace_size(int64_t bh, int64_t n, int d, int dv, size_t* bytes);
int sa_flash_causal_attention(const float* q, const float* k, const float* v, int64_t bh, int64_t n,
                              int d, int dv, float scale, float* out, void* workspace,
                              size_t workspace_bytes, void* stream);

/* ---- serving: windowed attention, a paged 4-bit cache, page plans, norm + rotation ----
 * No counterpart in the reference.  dtype is an SA_REP_* code, of every tensor
 * of elements in the call; strides are in elements and the last dimension is
 * contiguous.  The kernels check the contents of device-side index arrays
 * (offsets, slots, page tables, lengths): what is out of range is skipped and
 * recorded in the device's error word, which sa_serving_status reads.  No call
 * allocates; all may be captured into a graph. */

/* Synchronises `stream`, then returns SA_OK, or what the serving calls on this
 * device recorded first since the last read (SA_ERR_INVALID_ARG for bad index
 * contents, SA_ERR_TIMEOUT for a bounded wait that gave up) and clears it. */
int sa_serving_status(void* stream);

/* Attention with a sliding window and first tokens that stay visible:
 *   out_i = softmax over visible j of (scale q_i.k_j), times v_j,
 *   visible: j <= p and (j > p - window or j < sinks), p = m - n + i;
 * window 0 means no end.  A query that sees nothing gives zeros.  Query head h
 * reads key head h / (heads / kv_heads).
 * Dense (cu_q == cu_k == NULL): q [batch, heads, n, d], k [batch, kv_heads, m,
 * d], v [.., m, dv], out like q with dv; strides = {q_b, q_h, q_n, k_b, k_h,
 * k_n, v_b, v_h, v_n, o_b, o_h, o_n}.  Packed: cu_q, cu_k [batch + 1] are the
 * requests' first rows in q / out (n rows in all) and k / v (m rows in all),
 * p counts within the request, the *_b strides are 0; a request whose offsets
 * are out of order or range is reported and skipped.  Rows of no request, those
 * between a skipped one's offsets too, stay as they were or are zeroed
 * (zero_behind != 0).  d, dv <= 256.
 * Tensor cores: float16 / bfloat16 of d, dv <= 128 on 16-byte borders; dense
 * contiguous float32 (3xTF32) of d <= 64, dv <= 128 and long enough given a workspace of
 * sa_window_attention_workspace_size bytes (256-byte aligned; 0: none is used).
 * CUDA cores otherwise.  The 16-bit form does without a workspace, but uses one of
 * that size (packed: that of a dense call of batch 1 with as many queries and keys
 * as k has rows) to split few queries' many keys over the SMs, and to fold the sums
 * over more than 32768 keys, which the matrix units would pull towards zero. */
int sa_window_attention_workspace_size(int batch, int heads, int kv_heads, int64_t n, int64_t m, int d, int dv,
                                       int64_t window, int64_t sinks, int dtype, size_t* bytes);
int sa_window_attention(const void* q, const void* k, const void* v, void* out, const int64_t* strides, int batch,
                        int heads, int kv_heads, int64_t n, int64_t m, int d, int dv, int64_t window, int64_t sinks,
                        float scale, int dtype, const int32_t* cu_q, const int32_t* cu_k, int zero_behind, void* workspace,
                        size_t workspace_bytes, void* stream);

/* The cache: pages of page_size (16, 32, 64, 128 or 256) tokens; dp = d filled
 * up to 32, 64, 128 or 256 (d <= 256); byte b of a row holds column 2 b in its
 * low and 2 b + 1 in its high half:
 *   k_codes  uint8 [pages, heads, page_size, dp / 2]
 *   v_codes  uint8 [pages, heads, page_size / 4, dp / 2, 4]   (last: the token within four)
 *   k_params, v_params  bfloat16 [pages, heads, page_size, 2]: scale, least value
 * all contiguous and 16-byte aligned.  A row x is held as least = bf16(min x),
 * scale = bf16((max x - min x) / 15), code = clamp(rint((x - least) / scale), 0,
 * 15), and stands for scale * code + least; a row that holds NaN, an infinity
 * or a least value that bfloat16 cannot hold stands for NaN.
 * Slot = page * page_size + token within the page; negative: none. */

/* Quantises k, v [tokens, heads, d] (strides {k_t, k_h, v_t, v_h}) into their
 * slots [tokens]; each slot at most once per call. */
int sa_kv4_append(void* k_codes, void* k_params, void* v_codes, void* v_params, int64_t pages, int heads,
                  int page_size, int d, const void* k, const void* v, const int64_t* strides, const int32_t* slots,
                  int64_t tokens, int dtype, void* stream);

/* The values that the slots hold, k, v [tokens, heads, d] contiguous; zeros
 * for a negative slot. */
int sa_kv4_read(const void* k_codes, const void* k_params, const void* v_codes, const void* v_params, int64_t pages,
                int heads, int page_size, int d, void* k, void* v, const int32_t* slots, int64_t tokens, int dtype,
                void* stream);

/* Attention of each request's n newest tokens over the cache: q [requests, n,
 * heads, d] (strides {q_r, q_n, q_h}), out contiguous; request r holds
 * lengths[r] tokens (the new ones among them) in pages tables[r, 0..] (width
 * entries a row), query i stands at lengths[r] - n + i, visible as in
 * sa_window_attention.  Tokens behind a bad page id count as hidden. */
int sa_kv4_attend(const void* k_codes, const void* k_params, const void* v_codes, const void* v_params, int64_t pages,
                  int kv_heads, int page_size, int d, const void* q, void* out, const int64_t* strides,
                  const int32_t* tables, const int32_t* lengths, int requests, int n, int heads, int width,
                  int64_t window, int64_t sinks, float scale, int dtype, void* stream);

/* Room for fresh[r] (>= 0) new tokens of each of `requests` requests (at most
 * 16384): pages are taken in request order from the end of the free_count[0]
 * entries of free_pages and entered in tables [requests, width] (in place;
 * entries of pages held before stay).  lengths_out = lengths + fresh; offsets
 * [requests + 1] is the running sum of fresh; positions / slots [max_tokens]
 * give each packed new token's position in its request and its slot, -1 behind
 * the last token and where there is no page (per_request > 0: token i of
 * request r stands at r * per_request + i instead, max_tokens is requests *
 * per_request, and -1 fills the rows of requests with fewer new tokens); free_out[0] is what is left.
 * New tokens beyond the rows are reported; they count, and their pages are entered.
 * Page ids are below free_size.  No output overlaps an input. */
int sa_plan_kv_pages(const int32_t* lengths, const int32_t* fresh, int32_t* tables, const int32_t* free_pages,
                     const int32_t* free_count, int requests, int width, int free_size, int page_size, int max_tokens,
                     int per_request, int32_t* lengths_out, int32_t* offsets, int32_t* positions, int32_t* slots, int32_t* free_out,
                     void* stream);

/* sa_plan_kv_pages for packed prompts, whose tokens see one another and nothing
 * that their requests hold: new tokens of a request of lengths[r] > 0 are reported. */
int sa_plan_kv_prompts(const int32_t* lengths, const int32_t* fresh, int32_t* tables, const int32_t* free_pages,
                       const int32_t* free_count, int requests, int width, int free_size, int page_size, int max_tokens,
                       int32_t* lengths_out, int32_t* offsets, int32_t* positions, int32_t* slots, int32_t* free_out,
                       void* stream);

/* Returns the pages of the requests with drop[r] != 0 to the free list and
 * empties those requests (all in place). */
int sa_release_kv_pages(int32_t* lengths, int32_t* tables, const uint8_t* drop, int32_t* free_pages,
                        int32_t* free_count, int requests, int width, int free_size, int page_size, void* stream);

/* Root-mean-square norm of each head's row and its rotation by the token's
 * position, one pass: y = x / sqrt(mean(x^2) + eps) * weight (NULL: ones);
 * (y_a, y_b) -> (y_a cos - y_b sin, y_b cos + y_a sin) with angle
 * positions[t] * frequencies[i] (float64 [half]) and (a, b) = (i, i + half) or,
 * interleaved, (2 i, 2 i + 1).  q [tokens, heads, d], k [tokens, kv_heads, d];
 * strides = {q_t, q_h, k_t, k_h, qo_t, qo_h, ko_t, ko_h}; out may be the input
 * itself.  A token of negative position is left out: its output rows are zeroed
 * (zero_skipped != 0) or stay as they were.  d <= 256. */
int sa_qk_norm_rotary(const void* q, const void* k, void* q_out, void* k_out, const int32_t* positions,
                      const void* q_weight, const void* k_weight, const double* frequencies, const int64_t* strides,
                      int64_t tokens, int heads, int kv_heads, int d, int half, float eps, int interleaved,
                      int zero_skipped, int dtype, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* STREAMING_ATTENTION_H_ */
