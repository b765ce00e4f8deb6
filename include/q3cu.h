/*
 * q3cu.h -- C ABI of the B200 (sm_100a) fused Qwen3 layer kernels.
 *
 * This library replaces the operator backend that the qwen3.c-derived engine
 * calls once per op per layer: `MetalContext::execute*` in
 * src/metal/MetalContext.h:78-87 (Metal shaders under shaders/) and the CPU
 * helpers the engine runs between those calls (`quantize`, the embedding
 * gather).  Results follow the reference CPU engine src/cpu/qwen3_original.c:
 *
 *   - Q8_0 codes and scales, and the embedding dequant, are bit-exact;
 *   - RMSNorm (also the per-head QK-norm) and SwiGLU float outputs are
 *     bit-exact for f32 inputs (sequential sum of squares; an expf that
 *     reproduces the host libm's);
 *   - RoPE and softmax outputs are within 1e-5 relative / 1e-6 absolute (f32)
 *     and 1e-2 relative (bf16 inputs).
 *
 * Conventions
 *   - Device-pointer entry points (`q3cu_<op>`) take caller-owned device
 *     memory, run asynchronously on `stream` (NULL = the legacy default
 *     stream) and allocate nothing.  Row-major, contiguous rows.
 *   - Every entry point returns a q3cu_status; none exits or throws.  The
 *     message of the last failure on the calling thread is available from
 *     q3cu_last_error_string().
 *   - Errors found on the device (an out-of-range token or page id, a wait that
 *     gave up) set bits in a per-context status word and skip the affected row;
 *     q3cu_device_status() synchronises the stream and returns and clears
 *     them.
 *   - Q8_0 tensors are two arrays, as QuantizedTensor in
 *     src/cpu/qwen3_original.c:43-46: int8 codes [rows][n] and float scales
 *     [rows][n/64].  The group size is fixed at 64; n must be a multiple of 64.
 *   - The host-pointer entry points (`q3cu_execute_*`) keep the reference's
 *     signatures and are synchronous: copy in, run, copy out (the drop-in for
 *     MetalQwen3::metal_* -> MetalContext::execute*).
 *   - One context per device per host thread; a context is not thread-safe.
 */
#ifndef Q3CU_H
#define Q3CU_H

#include <stdint.h>
#include <stddef.h>

#ifdef __cplusplus
extern "C" {
#endif

typedef enum {
    Q3CU_OK = 0,
    Q3CU_ERR_INVALID = 1,    /* bad argument: NULL pointer, negative or zero size ...   */
    Q3CU_ERR_ALIGN = 2,      /* a pointer or row is not aligned as required             */
    Q3CU_ERR_GROUP = 3,      /* a Q8_0 length is not a multiple of the group size (64)  */
    Q3CU_ERR_CUDA = 4,       /* a CUDA runtime call failed                              */
    Q3CU_ERR_INDEX = 5,      /* device status: a token or page id was out of range      */
    Q3CU_ERR_TIMEOUT = 6,    /* device status: a bounded wait gave up                   */
    Q3CU_ERR_NOT_INIT = 7,   /* NULL or destroyed context                               */
    Q3CU_ERR_OOM = 8,        /* device or host allocation failed                        */
    Q3CU_ERR_DEVICE = 9,     /* no such device, or not an sm_100 device                 */
    Q3CU_ERR_FORMAT = 10     /* checkpoint header: bad magic, version or group size     */
} q3cu_status;

typedef enum {
    Q3CU_F32 = 0,
    Q3CU_BF16 = 1,
    Q3CU_Q8_0 = 8            /* of a paged cache only (q3cu_kv_cache_q8) */
} q3cu_dtype;

/* Bits of the device status word (q3cu_device_status). */
#define Q3CU_DEV_BAD_INDEX 0x1u
#define Q3CU_DEV_TIMEOUT   0x2u

#define Q3CU_GROUP_SIZE 64

typedef struct q3cu_ctx q3cu_ctx;
typedef void *q3cu_stream;               /* a cudaStream_t */

/* Mirrors the header fields of a v1 checkpoint (`Config`,
 * src/cpu/qwen3_original.c:28-41). */
typedef struct {
    int32_t magic_number, version, dim, hidden_dim, n_layers, n_heads, n_kv_heads,
            vocab_size, seq_len, head_dim, shared_classifier, group_size;
} q3cu_config;

/* ---- lifecycle (MetalContext::initialize/cleanup/isInitialized,
 *      src/metal/MetalContext.h:40-43) ------------------------------------- */
q3cu_status q3cu_init(int device, q3cu_ctx **out);
q3cu_status q3cu_destroy(q3cu_ctx *ctx);
int         q3cu_is_initialized(const q3cu_ctx *ctx);
const char *q3cu_last_error_string(void);
const char *q3cu_status_string(q3cu_status s);
int         q3cu_version(void);
/* Synchronises `stream`, returns the device status bits in *flags and clears
 * them.  Returns Q3CU_ERR_INDEX / Q3CU_ERR_TIMEOUT when the matching bit is set. */
q3cu_status q3cu_device_status(q3cu_ctx *ctx, q3cu_stream stream, uint32_t *flags);
/* Failure-path self-test (no counterpart in the reference): enqueues one CTA
 * whose threads wait on a shared-memory barrier that nothing completes, with
 * the same bounded wait the kernels use (about 2 s).  The wait gives up, sets
 * Q3CU_DEV_TIMEOUT in the status word and the kernel returns; nothing faults
 * and the context stays usable.  For testing a caller's handling of a
 * device-side timeout (read it with q3cu_device_status). */
q3cu_status q3cu_selftest_wait_timeout(q3cu_ctx *ctx, q3cu_stream stream);

/* Validates a checkpoint header (src/cpu/qwen3_original.c:236-244 exits on a bad
 * magic or version; this returns Q3CU_ERR_FORMAT instead). */
q3cu_status q3cu_check_header(const void *header, size_t bytes, q3cu_config *out);

/* ---- device-pointer ops ------------------------------------------------- */

/* RMSNorm of each row (src/cpu/qwen3_original.c:278-289;
 * shaders/rmsnorm.metal:23-66): out = w * (ss * x), ss = 1/sqrtf(sum(x^2)/dim + eps).
 * x, out: [rows][dim] of `dtype` (out may equal x); w: [dim] f32.
 * dim * sizeof(dtype) must be a multiple of 16 and x, out 16-byte aligned. */
q3cu_status q3cu_rmsnorm(q3cu_ctx *ctx, const void *x, q3cu_dtype dtype, const float *w,
                         int64_t rows, int dim, float eps, void *out, q3cu_stream stream);

/* RMSNorm fused with the Q8_0 quantize that follows it in the forward pass
 * (qwen3_original.c:353 then :356, :439 then :443, :462 then :465): the float
 * row never leaves the chip.  q: [rows][dim] int8, s: [rows][dim/64] f32. */
q3cu_status q3cu_rmsnorm_q8(q3cu_ctx *ctx, const void *x, q3cu_dtype dtype, const float *w,
                            int64_t rows, int dim, float eps, int8_t *q, float *s,
                            q3cu_stream stream);

/* Per-head QK-RMSNorm + rotate-half RoPE, in place (qwen3_original.c:361-393;
 * MetalContext::executeRoPE, src/metal/MetalContext.cpp:826-913;
 * shaders/rope.metal:6-77).  q: [rows][n_heads][head_dim],
 * k: [rows][n_kv][head_dim] of `dtype`; pos: [rows] int32 (device);
 * q_norm, k_norm: [head_dim] f32 (device).  freq_j = powf(theta, -j/(hd/2)) is
 * evaluated on the host with the C library's powf, as the reference does.
 * head_dim must be 128. */
q3cu_status q3cu_qk_norm_rope(q3cu_ctx *ctx, void *q, void *k, q3cu_dtype dtype,
                              const int32_t *pos, int64_t rows, int n_heads, int n_kv,
                              int head_dim, const float *q_norm, const float *k_norm,
                              float theta, float eps, q3cu_stream stream);

/* SwiGLU in place: hb = hb * (hb2 * (1/(1+expf(-hb)))) (qwen3_original.c:449-450;
 * MetalContext::executeSwiGLU, src/metal/MetalContext.cpp:772-824).
 * hb, hb2: [rows][hidden] of `dtype`; hidden * sizeof(dtype) % 16 == 0. */
q3cu_status q3cu_swiglu(q3cu_ctx *ctx, void *hb, const void *hb2, q3cu_dtype dtype,
                        int64_t rows, int hidden, q3cu_stream stream);

/* SwiGLU fused with the following Q8_0 quantize (qwen3_original.c:449-453). */
q3cu_status q3cu_swiglu_q8(q3cu_ctx *ctx, const void *hb, const void *hb2, q3cu_dtype dtype,
                           int64_t rows, int hidden, int8_t *q, float *s, q3cu_stream stream);

/* In-place softmax of ragged f32 rows (qwen3_original.c:291-308, called per
 * head at :416; MetalContext::executeSoftmax, src/metal/MetalContext.cpp:633-677).
 * Row r is x[row_off[r] .. row_off[r] + row_len[r]) (device arrays).
 * The running max starts at 0, as in the reference. */
q3cu_status q3cu_softmax_rows(q3cu_ctx *ctx, float *x, const int64_t *row_off,
                              const int32_t *row_len, int64_t rows, q3cu_stream stream);

/* Q8_0 quantize of each row (qwen3_original.c:147-168; engine copy
 * src/metal/MetalQwen3.cpp:308-329; shaders/quantize.metal:18-47). */
q3cu_status q3cu_quantize_q8(q3cu_ctx *ctx, const void *x, q3cu_dtype dtype, int64_t rows,
                             int n, int8_t *q, float *s, q3cu_stream stream);

/* Q8_0 dequantize (qwen3_original.c:142-145): x = q * s[i/64].  n = element count. */
q3cu_status q3cu_dequantize_q8(q3cu_ctx *ctx, const int8_t *q, const float *s, int64_t n,
                               float *x, q3cu_stream stream);

/* Embedding lookup from a Q8_0 table (qwen3_original.c:142-145 applied at load,
 * :203-205, then the row memcpy at :342; engine src/metal/MetalQwen3.cpp:228,362-365):
 * row i of the output is table row ids[i] dequantized, optionally re-quantized
 * to Q8_0 (:147-168).  tq: [vocab][dim] int8, ts: [vocab][dim/64] f32.
 * out_f32 [n][dim] may be NULL; out_q [n][dim] and out_s [n][dim/64] may both be
 * NULL.  An out-of-range id sets Q3CU_DEV_BAD_INDEX and leaves its row untouched. */
q3cu_status q3cu_embed_gather(q3cu_ctx *ctx, const int8_t *tq, const float *ts, int vocab,
                              int dim, const int32_t *ids, int64_t n, float *out_f32,
                              int8_t *out_q, float *out_s, q3cu_stream stream);

/* Q8_0 x Q8_0 matrix products for B token rows (qwen3_original.c:310-331
 * `matmul`, applied to each row; engine src/metal/MetalQwen3.cpp:530-533,
 * shaders/quantized_matmul.metal): out[b][i] = sum over the 64-groups j of row
 * i, in order, of RN(RN((float) dot(xq[b] group j, wq[i] group j) * ws[i][j])
 * * xs[b][j]) -- the reference's bits.  xq [B][n], xs [B][n/64]; wq [d][n],
 * ws [d][n/64] (row-major [out][in]); out [B][d].  n % 64 == 0; xq and wq
 * 32-byte aligned.  W is streamed once per block of up to 4 token rows. */
q3cu_status q3cu_matmul_q8(q3cu_ctx *ctx, const int8_t *xq, const float *xs, int B,
                           const int8_t *wq, const float *ws, int n, int d, float *out,
                           q3cu_stream stream);

/* Multi-head attention of one token over positions 0..pos
 * (qwen3_original.c:395-428; MetalContext::executeAttention,
 * src/metal/MetalContext.h:86-87, shaders/attention.metal): per query head h,
 * scores q_h . k_t / sqrtf(128) in index order, the reference's softmax (max
 * from 0), then xb_h = sum over t in order of att[t] * v_t; kv head h / kv_mul.
 * Device pointers: q [n_heads][128] (after QK-norm + RoPE); key_cache,
 * value_cache [pos + 1 or more][kv_dim] (this layer's rows); att
 * [n_heads][att_stride] is scratch for the scores (att_stride > pos); probs
 * (NULL, or a different buffer of the same shape) receives the probabilities,
 * the reference's att after its softmax; xb [n_heads][128].  head_dim is 128;
 * kv_dim % 4 == 0.  Any number of positions.  Same bits as the reference. */
q3cu_status q3cu_attention(q3cu_ctx *ctx, const float *q, const float *key_cache, const float *value_cache,
                           int pos, int n_heads, int kv_dim, int kv_mul, float *att, int att_stride, float *probs,
                           float *xb, q3cu_stream stream);

/* ---- a paged key-value cache shared by many sequences ---------------------
 * No counterpart in the reference, whose cache holds one sequence
 * (qwen3_original.c:403-404).  A cache is a pool of pages; a page holds
 * page_size consecutive positions of one sequence, and a table row per
 * sequence says which page holds its positions i * page_size ... .  Three
 * operators work on one layer's cache and one description of a batch:
 * append the batch's new token rows, then attend to the cache from the rows of
 * prompts, or from one new token per sequence. */
typedef struct {
    void *k, *v;             /* pages of [n_kv][page_size][head_dim], 16-byte aligned (device) */
    int64_t page_stride;     /* elements between the starts of two pages, of k and of v: at least
                                n_kv * page_size * head_dim, and a multiple of 8 */
    int32_t n_pages, n_kv;
    int32_t page_size;       /* 16, 32, 64, 128 or 256 */
    int32_t head_dim;        /* 128 */
    int32_t dtype;           /* q3cu_dtype of k and v */
} q3cu_kv_cache;

/* A cache of Q8_0 values: `codes` has dtype Q3CU_Q8_0, its k and v are pages of
 * int8 codes, its page_stride is a multiple of 16; every 64 codes of a row have
 * a scale beside them.  A position and kv head take 136 bytes of k and of v, where bf16
 * takes 256.  The calls below take it as &cache.codes: a q3cu_kv_cache of dtype
 * Q3CU_Q8_0 is always the first member of one of these.  A scale that is
 * infinite or NaN makes NaN of what it multiplies. */
typedef struct {
    q3cu_kv_cache codes;
    float *k_scale, *v_scale;    /* pages of [n_kv][page_size][2], 16-byte aligned (device) */
    int64_t scale_stride;        /* floats between the starts of two pages' scales: at least n_kv * page_size * 2,
                                    and a multiple of 4 */
} q3cu_kv_cache_q8;

/* The packed token rows of n_seqs sequences.  Sequence s owns rows row_off[s]
 * .. row_off[s+1]-1, the last of which is at position kv_len[s] - 1: kv_len
 * counts the sequence's positions with the new rows.  Rows at or behind
 * row_off[n_seqs] belong to no sequence and are left as they are.  A row whose
 * position would be negative is padding: nothing is appended for it, and its
 * attention is zero.  All three arrays are device memory, read when the
 * kernels run.  pages[s][i] is the page of positions i * page_size ...;
 * entries beyond the last position are not read. */
typedef struct {
    const int32_t *row_off;  /* [n_seqs + 1], rising from 0 to no more than the call's rows (not read by
                                q3cu_attention_paged) */
    const int32_t *kv_len;   /* [n_seqs] */
    const int32_t *pages;    /* [n_seqs][max_pages] */
    int32_t n_seqs;              /* at most 2^24 */
    int32_t max_pages;           /* max_pages * page_size <= 2^31 - 512 */
} q3cu_kv_batch;

/* QK-RMSNorm and rotation of the packed rows, keys and values into the cache
 * (the per-head operation of qwen3_original.c:361-393, for many rows).  q: [rows][n_heads][128] with q_stride elements
 * between rows, k and v: [rows][n_kv][128] with kv_stride, all of `dtype`
 * (one fused projection's output may hold all three).  q_norm, k_norm: [128]
 * f32, or NULL for the rotation alone.  q_out: [rows][n_heads][128] of
 * q_dtype; it may be q itself when the types agree and q_stride is
 * n_heads * 128.  n_heads 0 (q, q_out NULL) appends keys and values only.
 * The angle pos * theta^(-j/64) is formed in binary64: unlike
 * q3cu_qk_norm_rope, which keeps the reference's binary32 product, it is exact
 * at far positions.  Pointers 16-byte aligned, strides multiples of 16 bytes.
 * A page id outside the cache, or a position beyond the table, sets
 * Q3CU_DEV_BAD_INDEX and stores nothing for that row's keys and values. Two
 * rows of a call must not fall on the same page slot. */
q3cu_status q3cu_kv_append(q3cu_ctx *ctx, const q3cu_kv_cache *cache, const q3cu_kv_batch *batch, int64_t rows,
                           const void *q, const void *k, const void *v, q3cu_dtype dtype, int64_t q_stride,
                           int64_t kv_stride, int n_heads, const float *q_norm, const float *k_norm, float theta,
                           float eps, void *q_out, q3cu_dtype q_dtype, q3cu_stream stream);

/* How heads are rotated, where it is not the whole head by halves at one theta. */
typedef enum { Q3CU_ROPE_HALVES = 0, Q3CU_ROPE_PAIRS = 1 } q3cu_rope_layout;
typedef enum { Q3CU_ROPE_UNSCALED = 0, Q3CU_ROPE_LINEAR = 1, Q3CU_ROPE_YARN = 2 } q3cu_rope_scaling;
typedef struct {
    float theta;             /* pair j < dim / 2 turns by theta^(-2 j / dim) a position, before scaling */
    int32_t dim;             /* the first dim elements of a head are rotated: a multiple of 4 up to 128 */
    int32_t layout;          /* q3cu_rope_layout: pair j is elements (j, j + dim / 2), or (2 j, 2 j + 1) */
    int32_t scaling;         /* q3cu_rope_scaling: none; every frequency divided by factor; or YaRN (Peng et al., 2023):
                                pairs that turn more than beta_fast times over `original` positions keep their
                                frequency, those that turn less than beta_slow times have it divided by factor, with a
                                linear ramp over the pairs between (its ends rounded outwards to whole pairs, and cut to 0 and
                                dim - 1: where even pair 0 turns less than beta_slow times, it alone keeps its frequency) */
    float factor;            /* at least 1 (read when scaled) */
    float original;          /* positions trained on (YaRN) */
    float beta_fast, beta_slow;  /* YaRN: 32 and 1 usually */
    float gain;              /* factor of cosines and sines; 0: 1, and 0.1 ln(factor) + 1 with YaRN */
    const double *freq;      /* NULL, or [dim / 2] radians a position of each pair (host memory, read by the call), in
                                place of theta and scaling */
} q3cu_rope;

/* q3cu_kv_append with the rotation that `rope` describes (host memory).  Into a Q8_0 cache the rows are
 * quantised as they are written: the codes and scales are those that
 * q3cu_quantize_q8 makes of the f32 rows. */
q3cu_status q3cu_kv_append_rope(q3cu_ctx *ctx, const q3cu_kv_cache *cache, const q3cu_kv_batch *batch, int64_t rows,
                                const void *q, const void *k, const void *v, q3cu_dtype dtype, int64_t q_stride,
                                int64_t kv_stride, int n_heads, const float *q_norm, const float *k_norm,
                                const q3cu_rope *rope, float eps, void *q_out, q3cu_dtype q_dtype, q3cu_stream stream);

/* Reads the packed rows' keys and values back from the cache: k and v
 * [rows][n_kv][128] of `dtype` (f32 or bf16) with kv_stride elements between
 * rows.  A cache of any type; a Q8_0 code times its scale is rounded to f32, and
 * then to bf16 where that is asked for.  Padding rows, rows on a bad page or at a position beyond the
 * table (both flagged) are zeros; rows behind the last sequence are left as
 * they are.  Pointers 16-byte aligned, the stride a multiple of 16 bytes. */
q3cu_status q3cu_kv_read(q3cu_ctx *ctx, const q3cu_kv_cache *cache, const q3cu_kv_batch *batch, int64_t rows, void *k,
                         void *v, q3cu_dtype dtype, int64_t kv_stride, q3cu_stream stream);

/* Attention of one new token per sequence: row s of q ([n_seqs][n_heads][128]
 * of `dtype`, q_stride elements between rows) over positions 0..kv_len[s]-1 of
 * sequence s; query head h reads kv head h / (n_heads / n_kv), at most 16
 * query heads to a kv head.  Scores are scaled by 1/sqrt(128); the softmax is
 * the usual one (its maximum is the row's, where q3cu_softmax_rows' starts at
 * 0).  out: [n_seqs][n_heads][128] of `dtype`, other memory than q; zeros where kv_len is 0.  Any
 * mix of `dtype` and the cache's type; sums are binary32.  The caller's `work`
 * (device, 16-byte aligned, q3cu_attention_paged_workspace bytes, contents
 * irrelevant) holds partial results during the call: calls that may run at the
 * same time need one each.  What a page holds beyond a sequence's last
 * position is never used, NaN included.  A page id outside the cache sets
 * Q3CU_DEV_BAD_INDEX and reads as zeros; a kv_len beyond the table sets it and
 * is cut.  An infinite element at one of the sequence's own positions may make
 * results NaN that the formula gives another value: with a key those of its
 * heads, with a value those of its column. */
q3cu_status q3cu_attention_paged(q3cu_ctx *ctx, const q3cu_kv_cache *cache, const q3cu_kv_batch *batch,
                                 const void *q, q3cu_dtype dtype, int64_t q_stride, int n_heads, void *work,
                                 size_t work_bytes, void *out, q3cu_stream stream);
/* Bytes of `work` for the head counts, any batch. */
q3cu_status q3cu_attention_paged_workspace(q3cu_ctx *ctx, int n_heads, int n_kv, size_t *bytes);

/* Sequences that begin alike: sequences seq_off[g] .. seq_off[g+1]-1 of the
 * batch have their first len[g] positions in common, which are read from the
 * pages of the group's first sequence (the other sequences' entries for pages
 * that lie wholly before len[g] are not read).  Where that first sequence holds
 * fewer than len[g] positions, its kv_len being less, the group shares nothing,
 * and each sequence attends to the pages of its own table.  Device arrays, read when the kernels run. */
typedef struct {
    const int32_t *seq_off;  /* [n_groups + 1], rising within 0 .. n_seqs; sequences outside all groups share nothing */
    const int32_t *len;      /* [n_groups] */
    int32_t n_groups;        /* at most 2^24; may be 0 */
} q3cu_kv_prefix;

/* q3cu_attention_paged for a batch whose sequences share prefixes: the shared
 * positions are attended to once for the whole group, on the tensor cores.  The
 * result is that of q3cu_attention_paged over tables that list the first
 * sequence's pages for all of the group, but for the roundings of the shared
 * positions, which are q3cu_attention_prompt's (sums binary32).  A sequence
 * with fewer positions than are shared, or alone in its group, attends to its
 * own pages as if it were in none; a len beyond the table sets
 * Q3CU_DEV_BAD_INDEX and is cut.  A NaN or infinity at a shared position, where
 * the formula makes an infinity of it, may make a NaN; over a Q8_0 cache, values
 * more than 2^120 times those before may take these to 0.  q and out are bf16, the
 * cache bf16 or Q8_0; work: 32-byte aligned, q3cu_attention_shared_workspace
 * bytes for the batch's n_seqs (or more), used by one call at a time.  All else
 * as above. */
q3cu_status q3cu_attention_shared(q3cu_ctx *ctx, const q3cu_kv_cache *cache, const q3cu_kv_batch *batch,
                                  const q3cu_kv_prefix *prefix, const void *q, q3cu_dtype dtype, int64_t q_stride,
                                  int n_heads, void *work, size_t work_bytes, void *out, q3cu_stream stream);
/* Bytes of `work` for at most n_seqs sequences and the head counts. */
q3cu_status q3cu_attention_shared_workspace(q3cu_ctx *ctx, int n_seqs, int n_heads, int n_kv, size_t *bytes);

/* Causal attention of packed prompt rows over the cache, which holds their
 * keys and values already (q3cu_kv_append): a row at position p over positions
 * 0..p.  A whole prompt has kv_len equal to its rows; a chunk behind a cached
 * prefix has more.  q: [rows][n_heads][128] with q_stride elements between
 * rows; out: [rows][n_heads][128], other memory than q.  Both of the cache's
 * type, or bf16 over a Q8_0 cache: bf16 runs on the tensor cores with
 * probabilities rounded to bf16 (the sums binary32); over a Q8_0 cache they are
 * rounded to f16 instead, by 2^-11 of themselves or 2^-32 (2^-24 where a value
 * is smaller than those at positions before), and so are keys and
 * values, by 2^-10 of themselves or 2^-39 of the largest of 128 positions (so a
 * score moves by up to 2^-10 sum |q_i k_i| / sqrt(128), and a weight by that share
 * of itself: scores of several hundred give other weights than
 * q3cu_attention_paged, which takes the codes exactly); f32
 * runs with binary32's accuracy (elements below 2^-109 keep fewer bits).
 * Grouped heads, scale, softmax, empty rows, unused page space, bad
 * pages and alignment as above.  A NaN or infinity at a position changes no row
 * before it; where one would, the row is computed again by itself, at some 0.2 us
 * a key (a bf16 prompt does so for a second at most in one tile of rows; what is
 * left then stays NaN and Q3CU_DEV_TIMEOUT is set).  Over a Q8_0 cache that is
 * also done for a row behind which, among the 128 positions from a multiple of
 * 128 on where its last one lies, a scale is more than 2^24 times the largest
 * that it sees of them, and for one that sees values more than 2^120 times those
 * before; what is left there keeps a result of fewer bits.  Sequences with one row are
 * allowed, but q3cu_attention_paged is made for them. */
q3cu_status q3cu_attention_prompt(q3cu_ctx *ctx, const q3cu_kv_cache *cache, const q3cu_kv_batch *batch,
                                  int64_t rows, const void *q, q3cu_dtype dtype, int64_t q_stride, int n_heads,
                                  void *out, q3cu_stream stream);

/* ---- a checkpoint on the device and its decode step --------------------- */
typedef struct q3cu_model q3cu_model;

/* Loads a checkpoint image -- the file's bytes: 256-byte header, fp32 norms,
 * Q8_0 tensors (qwen3_original.c:185-248 read_checkpoint/memory_map_weights,
 * written by scripts/export.py:108-170) -- into device memory on ctx's device,
 * with a zeroed KV cache of seq_len positions (ctx_length > 0 caps seq_len as
 * :240-241 does).  The token table stays Q8_0: rows are dequantized on lookup
 * instead of keeping the reference's fp32 copy (:203-205).  head_dim must be
 * 128.  One device allocation, made here; a short image is Q3CU_ERR_FORMAT. */
q3cu_status q3cu_model_load(q3cu_ctx *ctx, const void *checkpoint, size_t bytes, int ctx_length,
                            q3cu_model **out);
q3cu_status q3cu_model_config(const q3cu_model *m, q3cu_config *out);
/* One decode step, `forward(token, pos)` (qwen3_original.c:333-468; the
 * library entry qwen3_forward, :1062): the token at `pos` attends to the KV
 * rows 0..pos written by earlier calls.  The logits [vocab] stay on the device
 * (q3cu_model_logits); with logits_host set they are also copied there and the
 * call synchronises `stream`.  Same bits as the reference.  Allocates nothing;
 * an out-of-range token or pos is Q3CU_ERR_INDEX. */
q3cu_status q3cu_model_forward(q3cu_model *m, int token, int pos, float *logits_host,
                               q3cu_stream stream);
const float *q3cu_model_logits(const q3cu_model *m);
q3cu_status q3cu_model_destroy(q3cu_model *m);

/* ---- host-pointer drop-in (synchronous), MetalContext signatures -------- */

/* MetalContext::executeRMSNorm (src/metal/MetalContext.h:79). */
q3cu_status q3cu_execute_rmsnorm(q3cu_ctx *ctx, float *output, const float *input,
                                 const float *weight, int size);
/* MetalContext::executeSoftmax (src/metal/MetalContext.h:80). */
q3cu_status q3cu_execute_softmax(q3cu_ctx *ctx, float *x, int size);
/* MetalContext::executeSwiGLU (src/metal/MetalContext.h:83). */
q3cu_status q3cu_execute_swiglu(q3cu_ctx *ctx, float *hb, const float *hb2, int hidden_dim);
/* MetalContext::executeRoPE (src/metal/MetalContext.h:84-85): QK-norm + RoPE
 * of one token's n_heads query heads and n_kv_heads key heads at `pos`. */
q3cu_status q3cu_execute_rope(q3cu_ctx *ctx, float *q, float *k, int head_dim, int pos,
                              int n_heads, int n_kv_heads, const float *q_norm_weights,
                              const float *k_norm_weights);
/* MetalContext::executeAttention (src/metal/MetalContext.h:86-87; called from
 * MetalQwen3::metal_attention, src/metal/MetalQwen3.cpp:639): one token's
 * attention over the layer's cache rows 0..pos at key_cache + loff and
 * value_cache + loff (row stride kv_dim), host pointers.  Writes xb
 * [n_heads][head_dim] and, as the reference's CPU loop does, the probabilities
 * into att [n_heads][seq_len] (columns 0..pos).  head_dim must be 128. */
q3cu_status q3cu_execute_attention(q3cu_ctx *ctx, float *xb, const float *q, float *att, float *key_cache,
                                   float *value_cache, int pos, int head_dim, int n_heads, int n_kv_heads,
                                   int seq_len, int kv_dim, uint64_t loff, int kv_mul);
/* The engine's CPU quantize (src/metal/MetalQwen3.cpp:308-329). */
q3cu_status q3cu_execute_quantize(q3cu_ctx *ctx, int8_t *q, float *s, const float *x, int n);
/* MetalContext::executeQuantizedMatMul (src/metal/MetalContext.h:81-82): one
 * token, W (d,n) @ x (n,) -> output (d,), all host pointers (copied in per
 * call, as the Metal path does).  group_size must be 64. */
q3cu_status q3cu_execute_quantized_matmul(q3cu_ctx *ctx, float *output, const int8_t *x_q,
                                          const float *x_s, const int8_t *w_q, const float *w_s,
                                          int n, int d, int group_size);
/* The engine's embedding row copy (src/metal/MetalQwen3.cpp:228) from a Q8_0
 * table row instead of a dequantized fp32 table. */
q3cu_status q3cu_execute_embedding(q3cu_ctx *ctx, float *out, const int8_t *q, const float *s,
                                   int token, int dim);

/* ---- allocation-free executeRMSNorm ----------------------------------------
 * No counterpart in the reference.  Same result as q3cu_execute_rmsnorm, for
 * callers that must not allocate device memory when they normalise a row: it
 * takes no context and stages x, w and the output in a fixed array inside the
 * library's device image (Q3CU_STATIC_SCRATCH_BYTES per device) instead of a
 * cudaMalloc'd buffer.  Synchronous on `stream` (NULL: the legacy default
 * stream) of the current device.
 *   - size must be 1..Q3CU_STATIC_RMSNORM_MAX; larger sizes return
 *     Q3CU_ERR_INVALID and touch nothing.
 *   - The first call on a device looks up the array's address (and loads the
 *     library's device code if that has not happened yet); make one call per
 *     device before any stream capture.
 *   - There is one array per device: calls that overlap on the same device
 *     (several host threads or streams) race and must be serialised by the
 *     caller. */
#define Q3CU_STATIC_RMSNORM_MAX 16384
#define Q3CU_STATIC_SCRATCH_BYTES (256 + 3 * 4 * Q3CU_STATIC_RMSNORM_MAX)
q3cu_status q3cu_execute_rmsnorm_static(float *output, const float *input, const float *weight,
                                        int size, q3cu_stream stream);

#ifdef __cplusplus
}
#endif
#endif /* Q3CU_H */
