/* C ABI of libtts_hip.so: the MI355X execution backend behind triton-shared's
 * plugin surface.  Plain pointers and sizes only; no Python, torch or C++ types.
 *
 * Every entry point returns a tts_status.  On a non-zero status
 * tts_last_error() (thread-local) holds a message.  Strings returned through
 * `char **out` are malloc'd by the library and released with tts_free().
 *
 * Each declaration cites the reference interface it replaces (paths relative to
 * the triton-shared source tree).
 */
#ifndef TTS_HIP_H
#define TTS_HIP_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

typedef enum tts_status {
  TTS_OK = 0,
  TTS_UNSUPPORTED = 1, /* the kernel is outside what this backend implements (NotImplementedError) */
  TTS_INVALID = 2,     /* malformed input or bad argument (ValueError / TypeError) */
  TTS_HIP_ERROR = 3    /* a HIP runtime call failed (RuntimeError) */
} tts_status;

/* One kernel argument, in the order of the tt.func signature (constexpr
 * parameters are not arguments).  Replaces the per-argument C parameters of the
 * generated kernel symbol, backend/driver.py:96-100,109-114: a pointer was
 * "int64_t rank, void *descriptor", a scalar was passed by value. */
typedef enum tts_arg_kind { TTS_ARG_PTR = 0, TTS_ARG_INT = 1, TTS_ARG_FLOAT = 2 } tts_arg_kind;
typedef struct tts_arg {
  int32_t kind; /* tts_arg_kind */
  int32_t reserved;
  union {
    void *ptr;  /* device pointer (may be NULL if the kernel never dereferences it) */
    int64_t i;  /* i1/i8/i16/i32/i64 and unsigned scalars, sign- or zero-extended */
    double f;   /* fp32/fp64 scalars */
  } v;
} tts_arg;

typedef struct tts_plan tts_plan;

/* TTIR text -> structured program text.
 * Replaces the `triton-shared-opt --triton-to-linalg-experimental` subprocess of
 * backend/compiler.py:48-67 (pipeline: lib/Conversion/TritonToLinalgExperimental/
 * TritonToLinalgExperimentalPass.cpp:52-88). */
tts_status tts_ttir_to_structured(const char *ttir_text, char **out);

/* Structured program text -> launch plan bytes (kernel family + bindings).
 * Replaces _ttsharedir_to_llir + _llir_to_bin, backend/compiler.py:75-175.
 * *out_name receives the kernel name (metadata["name"], compiler.py:133-136). */
tts_status tts_structured_to_plan(const char *structured_text, char **out_plan, size_t *out_len, char **out_name);

void tts_free(void *p);
const char *tts_last_error(void);

/* Plan bytes -> handle.  Replaces CPUUtils.load_binary, backend/driver.py:409-417
 * (there the "function" is the object file itself). */
tts_status tts_plan_load(const char *plan_bytes, size_t len, tts_plan **out);
void tts_plan_destroy(tts_plan *plan);
const char *tts_plan_kernel_name(const tts_plan *plan);
const char *tts_plan_family(const tts_plan *plan);   /* map1d, row_softmax, layernorm_fwd, gemm, gemm_w8a16 */
const char *tts_plan_signature(const tts_plan *plan); /* normalised op listing the family was recognised from */
int tts_plan_num_args(const tts_plan *plan);
/* kind of argument i: TTS_ARG_PTR / TTS_ARG_INT / TTS_ARG_FLOAT */
int tts_plan_arg_kind(const tts_plan *plan, int i);

/* Resolves the plan's bindings for one launch configuration without touching
 * the GPU and describes the kernel launch that tts_launch would issue, as
 * "key=value" lines.  Used by host-side tests; no counterpart in the reference. */
tts_status tts_plan_describe_launch(tts_plan *plan, int grid_x, int grid_y, int grid_z, const tts_arg *args,
                                    int num_args, char **out);

/* Enqueues the whole grid on `stream` (a hipStream_t; NULL = the null stream)
 * and returns without waiting.  Replaces _launch, backend/driver.py:116-133 (the
 * serial x/y/z loop over programs) together with the compiled kernel it calls.
 * A grid with zero volume is a no-op (driver.py:117). */
tts_status tts_launch(tts_plan *plan, int grid_x, int grid_y, int grid_z, void *stream, const tts_arg *args,
                      int num_args);

/* tts_launch for callers that cannot allocate device memory (code under HIP graph capture, tight serving loops,
 * harnesses that forbid hipMalloc).  No counterpart in the reference.  Same arguments and results as tts_launch, but
 * the call never allocates or frees device memory and never compiles: the split-K partial tiles and arrival counters
 * of the int8-weight product, and the partial sums of a matrix product that runs in K slices, live in a static device
 * array (8 MiB + 4096 counters per GPU, held until the process ends; its address is looked up with
 * hipGetSymbolAddress at the first call on each device).  A launch of the int8-weight product's decode kernels whose
 * partial tiles exceed that (the tiled kernel for more rows runs without slices instead), or
 * a launch that would need a run-time compiled kernel or a device-side table that no earlier tts_launch of the plan
 * has created yet, returns TTS_UNSUPPORTED with the reason; a matrix product runs in as many slices as fit there, or
 * without slices.  All calls on one GPU share the array:
 * calls that overlap in time on one GPU (two streams, two threads) race on it. */
tts_status tts_launch_noalloc(tts_plan *plan, int grid_x, int grid_y, int grid_z, void *stream, const tts_arg *args,
                              int num_args);

/* Name of the device kernel the last tts_launch on this plan used (for profiles). */
const char *tts_plan_last_kernel(const tts_plan *plan);
/* Into how many slices (workgroups per program or tile) the last tts_launch on this plan dealt a program's loop, or the K of a
 * product; 1: none.  *meet (may be NULL): 1 if the slices met in that kernel, 0 if a second kernel added them.  For tests.  (Of the
 * int8-weight product tts_plan_describe_launch tells.) */
int tts_plan_last_slices(const tts_plan *plan, int *meet);

/* ---- Operators whose weights are picked per row of activations: what a decode step does beside its shared projections.  No
 * counterpart in the reference.  They are calls of their own, without a Triton program or a plan; otherwise they behave as
 * tts_launch: asynchronous on `stream`, whose device has to be the current one, tensors borrowed until the stream has passed the call, nothing
 * compiled.  They allocate nothing (and so may be captured into a graph): scratch memory is the caller's, of the size that the
 * ..._workspace function of the same arguments says, 256-byte aligned, and free for other use once the stream has passed the call;
 * calls that may overlap in time need one each.  Every argument is checked on the host before anything is launched; what memory
 * holds (ids) is checked on the device.  Results do not depend on the order in which workgroups run.  A call for zero tokens does nothing. */

typedef enum tts_dtype { TTS_F32 = 0, TTS_F16 = 1, TTS_BF16 = 2, TTS_I8 = 3, TTS_I32 = 4 } tts_dtype;
/* A tensor in device memory; strides in elements, entries past `rank` are not read. */
typedef struct tts_tensor {
  void *ptr;
  int32_t dtype; /* tts_dtype */
  int32_t rank;
  int64_t shape[3];
  int64_t stride[3];
} tts_tensor;

typedef enum tts_scoring { TTS_SOFTMAX = 0, TTS_SIGMOID = 1 } tts_scoring;
typedef enum tts_activation { TTS_SILU = 0, TTS_GELU_TANH = 1, TTS_RELU = 2 } tts_activation;

/* The router of a mixture-of-experts layer.  logits [T, E] (f32, f16, bf16; E <= 1024), bias [E] f32 or NULL, ids [T, k] i32 and
 * weights [T, k] f32 (k <= 64) written; rows any distance apart, elements of a row neighbours.  With s = softmax or sigmoid of a
 * row's logits, ids are the k experts of the largest s + bias (without a bias: of the largest logits, which is the same order where
 * neither score has run into 0 or 1), in descending order, ties to the lowest expert, and weights are scale * s, divided by
 * the sum of the chosen s if `renormalize`: as the formula says also where all chosen s are too small for 32 bits, but 0 where s is
 * under e^-745 (a mask of the type's lowest value).  Logits of -inf are not chosen, nor is an s + bias that is
 * -inf or NaN; where fewer than k are left, ids are -1 and weights 0.  A row that holds a NaN has weights of NaN,
 * and so has the softmax of one that holds +inf (its ids are those of the limit of ever larger logits). */
tts_status tts_moe_route(const tts_tensor *logits, const tts_tensor *bias, int scoring, int renormalize, double scale,
                         const tts_tensor *ids, const tts_tensor *weights, void *stream);

/* The experts of a mixture-of-experts layer for a few tokens (T * k <= 4096):
 *   out[t] = sum over j of weights[t, j] * (h Wd[e]),  h = f(x[t] Wg[e]) * (x[t] Wu[e]),  e = ids[t, j],
 * x [T, H] f16 or bf16, ids [T, k] i32, weights [T, k] f32, w_up [E, H, 2 I] with Wg its first I columns and Wu the others, w_down
 * [E, I, O], out [T, O] of x's type (it may be x: all of x is read before any of out is written).  Not `gated`: w_up [E, H, I], h = f(x[t] W[e]).
 * Weights are of x's type, or i8 with s_up [E, 2 I] and s_down [E, O] f32 that multiply their columns (NULL otherwise); each matrix
 * has stride 1 along its inputs or along its outputs.  H, I, O >= 8, of i8 weights >= 16.  An id outside [0, E) contributes nothing; the same id
 * twice in a row contributes twice.  Sums, h and the weighted parts are held in 32 bits. */
tts_status tts_moe_experts_workspace(const tts_tensor *x, const tts_tensor *ids, const tts_tensor *w_up, const tts_tensor *w_down, int gated,
                                     size_t *bytes);
tts_status tts_moe_experts(const tts_tensor *x, const tts_tensor *ids, const tts_tensor *weights, const tts_tensor *w_up, const tts_tensor *s_up,
                           const tts_tensor *w_down, const tts_tensor *s_down, int activation, int gated, const tts_tensor *out,
                           void *workspace, size_t bytes, void *stream);

/* Low-rank adapters of many requests:
 *   out[t] = base[t] + scales[d] * (x[t] a[d]^T) b[d]^T,  d = ids[t];  out[t] = base[t], bit for bit, where d is not in [0, n).
 * base and out [T, N], x [T, K], a [n, r, K], b [n, N, r], all f16 or all bf16, the last dimension with stride 1; ids [T] i32, scales [n]
 * f32 or NULL (1); r <= 1024, T <= 2097120.  out may be base itself; otherwise it shares no memory with the inputs.  One request's adapter
 * (an infinity in it, say) does not reach another's rows.  Rows of one adapter next to each other read it once per 16 rows; in calls of more
 * than 1024 rows, a once per 64 and b once per 32. */
tts_status tts_lora_add_workspace(const tts_tensor *x, const tts_tensor *b, size_t *bytes);
tts_status tts_lora_add(const tts_tensor *base, const tts_tensor *x, const tts_tensor *a, const tts_tensor *b, const tts_tensor *ids,
                        const tts_tensor *scales, const tts_tensor *out, void *workspace, size_t bytes, void *stream);

/* ---- The attention part of a decode step over a cache held in 4 bits: page_slots -> qk_norm_rope -> kv4_write -> kv4_attention.  No counterpart in
 * the reference.  They behave as the operators above: asynchronous on `stream`, nothing allocated or compiled, scratch memory from the caller, arguments
 * checked on the host, what memory holds (lengths, pages, slots, positions) on the device.  Vectors have stride 1; the last dimension of what is a matrix or more has, too.
 * A step has T rows, the new tokens of one request after another; rows behind the last request's (a batch padded to what a graph was captured for) have no request. */

/* Block tables and slot maps.  table [B, M] i32: the pages of each request, in order; lengths [B] i32: the tokens that it has after this step, fresh [B]
 * i32: how many of them are new, its last ones (held between 0 and its length); free [F] i32: a stack of free pages, of which the first count[0] are on it, the last of them the
 * top.  B <= 4096.  Requests take the pages that they lack (to ceil(length / page), at most M) from the top of the stack, the first request first, each in the order of its
 * columns; those are written into the table, and nothing else of it; where the stack has run out, -1.  Written besides: slots [T] i32, table[b][position / page] * page + position %
 * page of each row, or -1 where there is no such page; positions [T]; owners [T], the row's request; -1 in all three for rows of no request; starts [B + 1], where the
 * requests' rows begin, and their end; left [1], how many pages are on the stack now.  If the requests have more than T rows, those behind have no slots here.  What is
 * written shares no memory with what is read. */
tts_status tts_page_slots(const tts_tensor *table, const tts_tensor *lengths, const tts_tensor *fresh, const tts_tensor *free, const tts_tensor *count, int page,
                          const tts_tensor *slots, const tts_tensor *positions, const tts_tensor *owners, const tts_tensor *starts, const tts_tensor *left, void *stream);

/* Norms of queries and keys for each head, and the rotation by position.  q [T, Hq, D], k [T, Hk, D] (f32, f16, bf16; D even, <= 512), tokens and heads any distance
 * apart (columns of one projection's rows, say).  Of each head y = x / sqrt(mean(x^2) + eps) * w, w_q and w_k [D] of q's type or f32 (both NULL: y = x); then of its first R
 * elements pairs (a, b) become (a cos - b sin, b cos + a sin): pair n is elements n and n + R / 2, or 2 n and 2 n + 1 if `interleaved`; cos_sin [P, R] f32 holds the cosines of a
 * position's R / 2 angles, then their sines; positions [T] i32.  Nothing of a row whose position is not in [0, P) is written, or zeros if `clear`.
 * Sums and products in 32 bits, rounded once.  q_out may be q itself and k_out k; otherwise what is written shares no memory with what is read. */
tts_status tts_qk_norm_rope(const tts_tensor *q, const tts_tensor *k, const tts_tensor *positions, const tts_tensor *cos_sin, const tts_tensor *w_q, const tts_tensor *w_k,
                            double eps, int interleaved, int clear, const tts_tensor *q_out, const tts_tensor *k_out, void *stream);

/* The cache [pages, Hk, page * (D + 8) / 2], f16 or bf16: for each page and head the keys and values of `page` tokens (a multiple of 16), of each element 4
 * bits and of each token's key and value a step and a lowest value of the cache's type; pages * page <= 2^31 - 1.  D is a multiple of 32 up to 256.  The last dimension has stride 1,
 * pages and heads are multiples of 16 bytes apart (8 elements).  Its inner layout is the library's own.
 * An element x of a head with lowest value l and largest h is held as c * s + l, s = (h - l) / 15 in 32 bits rounded to the type, c = how many of the borders
 * (n + 1/2) s, n = 0 .. 14, x - l is above.  A head that holds a NaN or an infinity, or whose h - l is not finite in 32 bits, is held as NaN.
 * write: k, v [T, Hk, D] of the cache's type into slots [T] i32 (page * tokens of a page + place in it); a row whose slot is not in the cache is not written.  The slots in
 * the cache are distinct: of two rows with the same one, parts of either are there afterwards.
 * read: what the slots hold, code * step + lowest rounded to the type; zeros for a slot that is not in the cache. */
tts_status tts_kv4_write(const tts_tensor *cache, const tts_tensor *k, const tts_tensor *v, const tts_tensor *slots, void *stream);
tts_status tts_kv4_read(const tts_tensor *cache, const tts_tensor *slots, const tts_tensor *k, const tts_tensor *v, void *stream);

/* Attention over the cache.  q [T, Hq, D], out the same (it may be q), Hq a multiple of Hk: head h reads the cache's head h / (Hq / Hk).  Rows starts[b] .. starts[b + 1] - 1 of q
 * are the last tokens of request b, which has lengths[b] tokens in the cache, in the pages table[b] (M columns, places for less than 2^30 tokens; starts [B + 1], lengths [B], table
 * [B, M] i32); the one at position i sees tokens j <= i, with a window (not 0) i - window < j, whose page is in the table and in [0, pages).  Where starts[B] is past T, the rows that
 * there are have the positions that page_slots gives them.
 *   out = sum over j of e^(z_j) v_j / sum of e^(z_j),  z_j = scale * q . k_j;  zeros for a row that sees none; rows of no request (before starts[0], behind starts[B])
 * are not written, or zeros if `clear`.
 * A row sees nothing of what others see alone: a NaN in a token's key or value reaches the rows that see it, and the largest values of tokens that it does not see leave it as it is.  Scores, sums and statistics are held in 32 bits, e^z times a
 * value's step in fp16 (2^-11 of it; of an fp16 cache as the sum of two of them, 2^-22), but for 2^-34 of the largest step so far among the tokens that it sees, q as it is but for
 * 2^-34 of its largest element, or 2^-147.   A row whose largest element times the scale is not finite in 32 bits may be NaN.
 * longest: no request has more tokens than that (0: as many as the table has places for); the number of workgroups follows it, and results do not depend on it but for the order of sums.  */
tts_status tts_kv4_attention_workspace(const tts_tensor *q, const tts_tensor *cache, const tts_tensor *table, int window, int64_t longest, size_t *bytes);
tts_status tts_kv4_attention(const tts_tensor *q, const tts_tensor *cache, const tts_tensor *table, const tts_tensor *lengths, const tts_tensor *starts, double scale, int window,
                             int64_t longest, int clear, const tts_tensor *out, void *workspace, size_t bytes, void *stream);

#ifdef __cplusplus
}
#endif
#endif /* TTS_HIP_H */
