/*
 * tricast_b200.h — C ABI of the B200 (sm_100a) backend for TriCast's emulation hot path.
 *
 * The library replaces TriCast's Triton backend module by module. Every entry point takes plain
 * device pointers, sizes and small POD descriptors; the caller (PyTorch in the Python shim, or any
 * C/ctypes caller) owns every buffer. Entry points are asynchronous on the given stream, never
 * allocate device memory except where a comment says so, and return a tc_status; the message of
 * the last failure on the calling host thread is available from tc_last_error().
 *
 * Reference interfaces each entry point replaces (paths inside the TriCast checkout):
 *   tc_cast              <- round_to_format_triton   src/tricast/kernels/quantize.py:161-178
 *                           (semantics: src/tricast/reference/cast.py:18-83)
 *   tc_quantize          <- quantize_triton          src/tricast/kernels/quantize.py:192-275
 *                           (semantics: src/tricast/reference/quantize.py:244-350)
 *   tc_gemm              <- gemm_triton              src/tricast/kernels/mma.py:821-886
 *                           (semantics: src/tricast/reference/mma.py:339-384)
 *   tc_error_stats       <- analysis._ErrorStats.update  src/tricast/analysis.py:37-50
 */
#ifndef TRICAST_B200_H
#define TRICAST_B200_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* Same type as cudaStream_t; 0 is the legacy default stream. */
typedef struct CUstream_st *tc_stream;

typedef enum tc_status {
  TC_OK = 0,
  TC_INVALID_ARGUMENT = 1,  /* bad shape, pointer, descriptor or size limit */
  TC_UNSUPPORTED = 2,       /* a valid TriCast spec this build does not implement */
  TC_CUDA_ERROR = 3,        /* a CUDA launch or runtime call failed */
  TC_WORKSPACE_TOO_SMALL = 4,
  TC_NONFINITE = 5          /* int_exact saw a NaN/Inf operand (reported by tc_gemm_check) */
} tc_status;

/* Container dtypes of values, inputs and outputs. */
typedef enum tc_dtype { TC_F32 = 0, TC_BF16 = 1, TC_F16 = 2 } tc_dtype;

/* Rounding codes (src/tricast/rounding.py:39). */
typedef enum tc_rounding { TC_RNE = 0, TC_RNA = 1, TC_RTZ = 2, TC_RUP = 3, TC_RDN = 4, TC_SR = 5 } tc_rounding;

/* A TriCast number format (src/tricast/formats.py:29-201): primary fields only; the library
 * derives emin/emax/max_normal itself. kind: 0 float (ExMy), 1 int (fixed point), 2 pow2 (E8M0).
 * special (floats): 0 ieee, 1 fn, 2 fnuz, 3 none. */
typedef struct tc_format {
  int32_t kind;
  int32_t ebits;       /* float, pow2 */
  int32_t mbits;       /* float */
  int32_t bias;        /* float, pow2 */
  int32_t special;     /* float */
  int32_t is_signed;   /* float, int */
  int32_t subnormals;  /* float */
  int32_t bits;        /* int */
  int32_t symmetric;   /* int */
  int32_t frac_bits;   /* int */
} tc_format;

/* QuantSpec (src/tricast/quant/spec.py:167-234). granularity: 0 tensor, 1 row, 2 group, 3 block.
 * scale_method: 0 absmax, 1 pow2_floor, 2 pow2_ceil, 3 mse, 4 percentile. zero_point: 0 none,
 * 1 int, 2 float. mse_search holds the MSE candidate ratios (already rounded to fp32) on the host. */
typedef struct tc_quant_spec {
  tc_format format;
  int32_t granularity;
  int32_t group_size;
  int32_t block_rows;
  int32_t block_cols;
  int32_t has_scale;
  tc_format scale_format;
  int32_t scale_method;
  int32_t scale_rounding;
  int32_t two_level;
  int32_t zero_point;
  int32_t rounding;
  int32_t sr_bits;
  int32_t saturate;
  float percentile;
  int32_t n_search;
  const float *mse_search;
} tc_quant_spec;

/* Outputs of tc_quantize. values (container dtype) and, when the spec has them, scale /
 * zero_point (scale layout, fp32) and global_scale (one fp32) are required; the rest are optional
 * extras written in the same pass (NULL to skip):
 *   codes       element codes: 4-bit formats two per byte (low nibble = even element), else one byte
 *   scale_codes scale-format codes, one byte per scale (E8M0: exponent + 127)
 *   dequant     fp32 dequantized values ((v - z) * s [+ z]) * d2, TriCast's QTensor.dequantize order */
typedef struct tc_quant_out {
  void *values;
  int32_t values_dtype;
  float *scale;
  float *zero_point;
  float *global_scale;
  uint8_t *codes;
  uint8_t *scale_codes;
  float *dequant;
} tc_quant_out;

/* One MMA operand (src/tricast/mma/operand.py:28-57): values [rows, K] row-major and contiguous.
 * scale_kind: 0 none, 1 tensor (scalar), 2 row ([rows]), 3 k ([rows, ceil(K / k_domain)]).
 * scale_fmt is used for scale_kind 3 only (has_scale_fmt 0 means fp32). alpha: device scalar or NULL. */
typedef struct tc_operand {
  const void *values;
  int32_t values_dtype;
  int64_t rows;
  int64_t K;
  tc_format fmt;
  const float *scale;
  int32_t scale_kind;
  int32_t has_scale_fmt;
  tc_format scale_fmt;
  int32_t k_domain;
  const float *alpha;
} tc_operand;

/* MMASpec (src/tricast/mma/spec.py:223-270) with scale_apply already resolved (TriCast's
 * resolve_scale_apply, src/tricast/reference/mma.py:184-202): 0 epilogue, 1 product, 2 group,
 * 3 promote, 4 operand. algorithm: 0 cofda, 1 gdfs, 2 fp32_fma, 3 fp64, 4 int_exact.
 * c_mode: 0 fused, 1 decoupled. norm_rounding: 0 rtz, 1 rne. out_dtype: container of out_format. */
typedef struct tc_mma_spec {
  int32_t algorithm;
  int32_t f_bits;
  int32_t chunk_size;
  int32_t c_mode;
  int32_t f2_bits;
  int32_t g_bits;
  int32_t group_size;
  int32_t k_tile;
  int32_t norm_rounding;
  int32_t scale_apply;
  int32_t promote_interval;
  tc_format out_format;
  int32_t out_dtype;
} tc_mma_spec;

/* Cast n fp32 values onto fmt's grid (TriCast round_to_format). noise: NULL or n uint32 values
 * (stochastic rounding). y may alias x. */
int tc_cast(const float *x, float *y, const uint32_t *noise, int64_t n, const tc_format *fmt,
            int32_t rounding, int32_t saturate, int32_t sr_bits, tc_stream stream);

/* Bytes of scratch tc_quantize needs for this shape and spec (0 when none). */
size_t tc_quantize_workspace(int64_t rows, int64_t K, const tc_quant_spec *spec);

/* Quantize x [rows, K] (x_dtype: TC_F32 / TC_BF16 / TC_F16) under spec, writing out. amax: NULL,
 * or a device fp32 scalar: for tensor granularity it overrides the tensor amax (TriCast's
 * quantize(amax=...)); for a two-level spec of finer granularity (NVFP4) it is the tensor amax the
 * global scale d2 is derived from, so that a shard of a larger tensor quantizes exactly as the same
 * rows of the whole tensor would (an extension: TriCast accepts amax for tensor granularity only);
 * other specs reject it. noise: NULL or rows*K uint32; scale_noise: NULL or one uint32 per scale. */
int tc_quantize(const void *x, int32_t x_dtype, int64_t rows, int64_t K, const tc_quant_spec *spec,
                const float *amax, const uint32_t *noise, const uint32_t *scale_noise,
                const tc_quant_out *out, void *workspace, size_t workspace_bytes, tc_stream stream);

/* The amax of x (n elements of x_dtype) as the bits of the fp32 |x| maximum, NaN-propagating (NaN
 * bits sort above Inf's), max-reduced into *bits (device uint32, cleared by the caller). A rank
 * holding a row shard of a tensor reduces its shard's bits with the other ranks' (integer max) and
 * passes the result, viewed as fp32, as tc_quantize's amax of a two-level spec. No counterpart in
 * TriCast, whose tensors are never sharded. */
int tc_tensor_amax_bits(const void *x, int32_t x_dtype, int64_t n, uint32_t *bits, tc_stream stream);

/* Bytes of scratch tc_gemm needs for these operands and spec. */
size_t tc_gemm_workspace(const tc_operand *a, const tc_operand *b, const tc_mma_spec *spec);

/* out [a.rows, b.rows] (spec.out_dtype) = a @ b^T under spec's accumulation rule, bias ([b.rows]
 * fp32) optional. Validation of TriCast's int64 headroom rules is the caller's (the Python shim
 * does it with TriCast's messages); this call checks pointers, shapes and size limits. */
int tc_gemm(const tc_operand *a, const tc_operand *b, const tc_mma_spec *spec, const float *bias, void *out,
            void *workspace, size_t workspace_bytes, tc_stream stream);

/* Pre-encoded B operands (weights). TriCast keeps a weight operand's packed K-major copy between
 * calls (src/tricast/mma/operand.py:66-75, nn/linear.py:216-224); these keep the fast path's own
 * encoding of B instead, so repeated GEMMs against one weight skip re-encoding it.
 * tc_encode_b_bytes: bytes of B's encoding for GEMMs of A operands like a (same format and scale
 * layout, and a row count on the same side of 16: more than 16 rows take the tiled kernels, at most
 * 16 the small-M ones) under spec; 0 when that path takes no pre-encoded B (the tiled GDFS-FP4 path
 * and the small-M CoFDA path take one). a's values are not read.
 * tc_encode_b: writes it into enc (device memory the caller owns, at least that many bytes); B's
 * values and scales are read, asynchronously on stream. A B the fast path cannot take is recorded in
 * the encoding and sends every GEMM on it to the exact kernel, as tc_gemm does.
 * tc_gemm_encoded: tc_gemm with B given by its encoding (b still describes B: shape, format, scales
 * for the exact kernel); workspace as tc_gemm_workspace(a, b, spec). The encoding must come from
 * tc_encode_b for this b, spec and an A like a; an encoding of another size is rejected with
 * TC_INVALID_ARGUMENT. */
size_t tc_encode_b_bytes(const tc_operand *a, const tc_operand *b, const tc_mma_spec *spec);
int tc_encode_b(const tc_operand *a, const tc_operand *b, const tc_mma_spec *spec, void *enc, size_t enc_bytes,
                tc_stream stream);
int tc_gemm_encoded(const tc_operand *a, const tc_operand *b, const void *b_enc, size_t b_enc_bytes,
                    const tc_mma_spec *spec, const float *bias, void *out, void *workspace, size_t workspace_bytes,
                    tc_stream stream);

/* tc_gemm for callers that cannot allocate device memory. No counterpart in TriCast: this entry point
 * exists for hosts that reach the library through a bare C FFI without a CUDA allocator of their own,
 * or that reserve all device memory up front, and so cannot hand tc_gemm a workspace. Same
 * arguments and result as tc_gemm minus the workspace; the scratch comes from a fixed 32 MiB array
 * inside the library (held on every GPU that loads the library, until exit). Operands whose
 * tc_gemm_workspace() exceeds 32 MiB are rejected with TC_INVALID_ARGUMENT. The first call on a
 * device looks up that array's device address, so make it before any stream capture. The array used is
 * the current device's: call with the device of out (and of stream) current; an out on another
 * device is rejected with TC_INVALID_ARGUMENT. All calls share the array: calls whose GPU work can
 * overlap race and must not be issued. Allocates nothing. */
int tc_gemm_noalloc(const tc_operand *a, const tc_operand *b, const tc_mma_spec *spec, const float *bias,
                    void *out, tc_stream stream);

/* Device-side check used before int_exact: writes 1 to *flag (device int32) when any value of the
 * operand is NaN/Inf, else leaves it unchanged. */
int tc_any_nonfinite(const void *values, int32_t dtype, int64_t n, int32_t *flag, tc_stream stream);

/* fp64 error sums of ref vs emu (n elements each, dtypes as tc_dtype) added into sums[6] on the
 * device: {sum x^2, sum y^2, sum (x-y)^2, sum x*y, max |x-y|, count of non-finite elements}. */
int tc_error_stats(const void *ref, int32_t ref_dtype, const void *emu, int32_t emu_dtype, int64_t n,
                   double *sums, tc_stream stream);

/* Message of the last failed call on this host thread ("" if none). */
const char *tc_last_error(void);

/* Number of kernels this library has launched in the process (all threads, all devices). */
uint64_t tc_launch_count(void);

/* How many times, on the current device, the exact generic GEMM kernel queued behind a fast kernel
 * has actually run (the fast kernel declined the operands or one of its waits ran out). Waits for the
 * device. */
int tc_exact_fallbacks(uint64_t *count);

/* Of those runs, how many followed a fast kernel whose bounded wait ran out (it set its status word,
 * drained its own copies and MMAs, freed its TMEM and returned). Waits for the device. No counterpart
 * in TriCast, whose Triton kernels have no bounded waits. */
int tc_wait_timeouts(uint64_t *count);

/* How many (output, K tile) steps of the tensor-core GDFS-FP4 kernel, on the current device, failed
 * the single-pass bounds and ran the exact two-pass step instead (exact either way; this counts how
 * often the slow step runs). Waits for the device. No counterpart in TriCast. */
int tc_exact_tile_steps(uint64_t *count);

/* Poll limit of the pipeline waits (on shared-memory barriers) of the staged GEMM kernels launched
 * from now on, process-wide; polls < 0 restores the defaults (about 2**16 suspended or 2**22 plain
 * polls, seconds). With polls = 0 every such wait gives up at once: the kernel takes its timeout path
 * and the exact kernel queued behind it recomputes the product, so results stay exact. The waits that
 * drain a kernel's own copies and MMAs before it exits keep the default limit. No counterpart in
 * TriCast: it exists to test the timeout path without hanging or faulting a GPU. */
int tc_set_wait_limit(int32_t polls);

/* Silicon probe, not part of the emulation API: out[M][N] = sum_k A[m][k] * B[n][k] computed by the
 * B200's own FP8 tensor-core MMA (tcgen05.mma kind::f8f6f4, fp32 accumulator, K issued 32 at a time
 * in order, no scales). a [M][K] and b [N][K] are row-major 8-bit codes, fmt 0 = E4M3, 1 = E5M2;
 * out is fp32 [M][N]. *status (device) is set non-zero if a wait inside the kernel ran out. Used to
 * test whether an emulated accumulation model reproduces the hardware; no reference interface. */
int tc_probe_mma_fp8(const uint8_t *a, const uint8_t *b, int64_t M, int64_t N, int64_t K, int32_t fmt, float *out,
                     int32_t *status, tc_stream stream);

/* Silicon probe, block-scaled FP4: out[M][N] = sum_k A[m][k] sA[m][k / V] * B[n][k] sB[n][k / V] by the
 * tensor core's tcgen05.mma kind::mxf4nvf4 (fp32 accumulator, K issued 64 at a time in order).
 * a [M][K/2] and b [N][K/2] are packed E2M1 codes (element 2i in the low nibble, 16-byte aligned);
 * sfa [M][K/V] and sfb [N][K/V] are scale bytes: scale_fmt 0 = UE4M3 with V = 16 (NVFP4),
 * 1 = E8M0 with V = 32 (MXFP4). K must be a multiple of 64. *status as for tc_probe_mma_fp8. */
int tc_probe_mma_fp4(const uint8_t *a, const uint8_t *b, const uint8_t *sfa, const uint8_t *sfb, int64_t M, int64_t N,
                     int64_t K, int32_t scale_fmt, float *out, int32_t *status, tc_stream stream);

/* ---- Serving operators: entry points without a TriCast counterpart ---- */

/* Root-mean-square norm with the residual's addition and an 8-bit output with scales: h = x + residual
 * (x where residual is NULL), y = h / sqrt(mean(h^2) + eps) * weight (no product where weight is NULL),
 * codes and scales as tc_quantize gives them for y in fp32. x and residual: [rows][K] of dtype with row
 * strides in elements. codes: [rows][K] bytes. scale: per row or per group of the row ([rows][groups]),
 * fp32, or one E8M0 byte each where the spec's scale format is E8M0. residual_out: NULL, or h [rows][K]
 * in dtype. spec: fp8_e4m3, fp8_e5m2 or int8 elements rounded to nearest even and saturating; row or group
 * granularity; fp32 absmax or E8M0 pow2_floor scales; anything else is TC_UNSUPPORTED. Only
 * residual_out may alias x or residual, and only in whole. */
int tc_rms_norm_quantize(const void *x, const void *residual, int32_t dtype, int64_t rows, int64_t K,
                         int64_t x_stride, int64_t residual_stride, const void *weight, int32_t weight_dtype, float eps,
                         const tc_quant_spec *spec, void *codes, void *scale, void *residual_out, tc_stream stream);

/* How a paged cache holds a key or value row (one token, one head): as it is; E4M3 or INT8 codes with one
 * fp32 absmax scale (the fp8_row / int8_row schemes of a [rows][head_dim] tensor); E2M1 codes, two a byte
 * (low nibble first), with one E8M0 scale byte per 32 elements (mxfp4). */
typedef enum tc_kv_scheme { TC_KV_NONE = 0, TC_KV_FP8_ROW = 1, TC_KV_INT8_ROW = 2, TC_KV_MXFP4 = 3 } tc_kv_scheme;

/* A paged key / value cache the caller owns: k and v hold [num_pages][kv_heads][page_size] rows of codes,
 * k_scale and v_scale the rows' scales in the same order (NULL for TC_KV_NONE). dtype is that of the keys,
 * values and queries outside the cache. page_size: a power of two in [8, 256]; head_dim: a multiple of 16
 * (TC_KV_MXFP4: 32) in [16, 256]. Slot s is token s % page_size of page s / page_size. */
typedef struct tc_kv_cache {
  void *k;
  void *v;
  void *k_scale;
  void *v_scale;
  int32_t scheme;
  int32_t dtype;
  int64_t num_pages;
  int32_t page_size;
  int32_t kv_heads;
  int32_t head_dim;
} tc_kv_cache;

/* Quantize the keys and values of `tokens` tokens ([tokens][kv_heads][head_dim] with token and head
 * strides in elements, head_dim contiguous) into their slots. Slots outside the cache (-1) are skipped;
 * the others must differ: tokens are written in no order and in pieces, so a slot that two of them name
 * may end with codes of one and scales of the other (no other slot is touched). */
int tc_kv_write(const tc_kv_cache *cache, const void *k, int64_t k_token_stride, int64_t k_head_stride, const void *v,
                int64_t v_token_stride, int64_t v_head_stride, const int64_t *slots, int64_t tokens, tc_stream stream);

/* Dequantize the tokens at `slots` into k and v, [tokens][kv_heads][head_dim] of the cache's dtype: code *
 * scale in fp32, rounded once. Slots outside the cache read as zeros. */
int tc_kv_read(const tc_kv_cache *cache, const int64_t *slots, int64_t tokens, void *k, void *v, tc_stream stream);

/* Bytes of scratch tc_paged_attention needs for these sizes (0 when none). */
size_t tc_paged_attention_workspace(const tc_kv_cache *cache, int32_t q_heads, int64_t total_q, int32_t batch,
                                    int32_t max_q_len, int32_t max_pages);

/* out = softmax(scale * q k^T) v over each sequence's cached keys and values, for the last tokens of the
 * sequence: q and out [total_q][q_heads][head_dim] of the cache's dtype (q with token and head strides in
 * elements, out contiguous), query head h reading key / value head h / (q_heads / kv_heads). cu_q
 * [batch + 1]: sequence b's new tokens are cu_q[b] .. cu_q[b + 1] - 1, of which the first max_q_len are
 * computed; NULL: one each. seq_lens [batch]: its context, the new tokens (already written) included; token i of n sits
 * at position seq_lens[b] - n + i. block_table [batch][max_pages] (row stride table_stride): the page of
 * each page_size positions; keys on a page outside the cache count as absent. causal: a token sees itself
 * and earlier positions, the last `window` of them where window > 0; otherwise the whole context. Scores,
 * softmax and sums are fp32. A row that sees no key gives zeros, and -Inf in lse (NULL, or the fp32
 * [total_q][q_heads] natural logarithms of the softmax sums), as does a token of no sequence (before
 * cu_q[0], from cu_q[batch] on) or beyond max_q_len. */
int tc_paged_attention(const tc_kv_cache *cache, const void *q, int64_t q_token_stride, int64_t q_head_stride,
                       int64_t total_q, int32_t q_heads, const int32_t *block_table, int64_t table_stride,
                       int32_t max_pages, const int32_t *seq_lens, const int32_t *cu_q, int32_t batch, int32_t max_q_len,
                       float scale, int32_t causal, int32_t window, void *out, float *lse, void *workspace,
                       size_t workspace_bytes, tc_stream stream);

/* Bytes of scratch tc_plan_pages / tc_release_pages need for this many sequences. */
size_t tc_plan_pages_workspace(int32_t batch);
size_t tc_release_pages_workspace(int32_t batch);

/* Pages and slots of a batch's new tokens. Sequence i has seq_lens[i] tokens in a paged cache and gets new_lens[i] more, the
 * batch's new tokens one after the other; those from `tokens` on are left out (the sequences they belong to get fewer), as are
 * those that would make a length of 2**31 or more. Pages of page_size (a power of two) tokens that a sequence lacks are taken
 * from the stack free_pages [num_free], whose entries from *taken on are free, in the order of sequences and positions, and
 * written into its row of block_table [batch][max_pages] (row stride table_stride); no other entry is touched. Where the stack
 * is empty the entry becomes -1, and pages beyond max_pages are not taken. Written: out_lens [batch], the lengths with the new
 * tokens; cu_q [batch + 1], where the sequences' new tokens begin; per new token ([tokens], -1 behind the last) its slot (-1
 * without a page), sequence and position; *out_taken, the stack's new top; *missing, pages that were lacking. Nothing else is
 * kept: a program copies out_lens and out_taken where its next call reads them. No output may alias an input. Lengths below 0
 * count as 0. */
int tc_plan_pages(const int32_t *seq_lens, const int32_t *new_lens, int32_t batch, int32_t *block_table, int64_t table_stride,
                  int32_t max_pages, const int32_t *free_pages, int64_t num_free, const int32_t *taken, int32_t page_size,
                  int64_t tokens, int32_t *out_lens, int32_t *cu_q, int64_t *slots, int32_t *sequence, int32_t *positions,
                  int32_t *out_taken, int32_t *missing, void *workspace, size_t workspace_bytes, tc_stream stream);

/* The pages (entries >= 0) of the sequences with ended[i] != 0 go back below the stack's top, in the order of sequences and
 * columns, and their rows of block_table become -1; *out_taken is the new top. A page must stand in one row only. */
int tc_release_pages(int32_t *block_table, int64_t table_stride, int32_t max_pages, const uint8_t *ended, int32_t batch,
                     int32_t *free_pages, int64_t num_free, const int32_t *taken, int32_t *out_taken, void *workspace,
                     size_t workspace_bytes, tc_stream stream);

/* What the x of tc_low_rank_add holds besides a tc_dtype: 8-bit codes with one fp32 scale a row. */
typedef enum tc_x_codes { TC_X_E4M3 = 3, TC_X_E5M2 = 4, TC_X_INT8 = 5 } tc_x_codes;

/* Bytes of scratch tc_low_rank_add needs for these sizes (0 when none). */
size_t tc_low_rank_add_workspace(int64_t tokens, int32_t x_kind, int32_t w_dtype, int32_t rank, int32_t y_dtype, int32_t out_dtype);

/* Low-rank adapters beside a projection: out[t] = y[t] + gain[i] * b[i] (a[i] x[t]) with i = index[t], and out[t] = y[t] where
 * i is not in [0, adapters). y [tokens][n] and x [tokens][k] have row strides in elements, out [tokens][n] has none; a
 * [adapters][rank][k] and b [adapters][n][rank] of w_dtype; gain fp32 [adapters] or NULL (1). x_kind: a tc_dtype, or a
 * tc_x_codes; x_scale: NULL, or fp32 [tokens], a factor of each row (codes need it). Sums are fp32, out is rounded once. rank
 * at most 1024. Weights of 16 bits with x of their type or 8-bit codes, y and out of their type or fp32, and ranks up to 128 go
 * through the tensor cores, everything else element by element. There a[i] x[t] enters the second product in 16-bit parts, two
 * where out has 16 bits (bf16: 2**-16 of it is left out), three where it has 32. out may not alias an input. */
int tc_low_rank_add(const void *y, int32_t y_dtype, int64_t y_stride, const void *x, int32_t x_kind, int64_t x_stride,
                    const float *x_scale, int64_t tokens, int64_t k, int64_t n, const void *a, const void *b, int32_t w_dtype,
                    int32_t adapters, int32_t rank, const float *gain, const int32_t *index, void *out, int32_t out_dtype,
                    void *workspace, size_t workspace_bytes, tc_stream stream);

/* The activation of tc_gated_quantize. */
typedef enum tc_activation { TC_SILU = 0, TC_GELU = 1, TC_GELU_TANH = 2, TC_RELU = 3 } tc_activation;

/* y = activation(gate) * up in fp32, codes and scales as tc_quantize gives them for y. INT8: every step of the formula is
 * rounded by itself; else the logistic function and the normal distribution are good to some 16 halves of an fp32 step, and a
 * scale or code follows where y lies that near a border. gate and up: [rows][K] of dtype with row strides in elements (two
 * halves of one projection's rows, say); codes, scale and spec as tc_rms_norm_quantize's. */
int tc_gated_quantize(const void *gate, int64_t gate_stride, const void *up, int64_t up_stride, int32_t dtype, int64_t rows,
                      int64_t K, int32_t activation, const tc_quant_spec *spec, void *codes, void *scale, tc_stream stream);

/* Tokens drawn from logits [rows][vocab] of dtype (row stride in elements) by given random numbers uniform [rows] in [0, 1):
 * w_i = exp((l_i - max l) / temperature), weights below 2**-126 counting as 0; of those the top_k largest (ties to the lower
 * index; <= 0: all); of those, in descending order, the fewest whose weights reach top_p of their sum (>= 1: all); of those
 * the ones with w_i >= min_p (<= 0: all; the largest always stays). tokens[r] is the first index at which the sum of the kept weights, in
 * index order, exceeds uniform[r] times their total; logprobs (or NULL) log(w / total). temperature <= 0: the first largest
 * logit, log-probability 0. A row without a logit above -Inf gives -1 and -Inf, one with a NaN -1 and NaN. Settings: one
 * a row where the array is given, else the value beside it; NaN settings bound nothing, a NaN temperature is 0, one between 0 and
 * 2**-100 is 2**-100. At most 2**27 rows and a vocabulary of 2**23. */
int tc_sample_tokens(const void *logits, int32_t dtype, int64_t rows, int64_t vocab, int64_t stride, const float *uniform,
                     const float *temperature, float all_temperature, const int32_t *top_k, int32_t all_top_k,
                     const float *top_p, float all_top_p, const float *min_p, float all_min_p, int64_t *tokens, float *logprobs,
                     tc_stream stream);

/* Library version string. */
const char *tc_version(void);

#ifdef __cplusplus
}
#endif

#endif /* TRICAST_B200_H */
