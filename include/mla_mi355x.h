/*
 * mla_mi355x.h -- C ABI of the MI355X (gfx950) weight-absorbed MLA decode:
 *
 *     O*[h, :] = softmax_t( Q*[h, :] . C[t, :] / sqrt(192) ) . C[t, :512]
 *
 * with Q* [num_heads x 576], the latent cache C [N x 576] (first 512 columns
 * are C_N, the last 64 the rope part) and O* [num_heads x 512], and of what a
 * serving loop runs around it on a paged cache: block tables, shared pages,
 * cache rows, prompts, drafted tokens.
 *
 * This is the drop-in boundary below the PyTorch extension: the reference's
 * extension (csrc/mla_api.cpp) calls raw-pointer launchers declared in
 * csrc/mla_decode.hpp; the entry points here are what it would bind instead.
 *
 * Conventions (all entry points):
 *  - Plain device pointers, row-major and contiguous, 16-byte aligned.
 *  - `stream` is a hipStream_t (NULL = the default stream). Work is enqueued
 *    asynchronously; nothing synchronises, nothing allocates.
 *  - The caller owns the workspace; query its size with the matching
 *    *_workspace_size function (same arguments, same current device).
 *    Calls that share one workspace must not overlap in time.
 *  - `num_splits` <= 0 picks the split count from the sequence length and
 *    the device's CU count; > 0 requests that many splits (clamped so every
 *    split holds at least one LDS block).
 *  - Return value: MLA_STATUS_SUCCESS (0) or one of the codes below; nothing
 *    is enqueued when a code other than 0 or MLA_STATUS_HIP_ERROR is
 *    returned. Thread-safe. Shared state: a per-device cache of the CU
 *    count and a per-device cache of the allocation-free entry point's
 *    scratch address (each written once per device). Per host thread: the
 *    last HIP error and the last few split plans.
 *  - num_heads must be a positive multiple of 16 (mla_append_kv_*: 0 to 4096).
 */
#ifndef MLA_MI355X_H
#define MLA_MI355X_H

#include <stddef.h>

#ifdef __cplusplus
extern "C" {
#endif

#define MLA_HEAD_DIM_K 576 /* mla.py:33 HEAD_DIM_K = HEAD_DIM_C + HEAD_DIM_ROPE */
#define MLA_HEAD_DIM_V 512 /* mla.py:31 HEAD_DIM_C */
#define MLA_ABI_VERSION 2 /* 2: mla_project_output_workspace_size takes d_model; status 5 added */

#define MLA_STATUS_SUCCESS 0
#define MLA_STATUS_INVALID_VALUE 1       /* null pointer or unsupported size */
#define MLA_STATUS_MISALIGNED 2          /* a pointer is not 16-byte aligned */
#define MLA_STATUS_WORKSPACE_TOO_SMALL 3 /* workspace_bytes below the size query */
#define MLA_STATUS_HIP_ERROR 4           /* a HIP launch failed: mla_last_hip_error() */
#define MLA_STATUS_SCRATCH_EXCEEDED 5    /* mla_decode_split_fp16_noalloc: partials exceed its scratch */

/* Size of the device array that holds the split partials of
 * mla_decode_split_fp16_noalloc (one per GPU the library runs on). */
#define MLA_NOALLOC_SCRATCH_BYTES (32u << 20)

/* Testing aid for mla_decode_split_fp16_ex: read the C_N^T operand of the
 * second product with scalar LDS loads instead of the LDS transpose read. */
#define MLA_FLAG_SCALAR_TRANSPOSE 1u

/* mla_decode_split_fp16_ex / _partials / _combine: keep the split partials
 * in fp32 instead of the input type (twice the partial traffic; the combine
 * must be given the same flag as the split phase). The workspace size
 * queries cover both precisions. */
#define MLA_FLAG_FP32_PARTIALS 4u

/* A single-sequence 16-bit call (mla_decode_split_fp16/_ex, _bf16, _fp8 and
 * the allocation-free entry point) whose plan has one split is ONE launch:
 * the split kernel writes the output itself, with no partials and no
 * combine (the planner prefers one split for short sequences, about
 * 200 tokens or fewer at 128 heads, for that reason). This flag keeps the
 * reference's two launches in that case too: split kernel, then the LSE
 * combine (csrc/mla_decode_splitk_fwd.cuh:973-978). */
#define MLA_FLAG_TWO_LAUNCHES 8u

/* Plan queries only (mla_decode_split_num_splits, _head_tile, _launches):
 * report the plan of the fp8-cache entry mla_decode_split_fp8 for these
 * sizes. Its cache streams half the bytes of a 16-bit one, so with few heads
 * and long sequences its plan can take more splits, or another head tile,
 * than the 16-bit plan. The decode entry points ignore it; mla_append_kv_*
 * takes it for a cache of E4M3FN bytes. */
#define MLA_FLAG_FP8_CACHE 16u

/* mla_append_kv_*: the rotation's pairs are values i and i + 32, not 2 i and
 * 2 i + 1. */
#define MLA_FLAG_ROPE_HALVES 32u

int mla_abi_version(void);
const char *mla_status_string(int status);
/* hipError_t of the last failed HIP call on this thread (0 if none). */
int mla_last_hip_error(void);

/* Number of splits (partial results per head) that mla_decode_split_fp16_ex
 * (with MLA_FLAG_FP8_CACHE: mla_decode_split_fp8) uses for these arguments
 * and flags on the current device; 0 for invalid sizes.
 * Replaces the fixed `num_splits = 4` of mla_decode_split
 * (csrc/mla_api.cpp:97). */
int mla_decode_split_num_splits(int num_heads, int seq_length, int num_splits,
                                unsigned flags);

/* Heads per workgroup (16, 32 or 64) of the plan that
 * mla_decode_split_fp16_ex (with MLA_FLAG_FP8_CACHE: mla_decode_split_fp8)
 * uses for these arguments and flags on the current device; 0 for invalid
 * sizes.
 * With an fp8 cache, tiles of 32 or 64 heads run the first product on fp8
 * MFMAs (Q* split in two fp8 parts), tiles of 16 convert C to fp16. No
 * counterpart in the reference. */
int mla_decode_split_head_tile(int num_heads, int seq_length, int num_splits,
                               unsigned flags);

/* Kernel launches (1 or 2, see MLA_FLAG_TWO_LAUNCHES) that
 * mla_decode_split_fp16_ex (with MLA_FLAG_FP8_CACHE: mla_decode_split_fp8)
 * makes for these arguments and flags on the current device; 0 for invalid sizes. No counterpart in the reference, whose
 * launcher always makes two (csrc/mla_decode_splitk_fwd.cuh:973-978). */
int mla_decode_split_launches(int num_heads, int seq_length, int num_splits,
                              unsigned flags);

/* Workspace for mla_decode_split_fp16 (split partials: O normalised by its
 * running sum in fp16, running max and sum in fp32). Replaces the
 * splits_max / splits_sum / splits_out buffers that mla_decode_split_
 * allocates per call (csrc/mla_api.cpp:71-75). Returns 0 for invalid sizes. */
size_t mla_decode_split_workspace_size(int num_heads, int seq_length,
                                       int num_splits);

/* fp16 split-KV decode: query [num_heads x 576] fp16, cache [seq_length x 576]
 * fp16 -> out [num_heads x 512] fp16; fp32 accumulation and softmax state,
 * fp16 normalised partials merged in fp32. Replaces run_mla_decode_splitk<at::Half>
 * (csrc/mla_decode.hpp:25-34; csrc/mla_decode_splitk_fwd_sm89.cu:26-47 ->
 * run_mla_decode_splitk_fp16, csrc/mla_decode_splitk_fwd.cuh:941-985), which
 * took three caller buffers, no stream, and required num_heads == 128 and
 * seq_length % 64 == 0. */
int mla_decode_split_fp16(const void *query, const void *cache, void *out,
                          void *workspace, size_t workspace_bytes,
                          int num_heads, int seq_length, int num_splits,
                          void *stream);

/* mla_decode_split_fp16 with flags (MLA_FLAG_*). */
int mla_decode_split_fp16_ex(const void *query, const void *cache, void *out,
                             void *workspace, size_t workspace_bytes,
                             int num_heads, int seq_length, int num_splits,
                             unsigned flags, void *stream);

/* mla_decode_split_fp16 without a workspace, for callers that cannot
 * allocate device memory (code under HIP graph capture, tight serving loops,
 * harnesses that forbid hipMalloc). No counterpart in the reference. The split
 * partials go to a file-scope device array of MLA_NOALLOC_SCRATCH_BYTES
 * (32 MiB) that each GPU holds until the process ends; its device address is
 * looked up (hipGetSymbolAddress) on the first call on each device. The call
 * allocates nothing and launches the same kernels with the same split plan
 * as mla_decode_split_fp16, so the results are identical. Every call on one
 * GPU shares that GPU's array: calls that overlap in time on one GPU (other
 * streams, other threads) race. Nothing in the array needs clearing: each
 * call writes every partial it reads. Returns MLA_STATUS_SCRATCH_EXCEEDED
 * when the plan's partials would not fit (not for any num_splits <= 0 plan
 * on a GPU of up to 256 CUs: those stay below 17 MiB). */
int mla_decode_split_fp16_noalloc(const void *query, const void *cache,
                                  void *out, int num_heads, int seq_length,
                                  int num_splits, void *stream);

/* The two launches of mla_decode_split_fp16, one at a time: the split-KV
 * kernel, which leaves its partials in the workspace, then the LSE combine,
 * which merges them into out. Called back to back on one stream with the
 * same num_heads / seq_length / num_splits they equal mla_decode_split_fp16
 * (the reference's launcher makes the same two launches,
 * csrc/mla_decode_splitk_fwd.cuh:973-978); apart, they let a caller place
 * other work or timing events between the phases. */
int mla_decode_split_fp16_partials(const void *query, const void *cache,
                                   void *workspace, size_t workspace_bytes,
                                   int num_heads, int seq_length,
                                   int num_splits, unsigned flags,
                                   void *stream);
int mla_decode_split_fp16_combine(const void *workspace,
                                  size_t workspace_bytes, void *out,
                                  int num_heads, int seq_length,
                                  int num_splits, unsigned flags,
                                  void *stream);

/* Workspace for mla_decode_fused_fp32. */
size_t mla_decode_fused_workspace_size(int num_heads, int seq_length,
                                       int num_splits);

/* fp32 decode: query [num_heads x head_dim_c] fp32, cache
 * [seq_length x head_dim_c] fp32 -> out [num_heads x 512] fp32, products
 * of fp32 precision whatever the values: chunks of 64 tokens or more multiply
 * operands split in three bf16 parts (all 24 bits; what lies below 2^-110, to
 * 2^-133) with fp32 sums, others run on fp32 MFMAs. head_dim_c must be 576. Replaces run_mla_decode_fused
 * (csrc/mla_decode.hpp:17-22; csrc/mla_decode_fused_fwd_sm89.cu:6-60), which
 * needed num_heads % 16 == 0 and seq_length % 16 == 0 and no workspace. */
int mla_decode_fused_fp32(const float *query, const float *cache, float *out,
                          void *workspace, size_t workspace_bytes,
                          int num_heads, int head_dim_c, int seq_length,
                          int num_splits, void *stream);

/* Workspace for mla_decode_split_batched_fp16. */
size_t mla_decode_split_batched_workspace_size(int batch, int num_heads,
                                               int total_tokens,
                                               int num_splits);

/* Batched variable-length fp16 decode (no reference counterpart: the
 * reference handles one sequence per call, csrc/mla_api.cpp:67-69).
 * query [batch x num_heads x 576] fp16; cache = the sequences' caches packed
 * back to back [total_tokens x 576] fp16; cu_seqlens [batch + 1] int32 on the
 * device with cu_seqlens[0] = 0, non-decreasing, cu_seqlens[batch] =
 * total_tokens (sequence b owns rows cu_seqlens[b] .. cu_seqlens[b+1]-1);
 * out [batch x num_heads x 512] fp16. Empty sequences give zero rows. The
 * splits are cut over the packed tokens, so work is balanced whatever the
 * length mix. Values of cu_seqlens outside [0, total_tokens] are clamped. */
int mla_decode_split_batched_fp16(const void *query, const void *cache,
                                  const int *cu_seqlens, void *out,
                                  void *workspace, size_t workspace_bytes,
                                  int batch, int num_heads, int total_tokens,
                                  int num_splits, void *stream);

/* The two launches of mla_decode_split_batched_fp16, one at a time, as
 * mla_decode_split_fp16_partials / _combine are for one sequence: the
 * split-KV kernel leaves the partials in the workspace, the combine merges
 * them into out. Called back to back on one stream with the same sizes they
 * equal mla_decode_split_batched_fp16. No reference counterpart (the
 * reference decodes one sequence per call). */
int mla_decode_split_batched_fp16_partials(const void *query,
                                           const void *cache,
                                           const int *cu_seqlens,
                                           void *workspace,
                                           size_t workspace_bytes, int batch,
                                           int num_heads, int total_tokens,
                                           int num_splits, void *stream);
int mla_decode_split_batched_fp16_combine(const void *workspace,
                                          size_t workspace_bytes,
                                          const int *cu_seqlens, void *out,
                                          int batch, int num_heads,
                                          int total_tokens, int num_splits,
                                          void *stream);

/* bf16 KV cache: mla_decode_split_fp16 and mla_decode_split_batched_fp16
 * with query, cache and out in bf16 (the same workspace sizes; bf16 MFMAs,
 * fp32 accumulation and softmax state, P and the normalised partials in
 * bf16). No reference counterpart: the reference lists bf16 as future work
 * (README.md:405-408) and its --bf16 flag is commented out (mla.py:163). */
int mla_decode_split_bf16(const void *query, const void *cache, void *out,
                          void *workspace, size_t workspace_bytes,
                          int num_heads, int seq_length, int num_splits,
                          void *stream);
int mla_decode_split_batched_bf16(const void *query, const void *cache,
                                  const int *cu_seqlens, void *out,
                                  void *workspace, size_t workspace_bytes,
                                  int batch, int num_heads, int total_tokens,
                                  int num_splits, void *stream);

/* Paged KV cache (no reference counterpart: the reference reads one
 * contiguous cache per call, csrc/mla_api.cpp:67-69). kv_cache is
 * [num_pages x page_size x 576] (fp16 or bf16); token l of sequence b is row
 * l % page_size of page block_table[b * block_table_stride + l / page_size]
 * (int32 on the device). cu_seqlens [batch + 1] (int32, device) holds the
 * prefix sums of the sequence lengths (cu_seqlens[0] = 0, cu_seqlens[batch]
 * = total_tokens), query [batch x num_heads x 576], out
 * [batch x num_heads x 512]; empty sequences give zero rows. page_size is a
 * power of two >= 32. Page ids outside [0, num_pages) and block-table
 * columns beyond block_table_stride are clamped (the result is then
 * meaningless but every access stays inside the caller's buffers). The same
 * split planner as the packed batched entry (head tiles of 16, 32 or 64).
 * total_tokens is not checked against cu_seqlens[batch] (that would need a
 * device read): every sequence's range is clipped to [0, total_tokens), so a
 * total_tokens below cu_seqlens[batch] silently truncates the trailing
 * sequences (their rows cover only their tokens below total_tokens, zeros if
 * none) and still returns MLA_STATUS_SUCCESS; a larger one only changes the
 * split plan. */
size_t mla_decode_paged_workspace_size(int batch, int num_heads,
                                       int total_tokens, int num_splits);
int mla_decode_paged_fp16(const void *query, const void *kv_cache,
                          const int *block_table, const int *cu_seqlens,
                          void *out, void *workspace, size_t workspace_bytes,
                          int batch, int num_heads, int total_tokens,
                          int page_size, int num_pages,
                          int block_table_stride, int num_splits,
                          void *stream);
int mla_decode_paged_bf16(const void *query, const void *kv_cache,
                          const int *block_table, const int *cu_seqlens,
                          void *out, void *workspace, size_t workspace_bytes,
                          int batch, int num_heads, int total_tokens,
                          int page_size, int num_pages,
                          int block_table_stride, int num_splits,
                          void *stream);

/* mla_decode_paged_* over a paged cache of OCP fp8 E4M3FN bytes that hold
 * C / cache_scale (a per-tensor scale > 0), as mla_append_kv_* writes it with
 * MLA_FLAG_FP8_CACHE: query and out in fp16 or bf16, everything else as there.
 * The cache is read at one byte per value; every E4M3FN value is a value of the
 * query's type, so the products see the cache as it stands. A query is held
 * whole where the plan's head tile is 16, else (num_heads a multiple of 32) as two
 * fp8 parts a head, 8 significant bits of each value: all that bf16 has, three
 * less than fp16's. The softmax weights and the split partials are in the query's type. Errors in the 2-norm, of N(0, 1)
 * queries: fp16 0.00033 with 16 heads and 0.00073 with 128 (rounding the
 * exact result once: 0.00021), bf16 0.0024 with 128 (0.0017). */
size_t mla_decode_paged_fp8_workspace_size(int batch, int num_heads,
                                           int total_tokens, int num_splits);
int mla_decode_paged_fp8_fp16(const void *query, const void *kv_cache_fp8,
                              float cache_scale, const int *block_table,
                              const int *cu_seqlens, void *out, void *workspace,
                              size_t workspace_bytes, int batch, int num_heads,
                              int total_tokens, int page_size, int num_pages,
                              int block_table_stride, int num_splits,
                              void *stream);
int mla_decode_paged_fp8_bf16(const void *query, const void *kv_cache_fp8,
                              float cache_scale, const int *block_table,
                              const int *cu_seqlens, void *out, void *workspace,
                              size_t workspace_bytes, int batch, int num_heads,
                              int total_tokens, int page_size, int num_pages,
                              int block_table_stride, int num_splits,
                              void *stream);

/* fp8 KV cache (no reference counterpart: the reference lists it as future
 * work, README.md:408): query [.. x num_heads x 576] fp16, cache
 * [tokens x 576] OCP fp8 E4M3FN bytes holding C / cache_scale (a per-tensor
 * scale > 0), out fp16. The decode reads the cache at one byte per value
 * (half the HBM traffic of fp16), keeps the bytes as they are in LDS and
 * converts each MFMA operand to fp16 after its LDS read (exact: every E4M3FN
 * value is an fp16 value); products and softmax as on the fp16 path. Workspace from
 * mla_decode_split_fp8_workspace_size(batch, num_heads, total_tokens,
 * num_splits) (batch = 1 for the single-sequence entry). cu_seqlens as for
 * mla_decode_split_batched_fp16. */
size_t mla_decode_split_fp8_workspace_size(int batch, int num_heads,
                                           int total_tokens, int num_splits);
int mla_decode_split_fp8(const void *query, const void *cache_fp8,
                         float cache_scale, void *out, void *workspace,
                         size_t workspace_bytes, int num_heads,
                         int seq_length, int num_splits, void *stream);
int mla_decode_split_batched_fp8(const void *query, const void *cache_fp8,
                                 float cache_scale, const int *cu_seqlens,
                                 void *out, void *workspace,
                                 size_t workspace_bytes, int batch,
                                 int num_heads, int total_tokens,
                                 int num_splits, void *stream);

/* The projections around the decode, completing an MLA attention block's
 * decode step (no reference code: the math is README.md:76-85, 104-110).
 * Weights in torch Linear layout: w_uk, w_uv [num_heads][128][512] (the key
 * and value halves of the latent up-projection), w_o [d_model][num_heads*128].
 *
 * mla_absorb_query_*: q_nope [batch][num_heads][128], q_rope
 *   [batch][num_heads][64] -> q_star [batch][num_heads][576] with
 *   q_star[..., :512] = q_nope W_UK[h] and q_star[..., 512:] = q_rope, the
 *   query of mla_decode_split_batched_* / mla_decode_paged_* (no softmax
 *   scale: the decode applies it).
 * mla_project_output_*: o_star [batch][num_heads][512] (the decode's output)
 *   -> out [batch][d_model] = concat_h(o_star[:, h] W_UV[h]^T) W_O^T, with
 *   the per-head values in a caller workspace of
 *   mla_project_output_workspace_size(batch, num_heads, d_model) bytes
 *   (the per-head values, then the output projection's fp32 K-part sums;
 *   the size never falls as the batch grows, so that a workspace for the largest
 *   batch serves every smaller one).
 * All three products are MFMA kernels of this library (fp32 accumulation)
 * and allocate nothing: W_UK and W_UV one workgroup per (head, column
 * slice, row group), W_O streamed from HBM through an LDS ring by at most one
 * workgroup per CU, in K-parts whose fp32 sums a second small kernel adds. */
size_t mla_project_output_workspace_size(int batch, int num_heads, int d_model);
int mla_absorb_query_fp16(const void *q_nope, const void *q_rope,
                          const void *w_uk, void *q_star, int batch,
                          int num_heads, void *stream);
int mla_absorb_query_bf16(const void *q_nope, const void *q_rope,
                          const void *w_uk, void *q_star, int batch,
                          int num_heads, void *stream);
int mla_project_output_fp16(const void *o_star, const void *w_uv,
                            const void *w_o, void *out, void *workspace,
                            size_t workspace_bytes, int batch, int num_heads,
                            int d_model, void *stream);
int mla_project_output_bf16(const void *o_star, const void *w_uv,
                            const void *w_o, void *out, void *workspace,
                            size_t workspace_bytes, int batch, int num_heads,
                            int d_model, void *stream);

/* Products in OCP fp8 (E4M3FN) with a scale for each block of 128, as the
 * projections before and after the attention hold their weights (no reference
 * code).
 *
 * mla_quantize_fp8_*: rows x [rows][inputs] (x_stride values apart) in fp16 or bf16 ->
 *   xq [rows][inputs] and scales [ceil(inputs / 128)][rows]: a block's scale is
 *   top / 448 with top = max(max |x|, 2^-100), its values xq = e4m3(448 x / top)
 *   (to nearest even). An infinity makes its block's values NaN and its scale
 *   infinite, a NaN stays one.
 * mla_linear_fp8_*: out [rows][outputs], in x's type, = x W^T:
 *   out[m][n] = sum_b xs[m][b] w_scale[n / 128][b] sum_{k in b} xq[m][k] w[n][k]
 *   with x quantised so, w [outputs][inputs] E4M3FN (w_stride bytes apart) and
 *   w_scale [ceil(outputs / 128)][ceil(inputs / 128)]; sums in fp32, rounded
 *   once, the product of two scales too, which has to be a finite fp32 value. The workspace holds the quantised rows, and fp32 sums where
 *   the inputs are split over workgroups (the same bits whatever is in it).
 * mla_linear_fp8_quantized_*: the same of rows that are quantised already, xq
 *   (x_stride bytes apart), and out in fp16 or bf16; the scale of row m and block b is
 *   x_scale[m scale_row_stride + b scale_block_stride] (1 and rows as mla_quantize_fp8_*
 *   leaves them, which is read fastest).
 * A NaN or infinity in a row of x makes its row of out NaN, a NaN in a row of w its
 * column. inputs must be a multiple of 16, strides of 8 values (16-bit rows) or 16 bytes, and
 * inputs and strides at most 2^22 (scale_row_stride: 2^20); rows and outputs at most 2^26,
 * their tiles of 16 x 16 less than 2^31, and the blocks of x, rows times
 * ceil(inputs / 128), at most 2^30 - 64. */
int mla_quantize_fp8_fp16(const void *x, void *xq, float *scales, int rows,
                          int inputs, long long x_stride, void *stream);
int mla_quantize_fp8_bf16(const void *x, void *xq, float *scales, int rows,
                          int inputs, long long x_stride, void *stream);
size_t mla_linear_fp8_workspace_size(int rows, int inputs, int outputs);
/* What a call of these sizes launches on the current device (quantized: of rows that are quantised already):
 * workgroups of tile_outputs x tile_rows, the inputs split over `splits` of them, in `launches` launches in all
 * (quantisation and sum of the splits among them). */
int mla_linear_fp8_plan(int rows, int inputs, int outputs, int quantized,
                        int *tile_outputs, int *tile_rows, int *splits,
                        int *launches);
int mla_linear_fp8_fp16(const void *x, const void *w, const float *w_scale,
                        void *out, void *workspace, size_t workspace_bytes,
                        int rows, int inputs, int outputs, long long x_stride,
                        long long w_stride, void *stream);
int mla_linear_fp8_bf16(const void *x, const void *w, const float *w_scale,
                        void *out, void *workspace, size_t workspace_bytes,
                        int rows, int inputs, int outputs, long long x_stride,
                        long long w_stride, void *stream);
int mla_linear_fp8_quantized_fp16(const void *xq, const float *x_scale,
                                  const void *w, const float *w_scale,
                                  void *out, void *workspace,
                                  size_t workspace_bytes, int rows, int inputs,
                                  int outputs, long long x_stride,
                                  long long w_stride,
                                  long long scale_row_stride,
                                  long long scale_block_stride, void *stream);
int mla_linear_fp8_quantized_bf16(const void *xq, const float *x_scale,
                                  const void *w, const float *w_scale,
                                  void *out, void *workspace,
                                  size_t workspace_bytes, int rows, int inputs,
                                  int outputs, long long x_stride,
                                  long long w_stride,
                                  long long scale_row_stride,
                                  long long scale_block_stride, void *stream);

/* Block table, slots and positions of one step's tokens, from the requests'
 * lengths (no reference counterpart). All pointers are on the device and
 * aligned to their type.
 *
 * Request b holds context_lens[b] tokens and gets new_lens[b] more (negative
 * values count as 0; new_lens beyond total_new tokens in all are clipped).
 * Its tokens' pages are columns 0, 1, .. of row b of block_table
 * [batch][block_table_stride]; those of its context are read from there. Each
 * page that the new tokens start takes the next id of free_pages [num_free],
 * request after request from index *free_start on, and is written to the table.
 *   cu_seqlens, cu_new [batch + 1]  prefix sums of the lengths with the new
 *                                   tokens, and of the new tokens alone
 *                                   (both stop at INT_MAX)
 *   slots, positions [total_new]    of the new tokens, in request order: the
 *                                   cache row page * page_size + offset, and
 *                                   the position in its request
 *   free_next                       *free_start + pages taken
 * Entries past the last new token are slot -1, position 0. Where the free list
 * or the table's columns end, or a context's page is negative, the token's slot
 * is -1 (and a page that the list no longer has is written as -1); free_next
 * then exceeds num_free by the pages missing. free_next must not be
 * free_start. page_size is a power of two from 32 to 2^20. One launch. */
int mla_paged_tables(const int *context_lens, const int *new_lens,
                     const int *free_pages, const int *free_start,
                     int *block_table, int *cu_seqlens, int *cu_new,
                     long long *slots, int *positions, int *free_next,
                     int batch, int total_new, int num_free, int page_size,
                     int block_table_stride, void *stream);

/* Rows of a block table taken over from others: requests sampled several times,
 * beams reordered, drafts rolled back, requests ended (no reference
 * counterpart). All pointers are on the device and aligned to their type.
 *
 * Row b of new_table [batch][block_table_stride] holds the first kept_lens[b]
 * tokens (NULL: all; clamped to 0 and what is there) of row parents[b] of
 * block_table [rows][block_table_stride], whose rows hold lens [rows] tokens
 * (clamped to 0 and the columns' room); a parent outside [0, rows) makes
 * an empty row. new_lens [batch] gets the tokens, columns behind a row's
 * last page -1. Rows share their whole pages. Of the rows that end inside a page the
 * lowest goes on writing it, if no new row holds the page whole and pinned
 * ([num_pages], NULL: none) is not positive for it; every other one takes
 * the next page of the free list, row after row, and copies [batch][3] gets
 * (page, page taken, rows to copy); (-1, -1, 0) for the other rows.
 * Pages that a row of block_table holds, no row of new_table holds and that
 * are not pinned are pushed to the free list before: with f of them,
 * free_pages [num_free] gets their ids, lowest first, from index
 * *free_start - f on, and pages are taken from there on. free_next gets
 * *free_start - f + pages taken. Where the list ends (below 0 or at num_free) nothing is
 * written, and a page taken is -1. Ids outside [0, num_pages) are passed on
 * and neither freed nor copied. pinned marks pages that others hold, a prompt
 * cache or another table. rows is at most 8192, num_pages at most 2^18,
 * block_table_stride at most 2^20, page_size a power of two from 32 to 2^20. new_table, new_lens and
 * free_next must not be their inputs. One launch. */
size_t mla_page_tables_workspace_size(int num_pages);
int mla_fork_tables(const int *block_table, const int *lens,
                    const int *parents, const int *kept_lens,
                    const int *pinned, int *free_pages, const int *free_start,
                    int *new_table, int *new_lens, int *copies, int *free_next,
                    void *workspace, size_t workspace_bytes, int rows,
                    int batch, int num_pages, int num_free, int page_size,
                    int block_table_stride, void *stream);

/* The used pages of a pool moved to its lowest ids, so that its tail can be given
 * back (no reference counterpart). Of the pages that a row of block_table
 * holds (not pinned) and the ids of free_pages [num_free] from *free_start on
 * (not held, not pinned, each counted once), the k-th highest held one moves to the
 * k-th lowest free one as long as that is lower: copies
 * [min(num_free, num_pages / 2)][3] gets (from, to, page_size) in that order,
 * (-1, -1, 0) behind the last move. new_table gets block_table with every page
 * where it went (columns behind a row's last page: -1), new_free_pages the
 * free ids in ascending order from *free_start on, -1 elsewhere. Workspace,
 * limits and other conditions as for mla_fork_tables. One or two launches. */
int mla_compact_tables(const int *block_table, const int *lens,
                       const int *pinned, const int *free_pages,
                       const int *free_start, int *new_table, int *copies,
                       int *new_free_pages, void *workspace,
                       size_t workspace_bytes, int rows, int num_pages,
                       int num_free, int page_size, int block_table_stride,
                       void *stream);

/* The rows that mla_fork_tables and mla_compact_tables ask for: in each of
 * `layers` caches [num_pages][page_size][576] back to back, of elements of
 * 1, 2 or 4 bytes, the first copies[i][2] rows of page copies[i][0] go to page
 * copies[i][1]. Entries with an id outside [0, num_pages) or no rows copy
 * nothing, more rows than page_size are page_size. A page must not be copied to twice,
 * nor both to and from (the tables above never ask for that). One launch. */
int mla_copy_pages(void *kv_cache, const int *copies, int count, int layers,
                   int num_pages, int page_size, int element_size,
                   void *stream);

/* A step's latent rows into the cache, and its queries' rotary parts (no
 * reference counterpart; the reference's cache comes ready made). Token t:
 *   kv_cache[slots[t]][:512] = kv[t][:512] norm_weight / sqrt(mean(kv[t][:512]^2) + eps)
 *   kv_cache[slots[t]][512:] = rotated kv[t][512:]
 *   q_rope_out[t][h]         = rotated q_rope[t][h]
 * computed in fp32 and rounded once; rows of any finite values, also such whose
 * squares leave fp32's range. The rotation turns pair i (values 2 i and
 * 2 i + 1, or i and i + 32 with MLA_FLAG_ROPE_HALVES) by the angle whose
 * cosine and sine are cos_sin[positions[t]][i] and [32 + i] (fp32
 * [num_positions][64]; positions are clamped to it). kv [tokens] rows of 576
 * values, kv_stride values apart; q_rope [tokens][num_heads] rows of 64,
 * q_token_stride and q_head_stride values apart (strides: multiples of 8),
 * q_rope_out contiguous; num_heads 0: no queries, both NULL. kv_cache holds
 * cache_rows rows of 576 values of the input's type, or with
 * MLA_FLAG_FP8_CACHE of E4M3FN bytes of value / cache_scale (to nearest even,
 * saturated at 448, NaN kept). Slots outside [0, cache_rows) are not written;
 * two tokens with one slot leave a mix of both rows in it. One launch. */
int mla_append_kv_fp16(const void *kv, const void *norm_weight,
                       const float *cos_sin, const int *positions,
                       const long long *slots, const void *q_rope,
                       void *kv_cache, void *q_rope_out, float eps,
                       float cache_scale, int tokens, int num_heads,
                       int num_positions, long long cache_rows,
                       long long kv_stride, long long q_token_stride,
                       long long q_head_stride, unsigned flags, void *stream);
int mla_append_kv_bf16(const void *kv, const void *norm_weight,
                       const float *cos_sin, const int *positions,
                       const long long *slots, const void *q_rope,
                       void *kv_cache, void *q_rope_out, float eps,
                       float cache_scale, int tokens, int num_heads,
                       int num_positions, long long cache_rows,
                       long long kv_stride, long long q_token_stride,
                       long long q_head_stride, unsigned flags, void *stream);

/* Decode of a tree of drafted tokens a request, over the paged cache (no
 * reference counterpart: the reference decodes one token). kv_cache,
 * block_table, cu_seqlens, page_size, total_tokens as for mla_decode_paged_*;
 * a request's drafted tokens are the last draft_lens[b] ones of its cache
 * (draft_lens [batch], clamped to [0, drafts]; NULL: drafts for every request),
 * already written. query [batch x drafts x num_heads x 576] -> out [batch x
 * drafts x num_heads x 512]. Drafted token i sees the request's whole context
 * and drafted token j where bit j of tree_mask[b][i] ([batch x drafts]) is set:
 * its ancestors and itself, or, with masks 2^(i+1) - 1, a plain chain. A row
 * that sees nothing, and the rows from draft_lens[b] on, are zeros. A row that
 * sees a drafted token with an infinity or NaN in its first 512 values is NaN;
 * what it does not see never reaches it. drafts is at most 64. num_splits <= 0 picks the splits of each request's tokens. */
size_t mla_decode_tree_workspace_size(int batch, int drafts, int num_heads,
                                      int total_tokens, int num_splits);
int mla_decode_tree_fp16(const void *query, const void *kv_cache,
                         const int *block_table, const int *cu_seqlens,
                         const long long *tree_mask, const int *draft_lens,
                         void *out, void *workspace, size_t workspace_bytes,
                         int batch, int drafts, int num_heads,
                         int total_tokens, int page_size, int num_pages,
                         int block_table_stride, int num_splits, void *stream);
int mla_decode_tree_bf16(const void *query, const void *kv_cache,
                         const int *block_table, const int *cu_seqlens,
                         const long long *tree_mask, const int *draft_lens,
                         void *out, void *workspace, size_t workspace_bytes,
                         int batch, int drafts, int num_heads,
                         int total_tokens, int page_size, int num_pages,
                         int block_table_stride, int num_splits, void *stream);

/* Causal attention of prompts, or chunks of prompts, in the expanded form (no
 * reference code; the math is README.md:64-85): with c_t, r_t the 512 latent
 * and 64 rotary values of cache row t,
 *   k[t][h] = [w_uk[h] c_t, r_t], v[t][h] = w_uv[h] c_t,
 *   out[i][h] = softmax_t( [q_nope, q_rope][i][h] . k[t][h] / sqrt(192) ) v[t][h].
 * Request b has the queries cu_q[b] .. cu_q[b + 1] - 1 of q_nope [queries x
 * num_heads x 128], q_rope [queries x num_heads x 64] and out [queries x
 * num_heads x 128], and the keys of its cache, cu_seqlens as for
 * mla_decode_split_batched_*; its queries are the last of its keys, and each
 * sees the keys up to its own position (zeros where there is none). kv_cache
 * is paged as for mla_decode_paged_*, or packed [total_tokens x 576] where
 * block_table is NULL (the page arguments are then ignored). Both prefix sums
 * start at 0 and are clamped to [0, queries] and [0, total_tokens]; rows of out
 * behind the last request's are zeros. w_uk, w_uv as for
 * mla_absorb_query_* / mla_project_output_*. K and V are rounded to the
 * inputs' type; a query that sees a key whose K or V is not finite then (fp16:
 * past 65504) gives NaN, and what it does not see never reaches it. The workspace holds K and V: 512
 * bytes a key and head, and partial results where few queries see many keys.
 * Two launches, three with partials. */
size_t mla_prefill_workspace_size(int batch, int num_heads, int queries,
                                  int total_tokens);
int mla_prefill_fp16(const void *q_nope, const void *q_rope, const void *w_uk,
                     const void *w_uv, const void *kv_cache,
                     const int *block_table, const int *cu_q,
                     const int *cu_seqlens, void *out, void *workspace,
                     size_t workspace_bytes, int batch, int num_heads,
                     int queries, int total_tokens, int page_size,
                     int num_pages, int block_table_stride, void *stream);
int mla_prefill_bf16(const void *q_nope, const void *q_rope, const void *w_uk,
                     const void *w_uv, const void *kv_cache,
                     const int *block_table, const int *cu_q,
                     const int *cu_seqlens, void *out, void *workspace,
                     size_t workspace_bytes, int batch, int num_heads,
                     int queries, int total_tokens, int page_size,
                     int num_pages, int block_table_stride, void *stream);

#ifdef __cplusplus
}
#endif

#endif /* MLA_MI355X_H */
