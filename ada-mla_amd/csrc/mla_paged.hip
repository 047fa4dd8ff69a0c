// What fills the paged latent cache that the decodes read:
//
//   mla_paged_tables   the block table's new pages, the prefix sums of the
//                      lengths, and each new token's slot and position, from
//                      the requests' lengths and a list of free pages;
//   mla_append_kv_*    the new tokens' latent rows, normalised and rotated,
//                      written to their slots, and their queries' rotary
//                      parts rotated.
//
// Both are bound by memory round trips (a step's few tokens) or by the bytes
// (prompts); each is one launch.
#include <algorithm>
#include <cstdint>

#include "mla_device.hpp"
#include "mla_internal.hpp"
#include "mla_mi355x.h"

namespace mla {
namespace {

bool aligned16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

// ---- tables -----------------------------------------------------------------

constexpr int kScan = 512;  // requests per scan tile: one per thread

// Sums that stop at `cap` (< 2^31): associative over values 0 .. cap, so the
// scans below hold whatever the lengths add up to.
__device__ __forceinline__ unsigned sat_add(unsigned a, unsigned b, unsigned cap) { return min(a + b, cap); }

// Inclusive scan of v over the workgroup's threads with sat_add, starting
// from `carry`; `last` receives the sum over all of them. s: a word of LDS a wave.
__device__ __forceinline__ unsigned block_scan(unsigned v, unsigned carry, unsigned cap, unsigned *s, unsigned &last)
{
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
        const unsigned u = __shfl_up(v, d);
        if (lane >= d)
            v = sat_add(u, v, cap);
    }
    if (lane == 63)
        s[wave] = v;
    __syncthreads();
    unsigned before = carry;
    last = carry;
#pragma unroll
    for (int w = 0; w < kScan / 64; ++w) {
        if (w == wave)
            before = last;
        last = sat_add(last, s[w], cap);
    }
    __syncthreads();
    return sat_add(before, v, cap);
}

// Request b holds context_lens[b] tokens and gets new_lens[b] more (clipped so
// that all of them together are at most total_new): its tokens' positions run
// on from its context, position p sits at row p mod page of page p / page, and
// the pages past ceil(context / page) come from the free list, request after
// request, from *free_start on. A new page starts with a new token, so the
// thread of that token writes the page's table entry, and a token's page is
// either an old entry of the table (nobody writes those) or computed from the
// prefix sums: no thread waits for another's table write.
// Every workgroup scans all the requests (a few KB from L2, kScan at a time) and
// takes tokens_per_wg tokens; their requests come from a binary search in LDS.
// That is one launch instead of three (sums, pages, slots), which is what a
// step's few tokens cost; workgroup 0 also writes the prefix sums. Bound by its
// chain of round trips: lengths, scans, page, store (64 requests of one token 3.5 us,
// 300000 tokens of 301 prompts 6.4 us, their 3.8 MB 0.8 us of it).
__global__ __launch_bounds__(kScan) void paged_tables_kernel(
    const int *__restrict__ context_lens, const int *__restrict__ new_lens, const int *__restrict__ free_pages,
    const int *__restrict__ free_start, int *block_table, int *__restrict__ cu_seqlens, int *__restrict__ cu_new,
    long long *__restrict__ slots, int *__restrict__ positions, int *__restrict__ free_next, int batch, int total_new,
    int num_free, int page_shift, int stride, int tokens_per_wg, int each)
{
    __shared__ unsigned s_scan[kScan / 64];
    __shared__ unsigned s_new[kScan + 1];  // prefix sums of the tile's new tokens
    __shared__ int s_context[kScan];
    __shared__ unsigned s_pages[kScan];  // pages taken before the request
    const int tid = threadIdx.x;
    const unsigned kMost = 0x7fffffffu;
    const unsigned mask = (1u << page_shift) - 1;
    const unsigned t_lo = blockIdx.x * (unsigned)tokens_per_wg;
    const unsigned t_hi = min(t_lo + tokens_per_wg, (unsigned)total_new);
    const long long start = *free_start;
    unsigned c_new = 0, c_len = 0, c_pages = 0;  // sums over the tiles before
    if (blockIdx.x == 0 && tid == 0)
        cu_seqlens[0] = cu_new[0] = 0;
    for (int b0 = 0; b0 < batch; b0 += kScan) {
        const int b = b0 + tid;
        unsigned context = 0, want = 0;
        if (b < batch) {
            context = (unsigned)max(context_lens[b], 0);
            want = (unsigned)min(max(new_lens[b], 0), total_new);
        }
        unsigned n_new, n_len, n_pages;
        const unsigned hi = block_scan(want, c_new, (unsigned)total_new, s_scan, n_new);
        s_new[tid + 1] = hi;
        if (tid == 0)
            s_new[0] = c_new;
        s_context[tid] = (int)context;
        __syncthreads();
        const unsigned lo = s_new[tid];
        const unsigned end = sat_add(context, hi - lo, kMost);
        const unsigned held = (context + mask) >> page_shift;
        const unsigned pages = b < batch ? ((end + mask) >> page_shift) - held : 0;
        const unsigned len = block_scan(b < batch ? end : 0, c_len, kMost, s_scan, n_len);
        const unsigned taken = block_scan(pages, c_pages, kMost, s_scan, n_pages);
        s_pages[tid] = taken - pages;
        if (blockIdx.x == 0 && b < batch) {
            cu_seqlens[b + 1] = (int)len;
            cu_new[b + 1] = (int)hi;
        }
        __syncthreads();
        // `each` tokens in a row per thread: one search, and mostly one page, for all
        for (unsigned first = t_lo + each * tid; first < min(t_hi, n_new); first += kScan * each) {
            unsigned t = max(first, c_new);
            const unsigned last = min(min(first + each, t_hi), n_new);
            if (t >= last)
                continue;
            int r = 0;  // the last request of the tile that starts at or before t
#pragma unroll
            for (int d = kScan / 2; d > 0; d /= 2)
                if (s_new[r + d] <= t)
                    r += d;
            int page = -1, page_col = -1, page_request = -1;
            for (; t < last; ++t) {
                while (s_new[r + 1] <= t)
                    ++r;
                const int ctx = s_context[r];
                const unsigned pos = sat_add((unsigned)ctx, t - s_new[r], kMost);
                const unsigned col = pos >> page_shift, first_col = ((unsigned)ctx + mask) >> page_shift;
                if (r != page_request || (int)col != page_col) {
                    page_request = r;
                    page_col = (int)col;
                    page = -1;
                    if (col < (unsigned)stride) {
                        int *entry = block_table + (size_t)(b0 + r) * stride + col;
                        if (col < first_col) {
                            page = *entry;
                        } else {
                            const long long i = start + s_pages[r] + (col - first_col);
                            if (i >= 0 && i < num_free)
                                page = free_pages[i];
                            if ((pos & mask) == 0)
                                *entry = page;
                        }
                    }
                }
                slots[t] = page < 0 ? -1 : ((long long)page << page_shift) + (pos & mask);
                positions[t] = (int)pos;
            }
        }
        __syncthreads();
        c_new = n_new;
        c_len = n_len;
        c_pages = n_pages;
    }
    for (unsigned t = max(t_lo, c_new) + tid; t < t_hi; t += kScan) {  // tokens of no request
        slots[t] = -1;
        positions[t] = 0;
    }
    if (blockIdx.x == 0 && tid == 0)
        *free_next = (int)min(max(start + (long long)c_pages, (long long)INT32_MIN), (long long)INT32_MAX);
}

// ---- cache rows -------------------------------------------------------------

constexpr int kLatent = 512, kRope = 64, kRow = 576;

// A rotation's 8 pairs of thread j (of 4): pairs 8j .. 8j+7. Interleaved, pair
// i is values 2i and 2i+1, so the thread's 16 values are two adjacent 16-byte
// chunks; in halves, pair i is values i and i + 32, chunks j and j + 4.
template <typename E>
struct Pairs {
    using E8 = typename Vec<E>::v8;
    float a[8], b[8];
    template <bool kHalves>
    __device__ __forceinline__ void load(const E *row, int j)
    {
        const E8 u = *(const E8 *)(row + (kHalves ? 8 * j : 16 * j));
        const E8 v = *(const E8 *)(row + (kHalves ? 32 + 8 * j : 16 * j + 8));
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            a[i] = kHalves ? (float)u[i] : i < 4 ? (float)u[2 * i] : (float)v[2 * i - 8];
            b[i] = kHalves ? (float)v[i] : i < 4 ? (float)u[2 * i + 1] : (float)v[2 * i - 7];
        }
    }
    __device__ __forceinline__ void rotate(const float *cos_sin_row, int j)
    {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const floatx4 c = *(const floatx4 *)(cos_sin_row + 8 * j + 4 * h);
            const floatx4 s = *(const floatx4 *)(cos_sin_row + 32 + 8 * j + 4 * h);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float x = a[4 * h + i], y = b[4 * h + i];
                a[4 * h + i] = x * c[i] - y * s[i];
                b[4 * h + i] = y * c[i] + x * s[i];
            }
        }
    }
    // the thread's 16 values in the order of its two chunks
    template <bool kHalves>
    __device__ __forceinline__ float at(int i) const
    {
        return kHalves ? (i < 8 ? a[i] : b[i - 8]) : (i & 1) ? b[i >> 1] : a[i >> 1];
    }
};

// 8 values as 8 bytes of OCP E4M3: to nearest even, saturated at +-448, NaN kept.
__device__ __forceinline__ uint2 to_fp8x8(const float *x)
{
    float y[8];
#pragma unroll
    for (int i = 0; i < 8; ++i)
        y[i] = x[i] != x[i] ? x[i] : fminf(fmaxf(x[i], -448.0f), 448.0f);
    int lo = __builtin_amdgcn_cvt_pk_fp8_f32(y[0], y[1], 0, false);
    lo = __builtin_amdgcn_cvt_pk_fp8_f32(y[2], y[3], lo, true);
    int hi = __builtin_amdgcn_cvt_pk_fp8_f32(y[4], y[5], 0, false);
    hi = __builtin_amdgcn_cvt_pk_fp8_f32(y[6], y[7], hi, true);
    return uint2{(unsigned)lo, (unsigned)hi};
}

// 8 values of a cache row at column col, rounded once to the cache's type.
template <typename E, bool kFp8>
__device__ __forceinline__ void store8(void *cache, size_t row, int col, const float *x, float cache_scale)
{
    if constexpr (kFp8) {
        float y[8];
#pragma unroll
        for (int i = 0; i < 8; ++i)
            y[i] = x[i] / cache_scale;
        *(uint2 *)((unsigned char *)cache + row * kRow + col) = to_fp8x8(y);
    } else {
        typename Vec<E>::v8 v;
#pragma unroll
        for (int i = 0; i < 8; ++i)
            v[i] = (E)x[i];
        *(typename Vec<E>::v8 *)((E *)cache + row * kRow + col) = v;
    }
}

// One wave per unit of work of a token: unit 0 is its latent row (a lane holds
// 8 of the 512 values: one 16-byte load, one wave sum of squares, one store;
// lanes 0 .. 3 rotate the key), the others 16 heads each of its queries (4
// threads a head). Everything a token's row needs is one wave's, so nothing
// goes through LDS. Many tokens are a memory stream (32768 tokens and 16 heads
// into an fp8 cache: 200 MB in 49 us, 4.0 TB/s, where a copy reaches 4.9; 45 us where the
// same inputs come again, part of them still in the 256 MB last-level cache); a step
// of 64 tokens and 128 heads is one round trip of loads (3.1 us).
template <typename E, bool kFp8, bool kHalves>
__global__ __launch_bounds__(256) void append_kv_kernel(const E *__restrict__ kv, const E *__restrict__ norm_weight,
                                                        const float *__restrict__ cos_sin,
                                                        const int *__restrict__ positions,
                                                        const long long *__restrict__ slots,
                                                        const E *__restrict__ q_rope, void *__restrict__ cache,
                                                        E *__restrict__ q_out, float eps, float cache_scale, int tokens,
                                                        int num_heads, int num_positions, long long cache_rows,
                                                        long long kv_stride, long long q_token_stride,
                                                        long long q_head_stride, int units)
{
    using E8 = typename Vec<E>::v8;
    const int lane = threadIdx.x & 63;
    const unsigned w = blockIdx.x * 4u + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int t = (int)(w / (unsigned)units), u = (int)(w % (unsigned)units);
    if (t >= tokens)
        return;
    const int pos = min(max(positions[t], 0), num_positions - 1);
    const float *angle = cos_sin + (size_t)pos * kRope;
    if (u > 0) {  // queries
        const int h = 16 * (u - 1) + (lane >> 2), j = lane & 3;
        if (h >= num_heads)
            return;
        Pairs<E> p;
        p.template load<kHalves>(q_rope + t * q_token_stride + h * q_head_stride, j);
        p.rotate(angle, j);
        E *out = q_out + ((size_t)t * num_heads + h) * kRope;
        E8 lo, hi;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            lo[i] = (E)p.template at<kHalves>(i);
            hi[i] = (E)p.template at<kHalves>(8 + i);
        }
        *(E8 *)(out + (kHalves ? 8 * j : 16 * j)) = lo;
        *(E8 *)(out + (kHalves ? 32 + 8 * j : 16 * j + 8)) = hi;
        return;
    }
    const long long slot = slots[t];
    if (slot < 0 || slot >= cache_rows)
        return;
    const E *row = kv + t * kv_stride;
    const E8 xv = *(const E8 *)(row + 8 * lane), wv = *(const E8 *)(norm_weight + 8 * lane);
    Pairs<E> p;
    if (lane < 4)
        p.template load<kHalves>(row + kLatent, lane);
    float x[8];
#pragma unroll
    for (int i = 0; i < 8; ++i)
        x[i] = (float)xv[i];
    auto mean_square = [&](float f) {  // of f x, the same in every lane
        float sum = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; ++i)
            sum += (f * x[i]) * (f * x[i]);
        sum = sum_over_lane_groups(sum);
#pragma unroll
        for (int d = 8; d > 0; d /= 2)
            sum += __shfl_xor(sum, d);
        return sum * (1.0f / kLatent);
    };
    float under_root = mean_square(1.0f) + eps, norm = 1.0f / sqrtf(under_root);
    // bf16 reaches further than its squares do in fp32. Where they may have left fp32's
    // range, rows and epsilon are squared again times a power of two: what then
    // vanishes is below 2^-24 of the sum.
    if (!(under_root > 0x1p-100f && under_root < 0x1p100f)) {
        const bool tiny = under_root < 1.0f;
        const float f = tiny ? 0x1p100f : 0x1p-100f;
        under_root = mean_square(f) + eps * f * f;
        norm = 1.0f / sqrtf(under_root) * (tiny ? 1.0f : f);
#pragma unroll
        for (int i = 0; i < 8; ++i)
            x[i] *= tiny ? f : 1.0f;  // 1 / norm may pass 2^128, each factor does not
    }
#pragma unroll
    for (int i = 0; i < 8; ++i)
        x[i] = x[i] * norm * (float)wv[i];
    store8<E, kFp8>(cache, (size_t)slot, 8 * lane, x, cache_scale);
    if (lane < 4) {
        p.rotate(angle, lane);
        float y[16];
#pragma unroll
        for (int i = 0; i < 16; ++i)
            y[i] = p.template at<kHalves>(i);
        store8<E, kFp8>(cache, (size_t)slot, kLatent + (kHalves ? 8 * lane : 16 * lane), y, cache_scale);
        store8<E, kFp8>(cache, (size_t)slot, kLatent + (kHalves ? 32 + 8 * lane : 16 * lane + 8), y + 8, cache_scale);
    }
}

template <typename E>
void launch_append(const void *kv, const void *norm_weight, const float *cos_sin, const int *positions,
                   const long long *slots, const void *q_rope, void *cache, void *q_out, float eps, float cache_scale,
                   int tokens, int num_heads, int num_positions, long long cache_rows, long long kv_stride,
                   long long q_token_stride, long long q_head_stride, unsigned flags, hipStream_t s)
{
    const int units = 1 + (num_heads + 15) / 16;
    const bool f8 = (flags & MLA_FLAG_FP8_CACHE) != 0, halves = (flags & MLA_FLAG_ROPE_HALVES) != 0;
    auto k = f8 ? (halves ? append_kv_kernel<E, true, true> : append_kv_kernel<E, true, false>)
                : (halves ? append_kv_kernel<E, false, true> : append_kv_kernel<E, false, false>);
    const long long waves = (long long)tokens * units;
    hipLaunchKernelGGL(k, dim3((unsigned)((waves + 3) / 4)), dim3(256), 0, s, static_cast<const E *>(kv),
                       static_cast<const E *>(norm_weight), cos_sin, positions, slots, static_cast<const E *>(q_rope),
                       cache, static_cast<E *>(q_out), eps, cache_scale, tokens, num_heads, num_positions, cache_rows,
                       kv_stride, q_token_stride, q_head_stride, units);
}

int append_kv(bool bf16, const void *kv, const void *norm_weight, const float *cos_sin, const int *positions,
              const long long *slots, const void *q_rope, void *cache, void *q_out, float eps, float cache_scale,
              int tokens, int num_heads, int num_positions, long long cache_rows, long long kv_stride,
              long long q_token_stride, long long q_head_stride, unsigned flags, void *stream)
{
    if (!kv || !norm_weight || !cos_sin || !positions || !slots || !cache || tokens < 1 || num_heads < 0 ||
        num_heads > 4096 || num_positions < 1 || cache_rows < 1 || kv_stride < 0 || !(eps >= 0.0f && eps < INFINITY) ||
        !(cache_scale > 0.0f && cache_scale < INFINITY) || (flags & ~(MLA_FLAG_FP8_CACHE | MLA_FLAG_ROPE_HALVES)) != 0 ||
        (num_heads > 0 && (!q_rope || !q_out || q_token_stride < 0 || q_head_stride < 0)) ||
        (int64_t)tokens * (1 + (num_heads + 15) / 16) > INT32_MAX)
        return MLA_STATUS_INVALID_VALUE;
    if (!aligned16(kv) || !aligned16(norm_weight) || !aligned16(cos_sin) || !aligned16(cache) || kv_stride % 8 != 0 ||
        (num_heads > 0 &&
         (!aligned16(q_rope) || !aligned16(q_out) || q_token_stride % 8 != 0 || q_head_stride % 8 != 0)))
        return MLA_STATUS_MISALIGNED;
    auto launch = bf16 ? launch_append<__bf16> : launch_append<_Float16>;
    launch(kv, norm_weight, cos_sin, positions, slots, q_rope, cache, q_out, eps, cache_scale, tokens, num_heads,
           num_positions, cache_rows, kv_stride, q_token_stride, q_head_stride, flags, static_cast<hipStream_t>(stream));
    const hipError_t e = hipPeekAtLastError();
    return e == hipSuccess ? MLA_STATUS_SUCCESS : record_hip_error(e);
}

}  // namespace
}  // namespace mla

extern "C" {

int mla_paged_tables(const int *context_lens, const int *new_lens, const int *free_pages, const int *free_start,
                     int *block_table, int *cu_seqlens, int *cu_new, long long *slots, int *positions, int *free_next,
                     int batch, int total_new, int num_free, int page_size, int block_table_stride, void *stream)
{
    if (!context_lens || !new_lens || !free_start || !block_table || !cu_seqlens || !cu_new || !free_next ||
        free_next == free_start || (!free_pages && num_free > 0) || ((!slots || !positions) && total_new > 0) ||
        batch < 1 || total_new < 0 || num_free < 0 || page_size < 32 || page_size > (1 << 20) ||
        (page_size & (page_size - 1)) != 0 || block_table_stride < 1)
        return MLA_STATUS_INVALID_VALUE;
    // Each workgroup scans every request again, so no more of them than 4 a CU;
    // its tokens are a multiple of its threads' runs.
    // A thread takes 4 tokens in a row where requests have as many on average (301
    // prompts, 300000 tokens: 6.4 us against 6.6 with one), else one: the
    // pages of 4 requests would be looked up one after another (64 requests
    // of one token: 3.4 us against 4.6).
    const int each = total_new / 4 >= batch ? 4 : 1;
    const int run = mla::kScan * each;
    const int runs = (int)(((int64_t)total_new + run - 1) / run);
    const int most = 4 * mla::current_cu_count();
    const int64_t per_wg = (int64_t)run * std::max(1, (runs + most - 1) / most);
    const int wgs = std::max(1, (int)(((int64_t)total_new + per_wg - 1) / per_wg));
    hipLaunchKernelGGL(mla::paged_tables_kernel, dim3(wgs), dim3(mla::kScan), 0, static_cast<hipStream_t>(stream),
                       context_lens, new_lens, free_pages, free_start, block_table, cu_seqlens, cu_new, slots, positions,
                       free_next, batch, total_new, num_free, __builtin_ctz((unsigned)page_size), block_table_stride,
                       (int)per_wg, each);
    const hipError_t e = hipPeekAtLastError();
    return e == hipSuccess ? MLA_STATUS_SUCCESS : mla::record_hip_error(e);
}

int mla_append_kv_fp16(const void *kv, const void *norm_weight, const float *cos_sin, const int *positions,
                       const long long *slots, const void *q_rope, void *kv_cache, void *q_rope_out, float eps,
                       float cache_scale, int tokens, int num_heads, int num_positions, long long cache_rows,
                       long long kv_stride, long long q_token_stride, long long q_head_stride, unsigned flags,
                       void *stream)
{
    return mla::append_kv(false, kv, norm_weight, cos_sin, positions, slots, q_rope, kv_cache, q_rope_out, eps,
                          cache_scale, tokens, num_heads, num_positions, cache_rows, kv_stride, q_token_stride,
                          q_head_stride, flags, stream);
}

int mla_append_kv_bf16(const void *kv, const void *norm_weight, const float *cos_sin, const int *positions,
                       const long long *slots, const void *q_rope, void *kv_cache, void *q_rope_out, float eps,
                       float cache_scale, int tokens, int num_heads, int num_positions, long long cache_rows,
                       long long kv_stride, long long q_token_stride, long long q_head_stride, unsigned flags,
                       void *stream)
{
    return mla::append_kv(true, kv, norm_weight, cos_sin, positions, slots, q_rope, kv_cache, q_rope_out, eps,
                          cache_scale, tokens, num_heads, num_positions, cache_rows, kv_stride, q_token_stride,
                          q_head_stride, flags, stream);
}

}  // extern "C"
