// PyTorch extension `ada_mla._C`: the Python surface of the reference's
// extension module `ada_mla` (csrc/mla_api.cpp:115-120), with the same
// function names and (query, cache) -> out contract, implemented over the
// C ABI in include/mla_mi355x.h.
//
// Differences from the reference, all on inputs it mishandled:
//  * inputs are validated (device, dtype, rank, 576 columns, num_heads a
//    multiple of 16, N >= 1) and made contiguous; errors raise instead of
//    being printf'd (reference TODOs csrc/mla_api.cpp:8, :18, :91).
//  * kernels run on torch's current HIP stream of the input's device, not
//    the legacy default stream.
//  * mla_decode_split accepts fp32 as well (the reference's fp32 split
//    launcher is an empty stub, csrc/mla_decode_splitk_fwd_sm89.cu:8-24, and
//    returned uninitialised memory); mla_decode_fused accepts fp16 as well
//    (the reference read any dtype as float*, csrc/mla_api.cpp:46-48).
//  * an optional num_splits keyword (default: chosen from N and the CU count).
//  * bf16 query/cache are accepted by mla_decode_split, mla_decode_fused and
//    mla_decode_split_batched (bf16 MFMAs; the reference lists bf16 as
//    future work, README.md:405-408).
//  * mla_decode_split and mla_decode_split_batched also take a float8_e4m3fn
//    cache with a float16 query: the cache holds C / cache_scale (keyword
//    cache_scale, default 1) and is read at one byte per value (fp8 is
//    future work in the reference too, README.md:408); mla_decode_paged takes
//    such a cache with float16 and bfloat16 queries.
#include <torch/extension.h>

#include <cmath>

#include <c10/hip/HIPStream.h>

#include "mla_mi355x.h"

namespace {

void check_status(int st, const char *fn)
{
    TORCH_CHECK(st == MLA_STATUS_SUCCESS, fn, ": ", mla_status_string(st),
                st == MLA_STATUS_HIP_ERROR ? " (hipError_t " + std::to_string(mla_last_hip_error()) + ")"
                                           : std::string());
}

// Shape and dtype are checked before the device so that every argument error
// is reported the same way whatever the tensors' device.
bool is_fp8_cache(const at::Tensor &query, const at::Tensor &cache)
{
    return cache.scalar_type() == at::kFloat8_e4m3fn && query.scalar_type() == at::kHalf;
}

void check_cache_scale(double cache_scale, const char *fn)
{
    TORCH_CHECK(std::isfinite(cache_scale) && cache_scale > 0, fn, ": cache_scale must be finite and > 0, got ",
                cache_scale);
}

void check_pair(const at::Tensor &query, const at::Tensor &cache, const char *fn)
{
    TORCH_CHECK(query.scalar_type() == cache.scalar_type() || is_fp8_cache(query, cache), fn,
                ": query and cache must have the same dtype (or a float16 query with a float8_e4m3fn cache)");
    TORCH_CHECK(query.scalar_type() == at::kHalf || query.scalar_type() == at::kBFloat16 ||
                    query.scalar_type() == at::kFloat,
                fn, ": dtype must be float16, bfloat16 or float32, got ", query.scalar_type());
    TORCH_CHECK(cache.dim() == 2 && cache.size(1) == MLA_HEAD_DIM_K, fn, ": cache must be [N, ",
                MLA_HEAD_DIM_K, "], got ", cache.sizes());
    TORCH_CHECK(cache.size(0) >= 1, fn, ": cache must hold at least one token");
    TORCH_CHECK(cache.size(0) <= INT32_MAX, fn, ": too many tokens");
    TORCH_CHECK(query.dim() == 2 && query.size(1) == MLA_HEAD_DIM_K, fn,
                ": query must be [num_heads, ", MLA_HEAD_DIM_K, "], got ", query.sizes());
    TORCH_CHECK(query.size(0) > 0 && query.size(0) % 16 == 0 && query.size(0) <= 4096, fn,
                ": num_heads must be a positive multiple of 16 (<= 4096), got ", query.size(0));
    TORCH_CHECK(query.is_cuda() && cache.is_cuda(), fn, ": query and cache must be GPU tensors");
    TORCH_CHECK(query.device() == cache.device(), fn, ": query and cache must be on the same device");
}

void check_heads(int64_t num_heads, const char *fn)
{
    TORCH_CHECK(num_heads > 0 && num_heads % 16 == 0 && num_heads <= 4096, fn,
                ": num_heads must be a positive multiple of 16 (<= 4096), got ", num_heads);
}

void *stream_of(const at::Tensor &t)
{
    return static_cast<void *>(c10::hip::getCurrentHIPStream(t.device().index()).stream());
}

at::Tensor workspace(size_t bytes, const at::Tensor &like)
{
    return at::empty({static_cast<int64_t>(bytes)}, like.options().dtype(at::kByte));
}

// Single sequence, dispatch on dtype.
at::Tensor decode_single(const at::Tensor &query_in, const at::Tensor &cache_in, int64_t num_splits,
                         double cache_scale, const char *fn)
{
    const bool fp8 = is_fp8_cache(query_in, cache_in);
    if (fp8)
        check_cache_scale(cache_scale, fn);
    check_pair(query_in, cache_in, fn);
    const at::OptionalDeviceGuard guard(query_in.device());
    const at::Tensor query = query_in.contiguous();
    const at::Tensor cache = cache_in.contiguous();
    const int nh = static_cast<int>(query.size(0));
    const int n = static_cast<int>(cache.size(0));
    const int splits = static_cast<int>(num_splits);
    at::Tensor out = at::empty({nh, MLA_HEAD_DIM_V}, query.options());
    int st;
    if (fp8) {
        const size_t ws_bytes = mla_decode_split_fp8_workspace_size(1, nh, n, splits);
        TORCH_CHECK(ws_bytes > 0, fn, ": unsupported sizes");
        at::Tensor ws = workspace(ws_bytes, query);
        st = mla_decode_split_fp8(query.data_ptr(), cache.data_ptr(), static_cast<float>(cache_scale),
                                  out.data_ptr(), ws.data_ptr(), ws_bytes, nh, n, splits, stream_of(query));
    } else if (query.scalar_type() != at::kFloat) {
        const size_t ws_bytes = mla_decode_split_workspace_size(nh, n, splits);
        TORCH_CHECK(ws_bytes > 0, fn, ": unsupported sizes");
        at::Tensor ws = workspace(ws_bytes, query);
        auto f = query.scalar_type() == at::kHalf ? mla_decode_split_fp16 : mla_decode_split_bf16;
        st = f(query.data_ptr(), cache.data_ptr(), out.data_ptr(), ws.data_ptr(), ws_bytes, nh, n, splits,
               stream_of(query));
    } else {
        const size_t ws_bytes = mla_decode_fused_workspace_size(nh, n, splits);
        TORCH_CHECK(ws_bytes > 0, fn, ": unsupported sizes");
        at::Tensor ws = workspace(ws_bytes, query);
        st = mla_decode_fused_fp32(query.data_ptr<float>(), cache.data_ptr<float>(), out.data_ptr<float>(),
                                   ws.data_ptr(), ws_bytes, nh, MLA_HEAD_DIM_K, n, splits,
                                   stream_of(query));
    }
    check_status(st, fn);
    return out;
}

// Reference: mla_decode_split (csrc/mla_api.cpp:86-113), the fp16 `-k fused`
// path of mla.py (mla.py:177-179).
at::Tensor mla_decode_split(const at::Tensor &query, const at::Tensor &cache, int64_t num_splits,
                            double cache_scale)
{
    return decode_single(query, cache, num_splits, cache_scale, "mla_decode_split");
}

// Reference: mla_decode_fused (csrc/mla_api.cpp:34-54), the `-k fused --fp32`
// path of mla.py (mla.py:174-176).
at::Tensor mla_decode_fused(const at::Tensor &query, const at::Tensor &cache, int64_t num_splits)
{
    TORCH_CHECK(cache.scalar_type() != at::kFloat8_e4m3fn, "mla_decode_fused: fp8 caches go through mla_decode_split");
    return decode_single(query, cache, num_splits, 1.0, "mla_decode_fused");
}

// No reference counterpart: B independent sequences packed back to back.
at::Tensor mla_decode_split_batched(const at::Tensor &query_in, const at::Tensor &cache_in,
                                    const at::Tensor &cu_seqlens_in, int64_t num_splits, double cache_scale)
{
    const char *fn = "mla_decode_split_batched";
    const bool fp8 = is_fp8_cache(query_in, cache_in);
    TORCH_CHECK(fp8 || (query_in.scalar_type() == cache_in.scalar_type() &&
                        (query_in.scalar_type() == at::kHalf || query_in.scalar_type() == at::kBFloat16)),
                fn, ": query and cache must both be float16 or both bfloat16 (or a float16 query with a "
                "float8_e4m3fn cache)");
    if (fp8)
        check_cache_scale(cache_scale, fn);
    TORCH_CHECK(cu_seqlens_in.scalar_type() == at::kInt && cu_seqlens_in.dim() == 1, fn,
                ": cu_seqlens must be a 1-D int32 tensor");
    TORCH_CHECK(query_in.dim() == 3 && query_in.size(2) == MLA_HEAD_DIM_K, fn,
                ": query must be [batch, num_heads, ", MLA_HEAD_DIM_K, "], got ", query_in.sizes());
    TORCH_CHECK(cache_in.dim() == 2 && cache_in.size(1) == MLA_HEAD_DIM_K, fn, ": cache must be [total, ",
                MLA_HEAD_DIM_K, "], got ", cache_in.sizes());
    TORCH_CHECK(query_in.size(0) >= 1 && cu_seqlens_in.size(0) == query_in.size(0) + 1, fn,
                ": cu_seqlens must have batch + 1 entries");
    TORCH_CHECK(cache_in.size(0) <= INT32_MAX, fn, ": too many tokens");
    check_heads(query_in.size(1), fn);
    TORCH_CHECK(query_in.is_cuda() && cache_in.is_cuda() && cu_seqlens_in.is_cuda(), fn,
                ": query, cache and cu_seqlens must be GPU tensors");
    TORCH_CHECK(query_in.device() == cache_in.device() && query_in.device() == cu_seqlens_in.device(), fn,
                ": all inputs must be on the same device");
    const at::OptionalDeviceGuard guard(query_in.device());
    const at::Tensor query = query_in.contiguous();
    const at::Tensor cache = cache_in.contiguous();
    const at::Tensor cu = cu_seqlens_in.contiguous();
    const int batch = static_cast<int>(query.size(0));
    const int nh = static_cast<int>(query.size(1));
    const int total = static_cast<int>(cache.size(0));
    const int splits = static_cast<int>(num_splits);
    at::Tensor out = at::empty({batch, nh, MLA_HEAD_DIM_V}, query.options());
    const size_t ws_bytes = fp8 ? mla_decode_split_fp8_workspace_size(batch, nh, total, splits)
                                : mla_decode_split_batched_workspace_size(batch, nh, total, splits);
    TORCH_CHECK(ws_bytes > 0, fn, ": unsupported sizes");
    at::Tensor ws = workspace(ws_bytes, query);
    const void *c = total > 0 ? cache.data_ptr() : nullptr;
    int st;
    if (fp8) {
        st = mla_decode_split_batched_fp8(query.data_ptr(), c, static_cast<float>(cache_scale), cu.data_ptr<int>(),
                                          out.data_ptr(), ws.data_ptr(), ws_bytes, batch, nh, total, splits,
                                          stream_of(query));
    } else {
        auto f = query.scalar_type() == at::kHalf ? mla_decode_split_batched_fp16 : mla_decode_split_batched_bf16;
        st = f(query.data_ptr(), c, cu.data_ptr<int>(), out.data_ptr(), ws.data_ptr(), ws_bytes, batch, nh, total,
               splits, stream_of(query));
    }
    check_status(st, fn);
    return out;
}

// No reference counterpart: a paged KV cache [num_pages, page_size, 576]
// addressed through block_table [batch, max_pages] (int32), with the
// sequences' lengths as prefix sums cu_seqlens [batch + 1] (int32).
// total_tokens (= cu_seqlens[batch]) is read from the device when not given,
// which synchronises the stream. A given total_tokens is not checked against
// cu_seqlens[batch]: sequences are clipped to [0, total_tokens), so a smaller
// value silently truncates the trailing sequences; a larger one only changes
// the split plan.
at::Tensor mla_decode_paged(const at::Tensor &query_in, const at::Tensor &kv_in,
                            const at::Tensor &block_table_in, const at::Tensor &cu_seqlens_in,
                            int64_t total_tokens, int64_t num_splits, double cache_scale)
{
    const char *fn = "mla_decode_paged";
    const bool fp8 = kv_in.scalar_type() == at::kFloat8_e4m3fn;
    TORCH_CHECK((fp8 || query_in.scalar_type() == kv_in.scalar_type()) &&
                    (query_in.scalar_type() == at::kHalf || query_in.scalar_type() == at::kBFloat16),
                fn, ": query and kv_cache must both be float16 or both bfloat16 (or a float8_e4m3fn kv_cache with "
                "either)");
    check_cache_scale(cache_scale, fn);
    TORCH_CHECK(fp8 || cache_scale == 1.0, fn, ": cache_scale is for a float8_e4m3fn cache");
    TORCH_CHECK(block_table_in.scalar_type() == at::kInt && block_table_in.dim() == 2, fn,
                ": block_table must be a 2-D int32 tensor");
    TORCH_CHECK(cu_seqlens_in.scalar_type() == at::kInt && cu_seqlens_in.dim() == 1, fn,
                ": cu_seqlens must be a 1-D int32 tensor");
    TORCH_CHECK(query_in.dim() == 3 && query_in.size(2) == MLA_HEAD_DIM_K, fn,
                ": query must be [batch, num_heads, ", MLA_HEAD_DIM_K, "], got ", query_in.sizes());
    TORCH_CHECK(kv_in.dim() == 3 && kv_in.size(2) == MLA_HEAD_DIM_K && kv_in.size(0) >= 1, fn,
                ": kv_cache must be [num_pages >= 1, page_size, ", MLA_HEAD_DIM_K, "], got ", kv_in.sizes());
    const int64_t page = kv_in.size(1);
    TORCH_CHECK(page >= 32 && (page & (page - 1)) == 0, fn, ": page_size must be a power of two >= 32, got ",
                page);
    TORCH_CHECK(kv_in.size(0) <= INT32_MAX, fn, ": too many pages");
    const int64_t batch = query_in.size(0);
    TORCH_CHECK(batch >= 1 && cu_seqlens_in.size(0) == batch + 1 && block_table_in.size(0) == batch, fn,
                ": cu_seqlens must have batch + 1 entries and block_table batch rows");
    TORCH_CHECK(block_table_in.size(1) >= 1, fn, ": block_table needs at least one column");
    check_heads(query_in.size(1), fn);
    TORCH_CHECK(query_in.is_cuda() && kv_in.is_cuda() && block_table_in.is_cuda() && cu_seqlens_in.is_cuda(), fn,
                ": all inputs must be GPU tensors");
    TORCH_CHECK(query_in.device() == kv_in.device() && query_in.device() == block_table_in.device() &&
                    query_in.device() == cu_seqlens_in.device(),
                fn, ": all inputs must be on the same device");
    const at::OptionalDeviceGuard guard(query_in.device());
    const at::Tensor query = query_in.contiguous();
    const at::Tensor kv = kv_in.contiguous();
    const at::Tensor bt = block_table_in.contiguous();
    const at::Tensor cu = cu_seqlens_in.contiguous();
    if (total_tokens < 0)
        total_tokens = cu[batch].item<int>();
    TORCH_CHECK(total_tokens >= 0 && total_tokens <= INT32_MAX, fn, ": bad total_tokens ", total_tokens);
    const int nh = static_cast<int>(query.size(1));
    const int total = static_cast<int>(total_tokens);
    const int splits = static_cast<int>(num_splits);
    at::Tensor out = at::empty({batch, nh, MLA_HEAD_DIM_V}, query.options());
    const size_t ws_bytes = (fp8 ? mla_decode_paged_fp8_workspace_size
                                 : mla_decode_paged_workspace_size)(static_cast<int>(batch), nh, total, splits);
    TORCH_CHECK(ws_bytes > 0, fn, ": unsupported sizes");
    at::Tensor ws = workspace(ws_bytes, query);
    const bool half = query.scalar_type() == at::kHalf;
    int st;
    if (fp8) {
        auto f = half ? mla_decode_paged_fp8_fp16 : mla_decode_paged_fp8_bf16;
        st = f(query.data_ptr(), kv.data_ptr(), static_cast<float>(cache_scale), bt.data_ptr<int>(), cu.data_ptr<int>(),
               out.data_ptr(), ws.data_ptr(), ws_bytes, static_cast<int>(batch), nh, total, static_cast<int>(page),
               static_cast<int>(kv.size(0)), static_cast<int>(bt.size(1)), splits, stream_of(query));
    } else {
        auto f = half ? mla_decode_paged_fp16 : mla_decode_paged_bf16;
        st = f(query.data_ptr(), kv.data_ptr(), bt.data_ptr<int>(), cu.data_ptr<int>(), out.data_ptr(),
               ws.data_ptr(), ws_bytes, static_cast<int>(batch), nh, total, static_cast<int>(page),
               static_cast<int>(kv.size(0)), static_cast<int>(bt.size(1)), splits, stream_of(query));
    }
    check_status(st, fn);
    return out;
}

void check_16bit(const at::Tensor &t, at::ScalarType dt, const char *fn, const char *name)
{
    TORCH_CHECK(t.scalar_type() == dt, fn, ": ", name, " must have the query's dtype (float16 or bfloat16)");
    TORCH_CHECK(t.is_cuda(), fn, ": ", name, " must be a GPU tensor");
}

// No reference code (the math is README.md:76-85): Q* = [q_nope W_UK[h], q_rope].
at::Tensor mla_absorb_query(const at::Tensor &q_nope_in, const at::Tensor &q_rope_in, const at::Tensor &w_uk_in)
{
    const char *fn = "mla_absorb_query";
    const auto dt = q_nope_in.scalar_type();
    TORCH_CHECK(dt == at::kHalf || dt == at::kBFloat16, fn, ": q_nope must be float16 or bfloat16");
    TORCH_CHECK(q_nope_in.dim() == 3 && q_nope_in.size(2) == 128 && q_nope_in.size(0) >= 1, fn,
                ": q_nope must be [batch, num_heads, 128], got ", q_nope_in.sizes());
    const int64_t b = q_nope_in.size(0), nh = q_nope_in.size(1);
    TORCH_CHECK(q_rope_in.dim() == 3 && q_rope_in.size(0) == b && q_rope_in.size(1) == nh && q_rope_in.size(2) == 64,
                fn, ": q_rope must be [batch, num_heads, 64], got ", q_rope_in.sizes());
    TORCH_CHECK(w_uk_in.dim() == 3 && w_uk_in.size(0) == nh && w_uk_in.size(1) == 128 && w_uk_in.size(2) == 512, fn,
                ": w_uk must be [num_heads, 128, 512], got ", w_uk_in.sizes());
    check_16bit(q_nope_in, dt, fn, "q_nope");
    check_16bit(q_rope_in, dt, fn, "q_rope");
    check_16bit(w_uk_in, dt, fn, "w_uk");
    const at::OptionalDeviceGuard guard(q_nope_in.device());
    const at::Tensor qn = q_nope_in.contiguous(), qr = q_rope_in.contiguous(), w = w_uk_in.contiguous();
    at::Tensor out = at::empty({b, nh, MLA_HEAD_DIM_K}, qn.options());
    auto f = dt == at::kHalf ? mla_absorb_query_fp16 : mla_absorb_query_bf16;
    check_status(f(qn.data_ptr(), qr.data_ptr(), w.data_ptr(), out.data_ptr(), static_cast<int>(b),
                   static_cast<int>(nh), stream_of(qn)),
                 fn);
    return out;
}

// No reference code (README.md:84-85): out = concat_h(O*[:, h] W_UV[h]^T) W_O^T.
at::Tensor mla_project_output(const at::Tensor &o_in, const at::Tensor &w_uv_in, const at::Tensor &w_o_in)
{
    const char *fn = "mla_project_output";
    const auto dt = o_in.scalar_type();
    TORCH_CHECK(dt == at::kHalf || dt == at::kBFloat16, fn, ": o_star must be float16 or bfloat16");
    TORCH_CHECK(o_in.dim() == 3 && o_in.size(2) == MLA_HEAD_DIM_V && o_in.size(0) >= 1, fn,
                ": o_star must be [batch, num_heads, 512], got ", o_in.sizes());
    const int64_t b = o_in.size(0), nh = o_in.size(1);
    TORCH_CHECK(w_uv_in.dim() == 3 && w_uv_in.size(0) == nh && w_uv_in.size(1) == 128 && w_uv_in.size(2) == 512, fn,
                ": w_uv must be [num_heads, 128, 512], got ", w_uv_in.sizes());
    TORCH_CHECK(w_o_in.dim() == 2 && w_o_in.size(1) == nh * 128 && w_o_in.size(0) >= 1, fn,
                ": w_o must be [d_model, num_heads * 128], got ", w_o_in.sizes());
    check_16bit(o_in, dt, fn, "o_star");
    check_16bit(w_uv_in, dt, fn, "w_uv");
    check_16bit(w_o_in, dt, fn, "w_o");
    const at::OptionalDeviceGuard guard(o_in.device());
    const at::Tensor o = o_in.contiguous(), wuv = w_uv_in.contiguous(), wo = w_o_in.contiguous();
    const int64_t d_model = wo.size(0);
    at::Tensor out = at::empty({b, d_model}, o.options());
    const size_t ws_bytes = mla_project_output_workspace_size(static_cast<int>(b), static_cast<int>(nh), static_cast<int>(d_model));
    TORCH_CHECK(ws_bytes > 0, fn, ": unsupported sizes");
    at::Tensor ws = workspace(ws_bytes, o);
    auto f = dt == at::kHalf ? mla_project_output_fp16 : mla_project_output_bf16;
    check_status(f(o.data_ptr(), wuv.data_ptr(), wo.data_ptr(), out.data_ptr(), ws.data_ptr(), ws_bytes,
                   static_cast<int>(b), static_cast<int>(nh), static_cast<int>(d_model), stream_of(o)),
                 fn);
    return out;
}

void check_int32(const at::Tensor &t, int64_t dim, const char *fn, const char *name)
{
    TORCH_CHECK(t.scalar_type() == at::kInt && t.dim() == dim, fn, ": ", name, " must be a ", dim, "-D int32 tensor");
}

void check_page_size(int64_t page, const char *fn)
{
    TORCH_CHECK(page >= 32 && page <= (1 << 20) && (page & (page - 1)) == 0, fn,
                ": page_size must be a power of two from 32 to 2^20, got ", page);
}

// Every tensor on the first one's GPU.
void check_devices(std::initializer_list<const at::Tensor *> tensors, const char *fn)
{
    const at::Tensor &first = **tensors.begin();
    for (const at::Tensor *t : tensors) {
        TORCH_CHECK(t->is_cuda(), fn, ": all inputs must be GPU tensors");
        TORCH_CHECK(t->device() == first.device(), fn, ": all inputs must be on the same device");
    }
}

// cu_seqlens[batch] where the caller has not given it (this waits for the stream).
int64_t given_total(int64_t total_tokens, const at::Tensor &cu, const char *fn)
{
    if (total_tokens < 0)
        total_tokens = cu[cu.size(0) - 1].item<int>();
    TORCH_CHECK(total_tokens >= 0 && total_tokens <= INT32_MAX, fn, ": bad total_tokens ", total_tokens);
    return total_tokens;
}

bool starts_aligned(const at::Tensor &t) { return reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0; }

// A contiguous tensor that starts at a multiple of 16 bytes: the same one, else a
// copy. (A contiguous view into a buffer may start anywhere, and contiguous()
// returns it as it is.)
at::Tensor readable(const at::Tensor &t)
{
    const at::Tensor c = t.contiguous();
    return starts_aligned(c) ? c : c.clone(at::MemoryFormat::Contiguous);
}

// A tensor whose rows the kernels can read in place: the last dimension
// contiguous, the others' strides multiples of 16 bytes, the start aligned;
// else a contiguous copy.
at::Tensor readable_rows(const at::Tensor &t)
{
    bool ok = starts_aligned(t) && t.stride(-1) == 1;
    for (int64_t d = 0; d + 1 < t.dim(); ++d)
        ok = ok && (t.size(d) == 1 || t.stride(d) % 8 == 0);
    return ok ? t : readable(t);
}

// A stride that the C ABI takes: that of a dimension of one entry is never used.
int64_t used_stride(const at::Tensor &t, int64_t d, int64_t least)
{
    return t.size(d) == 1 ? least : t.stride(d);
}

// A contiguous 1-D tensor of n entries in base's storage, `at` bytes into it: the small
// outputs of a call share one allocation, which costs a call as much host time as all of them.
at::Tensor part_of(const at::Tensor &base, size_t at_bytes, int64_t n, at::ScalarType type)
{
    at::Tensor t = at::detail::make_tensor<c10::TensorImpl>(c10::Storage(base.storage()), base.key_set(),
                                                            c10::scalarTypeToTypeMeta(type));
    t.unsafeGetTensorImpl()->set_sizes_contiguous({n});
    t.unsafeGetTensorImpl()->set_storage_offset(static_cast<int64_t>(at_bytes / c10::elementSize(type)));
    return t;
}

// No reference counterpart: block table, slots and positions of a step's tokens.
std::vector<at::Tensor> paged_tables(const at::Tensor &context_in, const at::Tensor &new_in, at::Tensor block_table,
                                         const at::Tensor &free_pages_in, const at::Tensor &free_start_in,
                                         int64_t page_size, int64_t total_new)
{
    const char *fn = "mla_paged_tables";
    check_int32(context_in, 1, fn, "context_lens");
    check_int32(new_in, 1, fn, "new_lens");
    check_int32(block_table, 2, fn, "block_table");
    check_int32(free_pages_in, 1, fn, "free_pages");
    check_int32(free_start_in, 1, fn, "free_start");
    const int64_t batch = context_in.size(0);
    TORCH_CHECK(batch >= 1 && batch <= INT32_MAX - 1 && new_in.size(0) == batch && block_table.size(0) == batch, fn,
                ": context_lens, new_lens and block_table must have one entry or row per request");
    TORCH_CHECK(block_table.size(1) >= 1 && block_table.size(1) <= INT32_MAX, fn, ": block_table needs at least one column");
    TORCH_CHECK(block_table.is_contiguous(), fn, ": block_table must be contiguous (it is written in place)");
    TORCH_CHECK(free_start_in.size(0) == 1, fn, ": free_start must have one entry");
    TORCH_CHECK(free_pages_in.size(0) <= INT32_MAX, fn, ": too many free pages");
    TORCH_CHECK(total_new >= 0 && total_new <= INT32_MAX, fn, ": bad total_new ", total_new);
    check_page_size(page_size, fn);
    check_devices({&context_in, &new_in, &block_table, &free_pages_in, &free_start_in}, fn);
    const at::OptionalDeviceGuard guard(context_in.device());
    const at::Tensor context = context_in.contiguous(), fresh = new_in.contiguous(), pages = free_pages_in.contiguous();
    // slots, then positions, cu_seqlens, cu_new and free_next, each from a multiple of 16 bytes on
    auto up = [](int64_t n) { return static_cast<size_t>((n + 15) / 16 * 16); };
    const size_t at_pos = up(8 * total_new), at_cu = at_pos + up(4 * total_new), at_new = at_cu + up(4 * (batch + 1));
    const size_t at_next = at_new + up(4 * (batch + 1));
    const at::Tensor all = workspace(at_next + 16, context);
    at::Tensor slots = part_of(all, 0, total_new, at::kLong), positions = part_of(all, at_pos, total_new, at::kInt);
    at::Tensor cu_seqlens = part_of(all, at_cu, batch + 1, at::kInt), cu_new = part_of(all, at_new, batch + 1, at::kInt);
    at::Tensor free_next = part_of(all, at_next, 1, at::kInt);
    check_status(mla_paged_tables(context.data_ptr<int>(), fresh.data_ptr<int>(), pages.data_ptr<int>(),
                                    free_start_in.data_ptr<int>(), block_table.data_ptr<int>(),
                                    cu_seqlens.data_ptr<int>(), cu_new.data_ptr<int>(),
                                    reinterpret_cast<long long *>(slots.data_ptr<int64_t>()), positions.data_ptr<int>(),
                                    free_next.data_ptr<int>(), static_cast<int>(batch), static_cast<int>(total_new),
                                    static_cast<int>(pages.size(0)), static_cast<int>(page_size),
                                    static_cast<int>(block_table.size(1)), stream_of(context)),
                 fn);
    return {cu_seqlens, cu_new, slots, positions, free_next};
}

// What fork and compaction check of a table and its pool.
void check_pool(const at::Tensor &table, const at::Tensor &lens, const at::Tensor &free_pages, const at::Tensor &free_start,
                const c10::optional<at::Tensor> &pinned, int64_t page_size, int64_t num_pages, const char *fn)
{
    check_int32(table, 2, fn, "block_table");
    check_int32(lens, 1, fn, "lens");
    check_int32(free_pages, 1, fn, "free_pages");
    check_int32(free_start, 1, fn, "free_start");
    TORCH_CHECK(table.size(0) >= 1 && table.size(0) <= 8192 && lens.size(0) == table.size(0), fn,
                ": lens and block_table must have one entry or row per request, 8192 at most");
    TORCH_CHECK(table.size(1) >= 1 && table.size(1) <= (1 << 20), fn, ": block_table needs at least one column (and 2^20 at most)");
    TORCH_CHECK(free_pages.size(0) <= INT32_MAX, fn, ": too many free pages");
    TORCH_CHECK(free_start.size(0) == 1, fn, ": free_start must have one entry");
    check_page_size(page_size, fn);
    TORCH_CHECK(num_pages >= 1 && num_pages <= (1 << 18), fn, ": num_pages must be 1 to 2^18, got ", num_pages);
    if (pinned) {
        check_int32(*pinned, 1, fn, "pinned");
        TORCH_CHECK(pinned->size(0) == num_pages, fn, ": pinned must have one entry per page");
    }
    check_devices({&table, &lens, &free_pages, &free_start, pinned ? &*pinned : &table}, fn);
}

// No reference counterpart: rows of a block table taken over from others.
std::vector<at::Tensor> fork_tables(const at::Tensor &table_in, const at::Tensor &lens_in, const at::Tensor &parents_in,
                                    at::Tensor free_pages, const at::Tensor &free_start, int64_t page_size,
                                    int64_t num_pages, const c10::optional<at::Tensor> &kept_in,
                                    const c10::optional<at::Tensor> &pinned_in)
{
    const char *fn = "mla_fork_tables";
    check_int32(parents_in, 1, fn, "parents");
    const int64_t batch = parents_in.size(0);
    TORCH_CHECK(batch >= 1 && batch <= INT32_MAX / 4, fn, ": parents must have at least one entry");
    if (kept_in) {
        check_int32(*kept_in, 1, fn, "kept_lens");
        TORCH_CHECK(kept_in->size(0) == batch, fn, ": kept_lens must have one entry per parent");
    }
    TORCH_CHECK(free_pages.is_contiguous(), fn, ": free_pages must be contiguous (it is written in place)");
    check_pool(table_in, lens_in, free_pages, free_start, pinned_in, page_size, num_pages, fn);
    check_devices({&table_in, &parents_in, kept_in ? &*kept_in : &table_in}, fn);
    const at::OptionalDeviceGuard guard(table_in.device());
    const at::Tensor table = table_in.contiguous(), lens = lens_in.contiguous(), parents = parents_in.contiguous();
    const at::Tensor kept = kept_in ? kept_in->contiguous() : at::Tensor();
    const at::Tensor pinned = pinned_in ? pinned_in->contiguous() : at::Tensor();
    const int64_t width = table.size(1);
    // the outputs and the workspace share one allocation, each from a multiple of 16 bytes on
    auto up = [](int64_t n) { return static_cast<size_t>((n + 15) / 16 * 16); };
    const size_t ws_bytes = mla_page_tables_workspace_size(static_cast<int>(num_pages));
    const size_t at_lens = up(4 * batch * width), at_copies = at_lens + up(4 * batch), at_next = at_copies + up(12 * batch);
    const at::Tensor all = workspace(at_next + 16, table), ws = workspace(ws_bytes, table);
    at::Tensor new_table = part_of(all, 0, batch * width, at::kInt).view({batch, width});
    at::Tensor new_lens = part_of(all, at_lens, batch, at::kInt);
    at::Tensor copies = part_of(all, at_copies, 3 * batch, at::kInt).view({batch, 3});
    at::Tensor free_next = part_of(all, at_next, 1, at::kInt);
    check_status(mla_fork_tables(table.data_ptr<int>(), lens.data_ptr<int>(), parents.data_ptr<int>(),
                                 kept_in ? kept.data_ptr<int>() : nullptr, pinned_in ? pinned.data_ptr<int>() : nullptr,
                                 free_pages.data_ptr<int>(), free_start.data_ptr<int>(), new_table.data_ptr<int>(),
                                 new_lens.data_ptr<int>(), copies.data_ptr<int>(), free_next.data_ptr<int>(), ws.data_ptr(),
                                 ws_bytes, static_cast<int>(table.size(0)), static_cast<int>(batch),
                                 static_cast<int>(num_pages), static_cast<int>(free_pages.size(0)),
                                 static_cast<int>(page_size), static_cast<int>(width), stream_of(table)),
                 fn);
    return {new_table, new_lens, copies, free_next};
}

// No reference counterpart: a pool's used pages moved to its lowest ids.
std::vector<at::Tensor> compact_tables(const at::Tensor &table_in, const at::Tensor &lens_in, const at::Tensor &free_in,
                                       const at::Tensor &free_start, int64_t page_size, int64_t num_pages,
                                       const c10::optional<at::Tensor> &pinned_in)
{
    const char *fn = "mla_compact_tables";
    check_pool(table_in, lens_in, free_in, free_start, pinned_in, page_size, num_pages, fn);
    const at::OptionalDeviceGuard guard(table_in.device());
    const at::Tensor table = table_in.contiguous(), lens = lens_in.contiguous(), free_pages = free_in.contiguous();
    const at::Tensor pinned = pinned_in ? pinned_in->contiguous() : at::Tensor();
    const int64_t num_free = free_pages.size(0), moves = std::min(num_free, num_pages / 2);
    at::Tensor new_table = at::empty(table.sizes(), table.options()), copies = at::empty({moves, 3}, table.options());
    at::Tensor new_free = at::empty({num_free}, table.options());
    const size_t ws_bytes = mla_page_tables_workspace_size(static_cast<int>(num_pages));
    const at::Tensor ws = workspace(ws_bytes, table);
    check_status(mla_compact_tables(table.data_ptr<int>(), lens.data_ptr<int>(), pinned_in ? pinned.data_ptr<int>() : nullptr,
                                    free_pages.data_ptr<int>(), free_start.data_ptr<int>(), new_table.data_ptr<int>(),
                                    copies.data_ptr<int>(), new_free.data_ptr<int>(), ws.data_ptr(), ws_bytes,
                                    static_cast<int>(table.size(0)), static_cast<int>(num_pages),
                                    static_cast<int>(num_free), static_cast<int>(page_size),
                                    static_cast<int>(table.size(1)), stream_of(table)),
                 fn);
    return {new_table, copies, new_free};
}

// No reference counterpart: the copies that either asks for, in every layer's cache.
void copy_pages(at::Tensor kv_cache, const at::Tensor &copies_in)
{
    const char *fn = "mla_copy_pages";
    TORCH_CHECK((kv_cache.dim() == 3 || kv_cache.dim() == 4) && kv_cache.size(-1) == MLA_HEAD_DIM_K && kv_cache.numel() > 0,
                fn, ": kv_cache must be [num_pages, page_size, ", MLA_HEAD_DIM_K, "] or [layers, num_pages, page_size, ",
                MLA_HEAD_DIM_K, "], got ", kv_cache.sizes());
    TORCH_CHECK(kv_cache.is_contiguous(), fn, ": kv_cache must be contiguous (it is written in place)");
    const int64_t size = kv_cache.element_size(), layers = kv_cache.dim() == 4 ? kv_cache.size(0) : 1;
    TORCH_CHECK(size == 1 || size == 2 || size == 4, fn, ": kv_cache must have elements of 1, 2 or 4 bytes");
    check_page_size(kv_cache.size(-2), fn);
    TORCH_CHECK(layers <= INT32_MAX && kv_cache.size(-3) <= INT32_MAX, fn, ": too many pages or layers");
    check_int32(copies_in, 2, fn, "copies");
    TORCH_CHECK(copies_in.size(1) == 3 && copies_in.size(0) <= INT32_MAX / 4, fn, ": copies must be [n, 3]");
    check_devices({&kv_cache, &copies_in}, fn);
    const at::OptionalDeviceGuard guard(kv_cache.device());
    const at::Tensor copies = copies_in.contiguous();
    check_status(mla_copy_pages(kv_cache.data_ptr(), copies.data_ptr<int>(), static_cast<int>(copies.size(0)),
                                static_cast<int>(layers), static_cast<int>(kv_cache.size(-3)),
                                static_cast<int>(kv_cache.size(-2)), static_cast<int>(size), stream_of(kv_cache)),
                 fn);
}

// No reference counterpart: a step's latent rows normalised, rotated and
// written to their slots of the cache, its queries' rotary parts rotated.
c10::optional<at::Tensor> mla_append_kv(const at::Tensor &kv_in, const at::Tensor &weight_in,
                                        const at::Tensor &cos_sin_in, const at::Tensor &positions_in,
                                        const at::Tensor &slots_in, at::Tensor kv_cache,
                                        const c10::optional<at::Tensor> &q_rope_in, double eps, double cache_scale,
                                        bool interleaved)
{
    const char *fn = "mla_append_kv";
    const auto dt = kv_in.scalar_type();
    TORCH_CHECK(dt == at::kHalf || dt == at::kBFloat16, fn, ": kv must be float16 or bfloat16");
    TORCH_CHECK(kv_in.dim() == 2 && kv_in.size(1) == MLA_HEAD_DIM_K && kv_in.size(0) <= INT32_MAX, fn,
                ": kv must be [tokens, ", MLA_HEAD_DIM_K, "], got ", kv_in.sizes());
    const int64_t tokens = kv_in.size(0);
    const bool fp8 = kv_cache.scalar_type() == at::kFloat8_e4m3fn;
    TORCH_CHECK(fp8 || kv_cache.scalar_type() == dt, fn, ": kv_cache must have kv's dtype or be float8_e4m3fn");
    TORCH_CHECK((kv_cache.dim() == 2 || kv_cache.dim() == 3) && kv_cache.size(-1) == MLA_HEAD_DIM_K &&
                    kv_cache.numel() > 0,
                fn, ": kv_cache must be [rows, ", MLA_HEAD_DIM_K, "] or [num_pages, page_size, ", MLA_HEAD_DIM_K,
                "], got ", kv_cache.sizes());
    TORCH_CHECK(kv_cache.is_contiguous(), fn, ": kv_cache must be contiguous (it is written in place)");
    TORCH_CHECK(weight_in.scalar_type() == dt && weight_in.dim() == 1 && weight_in.size(0) == MLA_HEAD_DIM_V, fn,
                ": norm_weight must be [", MLA_HEAD_DIM_V, "] of kv's dtype");
    TORCH_CHECK(cos_sin_in.scalar_type() == at::kFloat && cos_sin_in.dim() == 2 && cos_sin_in.size(1) == 64 &&
                    cos_sin_in.size(0) >= 1 && cos_sin_in.size(0) <= INT32_MAX,
                fn, ": cos_sin must be a float32 tensor [positions, 64]");
    check_int32(positions_in, 1, fn, "positions");
    TORCH_CHECK(slots_in.scalar_type() == at::kLong && slots_in.dim() == 1, fn, ": slots must be a 1-D int64 tensor");
    TORCH_CHECK(positions_in.size(0) == tokens && slots_in.size(0) == tokens, fn,
                ": positions and slots must have one entry per token");
    TORCH_CHECK(std::isfinite(eps) && eps >= 0, fn, ": eps must be finite and >= 0, got ", eps);
    check_cache_scale(cache_scale, fn);
    TORCH_CHECK(fp8 || cache_scale == 1.0, fn, ": cache_scale is for a float8_e4m3fn cache");
    int64_t heads = 0;
    if (q_rope_in) {
        TORCH_CHECK(q_rope_in->dim() == 3 && q_rope_in->size(0) == tokens && q_rope_in->size(2) == 64 &&
                        q_rope_in->size(1) >= 1 && q_rope_in->size(1) <= 4096,
                    fn, ": q_rope must be [tokens, num_heads (1 to 4096), 64], got ", q_rope_in->sizes());
        TORCH_CHECK(q_rope_in->scalar_type() == dt, fn, ": q_rope must have kv's dtype");
        heads = q_rope_in->size(1);
    }
    check_devices({&kv_in, &weight_in, &cos_sin_in, &positions_in, &slots_in, &kv_cache,
                   q_rope_in ? &*q_rope_in : &kv_in}, fn);
    const at::OptionalDeviceGuard guard(kv_in.device());
    c10::optional<at::Tensor> out;
    if (q_rope_in)
        out = at::empty({tokens, heads, 64}, q_rope_in->options().memory_format(at::MemoryFormat::Contiguous));
    if (tokens == 0)
        return out;
    const at::Tensor kv = readable_rows(kv_in), weight = readable_rows(weight_in), cos_sin = readable(cos_sin_in);
    const at::Tensor positions = positions_in.contiguous(), slots = slots_in.contiguous();
    const at::Tensor q = q_rope_in ? readable_rows(*q_rope_in) : at::Tensor();
    auto f = dt == at::kHalf ? mla_append_kv_fp16 : mla_append_kv_bf16;
    check_status(f(kv.data_ptr(), weight.data_ptr(), cos_sin.data_ptr<float>(), positions.data_ptr<int>(),
                   reinterpret_cast<const long long *>(slots.data_ptr<int64_t>()), heads ? q.data_ptr() : nullptr,
                   kv_cache.data_ptr(), heads ? out->data_ptr() : nullptr, static_cast<float>(eps),
                   static_cast<float>(cache_scale), static_cast<int>(tokens), static_cast<int>(heads),
                   static_cast<int>(cos_sin.size(0)), kv_cache.numel() / MLA_HEAD_DIM_K,
                   used_stride(kv, 0, MLA_HEAD_DIM_K), heads ? used_stride(q, 0, 64) : 0,
                   heads ? used_stride(q, 1, 64) : 0,
                   (fp8 ? MLA_FLAG_FP8_CACHE : 0u) | (interleaved ? 0u : MLA_FLAG_ROPE_HALVES), stream_of(kv)),
                 fn);
    return out;
}

// No reference counterpart: a tree of drafted tokens a request over the paged cache.
at::Tensor mla_decode_tree(const at::Tensor &query_in, const at::Tensor &kv_in, const at::Tensor &block_table_in,
                           const at::Tensor &cu_seqlens_in, const at::Tensor &tree_mask_in,
                           const c10::optional<at::Tensor> &draft_lens_in, int64_t total_tokens, int64_t num_splits)
{
    const char *fn = "mla_decode_tree";
    const auto dt = query_in.scalar_type();
    TORCH_CHECK(dt == kv_in.scalar_type() && (dt == at::kHalf || dt == at::kBFloat16), fn,
                ": query and kv_cache must both be float16 or both bfloat16");
    TORCH_CHECK(query_in.dim() == 4 && query_in.size(3) == MLA_HEAD_DIM_K, fn,
                ": query must be [batch, drafts, num_heads, ", MLA_HEAD_DIM_K, "], got ", query_in.sizes());
    const int64_t batch = query_in.size(0), drafts = query_in.size(1), heads = query_in.size(2);
    TORCH_CHECK(batch >= 1 && drafts >= 1 && drafts <= 64, fn, ": 1 to 64 drafted tokens a request, got ", drafts);
    check_heads(heads, fn);
    TORCH_CHECK(kv_in.dim() == 3 && kv_in.size(2) == MLA_HEAD_DIM_K && kv_in.size(0) >= 1, fn,
                ": kv_cache must be [num_pages >= 1, page_size, ", MLA_HEAD_DIM_K, "], got ", kv_in.sizes());
    check_page_size(kv_in.size(1), fn);
    TORCH_CHECK(kv_in.size(0) <= INT32_MAX, fn, ": too many pages");
    check_int32(block_table_in, 2, fn, "block_table");
    check_int32(cu_seqlens_in, 1, fn, "cu_seqlens");
    TORCH_CHECK(cu_seqlens_in.size(0) == batch + 1 && block_table_in.size(0) == batch && block_table_in.size(1) >= 1, fn,
                ": cu_seqlens must have batch + 1 entries and block_table batch rows and a column");
    TORCH_CHECK(tree_mask_in.scalar_type() == at::kLong && tree_mask_in.dim() == 2 && tree_mask_in.size(0) == batch &&
                    tree_mask_in.size(1) == drafts,
                fn, ": tree_mask must be an int64 tensor [batch, drafts]");
    if (draft_lens_in) {
        check_int32(*draft_lens_in, 1, fn, "draft_lens");
        TORCH_CHECK(draft_lens_in->size(0) == batch, fn, ": draft_lens must have one entry per request");
    }
    check_devices({&query_in, &kv_in, &block_table_in, &cu_seqlens_in, &tree_mask_in,
                   draft_lens_in ? &*draft_lens_in : &query_in}, fn);
    const at::OptionalDeviceGuard guard(query_in.device());
    const at::Tensor query = readable(query_in), kv = readable(kv_in), bt = block_table_in.contiguous();
    const at::Tensor cu = cu_seqlens_in.contiguous(), mask = tree_mask_in.contiguous();
    const at::Tensor lens = draft_lens_in ? draft_lens_in->contiguous() : at::Tensor();
    const int total = static_cast<int>(given_total(total_tokens, cu, fn));
    const int splits = static_cast<int>(num_splits);
    at::Tensor out = at::empty({batch, drafts, heads, MLA_HEAD_DIM_V}, query.options());
    const size_t ws_bytes = mla_decode_tree_workspace_size(static_cast<int>(batch), static_cast<int>(drafts),
                                                           static_cast<int>(heads), total, splits);
    TORCH_CHECK(ws_bytes > 0, fn, ": unsupported sizes");
    at::Tensor ws = workspace(ws_bytes, query);
    auto f = dt == at::kHalf ? mla_decode_tree_fp16 : mla_decode_tree_bf16;
    check_status(f(query.data_ptr(), kv.data_ptr(), bt.data_ptr<int>(), cu.data_ptr<int>(),
                   reinterpret_cast<const long long *>(mask.data_ptr<int64_t>()),
                   draft_lens_in ? lens.data_ptr<int>() : nullptr, out.data_ptr(), ws.data_ptr(), ws_bytes,
                   static_cast<int>(batch), static_cast<int>(drafts), static_cast<int>(heads), total,
                   static_cast<int>(kv.size(1)), static_cast<int>(kv.size(0)), static_cast<int>(bt.size(1)), splits,
                   stream_of(query)),
                 fn);
    return out;
}

// No reference code (the math is README.md:64-85): causal attention of prompts in the expanded form.
at::Tensor mla_prefill(const at::Tensor &q_nope_in, const at::Tensor &q_rope_in, const at::Tensor &w_uk_in,
                       const at::Tensor &w_uv_in, const at::Tensor &kv_in, const at::Tensor &cu_q_in,
                       const at::Tensor &cu_seqlens_in, const c10::optional<at::Tensor> &block_table_in,
                       int64_t total_tokens)
{
    const char *fn = "mla_prefill";
    const auto dt = q_nope_in.scalar_type();
    TORCH_CHECK(dt == at::kHalf || dt == at::kBFloat16, fn, ": q_nope must be float16 or bfloat16");
    TORCH_CHECK(q_nope_in.dim() == 3 && q_nope_in.size(2) == 128 && q_nope_in.size(0) >= 1 &&
                    q_nope_in.size(0) <= INT32_MAX,
                fn, ": q_nope must be [queries, num_heads, 128], got ", q_nope_in.sizes());
    const int64_t queries = q_nope_in.size(0), heads = q_nope_in.size(1);
    check_heads(heads, fn);
    TORCH_CHECK(q_rope_in.dim() == 3 && q_rope_in.size(0) == queries && q_rope_in.size(1) == heads &&
                    q_rope_in.size(2) == 64,
                fn, ": q_rope must be [queries, num_heads, 64], got ", q_rope_in.sizes());
    for (const at::Tensor *w : {&w_uk_in, &w_uv_in})
        TORCH_CHECK(w->dim() == 3 && w->size(0) == heads && w->size(1) == 128 && w->size(2) == MLA_HEAD_DIM_V, fn,
                    ": w_uk and w_uv must be [num_heads, 128, 512], got ", w->sizes());
    for (const at::Tensor *t : {&q_rope_in, &w_uk_in, &w_uv_in, &kv_in})
        TORCH_CHECK(t->scalar_type() == dt, fn, ": all inputs must have the queries' dtype");
    check_int32(cu_q_in, 1, fn, "cu_q");
    check_int32(cu_seqlens_in, 1, fn, "cu_seqlens");
    const int64_t batch = cu_q_in.size(0) - 1;
    TORCH_CHECK(batch >= 1 && cu_seqlens_in.size(0) == batch + 1, fn, ": cu_q and cu_seqlens must have batch + 1 entries");
    if (block_table_in) {
        TORCH_CHECK(kv_in.dim() == 3 && kv_in.size(2) == MLA_HEAD_DIM_K && kv_in.size(0) >= 1 &&
                        kv_in.size(0) <= INT32_MAX,
                    fn, ": a paged kv_cache must be [num_pages >= 1, page_size, ", MLA_HEAD_DIM_K, "], got ", kv_in.sizes());
        check_page_size(kv_in.size(1), fn);
        check_int32(*block_table_in, 2, fn, "block_table");
        TORCH_CHECK(block_table_in->size(0) == batch && block_table_in->size(1) >= 1, fn,
                    ": block_table must have batch rows and a column");
    } else {
        TORCH_CHECK(kv_in.dim() == 2 && kv_in.size(1) == MLA_HEAD_DIM_K && kv_in.size(0) <= INT32_MAX, fn,
                    ": a packed kv_cache must be [total, ", MLA_HEAD_DIM_K, "], got ", kv_in.sizes());
        TORCH_CHECK(total_tokens <= kv_in.size(0), fn, ": total_tokens exceeds the packed kv_cache's rows");
        if (total_tokens < 0)
            total_tokens = kv_in.size(0);
    }
    check_devices({&q_nope_in, &q_rope_in, &w_uk_in, &w_uv_in, &kv_in, &cu_q_in, &cu_seqlens_in,
                   block_table_in ? &*block_table_in : &q_nope_in}, fn);
    const at::OptionalDeviceGuard guard(q_nope_in.device());
    const at::Tensor qn = readable(q_nope_in), qr = readable(q_rope_in);
    const at::Tensor wuk = readable(w_uk_in), wuv = readable(w_uv_in), kv = readable(kv_in);
    const at::Tensor cu_q = cu_q_in.contiguous(), cu = cu_seqlens_in.contiguous();
    const at::Tensor bt = block_table_in ? block_table_in->contiguous() : at::Tensor();
    const int total = static_cast<int>(given_total(total_tokens, cu, fn));
    at::Tensor out = at::empty({queries, heads, 128}, qn.options());
    const size_t ws_bytes = mla_prefill_workspace_size(static_cast<int>(batch), static_cast<int>(heads),
                                                       static_cast<int>(queries), total);
    TORCH_CHECK(ws_bytes > 0, fn, ": unsupported sizes");
    at::Tensor ws = workspace(ws_bytes, qn);
    auto f = dt == at::kHalf ? mla_prefill_fp16 : mla_prefill_bf16;
    check_status(f(qn.data_ptr(), qr.data_ptr(), wuk.data_ptr(), wuv.data_ptr(), total > 0 ? kv.data_ptr() : nullptr,
                   bt.defined() ? bt.data_ptr<int>() : nullptr, cu_q.data_ptr<int>(), cu.data_ptr<int>(), out.data_ptr(),
                   ws.data_ptr(), ws_bytes, static_cast<int>(batch), static_cast<int>(heads), static_cast<int>(queries),
                   total, bt.defined() ? static_cast<int>(kv.size(1)) : 0, bt.defined() ? static_cast<int>(kv.size(0)) : 0,
                   bt.defined() ? static_cast<int>(bt.size(1)) : 0, stream_of(qn)),
                 fn);
    return out;
}

void check_inputs(int64_t inputs, const char *fn)
{
    TORCH_CHECK(inputs >= 16 && inputs % 16 == 0 && inputs <= (1 << 22), fn,
                ": the last dimension must be a positive multiple of 16 (<= 2^22), got ", inputs);
}

// x as rows [m, inputs] that the kernels can read in place (else a copy): the last dimension contiguous, rows `unit`
// values apart or a multiple of that.
at::Tensor as_rows(const at::Tensor &x, int64_t unit)
{
    const at::Tensor rows = x.dim() == 2 ? x : x.reshape({-1, x.size(-1)});
    const bool ok = starts_aligned(rows) && rows.stride(1) == 1 &&
                    (rows.size(0) == 1 || (rows.stride(0) % unit == 0 && rows.stride(0) <= (1 << 22)));
    return ok ? rows : readable(rows);
}

std::vector<int64_t> with_last(const at::Tensor &x, int64_t last)
{
    std::vector<int64_t> sizes = x.sizes().vec();
    sizes.back() = last;
    return sizes;
}

// No reference code: rows in e4m3 with a scale for each 128 values.
std::vector<at::Tensor> quantize_fp8(const at::Tensor &x_in)
{
    const char *fn = "mla_quantize_fp8";
    const auto dt = x_in.scalar_type();
    TORCH_CHECK(dt == at::kHalf || dt == at::kBFloat16, fn, ": x must be float16 or bfloat16");
    TORCH_CHECK(x_in.dim() >= 1, fn, ": x must be [..., inputs]");
    const int64_t inputs = x_in.size(-1), blocks = (inputs + 127) / 128, rows = inputs ? x_in.numel() / inputs : 0;
    check_inputs(inputs, fn);
    TORCH_CHECK(rows <= (1 << 26) && rows * blocks <= (1 << 30) - 64, fn, ": too many rows");
    check_devices({&x_in}, fn);
    const at::OptionalDeviceGuard guard(x_in.device());
    const auto options = x_in.options().memory_format(at::MemoryFormat::Contiguous);
    at::Tensor q = at::empty(x_in.sizes(), options.dtype(at::kFloat8_e4m3fn));
    // block by block in memory: [..., blocks] is a view of [blocks, ...]
    std::vector<int64_t> sizes = x_in.sizes().vec();
    sizes.pop_back();
    sizes.insert(sizes.begin(), blocks);
    at::Tensor scales = at::empty(sizes, options.dtype(at::kFloat));
    if (rows == 0)
        return {q, scales.movedim(0, -1)};
    const at::Tensor x = as_rows(x_in, 8);
    auto f = dt == at::kHalf ? mla_quantize_fp8_fp16 : mla_quantize_fp8_bf16;
    check_status(f(x.data_ptr(), q.data_ptr(), scales.data_ptr<float>(), static_cast<int>(rows), static_cast<int>(inputs),
                   used_stride(x, 0, inputs), stream_of(x)),
                 fn);
    return {q, scales.movedim(0, -1)};
}

// No reference code: y = x W^T with W in e4m3 and a scale for each 128 x 128 values.
at::Tensor linear_fp8(const at::Tensor &x_in, const at::Tensor &w_in, const at::Tensor &ws_in,
                      const c10::optional<at::Tensor> &xs_in, const c10::optional<at::ScalarType> &dtype)
{
    const char *fn = "mla_linear_fp8";
    const bool quantised = x_in.scalar_type() == at::kFloat8_e4m3fn;
    TORCH_CHECK(quantised || x_in.scalar_type() == at::kHalf || x_in.scalar_type() == at::kBFloat16, fn,
                ": x must be float16, bfloat16 or float8_e4m3fn");
    TORCH_CHECK(quantised == xs_in.has_value(), fn, ": x_scale comes with a float8_e4m3fn x, and only with one");
    const auto dt = dtype ? *dtype : quantised ? at::kBFloat16 : x_in.scalar_type();
    TORCH_CHECK(dt == at::kHalf || dt == at::kBFloat16, fn, ": dtype must be float16 or bfloat16");
    TORCH_CHECK(quantised || dt == x_in.scalar_type(), fn, ": dtype is for a float8_e4m3fn x (else out has x's)");
    TORCH_CHECK(x_in.dim() >= 1, fn, ": x must be [..., inputs]");
    const int64_t inputs = x_in.size(-1), blocks = (inputs + 127) / 128, rows = inputs ? x_in.numel() / inputs : 0;
    check_inputs(inputs, fn);
    TORCH_CHECK(w_in.scalar_type() == at::kFloat8_e4m3fn && w_in.dim() == 2 && w_in.size(1) == inputs && w_in.size(0) >= 1, fn,
                ": weight must be a float8_e4m3fn tensor [outputs, ", inputs, "], got ", w_in.sizes());
    const int64_t outputs = w_in.size(0);
    TORCH_CHECK(rows <= (1 << 26) && outputs <= (1 << 26) && rows * blocks <= (1 << 30) - 64, fn, ": too many rows or outputs");
    TORCH_CHECK(ws_in.scalar_type() == at::kFloat && ws_in.dim() == 2 && ws_in.size(0) == (outputs + 127) / 128 &&
                    ws_in.size(1) == blocks,
                fn, ": weight_scale must be a float32 tensor [", (outputs + 127) / 128, ", ", blocks, "], got ", ws_in.sizes());
    if (xs_in)
        TORCH_CHECK(xs_in->scalar_type() == at::kFloat && xs_in->sizes().vec() == with_last(x_in, blocks), fn,
                    ": x_scale must be a float32 tensor of x's shape with ", blocks, " in the last place, got ", xs_in->sizes());
    check_devices({&x_in, &w_in, &ws_in, xs_in ? &*xs_in : &x_in}, fn);
    const at::OptionalDeviceGuard guard(x_in.device());
    at::Tensor out = at::empty(with_last(x_in, outputs), x_in.options().dtype(dt).memory_format(at::MemoryFormat::Contiguous));
    if (rows == 0)
        return out;
    const at::Tensor x = as_rows(x_in, quantised ? 16 : 8), w = as_rows(w_in, 16), ws = ws_in.contiguous();
    const int m = static_cast<int>(rows), k = static_cast<int>(inputs), n = static_cast<int>(outputs);
    const int64_t x_stride = used_stride(x, 0, inputs), w_stride = used_stride(w, 0, inputs);
    const size_t ws_bytes = mla_linear_fp8_workspace_size(m, k, n);
    TORCH_CHECK(ws_bytes > 0, fn, ": unsupported sizes");
    const at::Tensor space = workspace(ws_bytes, x);
    if (quantised) {
        // rows and blocks any distance apart; leading dimensions that do not make one are copied
        at::Tensor xs = xs_in->dim() == 2 ? *xs_in : xs_in->reshape({-1, blocks});
        if (xs.size(0) > 1 && xs.stride(0) > (1 << 20))
            xs = xs.contiguous();
        auto f = dt == at::kHalf ? mla_linear_fp8_quantized_fp16 : mla_linear_fp8_quantized_bf16;
        check_status(f(x.data_ptr(), xs.data_ptr<float>(), w.data_ptr(), ws.data_ptr<float>(), out.data_ptr(), space.data_ptr(),
                       ws_bytes, m, k, n, x_stride, w_stride, used_stride(xs, 0, 0), used_stride(xs, 1, 0), stream_of(x)),
                     fn);
        return out;
    }
    auto f = dt == at::kHalf ? mla_linear_fp8_fp16 : mla_linear_fp8_bf16;
    check_status(f(x.data_ptr(), w.data_ptr(), ws.data_ptr<float>(), out.data_ptr(), space.data_ptr(), ws_bytes, m, k, n,
                   x_stride, w_stride, stream_of(x)),
                 fn);
    return out;
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m)
{
    m.doc() = "MI355X (gfx950) MLA decode: drop-in for the ada_mla extension's fused path";
    m.def("mla_decode_split", &mla_decode_split,
          "fp16 / bf16 (or fp32) split-KV MLA decode (query [n_h,576], cache [N,576]); a float8_e4m3fn "
          "cache (holding C / cache_scale) with a float16 query",
          pybind11::arg("query"), pybind11::arg("cache"), pybind11::arg("num_splits") = 0,
          pybind11::arg("cache_scale") = 1.0);
    m.def("mla_decode_fused", &mla_decode_fused, "fp32 MLA decode (query [n_h,576], cache [N,576])",
          pybind11::arg("query"), pybind11::arg("cache"), pybind11::arg("num_splits") = 0);
    m.def("mla_decode_split_batched", &mla_decode_split_batched,
          "batched fp16 / bf16 MLA decode (query [B,n_h,576], packed cache [sum N,576], cu_seqlens [B+1] int32); "
          "a float8_e4m3fn cache (holding C / cache_scale) with a float16 query",
          pybind11::arg("query"), pybind11::arg("cache"), pybind11::arg("cu_seqlens"),
          pybind11::arg("num_splits") = 0, pybind11::arg("cache_scale") = 1.0);
    m.def("mla_decode_paged", &mla_decode_paged,
          "paged-KV fp16 / bf16 MLA decode (query [B,n_h,576], kv_cache [pages,page_size,576], "
          "block_table [B,max_pages] int32, cu_seqlens [B+1] int32); total_tokens=-1 reads cu_seqlens[B] "
          "(synchronising); a given total_tokens is not checked: one below cu_seqlens[B] silently "
          "truncates the trailing sequences. kv_cache of the query's dtype, or float8_e4m3fn holding C / cache_scale (num_heads "
          "a multiple of 32: the query then to 8 significant bits)",
          pybind11::arg("query"), pybind11::arg("kv_cache"), pybind11::arg("block_table"),
          pybind11::arg("cu_seqlens"), pybind11::arg("total_tokens") = -1, pybind11::arg("num_splits") = 0,
          pybind11::arg("cache_scale") = 1.0);
    m.def("mla_absorb_query", &mla_absorb_query,
          "Q* [B,n_h,576] = [q_nope W_UK[h], q_rope] (q_nope [B,n_h,128], q_rope [B,n_h,64], w_uk [n_h,128,512])",
          pybind11::arg("q_nope"), pybind11::arg("q_rope"), pybind11::arg("w_uk"));
    m.def("mla_project_output", &mla_project_output,
          "out [B,d_model] = concat_h(O*[:,h] W_UV[h]^T) W_O^T (o_star [B,n_h,512], w_uv [n_h,128,512], "
          "w_o [d_model,n_h*128])",
          pybind11::arg("o_star"), pybind11::arg("w_uv"), pybind11::arg("w_o"));
    m.def("mla_quantize_fp8", &quantize_fp8,
          "(x in float8_e4m3fn, scales float32 [..., ceil(inputs/128)], block by block in memory) of float16 or bfloat16 x "
          "[..., inputs]: each 128 values' largest at 448",
          pybind11::arg("x"));
    m.def("mla_linear_fp8", &linear_fp8,
          "x W^T [..., outputs] of x [..., inputs] (float16 or bfloat16, quantised as mla_quantize_fp8 does; or "
          "float8_e4m3fn with x_scale, the result then in dtype, bfloat16 by default) and weight [outputs, inputs] "
          "float8_e4m3fn with weight_scale float32 [ceil(outputs/128), ceil(inputs/128)]; inputs a multiple of 16",
          pybind11::arg("x"), pybind11::arg("weight"), pybind11::arg("weight_scale"),
          pybind11::arg("x_scale") = pybind11::none(), pybind11::arg("dtype") = pybind11::none());
    m.def("mla_paged_tables", &paged_tables,
          "(cu_seqlens [B+1], cu_new [B+1], slots [total_new] int64, positions [total_new], free_next [1]) of a "
          "step's tokens from int32 context_lens and new_lens [B]; the pages that the new tokens start come from "
          "free_pages, from index free_start[0] on, and are written to block_table [B,max_pages] in place. "
          "Tokens that find no page, and entries past the last token, have slot -1",
          pybind11::arg("context_lens"), pybind11::arg("new_lens"), pybind11::arg("block_table"),
          pybind11::arg("free_pages"), pybind11::arg("free_start"), pybind11::arg("page_size"),
          pybind11::arg("total_new"));
    m.def("mla_fork_tables", &fork_tables,
          "(block_table [B,max_pages], lens [B], copies [B,3], free_next [1]): row b holds the first kept_lens[b] tokens "
          "(None: all) of row parents[b] of block_table (lens [R]); whole pages are shared, a last page that another row "
          "goes on writing is copied (copies: page, page taken, rows; for mla_copy_pages), pages that no row holds any "
          "more are pushed to free_pages in place, below free_start[0]. pinned [num_pages]: pages that others hold",
          pybind11::arg("block_table"), pybind11::arg("lens"), pybind11::arg("parents"), pybind11::arg("free_pages"),
          pybind11::arg("free_start"), pybind11::arg("page_size"), pybind11::arg("num_pages"),
          pybind11::arg("kept_lens") = pybind11::none(), pybind11::arg("pinned") = pybind11::none());
    m.def("mla_compact_tables", &compact_tables,
          "(block_table, copies [n,3], free_pages): the highest used pages that are not pinned moved to the lowest free "
          "ids (free_pages from free_start[0] on), as long as those are lower; copies for mla_copy_pages",
          pybind11::arg("block_table"), pybind11::arg("lens"), pybind11::arg("free_pages"), pybind11::arg("free_start"),
          pybind11::arg("page_size"), pybind11::arg("num_pages"), pybind11::arg("pinned") = pybind11::none());
    m.def("mla_copy_pages", &copy_pages,
          "the first copies[i][2] rows of page copies[i][0] of kv_cache [pages,page_size,576] or "
          "[layers,pages,page_size,576] to page copies[i][1], in place (copies [n,3] int32; ids out of range: nothing)",
          pybind11::arg("kv_cache"), pybind11::arg("copies"));
    m.def("mla_append_kv", &mla_append_kv,
          "latent rows kv [T,576] RMS-normalised (first 512 values, norm_weight [512]) and rotated (last 64, "
          "cos_sin [P,64] float32 at positions [T] int32), written to rows slots [T] int64 of kv_cache in place "
          "(negative: not written; the same slot twice: undefined); kv_cache of kv's dtype, or float8_e4m3fn "
          "holding values / cache_scale. Returns q_rope [T,n_h,64] rotated, or None. interleaved: pairs 2i, 2i+1, "
          "else i, i+32",
          pybind11::arg("kv"), pybind11::arg("norm_weight"), pybind11::arg("cos_sin"), pybind11::arg("positions"),
          pybind11::arg("slots"), pybind11::arg("kv_cache"), pybind11::arg("q_rope") = pybind11::none(),
          pybind11::arg("eps") = 1e-6, pybind11::arg("cache_scale") = 1.0, pybind11::arg("interleaved") = true);
    m.def("mla_decode_tree", &mla_decode_tree,
          "decode of a tree of drafted tokens (query [B,drafts,n_h,576], the last draft_lens[b] tokens of each "
          "request's paged cache; None: all drafts) -> [B,drafts,n_h,512]; drafted token i sees the context and the "
          "drafted tokens j whose bit j of tree_mask[b][i] (int64) is set. kv_cache, block_table, cu_seqlens and "
          "total_tokens as for mla_decode_paged",
          pybind11::arg("query"), pybind11::arg("kv_cache"), pybind11::arg("block_table"),
          pybind11::arg("cu_seqlens"), pybind11::arg("tree_mask"), pybind11::arg("draft_lens") = pybind11::none(),
          pybind11::arg("total_tokens") = -1, pybind11::arg("num_splits") = 0);
    m.def("mla_prefill", &mla_prefill,
          "causal attention of prompts in the expanded form (q_nope [T,n_h,128], q_rope [T,n_h,64], w_uk and w_uv "
          "[n_h,128,512]) -> [T,n_h,128]; request b's queries cu_q[b]..cu_q[b+1]-1 are the last of its cache's tokens "
          "(cu_seqlens [B+1]). kv_cache [total,576] packed, or [pages,page_size,576] with block_table; total_tokens "
          "(cu_seqlens[B]) is read from the device where a paged call does not give it",
          pybind11::arg("q_nope"), pybind11::arg("q_rope"), pybind11::arg("w_uk"), pybind11::arg("w_uv"),
          pybind11::arg("kv_cache"), pybind11::arg("cu_q"), pybind11::arg("cu_seqlens"),
          pybind11::arg("block_table") = pybind11::none(), pybind11::arg("total_tokens") = -1);
    m.attr("HEAD_DIM_C") = MLA_HEAD_DIM_V;
    m.attr("HEAD_DIM_ROPE") = MLA_HEAD_DIM_K - MLA_HEAD_DIM_V;
    m.attr("HEAD_DIM_K") = MLA_HEAD_DIM_K;
}
