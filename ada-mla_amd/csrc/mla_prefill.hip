// Causal attention of prompts, or of chunks of prompts behind a cached
// context, in the expanded form (mla_prefill_*):
//
//   k[t, h] = [W_UK[h] c_t, r_t],  v[t, h] = W_UV[h] c_t     (c_t, r_t: latent row t)
//   o[i, h] = softmax_t<=pos(i)( [q_nope, q_rope][i, h] . k[t, h] / sqrt(192) ) v[t, h]
//
// Against the absorbed form a (query, key, head) costs 192 + 128 products
// instead of 576 + 512, for 2 x 128 x 512 once per key and head: with more
// than some 340 queries a key the expanded form needs fewer.
//
// Two launches: expand_kernel writes K, V and the rotary parts to the
// workspace, tile by tile of 64 keys (each sequence starts a tile of its own);
// attend_kernel is one pass over them with a running maximum and sum.
// K and V are held in the inputs' 16-bit type, as a cache of expanded heads
// would hold them: a rounding of half a step on each, the products in fp32.
#include <algorithm>
#include <cmath>
#include <cstdint>

#include "mla_flash.hpp"
#include "mla_mi355x.h"

namespace mla {
namespace {

constexpr int kNope = 128, kRopeDim = 64, kLatent = 512;
constexpr int kTile = 64;      // keys per tile; sequences are padded to it in the workspace
constexpr int kQueries = 128;  // queries per workgroup: 32 a wave

bool aligned16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

struct PrefillArgs {
    const void *q_nope, *q_rope, *w_uk, *w_uv, *cache;
    const int *block_table;  // nullptr: a packed cache
    const int *cu_q, *cu_seqlens;
    void *out;
    void *k, *v;                // [head][padded key][128]
    void *rope;                 // [padded key][64]
    unsigned long long *flags;  // [head][tile][2]: keys whose V holds an infinity or NaN, by half of its columns
    int batch, num_heads, queries, total_tokens;
    int padded;  // keys of the workspace: whole tiles
    int q_slots;
    int page_shift, num_pages, bt_stride;
    float scale_log2;
};

__device__ __forceinline__ int clamped(const int *cu, int b, int most) { return min(max(cu[b], 0), most); }

// The last b < batch with cu[b] / unit + b <= slot, by the whole wave: the
// sequence that owns this slot where each takes the slots from cu[b] / unit +
// b on. That numbering needs no prefix sums of rounded lengths, and no two
// sequences' slots meet.
__device__ __forceinline__ int owner_of_slot(const int *cu, int batch, int most, int unit, int slot, int lane)
{
    int b = 0;
    for (int base = 0; base < batch; base += 64) {
        const int i = base + lane;
        const unsigned long long m = __builtin_amdgcn_ballot_w64(i < batch && clamped(cu, i, most) / unit + i <= slot);
        if (m != 0)
            b = base + 63 - __builtin_clzll(m);
        if (m != ~0ull)
            break;
    }
    return __builtin_amdgcn_readfirstlane(b);
}

// ---- expansion --------------------------------------------------------------
// One workgroup (4 waves): 128 keys x the 128 columns of K or of V of one head,
// k = 512 in steps of 64. Rows of 128 bytes in LDS, 16-byte chunk c of row r
// at c ^ (r mod 8).
constexpr int kStep = 64;
constexpr int kStepElems = 128 * kStep;  // of one operand

template <typename E>
__global__ __launch_bounds__(256) void expand_kernel(PrefillArgs a)
{
    using E8 = typename Vec<E>::v8;
    using E4 = typename Vec<E>::v4;
    __shared__ __attribute__((aligned(1024))) E s_buf[2][2][kStepElems];  // [stage][keys, weights]
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int r32 = lane & 31, hl = lane >> 5;
    // workgroup -> (head and side, key tile pair): an XCD takes one head's side
    // through all keys, so that its weights stay in that L2
    const int pairs = (a.padded / kTile + 1) / 2;
    const int hs = (blockIdx.x >> 3) / pairs * 8 + (blockIdx.x & 7);
    const int pair = (blockIdx.x >> 3) % pairs;
    const int h = hs >> 1, side = hs & 1;
    if (h >= a.num_heads)
        return;

    // the two tiles' sequences
    int seq[2], seq_lo[2], len[2], t0[2];
    bool any = false;
#pragma unroll
    for (int g = 0; g < 2; ++g) {
        const int tile = 2 * pair + g;
        const int b = owner_of_slot(a.cu_seqlens, a.batch, a.total_tokens, kTile, tile, lane);
        seq[g] = b;
        seq_lo[g] = clamped(a.cu_seqlens, b, a.total_tokens);
        len[g] = max(clamped(a.cu_seqlens, b + 1, a.total_tokens), seq_lo[g]) - seq_lo[g];
        t0[g] = (tile - seq_lo[g] / kTile - b) * kTile;  // the tile's first key within its sequence
        if (tile * kTile >= a.padded)
            len[g] = 0;
        any |= t0[g] < len[g];
    }
    if (!any)
        return;
    auto key_source = [&](int r) -> const E * {  // latent row of the pair's key r; keys past a sequence re-read a real one
        const int g = r >> 6;
        const int b = g ? seq[1] : seq[0], lo = g ? seq_lo[1] : seq_lo[0], n = g ? len[1] : len[0];
        const int t = max(min((g ? t0[1] : t0[0]) + (r & 63), n - 1), 0);
        size_t row;
        if (a.block_table) {
            const int col = min(t >> a.page_shift, a.bt_stride - 1);
            const int page = min(max(a.block_table[(size_t)b * a.bt_stride + col], 0), a.num_pages - 1);
            row = ((size_t)page << a.page_shift) + (t & ((1 << a.page_shift) - 1));
        } else {
            row = min(lo + t, a.total_tokens - 1);
        }
        return (const E *)a.cache + row * kDK;
    };
    const E *w = (const E *)(side ? a.w_uv : a.w_uk) + (size_t)h * kNope * kLatent;
    const E *src[8];  // the lane's place in the wave's 8 load units of 8 rows: 4 of keys, 4 of weights
#pragma unroll
    for (int u = 0; u < 4; ++u) {
        const int r = 32 * wave + 8 * u + (lane >> 3);
        const int c = (lane & 7) ^ (r & 7);
        src[u] = key_source(r) + 8 * c;
        src[4 + u] = w + (size_t)r * kLatent + 8 * c;
    }
    const unsigned lds = lds_address(s_buf);
    auto load_step = [&](int s) {
        const unsigned at = lds + (s & 1) * (4 * kStepElems) + 32 * wave * (kStep * 2);
#pragma unroll
        for (int u = 0; u < 8; ++u)
            gather_to_lds16(src[u] + s * kStep, at + (u >> 2) * (2 * kStepElems) + (u & 3) * 1024);
    };
    load_step(0);
    if (hs == 0) {  // the rotary parts: 8 chunks a key
        for (int i = threadIdx.x; i < 128 * 8; i += 256) {
            const int r = i >> 3, p = 2 * pair * kTile + r;
            if (p < a.padded)
                *(uint4 *)((E *)a.rope + (size_t)p * kRopeDim + 8 * (i & 7)) =
                    *(const uint4 *)(key_source(r) + kLatent + 8 * (i & 7));
        }
    }
    // wave (i, j): columns 64 i .. +63 of the head's 128, keys 64 j .. +63
    const int wi = wave >> 1, wj = wave & 1;
    floatx16 acc[2][2] = {};
    for (int s = 0; s < kLatent / kStep; ++s) {
        MLA_WAIT_VMCNT(0);
        lds_barrier();
        if (s + 1 < kLatent / kStep)
            load_step(s + 1);
        const unsigned at = lds + (s & 1) * (4 * kStepElems);
        auto operand = [&](unsigned base, int r, int k) -> E8 {
            return lds_load<E8>(base + r * (kStep * 2) + 16 * ((2 * k + hl) ^ (r & 7)));
        };
#pragma unroll
        for (int k = 0; k < kStep / 16; ++k) {
            E8 wv[2], cv[2];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                wv[i] = operand(at + 2 * kStepElems, 64 * wi + 32 * i + r32, k);
                cv[i] = operand(at, 64 * wj + 32 * i + r32, k);
            }
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
                for (int j = 0; j < 2; ++j)
                    acc[i][j] = mfma32x32x16(wv[i], cv[j], acc[i][j]);
        }
    }
    // lane: key 32 j + r32 of the wave's 64, columns 32 i + 8 k + 4 hl .. +3
    const int tile = 2 * pair + wj;
    const int t_first = wj ? t0[1] : t0[0], n = wj ? len[1] : len[0];
    if (t_first >= n)
        return;
    E *dst = (E *)(side ? a.v : a.k) + ((size_t)h * a.padded + (size_t)tile * kTile) * kNope + 64 * wi + 4 * hl;
    unsigned long long bad = 0;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        const bool real = t_first + 32 * j + r32 < n;  // keys past the sequence hold zeros
        bool lane_bad = false;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                E4 v;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    // V: what is not finite becomes 0 and flags its key, so
                    // that a query that must not see the key can meet it with
                    // weight 0
                    E x = real ? (E)acc[i][j][4 * k + e] : (E)0.0f;
                    if (side && not_finite<E>(__builtin_bit_cast(unsigned short, x))) {
                        x = (E)0.0f;
                        lane_bad = true;
                    }
                    v[e] = x;
                }
                *(E4 *)(dst + (size_t)(32 * j + r32) * kNope + 32 * i + 8 * k) = v;
            }
        }
        const unsigned long long m = __builtin_amdgcn_ballot_w64(lane_bad);
        bad |= (unsigned long long)((unsigned)m | (unsigned)(m >> 32)) << (32 * j);
    }
    if (side && lane == 0)
        a.flags[((size_t)h * (a.padded / kTile) + tile) * 2 + wi] = bad;
}

// ---- attention --------------------------------------------------------------

template <typename E>
__global__ __launch_bounds__(256, 2) void attend_kernel(PrefillArgs a)
{
    using E8 = typename Vec<E>::v8;
    using E4 = typename Vec<E>::v4;
    constexpr int kKElems = kTile * kNope, kRElems = kTile * kRopeDim;
    constexpr int kStage = 2 * kKElems + kRElems;  // K, V, rotary parts: 40 KB
    __shared__ __attribute__((aligned(1024))) E s_buf[2][kStage];
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int r32 = lane & 31, hl = lane >> 5;
    // workgroup -> (head, query tile): all tiles of a head on one XCD, whose L2
    // then holds its K and V, the last (longest) first
    const int li = blockIdx.x >> 3;
    const int h = li / a.q_slots * 8 + (blockIdx.x & 7);
    const int slot = a.q_slots - 1 - li % a.q_slots;
    if (h >= a.num_heads)
        return;
    const int b = owner_of_slot(a.cu_q, a.batch, a.queries, kQueries, slot, lane);
    const int q_lo = clamped(a.cu_q, b, a.queries);
    const int n_q = max(clamped(a.cu_q, b + 1, a.queries), q_lo) - q_lo;
    const int q0 = (slot - q_lo / kQueries - b) * kQueries;
    // the last sequence's tiles go on to the end of the output: rows behind it are zeros
    const int rows = b == a.batch - 1 ? a.queries - q_lo : n_q;
    if (q0 >= n_q) {
        for (int i = threadIdx.x; i < min(kQueries, rows - q0) * (kNope / 8); i += 256)
            *(uint4 *)((E *)a.out + ((size_t)(q_lo + q0 + i / (kNope / 8)) * a.num_heads + h) * kNope +
                       8 * (i % (kNope / 8))) = uint4{0, 0, 0, 0};
        return;
    }
    const int k_lo = clamped(a.cu_seqlens, b, a.total_tokens);
    const int n_k = max(clamped(a.cu_seqlens, b + 1, a.total_tokens), k_lo) - k_lo;
    const int shift = n_k - n_q;  // query i sees the keys 0 .. i + shift
    const int tile0 = k_lo / kTile + b;
    const int n_tiles = (min(n_k, min(q0 + kQueries, n_q) + shift) + kTile - 1) / kTile;

    const int row = q0 + 32 * wave + r32;
    const int last = min(row, n_q - 1) + shift;  // the lane's last key
    const size_t q_at = (size_t)(q_lo + min(row, n_q - 1)) * a.num_heads + h;
    E8 q[12];
#pragma unroll
    for (int k = 0; k < 8; ++k)
        q[k] = *(const E8 *)((const E *)a.q_nope + q_at * kNope + 16 * k + 8 * hl);
#pragma unroll
    for (int k = 0; k < 4; ++k)
        q[8 + k] = *(const E8 *)((const E *)a.q_rope + q_at * kRopeDim + 16 * k + 8 * hl);

    const unsigned lds = lds_address(s_buf);
    const E *ks = (const E *)a.k + ((size_t)h * a.padded + (size_t)tile0 * kTile) * kNope;
    const E *vs = (const E *)a.v + ((size_t)h * a.padded + (size_t)tile0 * kTile) * kNope;
    const E *rs = (const E *)a.rope + (size_t)tile0 * kTile * kRopeDim;
    const unsigned long long *flags = a.flags + ((size_t)h * (a.padded / kTile) + tile0) * 2;
    // 16 units of K and of V (4 rows each), 8 of the rotary parts (8 rows)
    auto load_tile = [&](int j) {
        const unsigned at = lds + (j & 1) * (kStage * 2);
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const int r = 16 * wave + 4 * u + (lane >> 4);
            const int off = r * (kNope * 2) + 16 * ((lane & 15) ^ row_swizzle(r));
            global_to_lds16_at(ks + (size_t)j * kKElems, off, at + (4 * wave + u) * 1024);
            global_to_lds16_at(vs + (size_t)j * kKElems, off, at + 2 * kKElems + (4 * wave + u) * 1024);
        }
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const int r = 16 * wave + 8 * u + (lane >> 3);
            global_to_lds16_at(rs + (size_t)j * kRElems, r * (kRopeDim * 2) + 16 * ((lane & 7) ^ rope_swizzle(r)),
                               at + 4 * kKElems + (2 * wave + u) * 1024);
        }
    };
    const int key = key_of_row(r32);
    const unsigned k_lane = key * (kNope * 2) + 16 * (hl ^ row_swizzle(key));
    const unsigned rope_lane = 4 * kKElems + key * (kRopeDim * 2) + 16 * (hl ^ rope_swizzle(key));
    unsigned v_lane[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int j = lane & 15, r = 8 * hl + 2 * (j >> 2) + i;
        v_lane[i] = 2 * kKElems + r * (kNope * 2) +
                    16 * ((2 * ((lane >> 4) & 1) + ((j & 3) >> 1)) ^ row_swizzle(r)) + 8 * (j & 1);
    }

    floatx16 o[4] = {};
    float m = -INFINITY, l = 0.0f;
    if (n_tiles > 0)
        load_tile(0);
    const int wave_last = min(q0 + 32 * wave + 31, n_q - 1) + shift;  // of the wave's queries
    const int wave_first = min(q0 + 32 * wave, n_q - 1) + shift;
    for (int j = 0; j < n_tiles; ++j) {
        MLA_WAIT_VMCNT(0);
        lds_barrier();  // tile j is there, and everyone is done with tile j - 1
        if (j + 1 < n_tiles)
            load_tile(j + 1);
        if (j * kTile > wave_last)
            continue;
        const unsigned at = lds + (j & 1) * (kStage * 2);
        floatx16 s[2];
#pragma unroll
        for (int g = 0; g < 2; ++g) {
            s[g] = floatx16{};
#pragma unroll
            for (int k = 0; k < 8; ++k)
                s[g] = mfma32x32x16(lds_load<E8>(((at + k_lane) ^ (32 * k)) + 32 * g * (kNope * 2)), q[k], s[g]);
#pragma unroll
            for (int k = 0; k < 4; ++k)
                s[g] = mfma32x32x16(lds_load<E8>(((at + rope_lane) ^ (32 * k)) + 32 * g * (kRopeDim * 2)), q[8 + k], s[g]);
        }
        if (j * kTile + kTile - 1 > wave_first) {
#pragma unroll
            for (int g = 0; g < 2; ++g)
#pragma unroll
                for (int r = 0; r < 16; ++r)
                    s[g][r] = j * kTile + 32 * g + key_of_reg(r, hl) <= last ? s[g][r] : -INFINITY;
        }
        float most = s[0][0];
#pragma unroll
        for (int r = 1; r < 32; ++r)
            most = fmaxf(most, s[r >> 4][r & 15]);
        most = reduce_halves(most, [](float x, float y) { return fmaxf(x, y); }) * a.scale_log2;
        if (__builtin_amdgcn_ballot_w64(most > m + kLazyRescale) != 0) {
            const float next = most > m + kLazyRescale ? most : m;  // each row by itself
            const float f = next == -INFINITY ? 1.0f : fast_exp2(m - next);
            m = next;
            l *= f;
#pragma unroll
            for (int c = 0; c < 4; ++c)
                o[c] *= f;
        }
        const float ref = m == -INFINITY ? 0.0f : m;
        float p[32];
#pragma unroll
        for (int r = 0; r < 32; ++r) {
            p[r] = fast_exp2(s[r >> 4][r & 15] * a.scale_log2 - ref);
            l += p[r];
        }
        const unsigned long long bad = scalar_load(flags + 2 * j) | scalar_load(flags + 2 * j + 1);
        if (bad != 0) {  // a query that sees a key whose V is not finite gives NaN
#pragma unroll
            for (int r = 0; r < 32; ++r) {
                const int t = 32 * (r >> 4) + key_of_reg(r & 15, hl);
                if (((bad >> t) & 1) != 0 && j * kTile + t <= last)
                    l = NAN;
            }
        }
#pragma unroll
        for (int ks4 = 0; ks4 < 4; ++ks4) {
            const E8 pb = p_operand<E>(p + 8 * ks4);
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                E4 part[2];
#pragma unroll
                for (int i = 0; i < 2; ++i)
                    part[i] = lds_load_tr16<E>(((at + v_lane[i]) ^ (64 * c)) + 16 * ks4 * (kNope * 2));
                const E8 v = {part[0][0], part[0][1], part[0][2], part[0][3], part[1][0], part[1][1], part[1][2], part[1][3]};
                o[c] = mfma32x32x16(v, pb, o[c]);
            }
        }
    }
    l = reduce_halves(l, [](float x, float y) { return x + y; });
    if (row >= rows)
        return;
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;  // a query that sees no key gives zeros
    E *out = (E *)a.out + ((size_t)(q_lo + row) * a.num_heads + h) * kNope + 4 * hl;
#pragma unroll
    for (int c = 0; c < 4; ++c)
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            E4 v;
#pragma unroll
            for (int e = 0; e < 4; ++e)
                v[e] = row < n_q ? (E)(o[c][4 * k + e] * inv) : (E)0.0f;
            *(E4 *)(out + 32 * c + 8 * k) = v;
        }
}

// ---- host -------------------------------------------------------------------

size_t align256(size_t n) { return (n + 255) / 256 * 256; }

struct PrefillPlan {
    int padded;
    size_t kv_bytes, rope_bytes, flag_bytes;
    size_t bytes() const { return 2 * kv_bytes + rope_bytes + flag_bytes; }
};

// Sequence b's keys start at tile cu[b] / 64 + b of the workspace.
PrefillPlan prefill_plan(int batch, int num_heads, int total_tokens)
{
    PrefillPlan p;
    p.padded = total_tokens / kTile * kTile + kTile * batch;
    p.kv_bytes = align256((size_t)num_heads * p.padded * kNope * 2);
    p.rope_bytes = align256((size_t)p.padded * kRopeDim * 2);
    p.flag_bytes = align256((size_t)num_heads * (p.padded / kTile) * 16);
    return p;
}

bool prefill_sizes_ok(int batch, int num_heads, int total_tokens)
{
    return batch >= 1 && num_heads > 0 && num_heads % 16 == 0 && num_heads <= 4096 && total_tokens >= 0 &&
           (int64_t)total_tokens + (int64_t)kTile * batch <= INT32_MAX - 4096;
}

template <typename E>
void launch_prefill(const PrefillArgs &a, hipStream_t s)
{
    if (a.total_tokens > 0) {
        const int pairs = (a.padded / kTile + 1) / 2;
        hipLaunchKernelGGL(expand_kernel<E>, dim3((unsigned)pairs * (2 * a.num_heads)), dim3(256), 0, s, a);
    }
    hipLaunchKernelGGL(attend_kernel<E>, dim3((unsigned)a.q_slots * a.num_heads), dim3(256), 0, s, a);
}

int prefill(bool bf16, const void *q_nope, const void *q_rope, const void *w_uk, const void *w_uv, const void *kv_cache,
            const int *block_table, const int *cu_q, const int *cu_seqlens, void *out, void *workspace,
            size_t workspace_bytes, int batch, int num_heads, int queries, int total_tokens, int page_size,
            int num_pages, int block_table_stride, void *stream)
{
    if (!prefill_sizes_ok(batch, num_heads, total_tokens) || queries < 1 || queries > INT32_MAX - 4096 || !q_nope ||
        !q_rope || !w_uk || !w_uv || (!kv_cache && total_tokens > 0) || !cu_q || !cu_seqlens || !out || !workspace ||
        (block_table && (page_size < 32 || page_size > (1 << 20) || (page_size & (page_size - 1)) != 0 ||
                         num_pages < 1 || block_table_stride < 1)))
        return MLA_STATUS_INVALID_VALUE;
    if (!aligned16(q_nope) || !aligned16(q_rope) || !aligned16(w_uk) || !aligned16(w_uv) || !aligned16(kv_cache) ||
        !aligned16(out) || !aligned16(workspace))
        return MLA_STATUS_MISALIGNED;
    const PrefillPlan p = prefill_plan(batch, num_heads, total_tokens);
    PrefillArgs a;
    a.q_slots = queries / kQueries + batch;
    if ((int64_t)(p.padded / kTile + 1) * num_heads > INT32_MAX / 256 ||
        (int64_t)a.q_slots * num_heads > INT32_MAX / 256)
        return MLA_STATUS_INVALID_VALUE;
    if (workspace_bytes < p.bytes())
        return MLA_STATUS_WORKSPACE_TOO_SMALL;
    a.q_nope = q_nope;
    a.q_rope = q_rope;
    a.w_uk = w_uk;
    a.w_uv = w_uv;
    a.cache = kv_cache;
    a.block_table = block_table;
    a.cu_q = cu_q;
    a.cu_seqlens = cu_seqlens;
    a.out = out;
    char *ws = static_cast<char *>(workspace);
    a.k = ws;
    a.v = ws + p.kv_bytes;
    a.rope = ws + 2 * p.kv_bytes;
    a.flags = reinterpret_cast<unsigned long long *>(ws + 2 * p.kv_bytes + p.rope_bytes);
    a.batch = batch;
    a.num_heads = num_heads;
    a.queries = queries;
    a.total_tokens = total_tokens;
    a.padded = p.padded;
    a.page_shift = block_table ? __builtin_ctz((unsigned)page_size) : 0;
    a.num_pages = num_pages;
    a.bt_stride = block_table_stride;
    a.scale_log2 = (float)(1.4426950408889634 / std::sqrt(192.0));
    if (bf16)
        launch_prefill<__bf16>(a, static_cast<hipStream_t>(stream));
    else
        launch_prefill<_Float16>(a, static_cast<hipStream_t>(stream));
    const hipError_t e = hipPeekAtLastError();
    return e == hipSuccess ? MLA_STATUS_SUCCESS : record_hip_error(e);
}

}  // namespace
}  // namespace mla

extern "C" {

size_t mla_prefill_workspace_size(int batch, int num_heads, int total_tokens)
{
    return mla::prefill_sizes_ok(batch, num_heads, total_tokens)
               ? mla::prefill_plan(batch, num_heads, total_tokens).bytes()
               : 0;
}

int mla_prefill_fp16(const void *q_nope, const void *q_rope, const void *w_uk, const void *w_uv, const void *kv_cache,
                     const int *block_table, const int *cu_q, const int *cu_seqlens, void *out, void *workspace,
                     size_t workspace_bytes, int batch, int num_heads, int queries, int total_tokens, int page_size,
                     int num_pages, int block_table_stride, void *stream)
{
    return mla::prefill(false, q_nope, q_rope, w_uk, w_uv, kv_cache, block_table, cu_q, cu_seqlens, out, workspace,
                        workspace_bytes, batch, num_heads, queries, total_tokens, page_size, num_pages,
                        block_table_stride, stream);
}

int mla_prefill_bf16(const void *q_nope, const void *q_rope, const void *w_uk, const void *w_uv, const void *kv_cache,
                     const int *block_table, const int *cu_q, const int *cu_seqlens, void *out, void *workspace,
                     size_t workspace_bytes, int batch, int num_heads, int queries, int total_tokens, int page_size,
                     int num_pages, int block_table_stride, void *stream)
{
    return mla::prefill(true, q_nope, q_rope, w_uk, w_uv, kv_cache, block_table, cu_q, cu_seqlens, out, workspace,
                        workspace_bytes, batch, num_heads, queries, total_tokens, page_size, num_pages,
                        block_table_stride, stream);
}

}  // extern "C"
