// Attention of a tree of drafted tokens over the paged latent cache, absorbed
// form (mla_decode_tree_*):
//
//   O*[b, i, h] = softmax_t( Q*[b, i, h] . C[t] / sqrt(192) ) C_N[t]
//
// over the tokens t that drafted token i of request b sees: all of its context
// and the drafted tokens of the request whose bit is set in tree_mask[b][i]
// (its ancestors and itself). The drafted tokens' latent rows are the last
// ones of the request's cache.
//
// Against the single-token decode, drafts x heads rows share each latent row,
// so from about 256 rows on the call is bound by the matrix units and, next,
// by LDS: a workgroup is 4 waves of one per SIMD, each owning 32 query rows
// whole (Q* 144 registers, O* 256 accumulators, P in registers, see
// mla_flash.hpp), so the waves meet only to hand over cache blocks.
//
// Measured: 32 drafts x 128 heads over 50021 tokens 403 us + 14 of merging (446
// GF: 1.11 PFLOP/s; a large matrix product reaches 1.3), bound by the LDS reads of
// the first product (16 bytes a lane each: 40 cycles a product instead of 32) and
// a clock of some 1.6 GHz; 48 requests of 5 x 16 rows over 12000 tokens 85 + 10 us,
// the cache at 4.5 TB/s; 7 x 16 rows over 1003 tokens 10 + 4 us, round trips.
// Rounded to 16 bits on the way: P, for the second product (p_operand). The error
// against 64 bits is then up to a quarter above that of rounding the result alone.
#include <algorithm>
#include <cmath>
#include <cstdint>

#include "mla_flash.hpp"
#include "mla_mi355x.h"

namespace mla {
namespace {

constexpr int kBlock = 32;                // tokens per cache block
constexpr int kWaves = 4;                 // waves per workgroup
constexpr int kRows = 32 * kWaves;        // query rows per workgroup
constexpr int kRing = 4;                  // LDS ring slots
constexpr int kSlotElems = kBlock * kDK;  // 36 KB
constexpr int kRopeDim = kDK - kDV;
constexpr int kRopeElems = kBlock * kDV;  // the rope part of a slot, after its C_N rows
constexpr int kUnitsPerWave = 9;          // 1 KB load units of a block per wave: 8 rows, 1 rope unit
constexpr int kAhead = 4;                 // products an operand is read ahead
constexpr int kMaxDrafts = 64;

bool aligned16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

struct TreeArgs {
    const void *q;
    const void *cache;
    const int *block_table;
    const int *cu_seqlens;
    const unsigned long long *tree_mask;
    const int *draft_lens;
    void *out;
    float *part_o;  // [part slot][row tile][wave][16 column tiles][4][64 lanes][4]
    float *part_m;  // [part slot][row tile * 128]
    float *part_l;
    int batch, drafts, num_heads, total_tokens;
    int chunk;      // tokens per split
    int row_tiles;  // of 128 rows, per request
    int n_slots;    // splits of the batch, at most: total_tokens / chunk + batch
    int pairs;      // how the splits' partials are numbered, see Request
    int by_xcd;     // 1: the workgroups of a split share an XCD
    int page_shift, num_pages, bt_stride;
    float scale_log2;
};

// Request b's tokens [lo, lo + len) of the packed numbering and its splits. The
// partials of a request of several splits take the part slots lo / chunk + b, ..., or
// with `pairs` 2 lo / chunk, ...: neither meets those of another request, whatever the
// lengths. (A request of several splits has len > chunk, so 2 len / chunk rounded
// down is at least len / chunk rounded up.) The second has fewer slots where most
// requests are shorter than a split.
struct Request {
    int lo, len, n_splits, slot0, drafts;
    __device__ __forceinline__ void read(const TreeArgs &a, int b)
    {
        lo = min(max(scalar_load(a.cu_seqlens + b), 0), a.total_tokens);
        len = min(max(scalar_load(a.cu_seqlens + b + 1), lo), a.total_tokens) - lo;
        n_splits = max(1, (len + a.chunk - 1) / a.chunk);
        slot0 = (int)(((unsigned)lo << a.pairs) / (unsigned)a.chunk) + (a.pairs ? 0 : b);
        drafts = a.draft_lens ? min(max(scalar_load(a.draft_lens + b), 0), a.drafts) : a.drafts;
    }
};

// kTiles: 32-column tiles of O* a workgroup computes, 16 (all) or 4. A quarter of
// the columns computes all logits again but takes a quarter of the second
// product's and the results' time: for calls that leave most of the CUs idle.
template <typename E, int kTiles>
__global__ __attribute__((amdgpu_flat_work_group_size(256, 256), amdgpu_waves_per_eu(1, 1))) void tree_kernel(TreeArgs a)
{
    constexpr int kParts = kDV / 32 / kTiles;
    using E8 = typename Vec<E>::v8;
    using E4 = typename Vec<E>::v4;
    __shared__ __attribute__((aligned(1024))) E s_ring[kRing * kSlotElems];
    __shared__ unsigned s_bad[kWaves];
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int r32 = lane & 31, hl = lane >> 5;
    const unsigned ring = lds_address(s_ring);

    // workgroup -> (split of a request, row tile, column part), the splits counted through
    // the batch. With by_xcd the workgroups of a split, which read the same tokens, get ids
    // equal mod 8, i.e. one XCD and its L2, and the splits go to the XCDs in turn. (Taken by
    // slot, of which requests leave some empty, 15 requests of 32 drafts x 128 heads fell on
    // half of the XCDs: 642 us against 379, 24 of 16 x 64 628 against 329.)
    const int per_split = a.row_tiles * kParts;
    const int id = a.by_xcd ? blockIdx.x >> 3 : blockIdx.x;
    const int nth = a.by_xcd ? id / per_split * 8 + (blockIdx.x & 7) : id / per_split;
    const int within = id % per_split;
    const int rt = within / kParts, part = within % kParts;
    int b = -1, split = 0, before = 0;  // the nth split's request, its place there, the splits of the requests before
    for (int base = 0; base < a.batch; base += 64) {
        const int i = min(base + lane, a.batch - 1);
        const int lo = min(max(a.cu_seqlens[i], 0), a.total_tokens);
        const int len = min(max(a.cu_seqlens[i + 1], lo), a.total_tokens) - lo;
        const int n = base + lane < a.batch ? max(1, (len + a.chunk - 1) / a.chunk) : 0;
        int sum = n;
#pragma unroll
        for (int d = 1; d < 64; d *= 2) {
            const int u = __shfl_up(sum, d);
            sum += lane >= d ? u : 0;
        }
        const unsigned long long m = __builtin_amdgcn_ballot_w64(before + sum > nth);
        if (m != 0) {
            const int k = __builtin_ctzll(m);
            b = base + k;
            split = nth - before - (__builtin_amdgcn_readlane(sum, k) - __builtin_amdgcn_readlane(n, k));
            break;
        }
        before += __builtin_amdgcn_readlane(sum, 63);
    }
    if (b < 0)
        return;
    b = __builtin_amdgcn_readfirstlane(b);
    Request rq;
    rq.read(a, b);
    const int slot = rq.slot0 + split;
    const int rows = a.drafts * a.num_heads;      // of the request's output
    const int live = rq.drafts * a.num_heads;     // of its drafted tokens
    const int row = rt * kRows + 32 * wave + r32; // this lane's
    E *out = (E *)a.out + (size_t)b * rows * kDV;
    if (rt * kRows >= live) {  // only padding rows
        if (rq.n_splits == 1 && part == 0)
            for (int i = threadIdx.x; i < min(kRows, rows - rt * kRows) * (kDV / 8); i += 256)
                *(uint4 *)(out + (size_t)rt * kRows * kDV + 8 * i) = uint4{0, 0, 0, 0};
        return;
    }
    const int context = rq.len - rq.drafts;
    const int t_lo = split * a.chunk, t_hi = min(t_lo + a.chunk, rq.len);
    const int n_blocks = (t_hi - t_lo + kBlock - 1) / kBlock;

    // Block i of the split goes into its ring slot in 9 load units a wave: 8
    // rows, and the rope parts of 8 rows. Every block lies in one page. Page
    // ids and columns are clamped, so a bad table gives wrong results and no
    // stray access; rows past the request's end re-read its last one.
    auto page_of = [&](int i) -> int {
        const int col = min((t_lo + i * kBlock) >> a.page_shift, a.bt_stride - 1);
        return scalar_load(a.block_table + (size_t)b * a.bt_stride + col);
    };
    auto block_source = [&](int i, int page) -> const E * {
        page = min(max(page, 0), a.num_pages - 1);
        return wave_uniform((const E *)a.cache +
                            (((size_t)page << a.page_shift) + ((t_lo + i * kBlock) & ((1 << a.page_shift) - 1))) * kDK);
    };
    auto load_unit = [&](const E *base, int i, int u) {
        const int lim = min(kBlock - 1, rq.len - 1 - (t_lo + i * kBlock));
        const unsigned dst = ring + (i & (kRing - 1)) * (kSlotElems * 2);
        int ln = lane;  // opaque: the offsets are formed at each load, not kept in registers
        asm volatile("" : "+v"(ln));
        if (u < 8) {
            const int r = 8 * wave + u;
            global_to_lds16_at(base, min(r, lim) * (kDK * 2) + 16 * (ln ^ key_swizzle(r)), dst + r * (kDV * 2));
        } else {
            const int r = 8 * wave + (ln >> 3);
            global_to_lds16_at(base, min(r, lim) * (kDK * 2) + 2 * (kDV + 8 * ((ln & 7) ^ rope_swizzle(r))),
                               dst + 2 * kRopeElems + 1024 * wave);
        }
    };

    // LDS addresses, less the slot's, of the lane's operands. A chunk's place
    // differs from chunk 0's in the same row only by an XOR of its low four
    // bits and an offset of the others, so one address each serves all chunks.
    const unsigned k_lane = r32 * (kDV * 2) + 16 * (hl ^ key_swizzle(r32));
    const unsigned rope_lane = 2 * kRopeElems + r32 * (kRopeDim * 2) + 16 * (hl ^ rope_swizzle(r32));
    unsigned v_lane[2];  // the two transpose reads that match a P operand, 4 keys each
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const int j = lane & 15, r = 8 * h + 4 * hl + (j >> 2);
        v_lane[h] = r * (kDV * 2) + 16 * ((2 * ((lane >> 4) & 1) + ((j & 3) >> 1)) ^ key_swizzle(r)) + 8 * (j & 1);
    }
    // Operand k of the 32 rows in a ring slot: values 16 k + 8 hl .. +7 of the lane's row.
    auto row_operand = [&](unsigned slot_at, int k) -> E8 {
        return k < kDV / 16 ? lds_load<E8>(((slot_at + k_lane) ^ (32 * (k & 7))) + 256 * (k >> 3))
                            : lds_load<E8>((slot_at + rope_lane) ^ (32 * (k - kDV / 16)));
    };

    // Q*: the B operand of S^T, whole rows in registers, staged through the
    // wave's own ring slot by whole rows like a cache block (loaded into
    // registers at once, every load touched 32 rows of memory).
    const bool busy = rt * kRows + 32 * wave < live;  // else all the wave's rows are padding
    E8 q[kDK / 16] = {};
    unsigned long long mask = 0;
    if (busy) {
        const int first = rt * kRows + 32 * wave, lim = min(31, live - 1 - first);  // rows past the drafts re-read the last
        const E *src = wave_uniform((const E *)a.q + ((size_t)b * rows + first) * kDK);
        const unsigned own = ring + wave * (kSlotElems * 2);
#pragma unroll
        for (int r = 0; r < 32; ++r)
            global_to_lds16_at(src, min(r, lim) * (kDK * 2) + 16 * (lane ^ key_swizzle(r)), own + r * (kDV * 2));
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const int r = 8 * u + (lane >> 3);
            global_to_lds16_at(src, min(r, lim) * (kDK * 2) + 2 * (kDV + 8 * ((lane & 7) ^ rope_swizzle(r))),
                               own + 2 * kRopeElems + 1024 * u);
        }
        mask = a.tree_mask[(size_t)b * a.drafts + min(row, live - 1) / a.num_heads];
        MLA_WAIT_VMCNT(0);
        asm volatile("" ::: "memory");
#pragma unroll
        for (int k = 0; k < kDK / 16; ++k)
            q[k] = row_operand(own, k);
    }
    // waited for here, by name: the compiler does not know of the loads to LDS
    // and would wait at the uses inside the loop, in every block
    in_registers(mask);
#pragma unroll
    for (int k = 0; k < kDK / 16; ++k)
        in_registers(q[k]);
    lds_barrier();  // the ring is free
    auto load_block = [&](int i, const E *src) {
#pragma unroll
        for (int u = 0; u < kUnitsPerWave; ++u)
            load_unit(src, i, u);
    };
    for (int i = 0; i < min(kRing - 1, n_blocks); ++i)
        load_block(i, block_source(i, page_of(i)));
    // A drafted token that a row does not see meets it with weight 0: 0 times
    // an infinity or NaN in its row would still be NaN, so those become 0 for
    // the second product, once every wave has block i's logits. Returns the
    // block's tokens that had one: a row that sees such a token gives NaN.
    auto drop_not_finite = [&](int i) -> unsigned {
        constexpr int kEach = kBlock * kDV / 8 / 256;  // 16-byte pieces of a thread
        uint4 *at = (uint4 *)(s_ring + (i & (kRing - 1)) * kSlotElems) + threadIdx.x;
        uint4 v[kEach];
#pragma unroll
        for (int u = 0; u < kEach; ++u)
            v[u] = at[256 * u];
        unsigned top = 0;  // the largest magnitude's bits, both halves
#pragma unroll
        for (int u = 0; u < kEach; ++u)
            for (unsigned w : {v[u].x, v[u].y, v[u].z, v[u].w})
                top = max_u16x2(top, w & 0x7fff7fffu);
        const bool lane_bad = not_finite<E>((unsigned short)top) || not_finite<E>((unsigned short)(top >> 16));
        unsigned bad = 0;
        if (__builtin_amdgcn_ballot_w64(lane_bad) != 0) {
#pragma unroll
            for (int u = 0; u < kEach; ++u) {  // the wave's pieces u are token 4 u + wave
                bool found = false;
                for (unsigned *w : {&v[u].x, &v[u].y, &v[u].z, &v[u].w}) {
                    const unsigned keep = (not_finite<E>((unsigned short)*w) ? 0u : 0xffffu) |
                                          (not_finite<E>((unsigned short)(*w >> 16)) ? 0u : 0xffff0000u);
                    found |= keep != ~0u;
                    *w &= keep;
                }
                at[256 * u] = v[u];
                bad |= __builtin_amdgcn_ballot_w64(found) != 0 ? 1u << (4 * u + wave) : 0u;
            }
        }
        if (lane == 0)
            s_bad[wave] = bad;
        lds_barrier();
        return s_bad[0] | s_bad[1] | s_bad[2] | s_bad[3];
    };
    // a block that holds drafted tokens, or the request's end
    auto is_edge = [&](int i) { return t_lo + (i + 1) * kBlock > context; };
    if (!busy) {  // loads its share, and passes the same barriers
        if (n_blocks > 0) {
            MLA_WAIT_VMCNT(0);
            lds_barrier();
        }
        for (int i = 0; i < n_blocks; ++i) {
            MLA_WAIT_VMCNT(0);
            lds_barrier();
            if (i + kRing - 1 < n_blocks)
                load_block(i + kRing - 1, block_source(i + kRing - 1, page_of(i + kRing - 1)));
            if (is_edge(i))
                drop_not_finite(i);
        }
        if (rq.n_splits == 1 && part == 0 && row < rows)
            for (int k = hl; k < kDV / 8; k += 2)
                *(uint4 *)(out + (size_t)row * kDV + 8 * k) = uint4{0, 0, 0, 0};
        return;
    }

    int next_page = kRing - 1 < n_blocks ? page_of(kRing - 1) : 0;

    floatx16 o[kTiles];
#pragma unroll
    for (int c = 0; c < kTiles; ++c) {
        o[c] = floatx16{};
        in_accumulators(o[c]);
    }
    float m = -INFINITY, l = 0.0f;

    // The same units of a block whose 32 rows are all there, in three instructions each.
    const int row_off = 16 * (lane ^ key_swizzle(8 * wave));
    const int rope_off = (lane >> 3) * (kDK * 2) + 2 * kDV + 16 * ((lane & 7) ^ rope_swizzle(8 * wave + (lane >> 3)));
    auto stream_unit = [&](const E *src, unsigned slot, auto unit) {  // src: the wave's first row
        constexpr int u = decltype(unit)::value;
        if constexpr (u < 8)
            stream_to_lds16<u * kDK * 2, u * kDV * 2, 0>(src, row_off ^ (64 * (u & 3)) ^ (16 * (u >> 2)), slot + 8192 * wave);
        else
            stream_to_lds16<0, 2 * kRopeElems, 0>(src, rope_off, slot + 1024 * wave);
    };

    // S^T of block i, with side(k) between the products: what does not depend
    // on them, in their shadow (a product takes 32 cycles and one issue slot of
    // 4). Each operand is read kAhead products before its own. The products go
    // to ordinary registers: O* fills the accumulation registers.
    auto logits = [&](int i, auto &&side) -> floatx16 {
        const unsigned blk = ring + (i & (kRing - 1)) * (kSlotElems * 2);
        auto k_operand = [&](int k) -> E8 { return row_operand(blk, k); };
        E8 kv[kAhead + 1];
        floatx16 s;
#pragma unroll
        for (int k = 0; k < kAhead; ++k)
            kv[k] = k_operand(k);
        for_constants(
            [&](auto product) {
                constexpr int k = decltype(product)::value;
                if constexpr (k + kAhead < kDK / 16)
                    kv[(k + kAhead) % (kAhead + 1)] = k_operand(k + kAhead);
                if constexpr (k == 0)
                    mfma32x32x16_first(s, kv[0], q[0]);
                else
                    mfma32x32x16_next(s, kv[k % (kAhead + 1)], q[k]);
                side(product);
                __builtin_amdgcn_sched_barrier(0);
            },
            std::make_integer_sequence<int, kDK / 16>{});
        mfma_settle(s);
        return s;
    };
    auto largest = [&](const floatx16 &s) {
        float most = s[0];
#pragma unroll
        for (int r = 1; r < 16; ++r)
            most = fmaxf(most, s[r]);
        return most;
    };

    floatx16 s = {};
    float most = -INFINITY;  // the lane's largest logit of block i
    if (n_blocks > 0) {
        if (n_blocks > 2)
            MLA_WAIT_VMCNT(2 * kUnitsPerWave);
        else if (n_blocks > 1)
            MLA_WAIT_VMCNT(kUnitsPerWave);
        else
            MLA_WAIT_VMCNT(0);
        lds_barrier();
        s = logits(0, [](auto) {});
        most = largest(s);
    }
    for (int i = 0; i < n_blocks; ++i) {
        // Block i: s holds its logits. Those of block i + 1 are computed
        // while block i's weights are, then O* takes block i.
        const bool more = i + 1 < n_blocks;
        if (i + 2 < n_blocks)
            MLA_WAIT_VMCNT(kUnitsPerWave);
        else
            MLA_WAIT_VMCNT(0);
        lds_barrier();  // block i + 1 is there, every wave has block i's logits, and block i - 1's slot is free
        const bool feed = i + kRing - 1 < n_blocks;
        const E *feed_src = block_source(i + kRing - 1, next_page);
        next_page = i + kRing < n_blocks ? page_of(i + kRing) : 0;

        const int t0 = t_lo + i * kBlock;
        if (is_edge(i)) {
            auto sees = [&](int t) -> bool {
                const unsigned bit = (unsigned)(mask >> ((t - context) & 63)) & 1u;
                return ((unsigned)(t < context) | ((unsigned)(t < rq.len) & bit)) != 0;
            };
#pragma unroll
            for (int r = 0; r < 16; ++r)
                s[r] = sees(t0 + key_of_reg(r, hl)) ? s[r] : -INFINITY;
            most = largest(s);
            const unsigned bad = drop_not_finite(i);
            if (bad != 0) {
#pragma unroll
                for (int r = 0; r < 16; ++r)
                    l = ((bad >> key_of_reg(r, hl)) & 1u) != 0 && sees(t0 + key_of_reg(r, hl)) ? NAN : l;
            }
        }
        most = reduce_halves(most, [](float x, float y) { return fmaxf(x, y); }) * a.scale_log2;
        // the reference moves only past kLazyRescale, so P is at most 2^8
        if (__builtin_amdgcn_ballot_w64(most > m + kLazyRescale) != 0) {
            const float next = most > m + kLazyRescale ? most : m;  // each row by itself
            const float f = next == -INFINITY ? 1.0f : fast_exp2(m - next);
            m = next;
            l *= f;
            if (i > 0) {  // before, O* is zero
#pragma unroll
                for (int c = 0; c < kTiles; ++c) {
                    in_accumulators(o[c]);
                    o[c] *= f;
                    in_accumulators(o[c]);
                    __builtin_amdgcn_sched_barrier(0);
                }
            }
        }
        const float ref = m == -INFINITY ? 0.0f : m;
        float p[16];
        auto weight = [&](int r) {
            p[r] = fast_exp2(s[r] * a.scale_log2 - ref);
            l += p[r];
        };
        // block i + 3, requested between the products where it is whole
        const bool whole = feed && t0 + kRing * kBlock <= rq.len;
        if (feed && !whole)
            load_block(i + kRing - 1, feed_src);
        floatx16 ahead = {};
        if (more && whole) {
            const E *src = feed_src + 8 * wave * kDK;
            const unsigned slot_at = ring + ((i + kRing - 1) & (kRing - 1)) * (kSlotElems * 2);
            ahead = logits(i + 1, [&](auto product) {
                constexpr int k = decltype(product)::value;
                if constexpr (k % 2 == 0 && k < 32)
                    weight(k / 2);
                if constexpr (k % 4 == 1)
                    stream_unit(src, slot_at, std::integral_constant<int, k / 4>{});
            });
        } else if (more) {
            ahead = logits(i + 1, [&](auto product) {
                constexpr int k = decltype(product)::value;
                if constexpr (k % 2 == 0 && k < 32)
                    weight(k / 2);
            });
        } else {
#pragma unroll
            for (int r = 0; r < 16; ++r)
                weight(r);
        }
        const E8 pb[2] = {p_operand<E>(p), p_operand<E>(p + 8)};

        const unsigned blk = ring + (i & (kRing - 1)) * (kSlotElems * 2);
        const unsigned v_at[2] = {blk + v_lane[0] + part * (kTiles * 64), blk + v_lane[1] + part * (kTiles * 64)};
        auto v_operand = [&](int u) -> E8 {  // 32 columns of tile c, keys 16 ks .. +15 in the order of P's registers
            const int ks = u / kTiles, c = u % kTiles;
            E4 part[2];
#pragma unroll
            for (int h = 0; h < 2; ++h)
                part[h] = lds_load_tr16<E>((v_at[h] ^ (64 * (c & 3))) + 256 * (c >> 2) + 16 * ks * (kDV * 2));
            return E8{part[0][0], part[0][1], part[0][2], part[0][3], part[1][0], part[1][1], part[1][2], part[1][3]};
        };
        constexpr int kOps = 2 * kTiles;
        E8 v[kAhead + 1];
#pragma unroll
        for (int u = 0; u < kAhead; ++u)
            v[u] = v_operand(u);
        most = ahead[0];
#pragma unroll
        for (int u = 0; u < kOps; ++u) {
            if (u + kAhead < kOps)
                v[(u + kAhead) % (kAhead + 1)] = v_operand(u + kAhead);
            floatx16 &acc = o[u % kTiles];
            acc = mfma32x32x16(v[u % (kAhead + 1)], pb[u / kTiles], acc);
            in_accumulators(acc);
#pragma unroll
            for (int r = u * 16 / kOps; r < (u + 1) * 16 / kOps; ++r)
                most = fmaxf(most, ahead[r]);
            __builtin_amdgcn_sched_barrier(0);
        }
        s = ahead;
    }

#pragma unroll
    for (int c = 0; c < kTiles; ++c)
        in_accumulators(o[c]);
    l = reduce_halves(l, [](float x, float y) { return x + y; });
    if (rq.n_splits == 1) {
        // a row that sees nothing has l = 0 and gives zeros
        const float inv = l == 0.0f || row >= live ? 0.0f : 1.0f / l;
        if (row < rows) {
#pragma unroll
            for (int c = 0; c < kTiles; ++c) {
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    E4 v;
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        v[j] = row < live ? (E)(o[c][4 * k + j] * inv) : (E)0.0f;
                    *(E4 *)(out + (size_t)row * kDV + 32 * (part * kTiles + c) + 8 * k + 4 * hl) = v;
                }
            }
        }
        return;
    }
    const size_t tile = (size_t)slot * a.row_tiles + rt;
    float *po = a.part_o + (tile * kWaves + wave) * (32 * kDV) + part * (kTiles * 1024);
#pragma unroll
    for (int c = 0; c < kTiles; ++c)
#pragma unroll
        for (int k = 0; k < 4; ++k)
            *(floatx4 *)(po + ((c * 4 + k) * 64 + lane) * 4) =
                floatx4{o[c][4 * k], o[c][4 * k + 1], o[c][4 * k + 2], o[c][4 * k + 3]};
    if (hl == 0 && part == 0) {
        a.part_m[tile * kRows + 32 * wave + r32] = m;
        a.part_l[tile * kRows + 32 * wave + r32] = l;
    }
}

// Merges the splits of a request (those of more than one). A workgroup takes 32
// rows x `tiles` times 32 columns; wave w the splits w, w + 4, .., and a lane the 16 values it
// would hold in the split kernel. The waves' sums meet in LDS. The order of the
// additions depends on the split count alone.
constexpr int kMany = 4;  // splits of a wave in flight together

template <typename E>
__global__ __launch_bounds__(256) void tree_combine_kernel(TreeArgs a, int tiles)
{
    using E4 = typename Vec<E>::v4;
    __shared__ float s_m[kWaves][32];
    __shared__ float s_l[kWaves][32];
    __shared__ floatx4 s_o[kWaves][4][64];
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int per_row = kDV / 32 / tiles;  // workgroups of 32 rows
    const int c0 = blockIdx.x % per_row * tiles, w = blockIdx.x / per_row & 3, rest = blockIdx.x / per_row >> 2;
    const int rt = rest % a.row_tiles, b = rest / a.row_tiles;
    Request rq;
    rq.read(a, b);
    if (rq.n_splits == 1)
        return;
    const int rows = a.drafts * a.num_heads, live = rq.drafts * a.num_heads;
    const int r32 = lane & 31, hl = lane >> 5;
    const int row = rt * kRows + 32 * w + r32;
    for (int c = c0; c < c0 + tiles; ++c) {
        if (c > c0)
            __syncthreads();  // everyone has read the sums of the tile before
        floatx4 acc[4] = {};
        float m = -INFINITY, l = 0.0f;
        if (rt * kRows + 32 * w < live) {  // else no wave has left partials of these rows
            // past the last split a wave repeats it with weight 0
            const size_t tile0 = (size_t)rq.slot0 * a.row_tiles + rt;
            auto at = [&](int s) { return tile0 + (size_t)min(s, rq.n_splits - 1) * a.row_tiles; };
            for (int s = wave; s < rq.n_splits; s += kWaves * kMany) {
                float ms[kMany], ls[kMany];
                floatx4 po[kMany][4];
#pragma unroll
                for (int k = 0; k < kMany; ++k) {
                    const size_t t = at(s + kWaves * k);
                    ms[k] = a.part_m[t * kRows + 32 * w + r32];
                    ls[k] = a.part_l[t * kRows + 32 * w + r32];
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        po[k][j] = *(const floatx4 *)(a.part_o + (t * kWaves + w) * (32 * kDV) + ((c * 4 + j) * 64 + lane) * 4);
                }
                float next = m;
#pragma unroll
                for (int k = 0; k < kMany; ++k)
                    next = fmaxf(next, ms[k]);
                const float ref = next == -INFINITY ? 0.0f : next;
                const float f0 = fast_exp2(m - ref);
                l *= f0;
#pragma unroll
                for (int j = 0; j < 4; ++j)
                    acc[j] *= f0;
#pragma unroll
                for (int k = 0; k < kMany; ++k) {
                    if (s + kWaves * k >= rq.n_splits)
                        continue;
                    const float f = fast_exp2(ms[k] - ref);
                    l += f * ls[k];
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        acc[j] += f * po[k][j];
                }
                m = next;
            }
        }
        if (hl == 0) {
            s_m[wave][r32] = m;
            s_l[wave][r32] = l;
        }
#pragma unroll
        for (int j = 0; j < 4; ++j)
            s_o[wave][j][lane] = acc[j];
        __syncthreads();
        // wave j: the 4 columns of quarter j of each lane
        float top = -INFINITY;
#pragma unroll
        for (int k = 0; k < kWaves; ++k)
            top = fmaxf(top, s_m[k][r32]);
        const float ref = top == -INFINITY ? 0.0f : top;
        floatx4 sum = {};
        l = 0.0f;
#pragma unroll
        for (int k = 0; k < kWaves; ++k) {
            const float f = fast_exp2(s_m[k][r32] - ref);
            l += f * s_l[k][r32];
            sum += f * s_o[k][wave][lane];
        }
        const float inv = l == 0.0f ? 0.0f : 1.0f / l;
        E4 v;
#pragma unroll
        for (int j = 0; j < 4; ++j)
            v[j] = row < live ? (E)(sum[j] * inv) : (E)0.0f;
        if (row < rows)
            *(E4 *)((E *)a.out + ((size_t)b * rows + row) * kDV + 32 * c + 8 * wave + 4 * hl) = v;
    }
}

size_t align256(size_t n) { return (n + 255) / 256 * 256; }

struct TreePlan {
    int row_tiles, chunk, n_slots, pairs;
    int parts;  // column parts: 1 or 4
    size_t o_bytes, ml_bytes;
    size_t bytes() const { return std::max<size_t>(256, o_bytes + 2 * ml_bytes); }  // 0 would say: unsupported
};

// Splits of a request of mean length, and column parts: those with the least
// modelled time. A workgroup costs its start and end (Q*, the first block, its
// results) besides its blocks, and one runs on a CU at a time. Workgroups that fit
// the CUs at once take one round; else those of one request come in whole
// rounds, and those of a batch, of unequal lengths, follow each other with about
// 0.7 of a round to fill at the end (a request's last split is a part of one:
// half a split more a request). Partials (fp32, written and read) and the second
// launch are the price of a split. The constants are fitted to call times
// measured at given splits of requests of 16 to 4096 rows.
struct PartCost {
    int parts;
    double start_us, block_us;
};
constexpr PartCost kPartCosts[2] = {{1, 7.0, 1.8}, {4, 5.0, 1.0}};
constexpr double kCombineUs = 3.5, kSplitUs = 0.06, kPartialUsPerByte = 0.2e-6;

TreePlan compute_tree_plan(int batch, int drafts, int num_heads, int total_tokens, int num_splits, int cu_count)
{
    TreePlan p;
    p.row_tiles = (drafts * num_heads + kRows - 1) / kRows;
    const int longest = (int)(((int64_t)total_tokens + batch - 1) / batch);  // mean
    const int blocks = std::max(1, (longest + kBlock - 1) / kBlock);
    int splits = 1;
    double best = 0.0;
    const int asked = std::min(num_splits, blocks);
    for (const PartCost &c : kPartCosts) {
        const int lo = asked > 0 ? asked : 1, hi = asked > 0 ? asked : std::min(blocks, 256);
        for (int n = lo; n <= hi; ++n) {
            const int per = (blocks + n - 1) / n;
            if (n > lo && (blocks + n - 2) / (n - 1) == per)
                continue;  // no shorter than the one before
            const double each = batch == 1 ? n : n == 1 ? 1.0 : n + 0.5;
            const double wgs = each * batch * p.row_tiles * c.parts / cu_count;
            const double rounds = wgs <= (batch == 1 ? 1.0 : 1.1) ? 1.0 : batch == 1 ? std::ceil(wgs) : wgs + 0.7;
            double us = rounds * (c.start_us + per * c.block_us);
            if (n > 1)
                us += kCombineUs + kSplitUs * n + kPartialUsPerByte * n * batch * drafts * num_heads * (kDV * 4.0);
            if (best == 0.0 || us < best) {
                best = us;
                splits = n;
                p.parts = c.parts;
            }
        }
    }
    int64_t chunk = (longest + splits - 1) / splits;
    chunk = std::max<int64_t>(kBlock, (chunk + kBlock - 1) / kBlock * kBlock);
    // Where the rows alone fill the CUs, requests up to kWholeTokens are not split for being
    // longer than the mean: 60 requests of 24 drafts x 128 heads over 1 to 40 tokens 284 ->
    // 165 us, 40 of 16 x 128 over up to 716 186 -> 142. (Twice the mean for longer ones
    // gained on some batches, 257 -> 214, and lost on others, 161 -> 187.)
    constexpr int kWholeTokens = 1024;
    if (splits == 1 && asked <= 0 && (int64_t)batch * p.row_tiles * p.parts >= cu_count)
        chunk = std::max<int64_t>(chunk, kWholeTokens);
    p.chunk = (int)chunk;
    p.n_slots = total_tokens / p.chunk + batch;
    // partials: none where no request can be longer than a split
    const int64_t by_pairs = 2 * (int64_t)total_tokens / p.chunk;
    p.pairs = by_pairs < p.n_slots;
    const size_t part_slots = total_tokens <= p.chunk ? 0 : p.pairs ? (size_t)by_pairs : (size_t)p.n_slots;
    const size_t tiles = part_slots * p.row_tiles;
    p.o_bytes = align256(tiles * kRows * kDV * sizeof(float));
    p.ml_bytes = align256(tiles * kRows * sizeof(float));
    return p;
}

// The last plan of each host thread: a call asks for it twice (the workspace's
// size, then the launch), and a decode loop repeats its sizes.
TreePlan tree_plan(int batch, int drafts, int num_heads, int total_tokens, int num_splits, int cu_count)
{
    thread_local int key[6] = {0, 0, 0, 0, 0, 0};
    thread_local TreePlan plan;
    const int now[6] = {batch, drafts, num_heads, total_tokens, num_splits, cu_count};
    if (!std::equal(key, key + 6, now)) {
        plan = compute_tree_plan(batch, drafts, num_heads, total_tokens, num_splits, cu_count);
        std::copy(now, now + 6, key);
    }
    return plan;
}

bool tree_sizes_ok(int batch, int drafts, int num_heads, int total_tokens)
{
    return batch >= 1 && drafts >= 1 && drafts <= kMaxDrafts && num_heads > 0 && num_heads % 16 == 0 &&
           num_heads <= 4096 && total_tokens >= 0 && total_tokens <= INT32_MAX - 4096;
}

// Slots from which on a split's workgroups share an XCD: 16 requests of 16 drafts
// x 128 heads 222 -> 164 us, 23 of 30 x 64 120 -> 94. With fewer splits the
// XCDs would take one or two each, or none: 32 drafts x 128 heads over 50021 tokens
// in 8 splits 441 us against 414, in one split 8.7 ms against 2.1.
constexpr int kMinSlotsByXcd = 16;

template <typename E>
void launch_tree(const TreeArgs &a, int parts, hipStream_t s)
{
    auto k = parts == 4 ? tree_kernel<E, 4> : tree_kernel<E, 16>;
    const unsigned slots = a.by_xcd ? (a.n_slots + 7) / 8 * 8 : a.n_slots;
    hipLaunchKernelGGL(k, dim3(slots * a.row_tiles * parts), dim3(256), 0, s, a);
    if (a.total_tokens > a.chunk) {
        // one 32 x 32 tile a workgroup, 4 where there are many rows: 16 requests of 16
        // drafts x 128 heads 18.0 us (most of 16384 workgroups find nothing to do)
        // against 16.0
        const unsigned groups = (unsigned)a.batch * a.row_tiles * kWaves;
        const int tiles = groups >= 512 ? 4 : 1;
        hipLaunchKernelGGL(tree_combine_kernel<E>, dim3(groups * (kDV / 32 / tiles)), dim3(256), 0, s, a, tiles);
    }
}

int decode_tree(bool bf16, const void *query, const void *kv_cache, const int *block_table, const int *cu_seqlens,
                const long long *tree_mask, const int *draft_lens, void *out, void *workspace, size_t workspace_bytes,
                int batch, int drafts, int num_heads, int total_tokens, int page_size, int num_pages,
                int block_table_stride, int num_splits, void *stream)
{
    if (!tree_sizes_ok(batch, drafts, num_heads, total_tokens) || !query || !kv_cache || !block_table || !cu_seqlens ||
        !tree_mask || !out || !workspace || page_size < 32 || page_size > (1 << 20) ||
        (page_size & (page_size - 1)) != 0 || num_pages < 1 || block_table_stride < 1)
        return MLA_STATUS_INVALID_VALUE;
    if (!aligned16(query) || !aligned16(kv_cache) || !aligned16(out) || !aligned16(workspace))
        return MLA_STATUS_MISALIGNED;
    const TreePlan p = tree_plan(batch, drafts, num_heads, total_tokens, num_splits, current_cu_count());
    if ((int64_t)(p.n_slots + 7) * p.row_tiles > INT32_MAX / (256 * 4) || (int64_t)batch * p.row_tiles > INT32_MAX / (256 * 64))
        return MLA_STATUS_INVALID_VALUE;
    if (workspace_bytes < p.bytes())
        return MLA_STATUS_WORKSPACE_TOO_SMALL;
    TreeArgs a;
    a.q = query;
    a.cache = kv_cache;
    a.block_table = block_table;
    a.cu_seqlens = cu_seqlens;
    a.tree_mask = reinterpret_cast<const unsigned long long *>(tree_mask);
    a.draft_lens = draft_lens;
    a.out = out;
    char *ws = static_cast<char *>(workspace);
    a.part_o = reinterpret_cast<float *>(ws);
    a.part_m = reinterpret_cast<float *>(ws + p.o_bytes);
    a.part_l = reinterpret_cast<float *>(ws + p.o_bytes + p.ml_bytes);
    a.batch = batch;
    a.drafts = drafts;
    a.num_heads = num_heads;
    a.total_tokens = total_tokens;
    a.chunk = p.chunk;
    a.row_tiles = p.row_tiles;
    a.n_slots = p.n_slots;
    a.pairs = p.pairs;
    a.by_xcd = p.n_slots >= kMinSlotsByXcd;
    a.page_shift = __builtin_ctz((unsigned)page_size);
    a.num_pages = num_pages;
    a.bt_stride = block_table_stride;
    a.scale_log2 = (float)(1.4426950408889634 / std::sqrt(192.0));
    if (bf16)
        launch_tree<__bf16>(a, p.parts, static_cast<hipStream_t>(stream));
    else
        launch_tree<_Float16>(a, p.parts, static_cast<hipStream_t>(stream));
    const hipError_t e = hipPeekAtLastError();
    return e == hipSuccess ? MLA_STATUS_SUCCESS : record_hip_error(e);
}

}  // namespace
}  // namespace mla

extern "C" {

size_t mla_decode_tree_workspace_size(int batch, int drafts, int num_heads, int total_tokens, int num_splits)
{
    if (!mla::tree_sizes_ok(batch, drafts, num_heads, total_tokens))
        return 0;
    return mla::tree_plan(batch, drafts, num_heads, total_tokens, num_splits, mla::current_cu_count()).bytes();
}

int mla_decode_tree_fp16(const void *query, const void *kv_cache, const int *block_table, const int *cu_seqlens,
                         const long long *tree_mask, const int *draft_lens, void *out, void *workspace,
                         size_t workspace_bytes, int batch, int drafts, int num_heads, int total_tokens, int page_size,
                         int num_pages, int block_table_stride, int num_splits, void *stream)
{
    return mla::decode_tree(false, query, kv_cache, block_table, cu_seqlens, tree_mask, draft_lens, out, workspace,
                            workspace_bytes, batch, drafts, num_heads, total_tokens, page_size, num_pages,
                            block_table_stride, num_splits, stream);
}

int mla_decode_tree_bf16(const void *query, const void *kv_cache, const int *block_table, const int *cu_seqlens,
                         const long long *tree_mask, const int *draft_lens, void *out, void *workspace,
                         size_t workspace_bytes, int batch, int drafts, int num_heads, int total_tokens, int page_size,
                         int num_pages, int block_table_stride, int num_splits, void *stream)
{
    return mla::decode_tree(true, query, kv_cache, block_table, cu_seqlens, tree_mask, draft_lens, out, workspace,
                            workspace_bytes, batch, drafts, num_heads, total_tokens, page_size, num_pages,
                            block_table_stride, num_splits, stream);
}

}  // extern "C"
