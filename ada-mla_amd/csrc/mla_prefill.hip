// Causal attention of prompts, or of chunks of prompts behind a cached
// context, in the expanded form (mla_prefill_*):
//
//   k[t, h] = [W_UK[h] c_t, r_t],  v[t, h] = W_UV[h] c_t     (c_t, r_t: latent row t)
//   o[i, h] = softmax_t<=pos(i)( [q_nope, q_rope][i, h] . k[t, h] / sqrt(192) ) v[t, h]
//
// Against the absorbed form a (query, key, head) costs 192 + 128 products
// instead of 576 + 512, for 2 x 128 x 512 once per key and head: with more
// than some 170 queries a key (a prompt of 340 tokens) the expanded form needs fewer.
//
// Two launches mostly: expand_kernel writes K, V and the rotary parts to the
// workspace, tile by tile of 64 keys (each sequence starts a tile of its own);
// attend_kernel is one pass over them with a running maximum and sum. Where few
// queries see long contexts it splits the keys, and merge_kernel joins the parts;
// small calls take narrow_kernel instead.
// K and V are held in the inputs' 16-bit type, as a model that expands its keys
// with a matrix product holds them: a rounding of half a step on each, the sums in
// fp32. With P's (p_operand) that makes three roundings before the result's own.
// Against 64 bits, in units of the error that rounding the result alone has, V's makes
// 1.37, K's 1.2, P's 1.2, all of them 1.35 (some keys) to 1.67 (hundreds). A second 16 bits of V
// would take 16 products more to a tile's 40 and half as much workspace again, fp32 K and
// V twice the workspace and three products for each one.
//
// Measured: 8192 queries at 64 heads 154 us + 1320 us (137 and 1375 GF: 0.9 and
// 1.04 PFLOP/s, where a large matrix product reaches 1.3); 6 prompts of up to 1500
// tokens at 128 heads 187 + 301 us; 197 queries at 16 heads 7.5 + 7.2 us.
#include <algorithm>
#include <cmath>
#include <cstdint>

#include "mla_flash.hpp"
#include "mla_mi355x.h"

namespace mla {
namespace {

constexpr int kNope = 128, kRopeDim = 64, kLatent = 512;
constexpr int kTile = 64;      // keys per tile; sequences are padded to it in the workspace
typedef unsigned long long ulong4x __attribute__((ext_vector_type(4)));
typedef unsigned uint4x __attribute__((ext_vector_type(4)));
constexpr int kQueries = 128;  // queries per workgroup: 32 a wave

bool aligned16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

struct PrefillArgs {
    const void *q_nope, *q_rope, *w_uk, *w_uv, *cache;
    const int *block_table;  // nullptr: a packed cache
    const int *cu_q, *cu_seqlens;
    void *out;
    void *k, *v;                // [head][tile][4 column blocks][64 keys][32]
    void *rope;                 // [padded key][64]
    float *part_o;              // [query tile][head][split][wave][4 column tiles][4][64 lanes][4]
    float *part_m, *part_l;     // [query tile][head][split][128]
    unsigned long long *flags;  // [head][tile][4]: keys whose V holds an infinity or NaN, by 32 of its columns
    int batch, num_heads, queries, total_tokens;
    int padded;  // keys of the workspace: whole tiles
    int q_slots;
    int narrow;        // 1: narrow_kernel
    int splits;        // of a query tile's keys, at most
    int split_tiles;   // key tiles a split, at least
    int key_groups;    // of 32 keys a wave in expand_kernel, 1 or 2
    int group_blocks;  // weight blocks of an expanding workgroup
    int page_shift, num_pages, bt_stride;
    float scale_log2;
};

__device__ __forceinline__ int clamped(const int *cu, int b, int most) { return min(max(cu[b], 0), most); }

// Sequence b's range in cu, and its range in another one.
struct Owner {
    int b, lo, hi, other_lo, other_hi;
};

// The last b < batch with cu[b] / unit + b <= slot, by the whole wave: the
// sequence that owns this slot where each takes the slots from cu[b] / unit +
// b on. That numbering needs no prefix sums of rounded lengths, and no two
// sequences' slots meet. The ranges come with it, in one round trip.
__device__ __forceinline__ Owner owner_of_slot(const int *cu, int most, const int *other, int other_most, int batch,
                                               int unit, int slot, int lane)
{
    Owner w = {};
    for (int base = 0; base < batch; base += 64) {
        const int i = min(base + lane, batch - 1);
        const int lo = clamped(cu, i, most), hi = max(clamped(cu, i + 1, most), lo);
        const int other_lo = clamped(other, i, other_most), other_hi = max(clamped(other, i + 1, other_most), other_lo);
        const unsigned long long m = __builtin_amdgcn_ballot_w64(base + lane < batch && lo / unit + i <= slot);
        if (m != 0) {
            const int k = 63 - __builtin_clzll(m);
            w.b = base + k;
            w.lo = __builtin_amdgcn_readlane(lo, k);
            w.hi = __builtin_amdgcn_readlane(hi, k);
            w.other_lo = __builtin_amdgcn_readlane(other_lo, k);
            w.other_hi = __builtin_amdgcn_readlane(other_hi, k);
        }
        if (m != ~0ull)
            break;
    }
    return w;
}

// ---- expansion --------------------------------------------------------------
// A product of [keys x 512] latents with [512 x 256 heads] weights, whose depth
// is short: with both operands streamed, a workgroup would spend as long on its
// first loads and its stores as on the product. So the keys stay: a wave keeps
// 64 of them (one tile of the workspace) whole in registers, 256 a workgroup,
// and the weights stream past in blocks of 32 rows through an LDS ring, each
// block read once for 256 keys (two products a LDS read). With the weights as
// the A operand a lane owns a key and, with the rows of a block read in the
// order of weight_row, two times 8 adjacent columns of it, the lane 32 on the 8
// beside them. The workspace holds a tile's 64 keys x 32 columns of a block in one
// piece, so that a block's four stores a wave fill 4 KB of whole lines: in rows of 256
// bytes they were what bound this kernel (8192 keys at 64 heads 156 us, 124 without them).
// kGroups: groups of 32 keys a wave, 2 or, for calls that leave most of the CUs
// idle, 1: half the time to load the keys, and one product a LDS read.
constexpr int kWeightRows = 32;                       // rows of W a block
constexpr int kWeightElems = kWeightRows * kLatent;   // 32 KB
constexpr int kWeightRing = 4;
constexpr int kExpandWaves = 4;
constexpr int kBlocksPerSide = kNope / kWeightRows;   // blocks of one head's W_UK or W_UV

// The row of a weight block in row rho = 8 q + 4 c + j of the product's tile:
// lane half c then holds columns 8 c .. 8 c + 7 in its registers 0 .. 7 and 16 + 8 c ..
// in the others.
__device__ __forceinline__ int weight_row(int rho)
{
    return 16 * (rho >> 4) + 8 * ((rho >> 2) & 1) + 4 * ((rho >> 3) & 1) + (rho & 3);
}

// 16-byte chunk c of row r sits at c ^ weight_swizzle(r): rho mod 16, so that
// 16 lanes that read one chunk of 16 successive rho meet 16 places.
__device__ __forceinline__ int weight_swizzle(int r)
{
    return 8 * ((r >> 2) & 1) + 4 * ((r >> 3) & 1) + (r & 3);
}

template <typename E, int kGroups>
__global__ __attribute__((amdgpu_flat_work_group_size(256, 256), amdgpu_waves_per_eu(1, 1))) void
expand_kernel(PrefillArgs a)
{
    using E8 = typename Vec<E>::v8;
    __shared__ __attribute__((aligned(1024))) E s_ring[kWeightRing * kWeightElems];
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int r32 = lane & 31, hl = lane >> 5;
    // workgroup -> (group of weight blocks, four key tiles): the key tiles of a
    // group get ids that differ by 8, one XCD, whose L2 then holds the group's weights
    constexpr int kPerTile = 2 / kGroups;  // waves
    const int tiles = a.padded / kTile, quads = (tiles * kPerTile + kExpandWaves - 1) / kExpandWaves;
    const int group = (blockIdx.x >> 3) / quads * 8 + (blockIdx.x & 7);
    const int unit = (blockIdx.x >> 3) % quads * kExpandWaves + wave;
    const int tile = unit / kPerTile, key0 = 32 * (unit % kPerTile);  // the wave's tile, and its first key there
    const int n_blocks = 2 * kBlocksPerSide * a.num_heads;
    const int blk0 = group * a.group_blocks, blk1 = min(blk0 + a.group_blocks, n_blocks);
    if (blk0 >= n_blocks)
        return;

    // Block i: rows 32 (i mod 4) .. of side (i / 4) mod 2 of head i / 8. The
    // wave's 8 load units are its rows of 1 KB, which follow each other in
    // memory and in LDS; a row's swizzle differs from the first one's by an XOR.
    const unsigned ring = lds_address(s_ring);
    const int w_off = 16 * (lane ^ weight_swizzle(kWeightRows / 4 * wave));
    // Past the group's last block it is loaded again, into a slot that nobody
    // reads: every block then has the same instructions and the same counts.
    auto block_source = [&](int i) -> const E * {
        i = min(i, blk1 - 1);
        const int h = i / (2 * kBlocksPerSide), rest = i % (2 * kBlocksPerSide);
        return wave_uniform((const E *)(rest >= kBlocksPerSide ? a.w_uv : a.w_uk) +
                            ((size_t)h * kNope + rest % kBlocksPerSide * kWeightRows + kWeightRows / 4 * wave) * kLatent);
    };
    auto slot_of = [&](int i) {
        return ring + ((i - blk0) & (kWeightRing - 1)) * (kWeightElems * 2) + kWeightRows / 4 * wave * (kLatent * 2);
    };
    auto load_unit = [&](const E *src, unsigned dst, auto unit) {
        constexpr int u = decltype(unit)::value;
        stream_to_lds16<4096 * (u >> 2), 4096 * (u >> 2), 1024 * (u & 3)>(src, w_off ^ (16 * (u & 3)) ^ (128 * (u >> 2)), dst);
    };
    auto load_block = [&](int i) {
        const E *src = block_source(i);
        const unsigned dst = slot_of(i);
        for_constants([&](auto unit) { load_unit(src, dst, unit); }, std::make_integer_sequence<int, kWeightRows / 4>{});
    };
    // The wave's keys: latent rows of 1 KB by direct loads into the wave's own
    // ring slot, 32 at a time, then into registers (chunk c of row r at c ^ (r
    // mod 16)). Loaded into registers at once, every load touched 32 rows: 18 us
    // a workgroup with all CUs loading. Rows past the sequence are zeros.
    const Owner w = owner_of_slot(a.cu_seqlens, a.total_tokens, a.cu_seqlens, a.total_tokens, a.batch, kTile, tile, lane);
    const int b = w.b, seq_lo = w.lo, len = w.hi - w.lo;
    const int t0 = (tile - seq_lo / kTile - b) * kTile + key0;
    const bool live = tile < tiles && t0 - key0 < len;  // else nobody reads this tile
    if (!__syncthreads_or(live))
        return;
    auto key_source = [&](int t) -> const E * {  // latent row t of the sequence; the 32 rows of a block follow it
        size_t row;
        if (a.block_table) {
            const int col = min(t >> a.page_shift, a.bt_stride - 1);
            const int page = min(max(scalar_load(a.block_table + (size_t)b * a.bt_stride + col), 0), a.num_pages - 1);
            row = ((size_t)page << a.page_shift) + (t & ((1 << a.page_shift) - 1));
        } else {
            row = seq_lo + t;
        }
        return (const E *)a.cache + row * kDK;
    };
    E8 key[kGroups][kLatent / 16];
#pragma unroll
    for (int g = 0; g < kGroups; ++g) {
        const int t = t0 + 32 * g;
        if (live && t < len) {
            const E *src = wave_uniform(key_source(t));
            const int lim = min(31, len - 1 - t);
            const unsigned own = ring + wave * (kWeightElems * 2);
#pragma unroll
            for (int r = 0; r < 32; ++r)
                global_to_lds16_at(src + (size_t)min(r, lim) * kDK, 16 * (lane ^ row_swizzle(r)), own + r * (kLatent * 2));
            if (group == 0) {  // the rotary parts: 8 chunks a key
#pragma unroll
                for (int u = 0; u < 4; ++u) {
                    const int r = 8 * u + (lane >> 3);
                    *(uint4 *)((E *)a.rope + ((size_t)tile * kTile + key0 + 32 * g + r) * kRopeDim + 8 * (lane & 7)) =
                        *(const uint4 *)(src + (size_t)min(r, lim) * kDK + kLatent + 8 * (lane & 7));
                }
            }
            MLA_WAIT_VMCNT(0);
            asm volatile("" ::: "memory");
            const unsigned at = own + r32 * (kLatent * 2) + 16 * (hl ^ row_swizzle(r32));
            const bool real = r32 <= lim;
#pragma unroll
            for (int k = 0; k < kLatent / 16; ++k) {
                const uint4x v = lds_load<uint4x>((at ^ (32 * (k & 7))) + 256 * (k >> 3));
                key[g][k] = __builtin_bit_cast(E8, real ? v : uint4x{0, 0, 0, 0});
            }
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        } else {
#pragma unroll
            for (int k = 0; k < kLatent / 16; ++k)
                key[g][k] = E8{};
        }
#pragma unroll
        for (int k = 0; k < kLatent / 16; ++k)
            in_acc_registers(key[g][k]);
    }
    lds_barrier();  // the ring is free
    for (int i = blk0; i < blk0 + kWeightRing - 1; ++i)
        load_block(i);

    const int row = weight_row(r32);
    const unsigned w_lane = row * (kLatent * 2) + 16 * (hl ^ weight_swizzle(row));
    unsigned bad[kGroups] = {};  // the wave's keys whose V is not finite, in the block of `store`
    const unsigned row_at = (key0 + r32) * (kWeightRows * 2) + 16 * hl;  // the lane's first 8 values in the block's rows
    // Rounds and stores quarter `part` of key group g of block i, whose sums
    // are in acc; v and top gather a group's four quarters.
    auto store = [&](int i, const floatx16 (&acc)[kGroups], int g, int part, unsigned &top, E8 (&v)[2]) {
        typedef float floatx4v __attribute__((ext_vector_type(4)));
        const auto x = __builtin_convertvector(
            (floatx4v{acc[g][4 * part], acc[g][4 * part + 1], acc[g][4 * part + 2], acc[g][4 * part + 3]}), typename Vec<E>::v4);
#pragma unroll
        for (int r = 0; r < 4; ++r)
            v[part >> 1][4 * (part & 1) + r] = x[r];
        const auto w = __builtin_bit_cast(uint4x, v[part >> 1]);
#pragma unroll
        for (int k = 0; k < 2; ++k)  // the largest magnitude's bits, both halves
            top = max_u16x2(top, w[2 * (part & 1) + k] & 0x7fff7fffu);
        if (part != 3)
            return;
        const int h = i / (2 * kBlocksPerSide), rest = i % (2 * kBlocksPerSide);
        const bool side = rest >= kBlocksPerSide;
        const bool lane_bad = not_finite<E>((unsigned short)top) || not_finite<E>((unsigned short)(top >> 16));
        const unsigned long long m = __builtin_amdgcn_ballot_w64(lane_bad);
        if (m != 0) {
            // V: what is not finite becomes 0 and flags its key, so that a
            // query that must not see the key can meet it with weight 0. K: it
            // becomes NaN, as an infinity that was a finite value before its rounding
            // to fp16 could make a logit of -inf, and the key would count for nothing.
            const E put = side ? (E)0.0f : (E)NAN;
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const E y = v[r >> 3][r & 7];
                v[r >> 3][r & 7] = not_finite<E>(__builtin_bit_cast(unsigned short, y)) ? put : y;
            }
            bad[g] |= (unsigned)m | (unsigned)(m >> 32);
        }
        char *dst = (char *)wave_uniform((const char *)(side ? a.v : a.k) +
                                         (((size_t)h * tiles + tile) * kBlocksPerSide + rest % kBlocksPerSide) *
                                             (kTile * kWeightRows * 2));
        if (i >= blk0 && live) {
            *(E8 *)(dst + (row_at + 32 * g * (kWeightRows * 2))) = v[0];
            *(E8 *)(dst + (row_at + 32 * g * (kWeightRows * 2) + 32)) = v[1];
            if (side && lane == 0)
                ((unsigned *)a.flags)[2 * (((size_t)h * tiles + tile) * kBlocksPerSide + rest % kBlocksPerSide) + key0 / 32 + g] =
                    bad[g];
        }
        bad[g] = 0;
    };
    // Block i into acc, while block i - 1, in prev, is rounded and stored
    // between the products, a quarter of a group after every 8 of the 64.
    auto block = [&](int i, floatx16 (&acc)[kGroups], floatx16 (&prev)[kGroups]) {
        // Block i's 8 loads went out during block i - 3. Behind the last of them
        // come, in order, that block's 2 stores of a second group (half of block i - 4's;
        // one more where it holds flags), then twice 8 loads (of blocks i + 1, i + 2)
        // and 2 stores a group: at least 26, or 20 of one group. The first blocks have fewer
        // stores behind them.
        if (live && i - blk0 >= 4)
            MLA_WAIT_VMCNT(2 * (kWeightRows / 4) + 2 * 2 * kGroups + 2 * (kGroups - 1));
        else
            MLA_WAIT_VMCNT(2 * (kWeightRows / 4));
        lds_barrier();  // block i is there, and block i - 1's slot is free
        const E *feed_src = block_source(i + kWeightRing - 1);
        const unsigned feed_at = slot_of(i + kWeightRing - 1);
        const unsigned at = ring + ((i - blk0) & (kWeightRing - 1)) * (kWeightElems * 2) + w_lane;
        auto operand = [&](int k) -> E8 { return lds_load<E8>((at ^ (32 * (k & 7))) + 256 * (k >> 3)); };
        constexpr int kAhead = 4;  // steps an operand is read ahead
        E8 w[kAhead + 1], v[kGroups][2];
        unsigned top[kGroups] = {};
#pragma unroll
        for (int k = 0; k < kAhead; ++k)
            w[k] = operand(k);
        for_constants(
            [&](auto step) {
                constexpr int k = decltype(step)::value;
                if constexpr (k + kAhead < kLatent / 16)
                    w[(k + kAhead) % (kAhead + 1)] = operand(k + kAhead);
#pragma unroll
                for (int g = 0; g < kGroups; ++g) {
                    if constexpr (k == 0)
                        mfma32x32x16_first_acc(acc[g], w[0], key[g][0]);
                    else
                        mfma32x32x16_next_acc(acc[g], w[k % (kAhead + 1)], key[g][k]);
                }
                if constexpr (k == 2)  // three products at least behind the last of block i - 1
#pragma unroll
                    for (int g = 0; g < kGroups; ++g)
                        in_registers(prev[g]);
                if constexpr (k % 4 == 1)
                    load_unit(feed_src, feed_at, std::integral_constant<int, k / 4>{});
                if constexpr (k % 4 == 3 && k / 16 < kGroups)
                    store(i - 1, prev, k / 16, k / 4 % 4, top[k / 16], v[k / 16]);
                __builtin_amdgcn_sched_barrier(0);
            },
            std::make_integer_sequence<int, kLatent / 16>{});
    };
    auto store_last = [&](floatx16 (&acc)[kGroups]) {
#pragma unroll
        for (int g = 0; g < kGroups; ++g) {
            mfma_settle(acc[g]);
            E8 v[2];
            unsigned top = 0;
#pragma unroll
            for (int part = 0; part < 4; ++part)
                store(blk1 - 1, acc, g, part, top, v);
        }
    };
    floatx16 even[kGroups] = {}, odd[kGroups] = {};
    for (int i = blk0; i < blk1; i += 2) {
        block(i, even, odd);
        if (i + 1 < blk1)
            block(i + 1, odd, even);
    }
    if ((blk1 - blk0) & 1)
        store_last(even);
    else
        store_last(odd);
    MLA_WAIT_VMCNT(0);  // no load to LDS outlives the workgroup
}

// ---- attention --------------------------------------------------------------
// 128 queries a workgroup, 32 a wave, so that Q, O, S and P fit 256 registers and two
// workgroups share a CU: one's softmax runs beside the other's products. With 64
// queries a wave, half the LDS reads a product and one workgroup a CU, 8192
// queries at 64 heads took 1454 us against 1300. Key tiles are double buffered (80 KB
// a workgroup). Bound by the matrix units, which the products fill 77% of a tile's
// cycles, at the clock of some 1.6 GHz that this load leaves; prompts of a few hundred tokens
// spend a third of the time in the workgroups' starts and ends.

// A workgroup's queries: q0 .. of one sequence, and its keys.
struct QueryTile {
    int q_lo, n_q, q0;  // the sequence's first query, its queries, the tile's first one
    int n_k, tile0;     // its keys, its first tile in the workspace
    int n_tiles;        // tiles with keys that the queries see (0 or less: none)
    int per, n_splits;  // key tiles a split, and the splits
    int rows;           // rows of out from q_lo on: the last sequence's go on to the end of it
};

template <int kUnit>  // queries of a tile
__device__ __forceinline__ QueryTile query_tile(const PrefillArgs &a, int slot, int lane)
{
    QueryTile t;
    const Owner w = owner_of_slot(a.cu_q, a.queries, a.cu_seqlens, a.total_tokens, a.batch, kUnit, slot, lane);
    t.q_lo = w.lo;
    t.n_q = w.hi - w.lo;
    t.q0 = (slot - t.q_lo / kUnit - w.b) * kUnit;
    t.rows = w.b == a.batch - 1 ? a.queries - t.q_lo : t.n_q;
    t.n_k = w.other_hi - w.other_lo;
    t.tile0 = w.other_lo / kTile + w.b;
    t.n_tiles = (min(t.n_k, min(t.q0 + kUnit, t.n_q) + t.n_k - t.n_q) + kTile - 1) / kTile;
    t.per = INT32_MAX / 2;
    t.n_splits = 1;
    if (a.splits > 1) {
        t.per = max(a.split_tiles, (t.n_tiles + a.splits - 1) / a.splits);
        t.n_splits = max(1, (t.n_tiles + t.per - 1) / t.per);
    }
    return t;
}

// A tile behind the last sequence's queries: zeros.
template <typename E, int kUnit>
__device__ __forceinline__ void zero_rows(const PrefillArgs &a, const QueryTile &t, int h)
{
    for (int i = threadIdx.x; i < min(kUnit, t.rows - t.q0) * (kNope / 8); i += 256)
        *(uint4 *)((E *)a.out + ((size_t)(t.q_lo + t.q0 + i / (kNope / 8)) * a.num_heads + h) * kNope +
                   8 * (i % (kNope / 8))) = uint4{0, 0, 0, 0};
}

// The wave's 32 rows from `first` on (relative to the sequence's first query): normalised, rounded, through
// the wave's 8 KB of LDS at `at`, stored by whole rows (as they lie in the registers, a store would touch 32
// rows). A query that sees no key (l = 0) gives zeros, as do the rows behind the last sequence's queries.
template <typename E>
__device__ __forceinline__ void store_rows(const PrefillArgs &a, const QueryTile &t, int h, int first, int lane, unsigned at,
                                           const floatx16 (&o)[4], float l)
{
    using E4 = typename Vec<E>::v4;
    const int r32 = lane & 31, hl = lane >> 5;
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    const unsigned row_at = at + r32 * (kNope * 2) + 16 * key_swizzle(r32) + 8 * hl;
#pragma unroll
    for (int c = 0; c < 4; ++c)
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            E4 v;
#pragma unroll
            for (int e = 0; e < 4; ++e)
                v[e] = first + r32 < t.n_q ? (E)(o[c][4 * k + e] * inv) : (E)0.0f;
            lds_store(row_at ^ (16 * (4 * c + k)), v);
        }
    E *out = (E *)a.out + ((size_t)(t.q_lo + first) * a.num_heads + h) * kNope + 8 * (lane & 15);
#pragma unroll
    for (int u = 0; u < 8; ++u) {
        const int r = 4 * u + (lane >> 4);
        const uint4x v = lds_load<uint4x>(at + r * (kNope * 2) + 16 * ((lane & 15) ^ key_swizzle(r)));
        if (first + r < t.rows)
            *(uint4x *)(out + (size_t)r * a.num_heads * kNope) = v;
    }
}

constexpr int kVAt = kTile * kNope * 2, kRopeAt = 2 * kVAt;         // bytes of a stage before V, before the rotary parts
constexpr int kStageBytes = kRopeAt + kTile * kRopeDim * 2;         // 40 KB

// One wave's work on a tile of 64 keys in LDS, for its 32 queries.

// S^T: the lane's logits. k_at and rope_at: the lane's operand 0 of the keys' own
// parts and of the rotary ones.
template <typename E>
__device__ __forceinline__ void tile_logits(unsigned k_at, unsigned rope_at, const typename Vec<E>::v8 (&q)[12], floatx16 (&s)[2])
{
    using E8 = typename Vec<E>::v8;
    // operand k of both 32-key blocks: 8 steps of the head's own part, 4 of the rotary one
    auto operand = [&](int g, int k) -> E8 {
        return k < 8 ? lds_load<E8>((k_at ^ (32 * k)) + 32 * g * (kNope * 2))
                     : lds_load<E8>((rope_at ^ (32 * (k - 8))) + 32 * g * (kRopeDim * 2));
    };
    E8 kv[2][2][2];
#pragma unroll
    for (int g = 0; g < 2; ++g)
#pragma unroll
        for (int i = 0; i < 2; ++i)
            kv[0][g][i] = operand(g, i);
#pragma unroll
    for (int k = 0; k < 12; k += 2) {
        if (k + 2 < 12) {
#pragma unroll
            for (int g = 0; g < 2; ++g)
#pragma unroll
                for (int i = 0; i < 2; ++i)
                    kv[(k / 2 + 1) & 1][g][i] = operand(g, k + 2 + i);
            __builtin_amdgcn_sched_barrier(0);
        }
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int g = 0; g < 2; ++g)
                s[g] = mfma32x32x16(kv[(k / 2) & 1][g][i], q[k + i], s[g]);
        __builtin_amdgcn_sched_barrier(0);
    }
}

// The weights p of keys t0 .. t0 + 63 from their logits, and the running maximum
// m, sum l and output o moved on. The lane's query sees the keys up to `last`, every
// query of the wave those up to `wave_first`.
template <typename E>
__device__ __forceinline__ void tile_weights(const PrefillArgs &a, int t0, int wave_first, int last, int hl, const ulong4x *flags,
                                             floatx16 (&s)[2], float (&p)[32], float &m, float &l, floatx16 (&o)[4])
{
    if (t0 + kTile - 1 > wave_first) {
#pragma unroll
        for (int g = 0; g < 2; ++g)
#pragma unroll
            for (int r = 0; r < 16; ++r)
                s[g][r] = t0 + 32 * g + key_of_reg(r, hl) <= last ? s[g][r] : -INFINITY;
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
#pragma unroll
    for (int r = 0; r < 32; ++r) {
        p[r] = fast_exp2(s[r >> 4][r & 15] * a.scale_log2 - ref);
        l += p[r];
    }
    const ulong4x f4 = scalar_load(flags);
    const unsigned long long bad = f4[0] | f4[1] | f4[2] | f4[3];
    if (bad != 0) {  // a query that sees a key whose V is not finite gives NaN
#pragma unroll
        for (int r = 0; r < 32; ++r) {
            const int t = 32 * (r >> 4) + key_of_reg(r & 15, hl);
            if (((bad >> t) & 1) != 0 && t0 + t <= last)
                l = NAN;
        }
    }
}

// O^T += V^T P^T. v_at0, v_at1: the lane's two transpose reads of the first operand.
template <typename E>
__device__ __forceinline__ void tile_values(unsigned v_at0, unsigned v_at1, const float (&p)[32], floatx16 (&o)[4])
{
    using E8 = typename Vec<E>::v8;
    using E4 = typename Vec<E>::v4;
    auto operand = [&](int ks, int c) -> E8 {  // columns 32 c .. of V^T, keys 16 ks .. +15 in P's order
        E4 part[2];
#pragma unroll
        for (int i = 0; i < 2; ++i)
            part[i] = lds_load_tr16<E>(((i ? v_at1 : v_at0) ^ (64 * c)) + 16 * ks * (kNope * 2));
        return E8{part[0][0], part[0][1], part[0][2], part[0][3], part[1][0], part[1][1], part[1][2], part[1][3]};
    };
    E8 v[2][4];
#pragma unroll
    for (int c = 0; c < 4; ++c)
        v[0][c] = operand(0, c);
#pragma unroll
    for (int ks = 0; ks < 4; ++ks) {
        if (ks + 1 < 4) {
#pragma unroll
            for (int c = 0; c < 4; ++c)
                v[(ks + 1) & 1][c] = operand(ks + 1, c);
            __builtin_amdgcn_sched_barrier(0);
        }
        const E8 pb = p_operand<E>(p + 8 * ks);
#pragma unroll
        for (int c = 0; c < 4; ++c)
            o[c] = mfma32x32x16(v[ks & 1][c], pb, o[c]);
        __builtin_amdgcn_sched_barrier(0);
    }
}

// The lane's LDS addresses in a stage (K at 0, V, the rotary parts), and its part
// of the load units' offsets in the workspace: 4 keys of 256 bytes in LDS are
// 4 times 64 bytes there, the swizzle's low bits changing from one unit to the next.
struct TileLanes {
    unsigned k, rope, v[2];
    int kv_off, rope_off;
    __device__ __forceinline__ explicit TileLanes(int lane)
    {
        const int r32 = lane & 31, hl = lane >> 5, j = lane & 15;
        k = r32 * (kNope * 2) + 16 * (hl ^ key_swizzle(r32));
        rope = kRopeAt + r32 * (kRopeDim * 2) + 16 * (hl ^ rope_swizzle(r32));
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int r = 8 * i + 4 * hl + (j >> 2);
            v[i] = kVAt + r * (kNope * 2) + 16 * ((2 * ((lane >> 4) & 1) + ((j & 3) >> 1)) ^ key_swizzle(r)) + 8 * (j & 1);
        }
        const int chunk = j ^ key_swizzle(lane >> 4);
        kv_off = (chunk >> 2) * (kTile * kWeightRows * 2) + (lane >> 4) * (kWeightRows * 2) + 16 * (chunk & 3);
        rope_off = (lane >> 3) * (kRopeDim * 2) + 16 * ((lane & 7) ^ rope_swizzle(lane >> 3));
    }
};

template <typename E>
__global__ __launch_bounds__(256, 2) void attend_kernel(PrefillArgs a)
{
    using E8 = typename Vec<E>::v8;
    __shared__ __attribute__((aligned(1024))) char s_buf[2][kStageBytes];
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int r32 = lane & 31, hl = lane >> 5;
    // workgroup -> (head, query tile, split): all tiles of a head on one XCD, whose L2
    // then holds its K and V, the last (longest) first
    const int li = blockIdx.x >> 3, tile = a.splits > 1 ? li / a.splits : li, split = li - tile * a.splits;
    const int h = tile / a.q_slots * 8 + (blockIdx.x & 7);
    const int slot = a.q_slots - 1 - tile % a.q_slots;
    if (h >= a.num_heads)
        return;
    const QueryTile t = query_tile<kQueries>(a, slot, lane);
    if (split >= t.n_splits)
        return;
    if (t.q0 >= t.n_q) {
        if (split == 0)
            zero_rows<E, kQueries>(a, t, h);
        return;
    }
    const int q0 = t.q0, n_q = t.n_q, tile0 = t.tile0;
    const int shift = t.n_k - n_q;  // query i sees the keys 0 .. i + shift
    const int j0 = split == 0 ? 0 : split * t.per, j1 = min(j0 + t.per, t.n_tiles);  // the split's key tiles

    const int row = q0 + 32 * wave + r32;
    const int last = min(row, n_q - 1) + shift;  // the lane's last key
    const unsigned lds = lds_address(s_buf);
    const TileLanes at_lane(lane);
    const E *ks = wave_uniform((const E *)a.k + ((size_t)h * a.padded + (size_t)tile0 * kTile) * kNope + 16 * wave * kWeightRows);
    const E *vs = wave_uniform((const E *)a.v + ((size_t)h * a.padded + (size_t)tile0 * kTile) * kNope + 16 * wave * kWeightRows);
    const E *rs = wave_uniform((const E *)a.rope + ((size_t)tile0 * kTile + 16 * wave) * kRopeDim);
    const ulong4x *flags = (const ulong4x *)a.flags + (size_t)h * (a.padded / kTile) + tile0;
    // A wave's 10 load units: 4 of K, 4 of V and 2 of the rotary parts (8 rows of 128 bytes).
    constexpr int kUnits = 10;
    auto load_tile = [&](int j) {
        const unsigned at = lds + ((j - j0) & 1) * kStageBytes;
        const E *k = ks + (size_t)j * (kTile * kNope), *v = vs + (size_t)j * (kTile * kNope);
        const E *r = rs + (size_t)j * (kTile * kRopeDim);
        for_constants(
            [&](auto unit) {
                constexpr int u = decltype(unit)::value;
                stream_to_lds16<4 * u * kWeightRows * 2, 1024 * u, 0>(k, at_lane.kv_off ^ (16 * u), at + 4096 * wave);
                stream_to_lds16<4 * u * kWeightRows * 2, kVAt + 1024 * u, 0>(v, at_lane.kv_off ^ (16 * u), at + 4096 * wave);
            },
            std::make_integer_sequence<int, 4>{});
        stream_to_lds16<0, kRopeAt, 0>(r, at_lane.rope_off, at + 2048 * wave);
        stream_to_lds16<0, kRopeAt, 1024>(r, at_lane.rope_off ^ 64, at + 2048 * wave);
    };
    // The queries, the B operand of S^T: their own part comes by whole rows
    // through the second stage, 8 KB a wave, while the first key tile is on its
    // way to the first one. Rows past the sequence's queries re-read the last one.
    E8 q[12];
    {
        const int lim = n_q - 1 - q0;
        const size_t q_at = (size_t)(t.q_lo + q0) * a.num_heads + h;
        const E *qn = wave_uniform((const E *)a.q_nope + q_at * kNope);
        const E *qr = (const E *)a.q_rope + (q_at + (size_t)min(32 * wave + r32, lim) * a.num_heads) * kRopeDim + 8 * hl;
        const unsigned own = lds + kStageBytes + wave * 8192;
#pragma unroll
        for (int u = 0; u < 8; ++u) {
            const int r = 4 * u + (lane >> 4);
            global_to_lds16_at(qn, min(32 * wave + r, lim) * (a.num_heads * (kNope * 2)) + 16 * ((lane & 15) ^ key_swizzle(r)),
                               own + 1024 * u);
        }
#pragma unroll
        for (int k = 0; k < 4; ++k)
            q[8 + k] = *(const E8 *)(qr + 16 * k);
        if (j0 < j1)
            load_tile(j0);
        if (j0 < j1)
            MLA_WAIT_VMCNT(kUnits);
        else
            MLA_WAIT_VMCNT(0);
        asm volatile("" ::: "memory");
#pragma unroll
        for (int k = 0; k < 8; ++k)
            q[k] = lds_load<E8>((own + at_lane.k) ^ (32 * k));
    }
    floatx16 o[4] = {};
    float m = -INFINITY, l = 0.0f;
    // the last key of the wave's queries; a wave without queries only loads
    const int wave_last = q0 + 32 * wave < n_q ? min(q0 + 32 * wave + 31, n_q - 1) + shift : -1;
    const int wave_first = min(q0 + 32 * wave, n_q - 1) + shift;
    for (int j = j0; j < j1; ++j) {
        MLA_WAIT_VMCNT(0);
        lds_barrier();  // tile j is there, and everyone is done with tile j - 1
        if (j + 1 < j1)
            load_tile(j + 1);
        if (j * kTile > wave_last)
            continue;
        const unsigned at = lds + ((j - j0) & 1) * kStageBytes;
        floatx16 s[2] = {};
        float p[32];
        tile_logits<E>(at + at_lane.k, at + at_lane.rope, q, s);
        tile_weights<E>(a, j * kTile, wave_first, last, hl, flags + j, s, p, m, l, o);
        tile_values<E>(at + at_lane.v[0], at + at_lane.v[1], p, o);
    }
    l = reduce_halves(l, [](float x, float y) { return x + y; });
    if (t.n_splits > 1) {
        const size_t part = ((size_t)slot * a.num_heads + h) * a.splits + split;
        float *po = a.part_o + (part * 4 + wave) * (32 * kNope);
#pragma unroll
        for (int c = 0; c < 4; ++c)
#pragma unroll
            for (int k = 0; k < 4; ++k)
                *(floatx4 *)(po + ((c * 4 + k) * 64 + lane) * 4) =
                    floatx4{o[c][4 * k], o[c][4 * k + 1], o[c][4 * k + 2], o[c][4 * k + 3]};
        if (hl == 0) {
            a.part_m[part * kQueries + 32 * wave + r32] = m;
            a.part_l[part * kQueries + 32 * wave + r32] = l;
        }
        return;
    }
    lds_barrier();  // everyone is done with the last tile
    store_rows<E>(a, t, h, q0 + 32 * wave, lane, lds + wave * 8192, o, l);
}

// The same for calls so small that 128 queries a workgroup leave most of the CUs idle:
// 32 queries a workgroup, and its waves take the key tiles in turn, each a stage of its own
// and its own running maximum and sum, which meet at the end. A wave's next K is on
// its way while the weights and O take a tile, its next V while the logits do.
constexpr int kNarrow = 32;

template <typename E>
__global__ __attribute__((amdgpu_flat_work_group_size(256, 256), amdgpu_waves_per_eu(1, 1))) void
narrow_kernel(PrefillArgs a)
{
    using E8 = typename Vec<E>::v8;
    using E4 = typename Vec<E>::v4;
    __shared__ __attribute__((aligned(1024))) char s_buf[4][kStageBytes];
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int r32 = lane & 31, hl = lane >> 5;
    const int li = blockIdx.x >> 3;
    const int h = li / a.q_slots * 8 + (blockIdx.x & 7);
    const int slot = a.q_slots - 1 - li % a.q_slots;
    if (h >= a.num_heads)
        return;
    const QueryTile t = query_tile<kNarrow>(a, slot, lane);
    if (t.q0 >= t.n_q) {
        zero_rows<E, kNarrow>(a, t, h);
        return;
    }
    const int shift = t.n_k - t.n_q;  // query i sees the keys 0 .. i + shift
    const int last = min(t.q0 + r32, t.n_q - 1) + shift, first = t.q0 + shift;
    const unsigned at = lds_address(s_buf) + wave * kStageBytes;
    const TileLanes at_lane(lane);
    const E *ks = wave_uniform((const E *)a.k + ((size_t)h * a.padded + (size_t)t.tile0 * kTile) * kNope);
    const E *vs = wave_uniform((const E *)a.v + ((size_t)h * a.padded + (size_t)t.tile0 * kTile) * kNope);
    const E *rs = wave_uniform((const E *)a.rope + (size_t)t.tile0 * kTile * kRopeDim);
    const ulong4x *flags = (const ulong4x *)a.flags + (size_t)h * (a.padded / kTile) + t.tile0;
    // a tile's load units: 16 of K and 8 of the rotary parts, then 16 of V
    constexpr int kKeyUnits = 24, kValueUnits = 16;
    auto load_keys = [&](int j) {
        const E *k = ks + (size_t)j * (kTile * kNope), *r = rs + (size_t)j * (kTile * kRopeDim);
        for_constants(
            [&](auto unit) {
                constexpr int u = decltype(unit)::value;
                stream_to_lds16<4 * u * kWeightRows * 2, 1024 * u, 0>(k, at_lane.kv_off ^ (16 * (u & 3)), at);
            },
            std::make_integer_sequence<int, 16>{});
        for_constants(
            [&](auto unit) {
                constexpr int u = decltype(unit)::value;
                stream_to_lds16<1024 * u, kRopeAt + 1024 * u, 0>(r, at_lane.rope_off ^ (64 * (u & 1)), at);
            },
            std::make_integer_sequence<int, 8>{});
    };
    auto load_values = [&](int j) {
        const E *v = vs + (size_t)j * (kTile * kNope);
        for_constants(
            [&](auto unit) {
                constexpr int u = decltype(unit)::value;
                stream_to_lds16<4 * u * kWeightRows * 2, kVAt + 1024 * u, 0>(v, at_lane.kv_off ^ (16 * (u & 3)), at);
            },
            std::make_integer_sequence<int, 16>{});
    };
    // the wave's reads of LDS have ended: what they read may be loaded over
    auto reads_done = [] { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); };

    floatx16 o[4] = {};
    float m = -INFINITY, l = 0.0f;
    if (wave < t.n_tiles) {
        // the queries through V's place, whole rows: 8 KB of their own part, 4 KB of the rotary one
        E8 q[12];
        const int lim = t.n_q - 1 - t.q0;
        const size_t q_at = (size_t)(t.q_lo + t.q0) * a.num_heads + h;
        const E *qn = wave_uniform((const E *)a.q_nope + q_at * kNope);
        const E *qr = wave_uniform((const E *)a.q_rope + q_at * kRopeDim);
        constexpr int kQRopeAt = 32 * kNope * 2;
#pragma unroll
        for (int u = 0; u < 8; ++u) {
            const int r = 4 * u + (lane >> 4);
            global_to_lds16_at(qn, min(r, lim) * (a.num_heads * (kNope * 2)) + 16 * ((lane & 15) ^ key_swizzle(r)),
                               at + kVAt + 1024 * u);
        }
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const int r = 8 * u + (lane >> 3);
            global_to_lds16_at(qr, min(r, lim) * (a.num_heads * (kRopeDim * 2)) + 16 * ((lane & 7) ^ rope_swizzle(r)),
                               at + kVAt + kQRopeAt + 1024 * u);
        }
        load_keys(wave);
        MLA_WAIT_VMCNT(kKeyUnits);
        asm volatile("" ::: "memory");
#pragma unroll
        for (int k = 0; k < 12; ++k)
            q[k] = k < 8 ? lds_load<E8>((at + kVAt + at_lane.k) ^ (32 * k))
                         : lds_load<E8>((at + kVAt + kQRopeAt + at_lane.rope - kRopeAt) ^ (32 * (k - 8)));
#pragma unroll
        for (int k = 0; k < 12; ++k)
            in_registers(q[k]);
        reads_done();
        load_values(wave);
        for (int j = wave; j < t.n_tiles; j += 4) {
            const bool more = j + 4 < t.n_tiles;
            MLA_WAIT_VMCNT(kValueUnits);  // K and the rotary parts are there, V may not be
            asm volatile("" ::: "memory");
            floatx16 s[2] = {};
            float p[32];
            tile_logits<E>(at + at_lane.k, at + at_lane.rope, q, s);
            reads_done();
            if (more)
                load_keys(j + 4);
            tile_weights<E>(a, j * kTile, first, last, hl, flags + j, s, p, m, l, o);
            if (more)
                MLA_WAIT_VMCNT(kKeyUnits);
            else
                MLA_WAIT_VMCNT(0);
            asm volatile("" ::: "memory");
            tile_values<E>(at + at_lane.v[0], at + at_lane.v[1], p, o);
            reads_done();
            if (more)
                load_values(j + 4);
        }
    }
    l = reduce_halves(l, [](float x, float y) { return x + y; });
    // the waves' parts, each in its own stage: O as it lies in the registers (16 KB), m and l
    constexpr int kMAt = 32 * kNope * 4;
#pragma unroll
    for (int c = 0; c < 4; ++c)
#pragma unroll
        for (int k = 0; k < 4; ++k)
            lds_store(at + (4 * c + k) * 1024 + 16 * lane,
                      floatx4{o[c][4 * k], o[c][4 * k + 1], o[c][4 * k + 2], o[c][4 * k + 3]});
    if (hl == 0) {
        lds_store(at + kMAt + 4 * r32, m);
        lds_store(at + kMAt + 128 + 4 * r32, l);
    }
    lds_barrier();
    // wave c: columns 32 c .. of the 32 rows
    const unsigned all = at - wave * kStageBytes;
    float top = -INFINITY;
#pragma unroll
    for (int w = 0; w < 4; ++w)
        top = fmaxf(top, lds_load<float>(all + w * kStageBytes + kMAt + 4 * r32));
    const float ref = top == -INFINITY ? 0.0f : top;
    floatx4 sum[4] = {};
    l = 0.0f;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
        const unsigned from = all + w * kStageBytes;
        const float f = fast_exp2(lds_load<float>(from + kMAt + 4 * r32) - ref);
        l += f * lds_load<float>(from + kMAt + 128 + 4 * r32);
#pragma unroll
        for (int k = 0; k < 4; ++k)
            sum[k] += f * lds_load<floatx4>(from + (4 * wave + k) * 1024 + 16 * lane);
    }
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    const int row = t.q0 + r32;
    if (row >= t.rows)
        return;
    E *out = (E *)a.out + ((size_t)(t.q_lo + row) * a.num_heads + h) * kNope + 32 * wave + 4 * hl;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        E4 v;
#pragma unroll
        for (int e = 0; e < 4; ++e)
            v[e] = row < t.n_q ? (E)(sum[k][e] * inv) : (E)0.0f;
        *(E4 *)(out + 8 * k) = v;
    }
}

// Merges the splits of the query tiles that have more than one. A workgroup takes 32
// rows of a head, wave c their columns 32 c .., and a lane the 16 values it would hold in
// attend_kernel. The splits are added in their order.
template <typename E>
__global__ __launch_bounds__(256) void merge_kernel(PrefillArgs a)
{
    using E4 = typename Vec<E>::v4;
    const int lane = threadIdx.x & 63;
    const int c = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int w = blockIdx.x & 3, h = (blockIdx.x >> 2) % a.num_heads, slot = (blockIdx.x >> 2) / a.num_heads;
    const QueryTile t = query_tile<kQueries>(a, slot, lane);
    const int first = t.q0 + 32 * w;
    if (t.n_splits == 1 || t.q0 >= t.n_q || first >= t.rows)
        return;
    const int r32 = lane & 31, hl = lane >> 5;
    const size_t part0 = ((size_t)slot * a.num_heads + h) * a.splits;
    constexpr int kMany = 4;  // splits in flight together
    floatx4 acc[4] = {};
    float m = -INFINITY, l = 0.0f;
    for (int s = 0; first < t.n_q && s < t.n_splits; s += kMany) {
        float ms[kMany], ls[kMany];
        floatx4 po[kMany][4];
#pragma unroll
        for (int k = 0; k < kMany; ++k) {  // past the last split it is read again, and not used
            const size_t part = part0 + min(s + k, t.n_splits - 1);
            ms[k] = a.part_m[part * kQueries + 32 * w + r32];
            ls[k] = a.part_l[part * kQueries + 32 * w + r32];
#pragma unroll
            for (int j = 0; j < 4; ++j)
                po[k][j] = *(const floatx4 *)(a.part_o + (part * 4 + w) * (32 * kNope) + ((c * 4 + j) * 64 + lane) * 4);
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
            if (s + k >= t.n_splits)
                continue;
            const float f = fast_exp2(ms[k] - ref);
            l += f * ls[k];
#pragma unroll
            for (int j = 0; j < 4; ++j)
                acc[j] += f * po[k][j];
        }
        m = next;
    }
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    const int row = first + r32;
    if (row >= t.rows)
        return;
    E *out = (E *)a.out + ((size_t)(t.q_lo + row) * a.num_heads + h) * kNope + 32 * c + 4 * hl;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        E4 v;
#pragma unroll
        for (int e = 0; e < 4; ++e)
            v[e] = row < t.n_q ? (E)(acc[j][e] * inv) : (E)0.0f;
        *(E4 *)(out + 8 * j) = v;
    }
}

// ---- host -------------------------------------------------------------------

size_t align256(size_t n) { return (n + 255) / 256 * 256; }

struct PrefillPlan {
    int padded;
    int q_slots, splits, split_tiles;
    bool narrow;  // narrow_kernel, and its query tiles
    size_t kv_bytes, rope_bytes, flag_bytes, o_bytes, ml_bytes;
    size_t bytes() const { return 2 * kv_bytes + rope_bytes + flag_bytes + o_bytes + 2 * ml_bytes; }
};

// Splits of the keys, where few query tiles see long contexts: those with the least
// modelled time, for requests of mean lengths. A workgroup costs its start and end
// and its tiles, more each where two run on a CU; partials (fp32, written and read) and a
// third launch are the price. A split has a given number of tiles, more where a request is
// longer than the splits then reach. Calls in one split and as planned: 1 query behind
// 8000 tokens at 16 heads 225 us and 76, 500 queries there 274 and 134, 1000 at 32
// heads 336 and 317, 100 behind 2000 at 16 heads 76 and 39.
//
// narrow_kernel competes with them: one workgroup a CU at a time, four tiles in each
// kNarrowTileUs; only the first round is taken to see all the keys. 197 queries at
// 16 heads 10.2 -> 7.0 us, 500 16.9 -> 9.8, 1000 29.4 -> 20.9; 200 at 128 heads 12.6 stay (23.5).
constexpr double kNarrowStartUs = 4.7, kNarrowTileUs = 2.2;
constexpr double kStartUs = 4.8, kTileUs = 1.5, kSharedTileUs = 2.0, kMergeUs = 4.0, kPartialUsPerByte = 0.4e-6;

void plan_attention(PrefillPlan &p, int batch, int num_heads, int queries, int total_tokens, int cu_count)
{
    const int64_t mean_q = ((int64_t)queries + batch - 1) / batch, mean_k = ((int64_t)total_tokens + batch - 1) / batch;
    const int64_t wgs = (mean_q + kQueries - 1) / kQueries * batch * num_heads;
    const int tiles = (int)std::max<int64_t>(1, (mean_k + kTile - 1) / kTile);
    p.splits = 1;
    p.split_tiles = INT32_MAX / 2;
    double best = 0.0;
    for (int n = 1; n <= std::min(tiles, 128); ++n) {
        const int per = (tiles + n - 1) / n;
        if (n > 1 && (tiles + n - 2) / (n - 1) == per)
            continue;  // no shorter than the one before
        const int64_t rounds = std::max<int64_t>(1, (wgs * n + 2 * cu_count - 1) / (2 * cu_count));
        double us = rounds * (kStartUs + per * (wgs * n > cu_count ? kSharedTileUs : kTileUs));
        if (n > 1)
            us += kMergeUs + kPartialUsPerByte * wgs * n * (kQueries * kNope * 4.0);
        if (n == 1 || us < best) {
            best = us;
            p.splits = n;
            p.split_tiles = n == 1 ? INT32_MAX / 2 : per;
        }
    }
    const int64_t small = (mean_q + kNarrow - 1) / kNarrow * batch * num_heads;
    const int64_t rounds = (small + cu_count - 1) / cu_count;
    const int steps = (tiles + 3) / 4, mean_steps = (int)(std::max<int64_t>(0, mean_k - mean_q / 2) / (4 * kTile) + 1);
    p.narrow = rounds * kNarrowStartUs + (steps + (rounds - 1) * std::min(steps, mean_steps)) * kNarrowTileUs < best;
    p.q_slots = queries / (p.narrow ? kNarrow : kQueries) + batch;
    if (p.narrow)
        p.splits = 1;
}

// Sequence b's keys start at tile cu[b] / 64 + b of the workspace.
PrefillPlan prefill_plan(int batch, int num_heads, int queries, int total_tokens)
{
    PrefillPlan p;
    plan_attention(p, batch, num_heads, queries, total_tokens, current_cu_count());
    const size_t parts = p.splits > 1 ? (size_t)p.q_slots * num_heads * p.splits : 0;
    p.o_bytes = align256(parts * kQueries * kNope * sizeof(float));
    p.ml_bytes = align256(parts * kQueries * sizeof(float));
    p.padded = total_tokens / kTile * kTile + kTile * batch;
    p.kv_bytes = align256((size_t)num_heads * p.padded * kNope * 2);
    p.rope_bytes = align256((size_t)p.padded * kRopeDim * 2);
    p.flag_bytes = align256((size_t)num_heads * (p.padded / kTile) * 32);
    return p;
}

// Weight blocks of an expanding workgroup, and its key groups a wave. It costs its key
// loads (about as long as kKeyBlocks blocks, half with one group) and its blocks (kOneGroupBlock
// of the time with one group), and one runs on a CU at a time: of the divisions into a multiple of 8
// groups of blocks (one XCD's workgroups take the same ones) that fill one round, two
// rounds, .., the one with the least time wins.
constexpr double kKeyBlocks = 6.0, kOneGroupBlock = 0.65;

void plan_expansion(PrefillArgs &a, int cu_count)
{
    // key tiles that hold keys, at most (workgroups without any leave at once)
    const int64_t tiles = ((int64_t)a.total_tokens + (int64_t)(kTile - 1) * a.batch) / kTile;
    const int blocks = 2 * kBlocksPerSide * a.num_heads;
    double best = 0.0;
    for (int key_groups = 2; key_groups >= 1; --key_groups) {
        const int64_t quads = std::max<int64_t>(1, (tiles * 2 / key_groups + kExpandWaves - 1) / kExpandWaves);
        const double start = kKeyBlocks / 2 * key_groups, each = key_groups == 2 ? 1.0 : kOneGroupBlock;
        auto consider = [&](int64_t rounds, int per) {
            const double cost = rounds * (per * each + start);
            if (best == 0.0 || cost < best) {
                best = cost;
                a.key_groups = key_groups;
                a.group_blocks = per;
            }
        };
        consider((quads * 8 + cu_count - 1) / cu_count, blocks / 8);
        for (int rounds = 1; rounds <= 16; ++rounds) {
            const int64_t groups = std::min<int64_t>(rounds * (int64_t)cu_count / quads / 8 * 8, blocks);
            if (groups >= 8)
                consider(rounds, (int)((blocks + groups - 1) / groups));
        }
    }
}

bool prefill_sizes_ok(int batch, int num_heads, int queries, int total_tokens)
{
    return batch >= 1 && queries >= 1 && queries <= INT32_MAX - 4096 && num_heads > 0 && num_heads % 16 == 0 && num_heads <= 4096 && total_tokens >= 0 &&
           (int64_t)total_tokens + (int64_t)kTile * batch <= INT32_MAX - 4096;
}

int64_t expand_workgroups(const PrefillArgs &a)
{
    const int64_t quads = ((int64_t)a.padded / kTile * (2 / a.key_groups) + kExpandWaves - 1) / kExpandWaves;
    const int groups = (2 * kBlocksPerSide * a.num_heads + a.group_blocks - 1) / a.group_blocks;
    return quads * ((groups + 7) / 8 * 8);
}

template <typename E>
void launch_prefill(const PrefillArgs &a, hipStream_t s)
{
    if (a.total_tokens > 0) {
        auto k = a.key_groups == 2 ? expand_kernel<E, 2> : expand_kernel<E, 1>;
        hipLaunchKernelGGL(k, dim3((unsigned)expand_workgroups(a)), dim3(256), 0, s, a);
    }
    auto k = a.narrow ? narrow_kernel<E> : attend_kernel<E>;
    hipLaunchKernelGGL(k, dim3((unsigned)a.q_slots * a.num_heads * a.splits), dim3(256), 0, s, a);
    if (a.splits > 1)
        hipLaunchKernelGGL(merge_kernel<E>, dim3((unsigned)a.q_slots * a.num_heads * 4), dim3(256), 0, s, a);
}

int prefill(bool bf16, const void *q_nope, const void *q_rope, const void *w_uk, const void *w_uv, const void *kv_cache,
            const int *block_table, const int *cu_q, const int *cu_seqlens, void *out, void *workspace,
            size_t workspace_bytes, int batch, int num_heads, int queries, int total_tokens, int page_size,
            int num_pages, int block_table_stride, void *stream)
{
    if (!prefill_sizes_ok(batch, num_heads, queries, total_tokens) || !q_nope || !q_rope || !w_uk || !w_uv ||
        (!kv_cache && total_tokens > 0) || !cu_q || !cu_seqlens || !out || !workspace ||
        (block_table && (page_size < 32 || page_size > (1 << 20) || (page_size & (page_size - 1)) != 0 ||
                         num_pages < 1 || block_table_stride < 1)))
        return MLA_STATUS_INVALID_VALUE;
    if (!aligned16(q_nope) || !aligned16(q_rope) || !aligned16(w_uk) || !aligned16(w_uv) || !aligned16(kv_cache) ||
        !aligned16(out) || !aligned16(workspace))
        return MLA_STATUS_MISALIGNED;
    const PrefillPlan p = prefill_plan(batch, num_heads, queries, total_tokens);
    PrefillArgs a;
    a.q_slots = p.q_slots;
    a.narrow = p.narrow;
    a.splits = p.splits;
    a.split_tiles = p.split_tiles;
    if ((int64_t)(p.padded / kTile + 1) * num_heads > INT32_MAX / 256 ||
        (int64_t)a.q_slots * num_heads * (p.splits > 1 ? std::max(4, p.splits) : 1) > INT32_MAX / 256)
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
    a.part_o = reinterpret_cast<float *>(ws + 2 * p.kv_bytes + p.rope_bytes + p.flag_bytes);
    a.part_m = a.part_o + p.o_bytes / sizeof(float);
    a.part_l = a.part_m + p.ml_bytes / sizeof(float);
    a.batch = batch;
    a.num_heads = num_heads;
    a.queries = queries;
    a.total_tokens = total_tokens;
    a.padded = p.padded;
    plan_expansion(a, current_cu_count());
    if (expand_workgroups(a) > INT32_MAX / 256)
        return MLA_STATUS_INVALID_VALUE;
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

size_t mla_prefill_workspace_size(int batch, int num_heads, int queries, int total_tokens)
{
    return mla::prefill_sizes_ok(batch, num_heads, queries, total_tokens)
               ? mla::prefill_plan(batch, num_heads, queries, total_tokens).bytes()
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
