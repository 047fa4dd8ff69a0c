// Pages of the latent cache that several requests share:
//
//   mla_fork_tables      rows of the block table taken over from others: a request's
//                        pages shared with its copies, copied where it goes on writing,
//                        freed where nobody holds them any more;
//   mla_compact_tables   a pool's used pages moved to its lowest ids;
//   mla_copy_pages       the rows of the pages that either asks for, in every layer.
//
// Who holds a page is not counted from call to call: a call finds it out from the table,
// one bit a page in LDS. The tables are bound by their chain of memory round trips, the
// copies by the bytes.
#include <algorithm>
#include <climits>
#include <cstdint>

#include "mla_device.hpp"
#include "mla_internal.hpp"
#include "mla_mi355x.h"

namespace mla {
namespace {

constexpr int kThreads = 1024, kWaves = kThreads / 64;
constexpr int kMostPages = 1 << 18;  // 32 KB of bits
constexpr int kMostRows = 8192;
constexpr int kWords = kMostPages / 32;

// Exclusive sums of v over the workgroup's threads; total: over all of them. s: a word of LDS a wave.
__device__ __forceinline__ int block_before(int v, int *s, int &total)
{
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int sum = v;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
        const int u = __shfl_up(sum, d);
        if (lane >= d)
            sum += u;
    }
    if (lane == 63)
        s[wave] = sum;
    __syncthreads();
    int before = 0;
    total = 0;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
        if (w < wave)
            before += s[w];
        total += s[w];
    }
    __syncthreads();
    return before + sum - v;
}

struct Table {
    const int *ids;  // [rows][stride]
    const int *lens;
    int rows, stride, page_shift;
    __device__ __forceinline__ int tokens(int row) const
    {
        const long long most = (long long)stride << page_shift;
        return (int)min((long long)max(lens[row], 0), most);
    }
    __device__ __forceinline__ int pages(int tokens) const
    {
        return (int)(((unsigned)tokens + (1u << page_shift) - 1) >> page_shift);
    }
};

__device__ __forceinline__ bool has(const unsigned *bits, int page) { return (bits[page >> 5] >> (page & 31)) & 1; }

// One bit a page: held by a row of the table, and (kFull) by one of the first full[row]
// columns of a row. A wave takes 64 rows x 16 columns at once, each lane a column of 16 rows in a row:
// 16 loads in flight, and the page that a row shares with the row above (a prompt's) is marked once.
// held, full: columns of each row, in LDS; most: the largest of held.
template <bool kFull>
__device__ __forceinline__ void mark_pages(const Table &t, const int *held, const int *full, int most, int num_pages,
                                           unsigned *held_bits, unsigned *full_bits)
{
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int chunks = (most + 15) / 16, tasks = (t.rows + 63) / 64 * chunks;
    for (int task = wave; task < tasks; task += kWaves) {
        const int row0 = task / chunks * 64 + (lane >> 4) * 16, col = task % chunks * 16 + (lane & 15);
        int id[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const int row = row0 + i;
            id[i] = row < t.rows && col < held[row] ? t.ids[(size_t)row * t.stride + col] : -1;
        }
        bool above_full = false;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const int row = row0 + i;
            if ((unsigned)id[i] < (unsigned)num_pages) {
                const bool again = i > 0 && id[i] == id[i > 0 ? i - 1 : 0];
                const unsigned bit = 1u << (id[i] & 31);
                if (!again)
                    atomicOr(held_bits + (id[i] >> 5), bit);
                if constexpr (kFull) {
                    const bool whole = col < full[row];
                    if (whole && !(again && above_full))
                        atomicOr(full_bits + (id[i] >> 5), bit);
                    above_full = whole;
                }
            } else {
                above_full = false;
            }
        }
    }
}

// bits <- one bit a page that `pinned` counts as held elsewhere (none if it is null); others <- 0.
__device__ __forceinline__ void clear_bits(const int *pinned, int num_pages, unsigned *bits, unsigned *others)
{
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    for (int base = 256 * wave; base < num_pages; base += 256 * kWaves) {
        int v[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int p = base + 64 * i + lane;
            v[i] = pinned && p < num_pages ? pinned[p] : 0;
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const unsigned long long m = __builtin_amdgcn_ballot_w64(v[i] > 0);
            if (lane < 2) {  // at most 7 words past the last page's; kWords is a multiple of 8
                bits[base / 32 + 2 * i + lane] = (unsigned)(m >> (32 * lane));
                others[base / 32 + 2 * i + lane] = 0;
            }
        }
    }
}

// ---- fork -------------------------------------------------------------------

struct Fork {
    Table old;
    const int *parents, *kept, *pinned, *free_start;
    int *free_pages, *table, *lens, *copies, *free_next, *first;
    int batch, num_pages, num_free;
};

struct NewRow {
    int parent, tokens, full, rest;  // rest: tokens in the last page, which it does not fill
    int last;                        // that page's id
};

__device__ __forceinline__ NewRow new_row(const Fork &f, int b)
{
    NewRow r;
    r.parent = f.parents[b];
    const int kept = f.kept ? max(f.kept[b], 0) : INT_MAX;
    const bool real = (unsigned)r.parent < (unsigned)f.old.rows;
    r.tokens = real ? min(kept, f.old.tokens(r.parent)) : 0;
    r.full = r.tokens >> f.old.page_shift;
    r.rest = r.tokens & ((1 << f.old.page_shift) - 1);
    r.last = r.rest ? f.old.ids[(size_t)r.parent * f.old.stride + r.full] : -1;
    return r;
}

// Row b of the new table holds the first tokens of row parents[b] of the old one, on the same pages. Of the rows that end
// inside a page, the lowest may go on writing it if no other row holds it whole and it is not pinned; each
// other one gets a page of its own from the free list, and its rows to be copied. Pages of the old table that the new
// one does not hold, and that are not pinned, are pushed to the free list, lowest id first, before those
// pages are taken from it: at most as many as were taken, below free_start.
//
// Workgroup 0 does what needs an order (who holds what, the ranks in the free list), with a bit a page in LDS;
// the others write the whole columns of the new rows meanwhile, which need none. One launch: its
// chain of round trips (parents, lengths, ids, marks, first row of each last page, ranks, ids taken) is
// what a call costs.
__global__ __launch_bounds__(kThreads) void fork_kernel(Fork f)
{
    __shared__ unsigned s_held[kWords], s_kept[kWords];
    __shared__ int s_pages[kMostRows], s_full[kMostRows];
    __shared__ int s_scan[kWaves], s_most;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const Table &t = f.old;
    if (blockIdx.x > 0) {
        // whole columns, and -1 behind the row's last page; a row's 256 columns at once a wave
        const int chunks = (t.stride + 255) / 256;
        const long long items = (long long)f.batch * chunks;
        for (long long i = (long long)(blockIdx.x - 1) * kWaves + wave; i < items; i += (long long)(gridDim.x - 1) * kWaves) {
            const int b = (int)(i / chunks), col0 = (int)(i % chunks) * 256;
            const NewRow r = new_row(f, b);
            const int *src = t.ids + (size_t)max(r.parent, 0) * t.stride;
            int *dst = f.table + (size_t)b * t.stride;
            int id[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const int col = col0 + 64 * k + lane;
                id[k] = col < r.full ? src[col] : -1;
            }
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const int col = col0 + 64 * k + lane;
                if (col < t.stride && !(col == r.full && r.rest))
                    dst[col] = id[k];
            }
        }
        return;
    }
    clear_bits(f.pinned, f.num_pages, s_kept, s_held);
    if (tid == 0)
        s_most = 0;
    __syncthreads();
    int most = 0;
    for (int row = tid; row < t.rows; row += kThreads) {
        const int pages = t.pages(t.tokens(row));
        s_pages[row] = pages;
        s_full[row] = 0;
        most = max(most, pages);
    }
    atomicMax(&s_most, most);
    __syncthreads();
    NewRow mine = {};  // the thread's first row; the others are read again
    for (int b = tid; b < f.batch; b += kThreads) {
        const NewRow r = new_row(f, b);
        if (b == tid)
            mine = r;
        f.lens[b] = r.tokens;
        if (r.full)
            atomicMax(&s_full[r.parent], r.full);
        if (r.rest && (unsigned)r.last < (unsigned)f.num_pages)
            __hip_atomic_store(f.first + r.last, INT_MAX, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    __syncthreads();
    mark_pages<true>(t, s_pages, s_full, s_most, f.num_pages, s_held, s_kept);
    __syncthreads();
    // s_kept: pinned, or held whole by a new row
    auto open = [&](const NewRow &r) { return r.rest && (unsigned)r.last < (unsigned)f.num_pages && !has(s_kept, r.last); };
    for (int b = tid; b < f.batch; b += kThreads) {
        const NewRow r = b == tid ? mine : new_row(f, b);
        if (open(r))
            __hip_atomic_fetch_min(f.first + r.last, b, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    __syncthreads();
    auto goes_on = [&](const NewRow &r, int b) {
        return open(r) && __hip_atomic_load(f.first + r.last, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == b;
    };
    bool mine_goes_on = false;
    for (int b = tid; b < f.batch; b += kThreads) {
        const NewRow r = b == tid ? mine : new_row(f, b);
        const bool on = goes_on(r, b);
        if (b == tid)
            mine_goes_on = on;
        if (on)
            atomicAnd(s_held + (r.last >> 5), ~(1u << (r.last & 31)));  // not to be freed
    }
    __syncthreads();
    // pages to free: each thread a run of words, lowest ids first
    const int words = (f.num_pages + 31) / 32, per = (words + kThreads - 1) / kThreads;
    const int w0 = min(tid * per, words), w1 = min(w0 + per, words);
    int count = 0;
    for (int w = w0; w < w1; ++w)
        count += __builtin_popcount(s_held[w] & ~s_kept[w]);
    int freed;
    const int rank = block_before(count, s_scan, freed);
    const long long start = (long long)*f.free_start - freed;
    long long at = start + rank;
    for (int w = w0; w < w1; ++w)
        for (unsigned m = s_held[w] & ~s_kept[w]; m; m &= m - 1, ++at)
            if (at >= 0 && at < f.num_free)
                f.free_pages[at] = 32 * w + __builtin_ctz(m);
    __syncthreads();
    int taken = 0;
    for (int b0 = 0; b0 < f.batch; b0 += kThreads) {
        const int b = b0 + tid;
        NewRow r = mine;
        bool on = mine_goes_on;
        if (b0 > 0) {
            r = b < f.batch ? new_row(f, b) : NewRow{};
            on = goes_on(r, b);
        }
        const bool takes = b < f.batch && r.rest && (unsigned)r.last < (unsigned)f.num_pages && !on;
        int all;
        const long long i = start + taken + block_before(takes ? 1 : 0, s_scan, all);
        taken += all;
        if (b >= f.batch)
            continue;
        const int page = takes ? (i >= 0 && i < f.num_free ? f.free_pages[i] : -1) : r.last;
        if (r.rest)
            f.table[(size_t)b * t.stride + r.full] = page;
        int *copy = f.copies + 3 * (size_t)b;
        copy[0] = takes ? r.last : -1;
        copy[1] = takes ? page : -1;
        copy[2] = takes ? r.rest : 0;
    }
    if (tid == 0)
        *f.free_next = (int)min(max(start + taken, (long long)INT_MIN), (long long)INT_MAX);
}

// ---- compaction -------------------------------------------------------------

struct Compact {
    Table old;
    const int *pinned, *free_pages, *free_start;
    int *table, *copies, *free_out;
    int *to;  // [num_pages + 2]: where each page goes; then the moves, and the ids in the list
    int num_pages, num_free, most_moves;
};

// Of the movable pages t (held by a row, not pinned) and the free ones f (listed, neither held nor pinned), the k-th
// highest t moves to the k-th lowest f as long as that is lower. So f is moved to where more t stand above
// it than f below it, and t moves where more f stand below it than t above it: each page finds its own
// move from two sums over the bits, and k is the number of t above it (of f below it).
// One workgroup, as in fork_kernel; remap_kernel then writes what needs no order.
__global__ __launch_bounds__(kThreads) void compact_kernel(Compact c)
{
    __shared__ unsigned s_held[kWords], s_pinned[kWords], s_free[kWords];
    __shared__ int s_pages[kMostRows];
    __shared__ int s_scan[kWaves], s_most;
    const int tid = threadIdx.x;
    const Table &t = c.old;
    clear_bits(c.pinned, c.num_pages, s_pinned, s_held);
    const int words = (c.num_pages + 31) / 32;
    for (int w = tid; w < words; w += kThreads)
        s_free[w] = 0;
    for (int p = tid; p < c.num_pages; p += kThreads)
        c.to[p] = p;
    if (tid == 0)
        s_most = 0;
    __syncthreads();
    int most = 0;
    for (int row = tid; row < t.rows; row += kThreads) {
        const int pages = t.pages(t.tokens(row));
        s_pages[row] = pages;
        most = max(most, pages);
    }
    atomicMax(&s_most, most);
    const int start = min(max(*c.free_start, 0), c.num_free);
    for (int i0 = start; i0 < c.num_free; i0 += 8 * kThreads) {
        int id[8];
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            const long long i = (long long)i0 + k * kThreads + tid;
            id[k] = i < c.num_free ? c.free_pages[i] : -1;
        }
#pragma unroll
        for (int k = 0; k < 8; ++k)
            if ((unsigned)id[k] < (unsigned)c.num_pages)
                atomicOr(s_free + (id[k] >> 5), 1u << (id[k] & 31));
        if (i0 > c.num_free - 8 * kThreads)
            break;  // (i0 would pass 2^31)
    }
    __syncthreads();
    mark_pages<false>(t, s_pages, nullptr, s_most, c.num_pages, s_held, nullptr);
    __syncthreads();
    const int per = (words + kThreads - 1) / kThreads;
    const int w0 = min(tid * per, words), w1 = min(w0 + per, words);
    int movable = 0, listed = 0;
    for (int w = w0; w < w1; ++w) {
        const unsigned p = s_pinned[w], h = s_held[w], m = h & ~p, l = s_free[w] & ~h & ~p;
        s_held[w] = m;
        s_free[w] = l;
        movable += __builtin_popcount(m);
        listed += __builtin_popcount(l);
    }
    int all_movable, all_free;
    const int t_first = block_before(movable, s_scan, all_movable), f_first = block_before(listed, s_scan, all_free);
    // visit(page, is t, moves, k) for the thread's pages, lowest first
    auto each = [&](auto &&visit) {
        int t_below = t_first, f_below = f_first;
        for (int w = w0; w < w1; ++w) {
            const unsigned held = s_held[w];
            for (unsigned m = held | s_free[w]; m; m &= m - 1) {
                const int bit = __builtin_ctz(m);
                if ((held >> bit) & 1) {
                    const int above = all_movable - 1 - t_below++;
                    visit(32 * w + bit, true, f_below > above, above);
                } else {
                    visit(32 * w + bit, false, all_movable - t_below > f_below, f_below);
                    ++f_below;
                }
            }
        }
    };
    int moves = 0, left = 0;
    each([&](int page, bool is_t, bool moves_it, int k) {
        if (moves_it) {
            int *copy = c.copies + 3 * (size_t)k;
            copy[is_t ? 0 : 1] = page;
            if (is_t)
                copy[2] = 1 << t.page_shift;
        }
        moves += is_t && moves_it;
        left += is_t == moves_it;
    });
    int all_moves, all_left;
    block_before(moves, s_scan, all_moves);
    long long at = start + block_before(left, s_scan, all_left);
    each([&](int page, bool is_t, bool moves_it, int k) {
        if (is_t && moves_it)
            c.to[page] = c.copies[3 * (size_t)k + 1];
        if (is_t == moves_it)
            c.free_out[at++] = page;
    });
    if (tid == 0) {
        c.to[c.num_pages] = all_moves;
        c.to[c.num_pages + 1] = all_left;
    }
}

// The table with every page where it went, -1 behind a row's last page; the moves that are none; the list's other entries.
__global__ __launch_bounds__(256) void remap_kernel(Compact c)
{
    const Table &t = c.old;
    const int lane = threadIdx.x & 63;
    const long long wave = blockIdx.x * 4ll + (threadIdx.x >> 6), waves = gridDim.x * 4ll;
    const int chunks = (t.stride + 255) / 256;
    const long long items = (long long)t.rows * chunks;
    for (long long i = wave; i < items; i += waves) {
        const int row = (int)(i / chunks), col0 = (int)(i % chunks) * 256;
        const int pages = t.pages(t.tokens(row));
        const size_t base = (size_t)row * t.stride;
        int id[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const int col = col0 + 64 * k + lane;
            id[k] = col < pages ? t.ids[base + col] : -1;
        }
#pragma unroll
        for (int k = 0; k < 4; ++k)
            if ((unsigned)id[k] < (unsigned)c.num_pages)
                id[k] = c.to[id[k]];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const int col = col0 + 64 * k + lane;
            if (col < t.stride)
                c.table[base + col] = id[k];
        }
    }
    const int start = min(max(*c.free_start, 0), c.num_free);
    const int moves = c.to[c.num_pages], end = start + c.to[c.num_pages + 1];
    const long long thread = blockIdx.x * 256ll + threadIdx.x, threads = gridDim.x * 256ll;
    for (long long i = 3ll * moves + thread; i < 3ll * c.most_moves; i += threads)
        c.copies[i] = i % 3 == 2 ? 0 : -1;
    for (long long i = thread; i < c.num_free; i += threads)
        if (i < start || i >= end)
            c.free_out[i] = -1;
}

// ---- copies -----------------------------------------------------------------

// A workgroup takes one page's next chunk of bytes at a time, four 16-byte loads a thread in
// flight before their stores.
__global__ __launch_bounds__(256) void copy_pages_kernel(unsigned char *__restrict__ cache, const int *__restrict__ copies,
                                                         int count, int layers, int num_pages, int page_size, int row_bytes,
                                                         int chunk, int chunks)
{
    const long long page_bytes = (long long)page_size * row_bytes, items = (long long)count * chunks * layers;
    for (long long i = blockIdx.x; i < items; i += gridDim.x) {
        const long long e = i / chunks;
        const int layer = (int)(e / count), entry = (int)(e % count);
        const int src = copies[3 * (size_t)entry], dst = copies[3 * (size_t)entry + 1];
        const int rows = min(copies[3 * (size_t)entry + 2], page_size);
        if ((unsigned)src >= (unsigned)num_pages || (unsigned)dst >= (unsigned)num_pages || src == dst || rows <= 0)
            continue;
        const long long first = (i % chunks) * chunk, end = min(first + chunk, (long long)rows * row_bytes);
        unsigned char *layer_base = cache + (size_t)layer * num_pages * page_bytes;
        const unsigned char *from = layer_base + (size_t)src * page_bytes;
        unsigned char *to = layer_base + (size_t)dst * page_bytes;
        for (long long o = first + threadIdx.x * 16; o < end; o += 4 * 4096) {
            uint4 v[4];
#pragma unroll
            for (int k = 0; k < 4; ++k)
                v[k] = *(const uint4 *)(from + min(o + 4096 * k, end - 16));
#pragma unroll
            for (int k = 0; k < 4; ++k)
                if (o + 4096 * k < end)
                    *(uint4 *)(to + o + 4096 * k) = v[k];
        }
    }
}

bool page_ok(int page_size) { return page_size >= 32 && page_size <= (1 << 20) && (page_size & (page_size - 1)) == 0; }

bool table_ok(const int *block_table, const int *lens, int rows, int num_pages, int page_size, int stride)
{
    return block_table && lens && rows >= 1 && rows <= kMostRows && num_pages >= 1 && num_pages <= kMostPages &&
           page_ok(page_size) && stride >= 1;
}

int launched()
{
    const hipError_t e = hipPeekAtLastError();
    return e == hipSuccess ? MLA_STATUS_SUCCESS : record_hip_error(e);
}

}  // namespace
}  // namespace mla

extern "C" {

size_t mla_page_tables_workspace_size(int num_pages)
{
    return num_pages < 1 || num_pages > mla::kMostPages ? 0 : (4 * ((size_t)num_pages + 2) + 255) / 256 * 256;
}

int mla_fork_tables(const int *block_table, const int *lens, const int *parents, const int *kept_lens, const int *pinned,
                    int *free_pages, const int *free_start, int *new_table, int *new_lens, int *copies, int *free_next,
                    void *workspace, size_t workspace_bytes, int rows, int batch, int num_pages, int num_free,
                    int page_size, int block_table_stride, void *stream)
{
    if (!mla::table_ok(block_table, lens, rows, num_pages, page_size, block_table_stride) || !parents || !free_start ||
        (!free_pages && num_free > 0) || !new_table || !new_lens || !copies || !free_next || !workspace ||
        new_table == block_table || new_lens == lens || free_next == free_start || batch < 1 || batch > (1 << 30) ||
        num_free < 0)
        return MLA_STATUS_INVALID_VALUE;
    if ((reinterpret_cast<uintptr_t>(workspace) & 15u) != 0)
        return MLA_STATUS_MISALIGNED;
    if (workspace_bytes < mla_page_tables_workspace_size(num_pages))
        return MLA_STATUS_WORKSPACE_TOO_SMALL;
    const mla::Fork f{{block_table, lens, rows, block_table_stride, __builtin_ctz((unsigned)page_size)},
                      parents, kept_lens, pinned, free_start, free_pages, new_table, new_lens, copies, free_next,
                      static_cast<int *>(workspace), batch, num_pages, num_free};
    const int64_t items = (int64_t)batch * ((block_table_stride + 255) / 256);
    const int writers = (int)std::min<int64_t>((items + mla::kWaves - 1) / mla::kWaves, mla::current_cu_count() - 1);
    hipLaunchKernelGGL(mla::fork_kernel, dim3(1 + writers), dim3(mla::kThreads), 0, static_cast<hipStream_t>(stream), f);
    return mla::launched();
}

int mla_compact_tables(const int *block_table, const int *lens, const int *pinned, const int *free_pages,
                       const int *free_start, int *new_table, int *copies, int *new_free_pages, void *workspace,
                       size_t workspace_bytes, int rows, int num_pages, int num_free, int page_size,
                       int block_table_stride, void *stream)
{
    const int moves = std::min(num_free, num_pages / 2);
    if (!mla::table_ok(block_table, lens, rows, num_pages, page_size, block_table_stride) || !free_start || !new_table ||
        !workspace || new_table == block_table || num_free < 0 ||
        (num_free > 0 && (!free_pages || !new_free_pages || new_free_pages == free_pages)) || (moves > 0 && !copies))
        return MLA_STATUS_INVALID_VALUE;
    if ((reinterpret_cast<uintptr_t>(workspace) & 15u) != 0)
        return MLA_STATUS_MISALIGNED;
    if (workspace_bytes < mla_page_tables_workspace_size(num_pages))
        return MLA_STATUS_WORKSPACE_TOO_SMALL;
    const mla::Compact c{{block_table, lens, rows, block_table_stride, __builtin_ctz((unsigned)page_size)},
                         pinned, free_pages, free_start, new_table, copies, new_free_pages,
                         static_cast<int *>(workspace), num_pages, num_free, moves};
    hipStream_t s = static_cast<hipStream_t>(stream);
    hipLaunchKernelGGL(mla::compact_kernel, dim3(1), dim3(mla::kThreads), 0, s, c);
    if (const int st = mla::launched())
        return st;
    const int64_t waves = std::max((int64_t)rows * ((block_table_stride + 255) / 256), ((int64_t)3 * moves + num_free) / 256);
    const int wgs = (int)std::min<int64_t>((waves + 3) / 4 + 1, 4 * mla::current_cu_count());
    hipLaunchKernelGGL(mla::remap_kernel, dim3(wgs), dim3(256), 0, s, c);
    return mla::launched();
}

int mla_copy_pages(void *kv_cache, const int *copies, int count, int layers, int num_pages, int page_size,
                   int element_size, void *stream)
{
    if (!kv_cache || (count > 0 && !copies) || count < 0 || layers < 1 || num_pages < 1 || !mla::page_ok(page_size) ||
        (element_size != 1 && element_size != 2 && element_size != 4))
        return MLA_STATUS_INVALID_VALUE;
    if ((reinterpret_cast<uintptr_t>(kv_cache) & 15u) != 0)
        return MLA_STATUS_MISALIGNED;
    if (count == 0)
        return MLA_STATUS_SUCCESS;
    // chunks of a page's bytes: about 16 KB, whole rounds of a workgroup's 4 KB
    const int row_bytes = mla::kDK * element_size;
    const int64_t page_bytes = (int64_t)page_size * row_bytes;
    const int chunks = (int)((page_bytes + 16383) / 16384);
    const int chunk = (int)(((page_bytes + chunks - 1) / chunks + 4095) / 4096 * 4096);
    const int64_t items = (int64_t)count * layers * chunks;
    const int wgs = (int)std::min<int64_t>(items, 16 * (int64_t)mla::current_cu_count());
    hipLaunchKernelGGL(mla::copy_pages_kernel, dim3(wgs), dim3(256), 0, static_cast<hipStream_t>(stream),
                       static_cast<unsigned char *>(kv_cache), copies, count, layers, num_pages, page_size, row_bytes, chunk,
                       chunks);
    return mla::launched();
}

}  // extern "C"
