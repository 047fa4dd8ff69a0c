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
constexpr int kMostColumns = 1 << 20;  // 64 rows' offsets stay within 32 bits
constexpr int kWords = kMostPages / 32;
constexpr int kRemapHere = 12288;

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

// The largest v of the workgroup's threads, added to *s by each wave.
__device__ __forceinline__ void block_most(int v, int *s)
{
#pragma unroll
    for (int d = 32; d > 0; d /= 2)
        v = max(v, __shfl_xor(v, d));
    if ((threadIdx.x & 63) == 0)
        atomicMax(s, v);
}

struct Table {
    const int *ids;  // [rows][stride]
    const int *lens;
    int rows, stride, page_shift;
    __device__ __forceinline__ int within(int length) const
    {
        const long long most = (long long)stride << page_shift;
        return (int)min((long long)max(length, 0), most);
    }
    __device__ __forceinline__ int tokens(int row) const { return within(lens[row]); }
    __device__ __forceinline__ int pages(int tokens) const
    {
        return (int)(((unsigned)tokens + (1u << page_shift) - 1) >> page_shift);
    }
};

// One bit a page that a row of the table holds: in bits[w], or (kFull) in bits[2 w], with one in bits[2 w + 1] for a page
// in the first full columns of a row. A wave takes pieces of 32 rows x 32 columns, each lane four columns (one load) of 4
// rows in a row, kPieces of them at once; a page that the four rows share (a prompt's) is marked once. No load
// stands under a condition: the last pieces' rows and columns overlap the others' (a mark may be made twice). The
// first pieces' loads (fetch) need no length, so that a caller has them on their way before it knows any.
// One CU does all of it, in the end at the rate it reads new lines: 1024 rows of 75 columns, of which four share 62 pages,
// 300 KB in 8 us (10 with each entry compared to the one above it, 14 with one column a load, 20 with a condition around
// each load).
// held: of each row its pages, or (kFull) its pages and its full columns; in LDS, zeros from t.rows to the next
// multiple of 64. most: the largest row's pages. kNarrow: fewer than four columns, loaded one by one.
template <bool kFull, bool kNarrow>
struct Marks {
    typedef int Ids __attribute__((ext_vector_type(4), aligned(4)));
    static constexpr int kPieces = 4, kStep = kFull ? 2 : 1;
    const Table &t;
    const int lane, wave, row_pieces, above;  // above: the lane's first row in a piece
    Ids id[kPieces][4];

    __device__ __forceinline__ explicit Marks(const Table &table)
        : t(table), lane(threadIdx.x & 63), wave(__builtin_amdgcn_readfirstlane(threadIdx.x >> 6)),
          row_pieces((t.rows + 31) / 32), above(min(lane >> 3 << 2, max(t.rows - 4, 0)))
    {
    }
    // a piece's first row and the lane's first column
    __device__ __forceinline__ int row_of(int piece) const { return min(piece % row_pieces * 32, max(t.rows - 32, 0)); }
    __device__ __forceinline__ int col_of(int piece) const
    {
        return min((piece / row_pieces * 8 + (lane & 7)) * 4, max(t.stride - 4, 0));
    }
    // pieces first, first + kWaves, ..
    __device__ __forceinline__ void fetch(int first)
    {
        const int last = row_pieces * ((t.stride + 31) / 32) - 1;
#pragma unroll
        for (int k = 0; k < kPieces; ++k) {
            const int piece = min(first + k * kWaves, last);
            const int *base = t.ids + (size_t)row_of(piece) * t.stride;
            const int offset = above * t.stride + col_of(piece);
            if constexpr (!kNarrow) {
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    id[k][i] = *(const Ids *)(base + (size_t)min(i, t.rows - 1) * t.stride + offset);
            } else {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int *row = base + (size_t)min(i, t.rows - 1) * t.stride + offset;
                    id[k][i] = Ids{row[0], row[min(1, t.stride - 1)], row[min(2, t.stride - 1)], -1};
                }
            }
        }
    }
    // all pieces, the first kPieces of the wave fetched already
    __device__ __forceinline__ void mark(const int *held, int most, int num_pages, unsigned *bits)
    {
        const int pieces = row_pieces * ((most + 31) / 32);
        for (int first = wave; first < pieces; first += kPieces * kWaves) {
            if (first != wave)
                fetch(first);
#pragma unroll
            for (int k = 0; k < kPieces; ++k) {
                const int piece = first + k * kWaves;
                if (piece >= pieces)
                    break;
                const int first_col = col_of(piece);
                const int *rows = held + kStep * (row_of(piece) + above);
                int reached[4], whole[4], reached_most = 0, whole_most = 0;  // columns of the lane's rows
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    reached[i] = rows[kStep * i];
                    whole[i] = kFull ? rows[kStep * i + kStep - 1] : 0;
                    reached_most = max(reached_most, reached[i]);
                    whole_most = max(whole_most, whole[i]);
                }
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    const int col = first_col + c;
                    auto bit = [&](int page, int reach, int full) {
                        if (col < reach && (unsigned)page < (unsigned)num_pages) {
                            const unsigned one = 1u << (page & 31);
                            if constexpr (kFull)
                                atomicOr(reinterpret_cast<unsigned long long *>(bits) + (page >> 5),
                                         one | (unsigned long long)(col < full ? one : 0u) << 32);
                            else
                                atomicOr(bits + (page >> 5), one);
                        }
                    };
                    const bool same = id[k][0][c] == id[k][1][c] && id[k][1][c] == id[k][2][c] && id[k][2][c] == id[k][3][c];
                    bit(id[k][0][c], same ? reached_most : reached[0], same ? whole_most : whole[0]);
                    if (!same) {
#pragma unroll
                        for (int i = 1; i < 4; ++i)
                            bit(id[k][i][c], reached[i], whole[i]);
                    }
                }
            }
        }
    }
};

// One bit a page that `pinned` counts as held elsewhere (none if it is null), in bits[step w]; others[step w] <- 0.
// (Without pins the loads read `any` instead: under a condition each would be waited for by itself, which made 17 us
// of 21 700 pages, now 7 with the list and the first ids.)
template <int step>
__device__ __forceinline__ void clear_bits(const int *pinned, const int *any, int num_pages, unsigned *bits, unsigned *others)
{
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int last = num_pages - 1, last_read = pinned ? last : 0;
    const int *from = pinned ? pinned : any;
    const int least = pinned ? 0 : INT_MAX;
    for (int base = 1024 * wave; base < num_pages; base += 1024 * kWaves) {
        int v[16];
#pragma unroll
        for (int i = 0; i < 16; ++i)
            v[i] = from[min(base + 64 * i + lane, last_read)];
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const unsigned long long m = __builtin_amdgcn_ballot_w64(v[i] > least && base + 64 * i + lane <= last);
            if (lane < 2) {  // up to 31 words past the last page's: kWords is a multiple of 32
                bits[step * (base / 32 + 2 * i + lane)] = (unsigned)(m >> (32 * lane));
                others[step * (base / 32 + 2 * i + lane)] = 0;
            }
        }
    }
}

// held[step row] <- the row's pages, in LDS, the step's others 0; zeros up to the next multiple of 64 rows; the most of
// a row into *most. length: lens[row] of the thread's first row, or of any if it has none.
template <int step>
__device__ __forceinline__ void row_pages(const Table &t, int length, int *held, int *most)
{
    int largest = 0;
    for (int row = threadIdx.x; row < (t.rows + 63) / 64 * 64; row += kThreads) {
        if (row >= kThreads)
            length = t.lens[min(row, t.rows - 1)];
        const int pages = row < t.rows ? t.pages(t.within(length)) : 0;
        held[step * row] = pages;
        if constexpr (step == 2)
            held[step * row + 1] = 0;
        largest = max(largest, pages);
    }
    block_most(largest, most);
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
// chain of round trips (lengths, ids and pins; parents; marks; first row of each last page; ranks; ids taken) is
// what a call costs: 8.5 us of 64 rows of 11 pages, 20.2 of 1024 of 75, whose marks are 8.
template <bool kNarrow>
__global__ __launch_bounds__(kThreads) void fork_kernel(Fork f)
{
    __shared__ __attribute__((aligned(16))) unsigned s_bits[2 * kWords];  // of 32 pages: held before; pinned, or held whole by a new row
    __shared__ __attribute__((aligned(16))) int s_rows[2 * kMostRows];  // of a row: its pages, the most of them that a new row holds whole
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
    const int free_start = *f.free_start;
    auto held = [&](int w) -> unsigned & { return s_bits[2 * w]; };
    auto kept = [&](int w) -> unsigned & { return s_bits[2 * w + 1]; };
    Marks<true, kNarrow> marks(t);
    // what needs nothing read before it is on its way at once: lengths, ids, pins
    const int length = t.lens[min(tid, t.rows - 1)];
    marks.fetch(marks.wave);
    if (tid == 0)
        s_most = 0;
    clear_bits<2>(f.pinned, t.lens, f.num_pages, s_bits + 1, s_bits);
    const long long ahead = (long long)free_start + tid;
    const int near = f.num_free > 0 ? f.free_pages[min(max(ahead, 0ll), (long long)f.num_free - 1)] : 0;
    __syncthreads();
    row_pages<2>(t, length, s_rows, &s_most);
    NewRow mine = {};  // the thread's first row; the others are read again
    if (tid < f.batch)
        mine = new_row(f, tid);
    __syncthreads();
    for (int b = tid; b < f.batch; b += kThreads) {
        const NewRow r = b == tid ? mine : new_row(f, b);
        f.lens[b] = r.tokens;
        if (r.full)
            atomicMax(&s_rows[2 * r.parent + 1], r.full);
        if (r.rest && (unsigned)r.last < (unsigned)f.num_pages)
            __hip_atomic_store(f.first + r.last, INT_MAX, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    __syncthreads();
    asm volatile("" : : "v"(near));  // the free list where it will be read, brought to the cache
    marks.mark(s_rows, s_most, f.num_pages, s_bits);
    __syncthreads();
    auto open = [&](const NewRow &r) {
        return r.rest && (unsigned)r.last < (unsigned)f.num_pages && !((kept(r.last >> 5) >> (r.last & 31)) & 1);
    };
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
            atomicAnd(&held(r.last >> 5), ~(1u << (r.last & 31)));  // not to be freed
    }
    __syncthreads();
    // pages to free: each thread a run of words, lowest ids first
    const int words = (f.num_pages + 31) / 32, per = (words + kThreads - 1) / kThreads;
    const int w0 = min(tid * per, words), w1 = min(w0 + per, words);
    int count = 0;
    for (int w = w0; w < w1; ++w)
        count += __builtin_popcount(held(w) & ~kept(w));
    int freed;
    const int rank = block_before(count, s_scan, freed);
    const long long start = (long long)free_start - freed;
    long long at = start + rank;
    for (int w = w0; w < w1; ++w)
        for (unsigned m = held(w) & ~kept(w); m; m &= m - 1, ++at)
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
    int *move;  // [num_pages + 3]: of a page that moves, which move; then the moves, the ids in the list, the lowest page that moves
    int num_pages, num_free, most_moves;
    int remaps;  // the one workgroup that finds the moves writes the table too
};

// The table with every page where it went, -1 behind a row's last page; the moves that are none; the list's other entries.
// By `waves` waves, of which this is number `wave`, with so many threads.
__device__ __forceinline__ void remap(const Compact &c, int moves, int all_free, int lowest, long long wave, long long waves,
                                      long long thread, long long threads)
{
    const Table &t = c.old;
    const int lane = threadIdx.x & 63;
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
        for (int k = 0; k < 4; ++k)  // every held page from the lowest that moves on does, unless it is pinned
            if (id[k] >= lowest && id[k] < c.num_pages && !(c.pinned && c.pinned[id[k]] > 0))
                id[k] = c.copies[3 * (size_t)c.move[id[k]] + 1];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const int col = col0 + 64 * k + lane;
            if (col < t.stride)
                c.table[base + col] = id[k];
        }
    }
    const int start = min(max(*c.free_start, 0), c.num_free), end = start + all_free;
    for (long long i = 3ll * moves + thread; i < 3ll * c.most_moves; i += threads)
        c.copies[i] = i % 3 == 2 ? 0 : -1;
    for (long long i = thread; i < c.num_free; i += threads)
        if (i < start || i >= end)
            c.free_out[i] = -1;
}

// Of the movable pages t (held by a row, not pinned) and the free ones f (listed, neither held nor pinned), the k-th
// highest t moves to the k-th lowest f as long as that is lower. So f is moved to where more t stand above
// it than f below it, and t moves where more f stand below it than t above it: each page finds its own
// move from two sums over the bits, and k is the number of t above it (of f below it). With m moves, the list
// afterwards is the free pages but the m lowest, and the m highest movable ones, each page's place again a sum.
// One workgroup, as in fork_kernel, a lane a page; remap_kernel then writes what needs no order, where that is enough
// for a launch. 21 700 pages
// take 23 us, 9 of them for the two passes over the pages, whose scattered stores one CU makes; 700 pages and their table 11.
template <bool kNarrow>
__global__ __launch_bounds__(kThreads) void compact_kernel(Compact c)
{
    __shared__ __attribute__((aligned(8))) unsigned s_held[kWords], s_pinned[kWords], s_free[kWords];
    __shared__ __attribute__((aligned(16))) int s_rows[kMostRows];  // pages of each row, then the pages below each 64: movable, free
    __shared__ int s_scan[kWaves], s_most, s_moves, s_lowest;
    static_assert(kMostRows >= 2 * (kMostPages / 64), "the sums take the rows' place");
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const Table &t = c.old;
    const int start = min(max(*c.free_start, 0), c.num_free);
    if (tid == 0) {
        s_most = s_moves = 0;
        s_lowest = INT_MAX;
    }
    // the list's first ids are on their way with the rows' lengths and the pins
    constexpr int kIds = 16;
    const int *list = c.num_free > 0 ? c.free_pages : t.lens;  // (one entry is read of an empty list too)
    int id[kIds];
    auto fetch = [&](int i0) {
#pragma unroll
        for (int k = 0; k < kIds; ++k) {
            const long long i = min((long long)i0 + k * kThreads + tid, (long long)c.num_free - 1);
            id[k] = list[max(i, 0ll)];
        }
    };
    fetch(start);
    const int length = t.lens[min(tid, t.rows - 1)];
    Marks<false, kNarrow> marks(t);
    marks.fetch(marks.wave);
    const int groups = (c.num_pages + 63) / 64;
    for (int w = tid; w < 2 * groups; w += kThreads)
        s_free[w] = 0;
    clear_bits<1>(c.pinned, t.lens, c.num_pages, s_pinned, s_held);
    __syncthreads();
    row_pages<1>(t, length, s_rows, &s_most);
    for (int i0 = start;;) {
#pragma unroll
        for (int k = 0; k < kIds; ++k)
            if ((long long)i0 + k * kThreads + tid < c.num_free && (unsigned)id[k] < (unsigned)c.num_pages)
                atomicOr(s_free + (id[k] >> 5), 1u << (id[k] & 31));
        if (i0 >= c.num_free - kIds * kThreads)
            break;
        fetch(i0 += kIds * kThreads);
    }
    __syncthreads();
    marks.mark(s_rows, s_most, c.num_pages, s_held);
    __syncthreads();
    const int per = (groups + kThreads - 1) / kThreads, g0 = min(tid * per, groups), g1 = min(g0 + per, groups);
    int movable = 0, listed = 0;
    for (int w = 2 * g0; w < 2 * g1; ++w) {
        const unsigned p = s_pinned[w], h = s_held[w], m = h & ~p, l = s_free[w] & ~h & ~p;
        s_held[w] = m;
        s_free[w] = l;
        movable += __builtin_popcount(m);
        listed += __builtin_popcount(l);
    }
    int all_movable, all_free;
    int t_below = block_before(movable, s_scan, all_movable), f_below = block_before(listed, s_scan, all_free);
    for (int g = g0; g < g1; ++g) {
        s_rows[2 * g] = t_below;
        s_rows[2 * g + 1] = f_below;
        t_below += __builtin_popcount(s_held[2 * g]) + __builtin_popcount(s_held[2 * g + 1]);
        f_below += __builtin_popcount(s_free[2 * g]) + __builtin_popcount(s_free[2 * g + 1]);
    }
    __syncthreads();
    // visit(page, is movable, is free, movable ones below it, free ones below it), a lane a page
    auto each = [&](auto &&visit) {
        constexpr int kAtOnce = 4;  // groups read before they are visited
        for (int first = wave; first < groups; first += kAtOnce * kWaves) {
            uint2 held[kAtOnce], free[kAtOnce];
            int2 before[kAtOnce];
#pragma unroll
            for (int k = 0; k < kAtOnce; ++k) {
                const int g = min(first + k * kWaves, groups - 1);
                held[k] = *(const uint2 *)(s_held + 2 * g);
                free[k] = *(const uint2 *)(s_free + 2 * g);
                before[k] = *(const int2 *)(s_rows + 2 * g);
            }
#pragma unroll
            for (int k = 0; k < kAtOnce; ++k) {
                const int g = first + k * kWaves;
                if (g >= groups)
                    break;
                auto word = [](uint2 v) {
                    return (unsigned long long)(unsigned)__builtin_amdgcn_readfirstlane((int)v.y) << 32 |
                           (unsigned)__builtin_amdgcn_readfirstlane((int)v.x);
                };
                const unsigned long long h = word(held[k]), f = word(free[k]);
                auto below = [](unsigned long long m, int n) {
                    return (int)__builtin_amdgcn_mbcnt_hi((unsigned)(m >> 32), __builtin_amdgcn_mbcnt_lo((unsigned)m, (unsigned)n));
                };
                visit(64 * g + lane, __builtin_amdgcn_inverse_ballot_w64(h), __builtin_amdgcn_inverse_ballot_w64(f),
                      below(h, before[k].x), below(f, before[k].y));
            }
        }
    };
    int moves = 0, lowest = INT_MAX;
    each([&](int page, bool is_t, bool is_f, int tb, int fb) {
        const int above = all_movable - 1 - tb;
        if (is_t && fb > above) {
            c.copies[3u * above] = page;
            c.copies[3u * above + 2] = 1 << t.page_shift;
            c.move[page] = above;
            lowest = min(lowest, page);
            ++moves;
        } else if (is_f && all_movable - tb > fb) {
            c.copies[3u * fb + 1] = page;
        }
    });
#pragma unroll
    for (int d = 32; d > 0; d /= 2) {
        moves += __shfl_xor(moves, d);
        lowest = min(lowest, __shfl_xor(lowest, d));
    }
    if (lane == 0) {
        atomicAdd(&s_moves, moves);
        atomicMin(&s_lowest, lowest);
    }
    __syncthreads();
    const int all_moves = s_moves;
    int *const list_out = c.free_out + start - all_moves;
    each([&](int page, bool is_t, bool is_f, int tb, int fb) {
        const int moved_below = max(0, tb - (all_movable - all_moves));
        if (is_t ? tb >= all_movable - all_moves : is_f && fb >= all_moves)
            list_out[fb + moved_below] = page;
    });
    if (c.remaps) {
        __syncthreads();
        remap(c, all_moves, all_free, s_lowest, wave, kWaves, tid, kThreads);
    } else if (tid == 0) {
        c.move[c.num_pages] = all_moves;
        c.move[c.num_pages + 1] = all_free;
        c.move[c.num_pages + 2] = s_lowest;
    }
}

__global__ __launch_bounds__(256) void remap_kernel(Compact c)
{
    const int *found = c.move + c.num_pages;
    remap(c, found[0], found[1], found[2], blockIdx.x * 4ll + (threadIdx.x >> 6), gridDim.x * 4ll,
          blockIdx.x * 256ll + threadIdx.x, gridDim.x * 256ll);
}

// ---- copies -----------------------------------------------------------------

// A workgroup takes one chunk of a page at a time, four 16-byte loads a thread in flight before their stores (as
// vectors by themselves: an array of them went to LDS). Bound by HBM: 349 MB in 68 us, 5.1 TB/s.
__global__ __launch_bounds__(256) void copy_pages_kernel(unsigned char *__restrict__ cache, const int *__restrict__ copies,
                                                         unsigned count, unsigned per_entry, unsigned chunks, int num_pages,
                                                         int page_size, int row_bytes, int chunk)
{
    typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
    const size_t page_bytes = (size_t)page_size * row_bytes;
    // entry blockIdx.x / per_entry first, per_entry = layers x chunks: an entry's chunks are neighbours
    for (unsigned long long i = blockIdx.x; i < (unsigned long long)count * per_entry; i += gridDim.x) {
        const unsigned entry = (unsigned)(i / per_entry), part = (unsigned)(i - (unsigned long long)entry * per_entry);
        const int src = copies[3 * (size_t)entry], dst = copies[3 * (size_t)entry + 1];
        const int rows = min(copies[3 * (size_t)entry + 2], page_size);
        if ((unsigned)src >= (unsigned)num_pages || (unsigned)dst >= (unsigned)num_pages || src == dst || rows <= 0)
            continue;
        const unsigned layer = part / chunks;
        const size_t first = (size_t)(part - layer * chunks) * chunk, end = min(first + chunk, (size_t)rows * row_bytes);
        unsigned char *layer_base = cache + (size_t)layer * num_pages * page_bytes;
        const unsigned char *from = layer_base + (size_t)src * page_bytes;
        unsigned char *to = layer_base + (size_t)dst * page_bytes;
        for (size_t o = first + threadIdx.x * 16; o < end; o += 4 * 4096) {
            const size_t o1 = o + 4096, o2 = o + 2 * 4096, o3 = o + 3 * 4096, last = end - 16;
            const u32x4 a = *(const u32x4 *)(from + o), b = *(const u32x4 *)(from + min(o1, last));
            const u32x4 c = *(const u32x4 *)(from + min(o2, last)), d = *(const u32x4 *)(from + min(o3, last));
            *(u32x4 *)(to + o) = a;
            if (o1 < end)
                *(u32x4 *)(to + o1) = b;
            if (o2 < end)
                *(u32x4 *)(to + o2) = c;
            if (o3 < end)
                *(u32x4 *)(to + o3) = d;
        }
    }
}

bool page_ok(int page_size) { return page_size >= 32 && page_size <= (1 << 20) && (page_size & (page_size - 1)) == 0; }

bool table_ok(const int *block_table, const int *lens, int rows, int num_pages, int page_size, int stride)
{
    return block_table && lens && rows >= 1 && rows <= kMostRows && num_pages >= 1 && num_pages <= kMostPages &&
           page_ok(page_size) && stride >= 1 && stride <= kMostColumns;
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
    return num_pages < 1 || num_pages > mla::kMostPages ? 0 : (4 * ((size_t)num_pages + 3) + 255) / 256 * 256;
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
    const auto kernel = block_table_stride < 4 ? mla::fork_kernel<true> : mla::fork_kernel<false>;
    hipLaunchKernelGGL(kernel, dim3(1 + writers), dim3(mla::kThreads), 0, static_cast<hipStream_t>(stream), f);
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
    // Entries of the table, the moves and the list: up to kRemapHere the first workgroup writes them itself (us a call,
    // in one launch and in two: 1760 entries 10.3, 12.1; 8320 12.6, 13.4; 12 800 14.0, 14.4; 19 200 16.6, 15.5;
    // 38 400 24.0, 20.6).
    const int64_t entries = (int64_t)rows * block_table_stride + (int64_t)3 * moves + num_free;
    const int here = entries <= mla::kRemapHere;
    const mla::Compact c{{block_table, lens, rows, block_table_stride, __builtin_ctz((unsigned)page_size)},
                         pinned, free_pages, free_start, new_table, copies, new_free_pages,
                         static_cast<int *>(workspace), num_pages, num_free, moves, here};
    hipStream_t s = static_cast<hipStream_t>(stream);
    const auto kernel = block_table_stride < 4 ? mla::compact_kernel<true> : mla::compact_kernel<false>;
    hipLaunchKernelGGL(kernel, dim3(1), dim3(mla::kThreads), 0, s, c);
    if (const int st = mla::launched(); st || here)
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
    const int64_t per_entry = (int64_t)layers * chunks, items = (int64_t)count * per_entry;
    if (per_entry > INT32_MAX)
        return MLA_STATUS_INVALID_VALUE;
    const int wgs = (int)std::min<int64_t>(items, 64 * (int64_t)mla::current_cu_count());
    hipLaunchKernelGGL(mla::copy_pages_kernel, dim3(wgs), dim3(256), 0, static_cast<hipStream_t>(stream),
                       static_cast<unsigned char *>(kv_cache), copies, (unsigned)count, (unsigned)per_entry, (unsigned)chunks,
                       num_pages, page_size, row_bytes, chunk);
    return mla::launched();
}

}  // extern "C"
