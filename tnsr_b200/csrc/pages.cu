// Pages of key-value caches: who holds which page, and the pages' contents.  A book is a table [sequences, table_ld] of pages, the rows
// that each sequence has, and for each page of the pool how many live table entries hold it (0: the page is free).  Entries behind a
// sequence's last page are not read.
//
//   fork      sequence i becomes what parents[i] was: table rows change, no page is copied
//   reserve   room for new rows: free pages, the lowest first, in order of the sequences; a part-filled last page that others hold too is
//             copied first (one of its writers keeps it, if every holder is one: the first)
//   release   sequences end, their pages lose a holder
//   compact   live pages behind the first `live` ones move into the gaps before, in order
//   copy      pages onto others
//
// The bookkeeping is integers: counters by atomics (sums do not depend on their order), choices by ranks (prefix sums in order of sequences and
// pages), so a call's result is a function of its inputs.  What has an order runs in one block: 16 sequences x 4 beams with 40 entries each take
// a few us, which is the latency of a chain of dependent reads, and the search for free pages ends at the last one that is needed.
// What bounds a call that copies is the copying: 16-byte loads, eight on their way per thread (compaction of 512 MB: 117 us, of which the copying takes 102, 5.3 TB/s read and written, and
// the plan before it the rest; 4 or 16 blocks an SM are level with 8).  Fork and reserve of 64 sequences with 24 pools: 18.5 us, three launches that wait for one another.
//
// Also here: rows appended to caches in pages, and states reordered to their sequences' parents.
#include <algorithm>

#include "pages.cuh"

namespace tb {

constexpr uint32_t PG_NONE = 0xffffffffu;
constexpr uint32_t PG_THREADS = 1024;

// Workspace in u32: [0] pairs to copy, [1] ticket of fork, zero between calls; then lists that every call fills for itself, for their places follow the book's sizes.
struct PageScratch {
    uint32_t *header, *keeper, *writers, *pages, *from, *to, *need, *copy, *source;
};
static PageScratch page_scratch(void* ws, uint32_t sequences, uint32_t pool_pages) {
    uint32_t* p = reinterpret_cast<uint32_t*>(ws);
    PageScratch s;
    s.header = p;
    s.keeper = s.header + 16;
    s.writers = s.keeper + pool_pages;
    s.pages = s.writers + pool_pages;        // free pages in order, or where a page went
    s.from = s.pages + pool_pages;
    s.to = s.from + pool_pages;
    s.need = s.to + pool_pages;              // [sequences + 1] pages before a sequence's
    s.copy = s.need + sequences + 1;         // [sequences] copies before a sequence's
    s.source = s.copy + sequences;           // [sequences] page to be copied
    return s;
}
uint64_t pages_workspace_bytes(uint32_t sequences, uint32_t pool_pages) { return 4ull * (16 + 5ull * pool_pages + 3ull * sequences + 1); }

static __device__ __forceinline__ uint32_t pages_of(uint32_t rows, uint32_t page_rows) { return rows / page_rows + (rows % page_rows != 0); }
// Pages of sequence s; more than its table row has room for is the caller's mistake, and told.
static __device__ __forceinline__ uint32_t live_pages(const PageBook& b, uint32_t s) {
    const uint32_t n = pages_of(b.lengths[s], b.page_rows);
    if (n > b.table_ld) report(b.d_status, DEV_BAD_LENGTH);
    return min(n, b.table_ld);
}

// Exclusive prefix sum over the block in thread order, and the total.
__device__ __forceinline__ uint32_t block_scan(uint32_t v, uint32_t& total) {
    __shared__ uint32_t warps[32];
    const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5, count = blockDim.x >> 5;
    uint32_t x = v;
#pragma unroll
    for (int d = 1; d < 32; d *= 2) {
        const uint32_t y = __shfl_up_sync(0xffffffffu, x, d);
        if (lane >= d) x += y;
    }
    __syncthreads();
    if (lane == 31) warps[warp] = x;
    __syncthreads();
    uint32_t w = lane < count ? warps[lane] : 0u;
#pragma unroll
    for (int d = 1; d < 32; d *= 2) {
        const uint32_t y = __shfl_up_sync(0xffffffffu, w, d);
        if (lane >= d) w += y;
    }
    total = __shfl_sync(0xffffffffu, w, 31);
    const uint32_t before = __shfl_sync(0xffffffffu, w, warp ? warp - 1 : 0);
    return x - v + (warp ? before : 0u);
}

// ---- fork -----------------------------------------------------------------------------------------------------------------
// A block has `columns` columns of the whole table in shared memory, so that rows can trade places, and beside them what everybody's length and parent is; the last
// block that has read the lengths writes them.
__global__ void __launch_bounds__(256) pages_fork_kernel(PageBook b, const uint32_t* parents, uint32_t columns, uint32_t* ticket) {
    extern __shared__ uint32_t staged[];       // [sequences][columns], [sequences] lengths, [sequences] parents
    __shared__ uint32_t s_last;
    uint32_t *lengths = staged + columns * b.sequences, *from = lengths + b.sequences;
    pdl_wait();
    pdl_trigger();
    const uint32_t column0 = blockIdx.x * columns, here = min(columns, b.table_ld - column0), cells = b.sequences * here;
    for (uint32_t s = threadIdx.x; s < b.sequences; s += blockDim.x) {
        lengths[s] = b.lengths[s];
        if (blockIdx.x == 0 && pages_of(lengths[s], b.page_rows) > b.table_ld) report(b.d_status, DEV_BAD_LENGTH);
        uint32_t p = parents[s];
        if (p >= b.sequences) {
            if (blockIdx.x == 0) report(b.d_status, DEV_BAD_PARENT);
            p = s;
        }
        from[s] = p;
    }
    __syncthreads();
    auto live = [&](uint32_t s) { return min(pages_of(lengths[s], b.page_rows), b.table_ld); };
    for (uint32_t i = threadIdx.x; i < cells; i += blockDim.x) {
        const uint32_t s = i / here, c = i % here;
        staged[i] = column0 + c < live(s) ? b.table[(size_t)s * b.table_ld + column0 + c] : PG_NONE;
    }
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < cells; i += blockDim.x) {
        const uint32_t s = i / here, c = i % here, p = from[s];
        if (p == s) continue;
        const bool was = column0 + c < live(s), is = column0 + c < live(p);
        const uint32_t before = staged[i], page = staged[p * here + c];
        if (is) b.table[(size_t)s * b.table_ld + column0 + c] = page;
        if (was && is && before == page) continue;
        if ((was && before >= b.pool_pages) || (is && page >= b.pool_pages)) report(b.d_status, DEV_BAD_PAGE);
        if (was && before < b.pool_pages) atomicSub(b.holders + before, 1u);
        if (is && page < b.pool_pages) atomicAdd(b.holders + page, 1u);
    }
    if (threadIdx.x == 0) s_last = atomicAdd(ticket, 1u) + 1 == gridDim.x;      // lengths were read before the first barrier
    __syncthreads();
    if (!s_last) return;
    for (uint32_t s = threadIdx.x; s < b.sequences; s += blockDim.x)
        if (from[s] != s) b.lengths[s] = lengths[from[s]];
    if (threadIdx.x == 0) *ticket = 0;
}

int launch_pages_fork(const PageBook& b, const uint32_t* parents, cudaStream_t stream) {
    if (b.sequences == 0) return TNSR_B200_OK;
    // Columns of a block: with few sequences two, for less to do one thing behind the other; with more than 48 KB of them fewer, down to one: 12 bytes a sequence
    uint32_t columns = b.sequences > 256 ? 8 : 2;
    while (columns > 1 && (uint64_t)(columns + 2) * b.sequences > 12288) columns /= 2;
    if (int rc = allow_shared<pages_fork_kernel>(3 * PAGES_MAX_SEQUENCES * 4, "pages_fork attribute")) return rc;
    const PageScratch ws = page_scratch(b.workspace, b.sequences, b.pool_pages);
    launch_kernel(pages_fork_kernel, dim3(ceil_div(b.table_ld, columns)), dim3(256), (size_t)(columns + 2) * b.sequences * 4, stream, b, parents, columns,
                  ws.header + 1);
    count_launch();
    return check_launch("pages_fork");
}

// ---- contents of pages ------------------------------------------------------------------------------------------------------
constexpr uint32_t PG_POOLS = 64;                // pools of a launch: their pointers travel as parameters
constexpr uint32_t PG_PIECE = 32768;             // bytes that a block copies at a time: eight 16-byte loads a thread
struct PoolList {
    uint8_t* at[PG_POOLS];
    uint64_t bytes[PG_POOLS];
    uint32_t pieces[PG_POOLS];       // of a page
    uint32_t count, pieces_all;      // of a page in all pools
    bool wide;                       // 16-byte units
};

__device__ __forceinline__ void copy_piece(uint8_t* __restrict__ to, const uint8_t* from, uint64_t bytes, bool wide) {
    if (wide) {
        const uint4* src = reinterpret_cast<const uint4*>(from);
        uint4* dst = reinterpret_cast<uint4*>(to);
        const uint32_t n = (uint32_t)(bytes / 16);
        uint4 v[8];
        for (uint32_t i = threadIdx.x; i < n; i += 8 * 256) {
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (i + j * 256 < n) v[j] = src[i + j * 256];
#pragma unroll
            for (int j = 0; j < 8; ++j)
                if (i + j * 256 < n) dst[i + j * 256] = v[j];
        }
    } else {
        for (uint64_t i = threadIdx.x; i < bytes; i += blockDim.x) to[i] = from[i];
    }
}

// Pages from[i] -> to[i] of every pool; *d_pairs of them where d_pairs is set.  `moved`: table entries of pages from `keep_below` on become moved[entry].
__global__ void __launch_bounds__(256) pages_copy_kernel(const __grid_constant__ PoolList pools, const uint32_t* from, const uint32_t* to, uint32_t pairs,
                                                         const uint32_t* d_pairs, uint32_t pool_pages, int* d_status, PageBook b, const uint32_t* moved,
                                                         const uint32_t* d_live) {
    pdl_wait();
    pdl_trigger();
    const uint32_t n = d_pairs ? *d_pairs : pairs;
    if (moved && n) {
        const uint32_t live = *d_live;
        for (uint64_t i = (uint64_t)blockIdx.x * blockDim.x + threadIdx.x; i < (uint64_t)b.sequences * b.table_ld; i += (uint64_t)gridDim.x * blockDim.x) {
            const uint32_t s = (uint32_t)(i / b.table_ld), c = (uint32_t)(i % b.table_ld);
            if (c >= live_pages(b, s)) continue;
            const uint32_t page = b.table[i];
            if (page >= b.pool_pages) report(b.d_status, DEV_BAD_PAGE);
            else if (page >= live) b.table[i] = moved[page];
        }
    }
    // pair by pair in pieces of all pools; the next item's pages are asked for before the copy
    const uint64_t items = (uint64_t)n * pools.pieces_all;
    const uint32_t pairs_on = gridDim.x / max(pools.pieces_all, 1u), pieces_on = gridDim.x - pairs_on * pools.pieces_all;
    uint32_t pair = blockIdx.x / max(pools.pieces_all, 1u), at = blockIdx.x - pair * pools.pieces_all, next_src = 0, next_dst = 0;
    if (blockIdx.x < items) {
        next_src = from[pair];
        next_dst = to[pair];
    }
    for (uint64_t item = blockIdx.x; item < items; item += gridDim.x) {
        const uint32_t src = next_src, dst = next_dst;
        uint32_t piece = at, t = 0;
        while (piece >= pools.pieces[t]) piece -= pools.pieces[t++];
        pair += pairs_on;
        at += pieces_on;
        if (at >= pools.pieces_all) {
            at -= pools.pieces_all;
            ++pair;
        }
        if (item + gridDim.x < items) {
            next_src = from[pair];
            next_dst = to[pair];
        }
        if (src >= pool_pages || dst >= pool_pages) {
            if (threadIdx.x == 0) report(d_status, DEV_BAD_PAGE);
            continue;
        }
        const uint64_t first = (uint64_t)piece * PG_PIECE, bytes = pools.bytes[t];
        copy_piece(pools.at[t] + dst * bytes + first, pools.at[t] + src * bytes + first, min((uint64_t)PG_PIECE, bytes - first), pools.wide);
    }
}

// `most`: pairs at the most, for the grid.
static int launch_copies(const PagePools& pools, const uint32_t* from, const uint32_t* to, uint32_t pairs, const uint32_t* d_pairs, uint64_t most,
                         uint32_t pool_pages, int* d_status, const PageBook& b, const uint32_t* moved, const uint32_t* d_live, cudaStream_t stream) {
    bool launched = false;
    for (uint32_t first = 0; first < std::max(1u, pools.count); first += PG_POOLS) {
        PoolList list = {};
        list.wide = true;
        for (uint32_t t = first; t < std::min(pools.count, first + PG_POOLS); ++t) {
            list.at[list.count] = (uint8_t*)pools.tensors[t];
            list.bytes[list.count] = pools.page_bytes[t];
            list.pieces[list.count] = (uint32_t)ceil_div64(pools.page_bytes[t], PG_PIECE);
            list.pieces_all += list.pieces[list.count++];
            list.wide = list.wide && (reinterpret_cast<uintptr_t>(pools.tensors[t]) | pools.page_bytes[t]) % 16 == 0;
        }
        // eight blocks of 256 threads fill an SM
        const uint64_t items = std::max<uint64_t>(most * list.pieces_all, first || !moved ? 0 : ceil_div64((uint64_t)b.sequences * b.table_ld, 256));
        if (items == 0) continue;
        launch_kernel(pages_copy_kernel, dim3((unsigned)std::min<uint64_t>(items, 148 * 8)), dim3(256), 0, stream, list, from, to, pairs, d_pairs, pool_pages,
                      d_status, b, first ? nullptr : moved, d_live);
        count_launch();
        launched = true;
    }
    return launched ? check_launch("pages_copy") : TNSR_B200_OK;
}

int launch_pages_copy(const PagePools& pools, const uint32_t* from, const uint32_t* to, uint32_t pairs, uint32_t pool_pages, int* d_status, cudaStream_t stream) {
    return launch_copies(pools, from, to, pairs, nullptr, pairs, pool_pages, d_status, PageBook{}, nullptr, nullptr, stream);
}

// ---- reserve -----------------------------------------------------------------------------------------------------------------
// Writes the pages p of [0, pool) for which want(holders[p], p) holds to out[0 ..], up to `most` of them, in order; returns how many there were (counting
// ends with the block's sweep in which `most` was reached).  Sixteen pages per thread and sweep.
template <typename Want>
__device__ uint32_t list_pages(const uint32_t* holders, uint32_t pool, uint32_t most, uint32_t* out, Want want) {
    uint32_t found = 0;
    const bool wide = (reinterpret_cast<uintptr_t>(holders) & 15) == 0;
    for (uint32_t base = 0; base < pool && found < most; base += PG_THREADS * 16) {
        const uint32_t first = base + threadIdx.x * 16;
        uint32_t hits = 0;
        if (wide && first + 16 <= pool) {
            uint4 v[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) v[j] = reinterpret_cast<const uint4*>(holders + first)[j];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                hits |= (uint32_t)want(v[j].x, first + 4 * j) << (4 * j) | (uint32_t)want(v[j].y, first + 4 * j + 1) << (4 * j + 1) |
                        (uint32_t)want(v[j].z, first + 4 * j + 2) << (4 * j + 2) | (uint32_t)want(v[j].w, first + 4 * j + 3) << (4 * j + 3);
            }
        } else {
            for (uint32_t j = 0; j < 16 && first + j < pool; ++j) hits |= (uint32_t)want(holders[first + j], first + j) << j;
        }
        uint32_t total, at = found + block_scan(__popc(hits), total);
        for (; hits && at < most; hits &= hits - 1) {
            if (out) out[at] = first + __ffs(hits) - 1;
            ++at;
        }
        found += total;
    }
    return found;
}

__global__ void __launch_bounds__(PG_THREADS) pages_reserve_kernel(PageBook b, const uint32_t* rows, uint32_t rows_each, PageScratch ws) {
    __shared__ uint32_t s_bad;
    __shared__ uint32_t s_many;                  // wanted pages in units of 8192, rounded down per thread
    pdl_wait();
    pdl_trigger();
    if (threadIdx.x == 0) {
        s_bad = 0;
        s_many = 0;
        ws.header[0] = 0;
    }
    __syncthreads();
    // sequences that will write to a page which others hold too: how many per page, and the first of them
    auto last_entry = [&](uint32_t s, uint32_t length) { return b.table + (size_t)s * b.table_ld + length / b.page_rows; };
    const uint64_t room = min((uint64_t)b.table_ld * b.page_rows, (uint64_t)PAGED_MAX_KEYS);
    const uint32_t share = (b.sequences + PG_THREADS - 1) / PG_THREADS;
    const uint32_t s0 = min(b.sequences, threadIdx.x * share), s1 = min(b.sequences, s0 + share);
    for (uint32_t s = s0; s < s1; ++s) {
        const uint32_t length = b.lengths[s], n = rows ? rows[s] : rows_each;
        ws.source[s] = PG_NONE;
        if ((uint64_t)length + n > room) {
            atomicMax(&s_bad, (uint32_t)DEV_BAD_LENGTH);
            continue;
        }
        if (n == 0 || length % b.page_rows == 0) continue;
        const uint32_t page = *last_entry(s, length);
        if (page >= b.pool_pages) {
            atomicMax(&s_bad, (uint32_t)DEV_BAD_PAGE);
            continue;
        }
        if (b.holders[page] < 2) continue;
        ws.source[s] = page;
        ws.writers[page] = ws.keeper[page] = 0;
    }
    __syncthreads();
    for (uint32_t s = s0; s < s1; ++s) {
        const uint32_t page = ws.source[s];
        if (page == PG_NONE) continue;
        atomicAdd(ws.writers + page, 1u);
        atomicMax(ws.keeper + page, ~s);
    }
    __syncthreads();
    const uint32_t bad = s_bad;
    uint64_t want = 0;
    uint32_t copies = 0;
    for (uint32_t s = s0; s < s1; ++s) {
        const uint32_t page = ws.source[s];
        if (page != PG_NONE && __ldcg(ws.writers + page) == b.holders[page] && __ldcg(ws.keeper + page) == ~s) ws.source[s] = PG_NONE;   // keeps it
    }
    __syncthreads();
    for (uint32_t s = s0; s < s1 && !bad; ++s) {
        const uint32_t length = b.lengths[s], n = rows ? rows[s] : rows_each;
        const bool copy = ws.source[s] != PG_NONE;
        want += pages_of(length + n, b.page_rows) - pages_of(length, b.page_rows) + copy;
        copies += copy;
    }
    // Twelve sequences of 2^31 pages a thread at the most.  Above 2^18 units there are more than a pool's 2^30 pages; else there are fewer than 2^32 in all, and the sums
    // below are exact.
    if (want >> 13) atomicAdd(&s_many, (uint32_t)(want >> 13));
    uint32_t all, all_copies;
    uint32_t at = block_scan((uint32_t)want, all), copy_at = block_scan(copies, all_copies);      // with barriers
    // appended rows would go over old ones: whoever appends behind this call asks the word
    auto outcome = [&](uint32_t what) {
        if (threadIdx.x) return;
        if (what) report(b.d_status, (int)what);
        if (b.refused) *b.refused = what;
    };
    if (bad) {
        outcome(bad);
        return;
    }
    for (uint32_t s = s0; s < s1; ++s) {
        const uint32_t length = b.lengths[s], n = rows ? rows[s] : rows_each;
        const bool copy = ws.source[s] != PG_NONE;
        ws.need[s] = at;
        ws.copy[s] = copy_at;
        at += pages_of(length + n, b.page_rows) - pages_of(length, b.page_rows) + copy;
        copy_at += copy;
    }
    if (s_many > 1u << 18 || all > b.pool_pages || list_pages(b.holders, b.pool_pages, all, ws.pages, [](uint32_t h, uint32_t) { return h == 0; }) < all) {
        outcome(DEV_NO_PAGES);
        return;
    }
    __syncthreads();
    for (uint32_t j = threadIdx.x; j < all; j += PG_THREADS) {
        uint32_t low = 0, high = b.sequences;        // the last sequence whose pages start at or before j: it has some
        while (high - low > 1) {
            const uint32_t mid = (low + high) / 2;
            if (ws.need[mid] <= j) low = mid; else high = mid;
        }
        const uint32_t length = b.lengths[low], page = ws.pages[j], source = ws.source[low];
        uint32_t i = j - ws.need[low];
        b.holders[page] = 1;
        if (source != PG_NONE) {
            if (i == 0) {
                *last_entry(low, length) = page;
                atomicSub(b.holders + source, 1u);
                ws.from[ws.copy[low]] = source;
                ws.to[ws.copy[low]] = page;
                continue;
            }
            --i;
        }
        b.table[(size_t)low * b.table_ld + pages_of(length, b.page_rows) + i] = page;
    }
    __syncthreads();
    for (uint32_t s = s0; s < s1; ++s) b.lengths[s] += rows ? rows[s] : rows_each;
    if (threadIdx.x == 0) ws.header[0] = all_copies;
    outcome(0);
}

int launch_pages_reserve(const PageBook& b, const PagePools& pools, const uint32_t* rows, uint32_t rows_each, cudaStream_t stream) {
    if (b.sequences == 0) return TNSR_B200_OK;
    const PageScratch ws = page_scratch(b.workspace, b.sequences, b.pool_pages);
    launch_kernel(pages_reserve_kernel, dim3(1), dim3(PG_THREADS), 0, stream, b, rows, rows_each, ws);
    count_launch();
    if (int rc = check_launch("pages_reserve")) return rc;
    return launch_copies(pools, ws.from, ws.to, 0, ws.header, std::min(b.sequences, b.pool_pages), b.pool_pages, b.d_status, b, nullptr, nullptr, stream);
}

// ---- release -----------------------------------------------------------------------------------------------------------------
__global__ void __launch_bounds__(128) pages_release_kernel(PageBook b, const uint8_t* gone) {
    pdl_wait();
    pdl_trigger();
    const uint32_t s = blockIdx.x;
    if (!gone[s]) return;
    const uint32_t n = live_pages(b, s);
    for (uint32_t c = threadIdx.x; c < n; c += blockDim.x) {
        const uint32_t page = b.table[(size_t)s * b.table_ld + c];
        if (page < b.pool_pages) atomicSub(b.holders + page, 1u);
        else report(b.d_status, DEV_BAD_PAGE);
    }
    __syncthreads();
    if (threadIdx.x == 0) b.lengths[s] = 0;
}

int launch_pages_release(const PageBook& b, const uint8_t* gone, cudaStream_t stream) {
    if (b.sequences == 0) return TNSR_B200_OK;
    launch_kernel(pages_release_kernel, dim3(b.sequences), dim3(128), 0, stream, b, gone);
    count_launch();
    return check_launch("pages_release");
}

// ---- compact -----------------------------------------------------------------------------------------------------------------
__global__ void __launch_bounds__(PG_THREADS) pages_compact_kernel(PageBook b, PageScratch ws, uint32_t* live_out) {
    pdl_wait();
    pdl_trigger();
    const uint32_t live = list_pages(b.holders, b.pool_pages, PG_NONE, nullptr, [](uint32_t h, uint32_t) { return h != 0; });
    // gaps before `live`, and pages behind it: equally many
    const uint32_t gaps = list_pages(b.holders, live, PG_NONE, ws.to, [](uint32_t h, uint32_t) { return h == 0; });
    list_pages(b.holders, b.pool_pages, gaps, ws.from, [live](uint32_t h, uint32_t p) { return h != 0 && p >= live; });
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < gaps; i += PG_THREADS) {
        const uint32_t from = ws.from[i], to = ws.to[i];
        ws.pages[from] = to;
        b.holders[to] = b.holders[from];
        b.holders[from] = 0;
    }
    if (threadIdx.x == 0) {
        ws.header[0] = gaps;
        ws.header[2] = live;
        if (live_out) *live_out = live;
    }
}

int launch_pages_compact(const PageBook& b, const PagePools& pools, uint32_t* live_out, cudaStream_t stream) {
    const PageScratch ws = page_scratch(b.workspace, b.sequences, b.pool_pages);
    launch_kernel(pages_compact_kernel, dim3(1), dim3(PG_THREADS), 0, stream, b, ws, live_out);
    count_launch();
    if (int rc = check_launch("pages_compact")) return rc;
    return launch_copies(pools, ws.from, ws.to, 0, ws.header, b.pool_pages / 2, b.pool_pages, b.d_status, b, ws.pages, ws.header + 2, stream);
}

// ---- new rows into pages --------------------------------------------------------------------------------------------------------
template <typename U>
__global__ void __launch_bounds__(256) paged_append_kernel(PagedParams p, PagedAppend a, uint32_t k_units, uint32_t v_units, uint32_t per_unit) {
    pdl_wait();
    pdl_trigger();
    if (a.refused && *a.refused) return;                         // no room for the rows: what lies at their places is older
    const uint32_t row = blockIdx.x;
    uint32_t s = row / a.chunk;
    if (a.row_starts) {           // the last sequence that starts at or before the row
        uint32_t low = 0, high = a.sequences;
        while (high - low > 1) {
            const uint32_t mid = (low + high) / 2;
            if (a.row_starts[mid] <= row) low = mid; else high = mid;
        }
        s = low;
    }
    const PagedSequence q = paged_sequence(p, s);
    const uint32_t i = row - q.start;
    if (row < q.start || i >= q.count) return;                  // behind the last sequence
    // cut lengths and counts (told by now) would put rows where others are
    if (a.lengths[s] > p.capacity || (a.row_starts && min(a.row_starts[s + 1], a.rows) - q.start > a.chunk)) return;
    if (q.length < q.count - i) {                               // the cache has no such row
        if (threadIdx.x == 0) report(a.d_status, DEV_BAD_LENGTH);
        return;
    }
    uint32_t page, r;
    if (!paged_key(p, a.table + (size_t)s * a.table_ld, q.length - q.count + i, page, r)) {
        if (threadIdx.x == 0) report(a.d_status, DEV_BAD_PAGE);
        return;
    }
    // units of a head, then heads
    const uint32_t all = a.kv_heads * (k_units + v_units);
    for (uint32_t u = threadIdx.x; u < all; u += blockDim.x) {
        const bool key = u < a.kv_heads * k_units;
        const uint32_t x = key ? u : u - a.kv_heads * k_units, units = key ? k_units : v_units, h = x / units, c = x % units;
        const U* src = reinterpret_cast<const U*>(key ? a.k : a.v) + ((size_t)row * (key ? a.k_ld : a.v_ld)) / per_unit + x;
        U* dst = reinterpret_cast<U*>(key ? a.k_pool : a.v_pool) +
                 ((key ? a.k_page : a.v_page) * page + (key ? a.k_row : a.v_row) * r + (key ? a.k_head : a.v_head) * h) / per_unit + c;
        *dst = *src;
    }
}

int launch_paged_append(const PagedAppend& a, int dtype, cudaStream_t stream) {
    if (a.rows == 0 || a.sequences == 0) return TNSR_B200_OK;
    PagedParams p = {};
    p.a.lengths = a.lengths;
    p.a.row_starts = a.row_starts;
    p.a.d_status = a.d_status;
    p.a.chunk = a.chunk;
    p.a.rows = a.rows;
    p.a.pool_pages = a.pool_pages;
    p.page = fast_div(a.page_rows);
    p.capacity = (uint32_t)std::min<uint64_t>((uint64_t)a.table_ld * a.page_rows, PAGED_MAX_KEYS);
    const uint32_t size = dtype == TNSR_B200_F32 ? 4 : 2, per = 16 / size;
    // 16-byte units where every address is a multiple of one
    const uint64_t all = (uint64_t)a.dim | a.vdim | a.k_ld | a.v_ld | a.k_page | a.k_row | a.k_head | a.v_page | a.v_row | a.v_head;
    const uintptr_t at = (uintptr_t)a.k | (uintptr_t)a.v | (uintptr_t)a.k_pool | (uintptr_t)a.v_pool;
    const dim3 grid(a.rows);
    auto threads = [&](uint32_t units) { return dim3(std::min(256u, ceil_div(units, 32u) * 32u)); };
    if (all % per == 0 && at % 16 == 0) {
        launch_kernel(paged_append_kernel<uint4>, grid, threads(a.kv_heads * (a.dim + a.vdim) / per), 0, stream, p, a, a.dim / per, a.vdim / per, per);
    } else if (size == 4) {
        launch_kernel(paged_append_kernel<uint32_t>, grid, threads(a.kv_heads * (a.dim + a.vdim)), 0, stream, p, a, a.dim, a.vdim, 1u);
    } else {
        launch_kernel(paged_append_kernel<uint16_t>, grid, threads(a.kv_heads * (a.dim + a.vdim)), 0, stream, p, a, a.dim, a.vdim, 1u);
    }
    count_launch();
    return check_launch("paged_append");
}

// ---- states to their sequences' parents -------------------------------------------------------------------------------------------
// A thread has the same unit of every row of a group: it reads what moves, then writes, so the rows trade places without a copy of them
// and without waiting for anybody.  Rows that stay are neither read nor written.  Bound by HBM: 247 MB moved, 46 to 50 us = 4.9 to 5.4 TB/s.
constexpr uint32_t RO_TENSORS = 64;
struct StateList {
    uint8_t* at[RO_TENSORS];
    uint64_t units[RO_TENSORS], pitch[RO_TENSORS];      // units of a row, bytes between rows
};

template <typename U, int MAX>
__global__ void __launch_bounds__(128) reorder_states_kernel(const __grid_constant__ StateList list, const uint32_t* parents, uint32_t groups, uint32_t beams,
                                                             int* d_status) {
    pdl_wait();
    pdl_trigger();
    const uint64_t unit = (uint64_t)blockIdx.x * blockDim.x + threadIdx.x;
    uint8_t* base = list.at[blockIdx.z];
    const uint64_t pitch = list.pitch[blockIdx.z];
    for (uint32_t g = blockIdx.y; g < groups; g += gridDim.y) {
        uint32_t from[MAX];
        const uint32_t first = g * beams;
#pragma unroll
        for (int i = 0; i < MAX; ++i) {
            from[i] = PG_NONE;
            if (i < beams) {
                const uint32_t p = parents[first + i];
                if (p - first >= beams) {
                    if (unit == 0 && blockIdx.z == 0) report(d_status, DEV_BAD_PARENT);
                } else if (p != first + i) {
                    from[i] = p;
                }
            }
        }
        if (unit >= list.units[blockIdx.z]) continue;
        U v[MAX];
#pragma unroll
        for (int i = 0; i < MAX; ++i)
            if (from[i] != PG_NONE) v[i] = *reinterpret_cast<const U*>(base + from[i] * pitch + unit * sizeof(U));
#pragma unroll
        for (int i = 0; i < MAX; ++i)
            if (from[i] != PG_NONE) *reinterpret_cast<U*>(base + (first + i) * pitch + unit * sizeof(U)) = v[i];
    }
}

template <typename U>
static void launch_reorder(const StateList& list, uint32_t count, uint64_t most, const uint32_t* parents, uint32_t groups, uint32_t beams, int* d_status,
                           cudaStream_t stream) {
    const dim3 grid((unsigned)ceil_div64(most, 128), std::min(groups, 65535u), count);
    if (beams <= 4) launch_kernel(reorder_states_kernel<U, 4>, grid, dim3(128), 0, stream, list, parents, groups, beams, d_status);
    else if (beams <= 8) launch_kernel(reorder_states_kernel<U, 8>, grid, dim3(128), 0, stream, list, parents, groups, beams, d_status);
    else launch_kernel(reorder_states_kernel<U, (int)REORDER_MAX_BEAMS>, grid, dim3(128), 0, stream, list, parents, groups, beams, d_status);
}

int launch_reorder_states(void* const* tensors, const uint64_t* row_bytes, const uint64_t* pitches, uint32_t count, const uint32_t* parents,
                          uint32_t groups, uint32_t beams, int* d_status, cudaStream_t stream) {
    if (groups == 0 || (beams == 1 && !d_status)) return TNSR_B200_OK;        // a row alone stays; a parent outside is still told
    for (uint32_t first = 0; first < count; first += RO_TENSORS) {
        const uint32_t n = std::min(count - first, RO_TENSORS);
        uint64_t bits = 0, most = 0;
        for (uint32_t t = first; t < first + n; ++t) {
            bits |= (uint64_t)(uintptr_t)tensors[t] | row_bytes[t] | pitches[t];
            most = std::max(most, row_bytes[t]);
        }
        if (most == 0) continue;
        const uint32_t unit = bits % 16 == 0 ? 16 : bits % 4 == 0 ? 4 : 1;
        StateList list = {};
        for (uint32_t t = 0; t < n; ++t) {
            list.at[t] = (uint8_t*)tensors[first + t];
            list.units[t] = row_bytes[first + t] / unit;
            list.pitch[t] = pitches[first + t];
        }
        if (unit == 16) launch_reorder<uint4>(list, n, most / unit, parents, groups, beams, d_status, stream);
        else if (unit == 4) launch_reorder<uint32_t>(list, n, most / unit, parents, groups, beams, d_status, stream);
        else launch_reorder<uint8_t>(list, n, most / unit, parents, groups, beams, d_status, stream);
        count_launch();
        if (int rc = check_launch("reorder_states")) return rc;
    }
    return TNSR_B200_OK;
}

}  // namespace tb
