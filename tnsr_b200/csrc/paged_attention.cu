// Attention over key-value caches in pages, rows of any number per sequence: out = softmax(scale q . k) v over the keys a row sees.  A row at
// position p sees keys j <= p with j > p - window, and the first `sinks` ones beside the window; window 0: all of them.  The rows of a
// sequence are the last of its keys; a row before its first key sees nothing and gives zeros.
#include <algorithm>
#include <type_traits>

#include "mixers.cuh"
#include "paged.cuh"
#include "tc_common.cuh"

namespace tb {

// The sequence of a row, and the row's place in it.
__device__ __forceinline__ uint32_t sequence_of(const PagedAttention& a, uint32_t row) {
    if (!a.row_starts) return row / a.chunk;
    uint32_t low = 0, high = a.sequences;        // the last one that starts at or before the row: the one that has it
    while (high - low > 1) {
        const uint32_t mid = (low + high) / 2;
        if (a.row_starts[mid] <= row) low = mid; else high = mid;
    }
    return low;
}

// ---- any widths, strides and alignment ------------------------------------------------------------------------------------------
template <typename T>
__global__ void __launch_bounds__(128) paged_rows_kernel(PagedParams p) {
    pdl_wait();
    pdl_trigger();
    const uint64_t item = (uint64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
    if (item >= (uint64_t)p.a.rows * p.a.heads) return;
    const uint32_t row = (uint32_t)(item / p.a.heads), h = (uint32_t)(item % p.a.heads);
    const uint32_t s = sequence_of(p.a, row);
    const PagedSequence seq = paged_sequence(p, s);
    if (row < seq.start || row - seq.start >= seq.count) return;      // behind the last sequence
    paged_row<T>(p, s, seq, row, h, threadIdx.x & 31);
}

// ---- few rows: keys divided over blocks -------------------------------------------------------------------------------------------
// A unit is 16 rows (tokens x query heads) of one sequence and key/value head; its tiles are the TK keys each that some of the rows see: those of
// the first keys, then those from the first row's window on.  All tiles of all units, one unit behind the other, are divided into equal runs,
// a run per block, so that no block waits for a long sequence: a unit whose tiles lie in several runs leaves a partial result (numerators,
// maximum, sum) per block, and the block that arrives last joins them in the order of the runs.  A block finds its run by itself from the
// lengths (a prefix sum over the sequences), so nothing is planned on the host and a captured call follows its lengths.
// Bound by HBM where there are many keys (16 sequences of up to 32768, 1.39 GB: 208 us = 6.7 TB/s; 32 of up to 4096, 342 MB: 61 us = 5.6 TB/s), else by the
// chain plan, first tile, join (one sequence of 700 keys: 7.4 us).
struct FewUnit {
    PagedSequence seq;
    uint32_t s, kvh, rt, row_tiles;
    uint32_t row0, rows;         // first row and how many
    int32_t first, last;         // positions of the first and the last row's token
    uint32_t tiles, head_tiles, gap;    // tiles; those of the first keys; tile of the window's first key
};

template <uint32_t TK>
__device__ __forceinline__ void unit_tiles(const PagedParams& p, FewUnit& u) {
    u.row0 = u.rt * 16;
    u.rows = min(16u, u.seq.count * p.per.d - u.row0);
    const int32_t base = (int32_t)u.seq.length - (int32_t)u.seq.count;
    u.first = base + (int32_t)p.per.div(u.row0);
    u.last = base + (int32_t)p.per.div(u.row0 + u.rows - 1);
    u.head_tiles = u.gap = 0;
    if (u.last < 0) {            // nothing to see: one tile, all hidden, so that somebody writes the zeros
        u.tiles = 1;
        return;
    }
    if (p.a.window && u.first >= (int32_t)p.a.window) {
        u.gap = (uint32_t)(u.first + 1 - (int32_t)p.a.window) / TK;
        u.head_tiles = min((min(p.a.sinks, (uint32_t)u.last + 1) + TK - 1) / TK, u.gap);
    }
    u.tiles = u.head_tiles + (uint32_t)u.last / TK - u.gap + 1;
}
template <uint32_t TK>
__device__ __forceinline__ void load_sequence(const PagedParams& p, FewUnit& u) {
    u.seq = paged_sequence(p, u.s);
    u.row_tiles = (u.seq.count * p.per.d + 15) / 16;
}
// Tiles of all units of one key/value head of the sequence.
template <uint32_t TK>
__device__ __forceinline__ uint32_t head_tiles(const PagedParams& p, FewUnit u) {
    uint32_t n = 0;
    for (u.rt = 0; u.rt < u.row_tiles; ++u.rt) {
        unit_tiles<TK>(p, u);
        n += u.tiles;
    }
    return n;
}

// Where a block stands: a unit and a tile of it.
template <uint32_t TK>
struct FewCursor {
    FewUnit u;
    uint32_t tile;
    uint64_t at;                 // tiles before this one, of all units
    __device__ __forceinline__ void next_unit(const PagedParams& p) {
        tile = 0;
        if (++u.rt == u.row_tiles) {
            u.rt = 0;
            if (++u.kvh == p.a.kv_heads) {
                u.kvh = 0;
                do {
                    if (++u.s >= p.a.sequences) return;
                    load_sequence<TK>(p, u);
                } while (u.row_tiles == 0);
            }
        }
        unit_tiles<TK>(p, u);
    }
    __device__ __forceinline__ void next(const PagedParams& p) {
        ++at;
        if (++tile == u.tiles) next_unit(p);
    }
    __device__ __forceinline__ uint32_t key0() const { return (tile < u.head_tiles ? tile : u.gap + tile - u.head_tiles) * TK; }
};

// The four warps that compute; a fifth one feeds them.
__device__ __forceinline__ void few_sync() { asm volatile("bar.sync 1, 128;" ::: "memory"); }
__device__ __forceinline__ bool few_any(bool x) {
    uint32_t any;
    asm volatile(
        "{\n\t.reg .pred p, q;\n\t"
        "setp.ne.u32 p, %1, 0;\n\t"
        "bar.red.or.pred q, 1, 128, p;\n\t"
        "selp.u32 %0, 1, 0, q;\n\t}"
        : "=r"(any) : "r"((uint32_t)x) : "memory");
    return any != 0;
}

// x / y, by 32 bits where they do: 64 take some hundred instructions, and every block divides when it plans.
__device__ __forceinline__ uint64_t few_div(uint64_t x, uint64_t y) {
    return (x | y) >> 32 ? x / y : (uint64_t)((uint32_t)x / (uint32_t)y);
}

struct FewRun {
    uint64_t begin, end, length;         // of this block; tiles of a run
};

// Prefix sums over the first 128 threads.
__device__ __forceinline__ uint64_t scan128(uint64_t v, uint64_t* warps, uint64_t& total) {
    const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    uint64_t x = v;
#pragma unroll
    for (int d = 1; d < 32; d *= 2) {
        const uint64_t y = __shfl_up_sync(0xffffffffu, x, d);
        if (lane >= d) x += y;
    }
    if (lane == 31 && warp < 4) warps[warp] = x;
    __syncthreads();
    uint64_t before = 0;
    total = 0;
#pragma unroll
    for (uint32_t w = 0; w < 4; ++w) {
        if (w < warp) before += warps[w];
        total += warps[w];
    }
    return before + x - v;
}

// This block's run and its first tile; false: there is none.  `whole`: runs end where units do.
template <uint32_t TK>
__device__ __forceinline__ bool few_plan(const PagedParams& p, bool whole, FewRun& run, FewCursor<TK>& c) {
    __shared__ uint64_t warps[4], s_at;
    __shared__ uint32_t s_sequence, s_per_head;
    __shared__ PagedSequence s_found;
    const uint32_t share = (p.a.sequences + 127) / 128, s0 = threadIdx.x < 128 ? min(p.a.sequences, threadIdx.x * share) : p.a.sequences, s1 = min(p.a.sequences, s0 + share);
    uint64_t mine = 0;
    uint32_t per_head = 0;
    for (c.u.s = s0; c.u.s < s1; ++c.u.s) {
        load_sequence<TK>(p, c.u);
        per_head = head_tiles<TK>(p, c.u);
        mine += (uint64_t)per_head * p.a.kv_heads;
    }
    uint64_t total;
    uint64_t before = scan128(mine, warps, total);
    run.length = max((uint64_t)1, few_div(total + gridDim.x - 1, gridDim.x));
    run.begin = blockIdx.x * run.length;
    run.end = min(total, run.begin + run.length);
    if (run.begin >= total) return false;
    if (run.begin >= before && run.begin < before + mine) {
        c.u.s = s0;
        if (share > 1)
            for (;; ++c.u.s) {
                load_sequence<TK>(p, c.u);
                per_head = head_tiles<TK>(p, c.u);
                const uint64_t n = (uint64_t)per_head * p.a.kv_heads;
                if (run.begin < before + n) break;
                before += n;
            }
        s_sequence = c.u.s;
        s_found = c.u.seq;
        s_per_head = per_head;
        s_at = before;
    }
    __syncthreads();
    c.u.s = s_sequence;
    c.u.seq = s_found;
    c.u.row_tiles = (c.u.seq.count * p.per.d + 15) / 16;
    per_head = s_per_head;
    const uint64_t rest = run.begin - s_at;
    c.u.kvh = (uint32_t)few_div(rest, per_head);
    uint32_t r = (uint32_t)(rest - (uint64_t)c.u.kvh * per_head);
    for (c.u.rt = 0;; ++c.u.rt) {
        unit_tiles<TK>(p, c.u);
        if (r < c.u.tiles) break;
        r -= c.u.tiles;
    }
    c.tile = r;
    c.at = run.begin;
    if (whole && c.tile) {                       // the block before has this unit
        c.at += c.u.tiles - c.tile;
        c.next_unit(p);
        if (c.at >= run.end) return false;
    }
    return true;
}
__device__ __forceinline__ bool row_sees(const PagedParams& p, int32_t at, uint32_t key) {
    return (int32_t)key <= at && (!p.a.window || key < p.a.sinks || (int64_t)key + p.a.window > at);
}
// Whether any row of the unit sees the key: what nobody sees is not looked up.
__device__ __forceinline__ bool unit_sees(const PagedParams& p, const FewUnit& u, uint32_t key) {
    return (int32_t)key <= u.last && (!p.a.window || key < p.a.sinks || (int64_t)key + p.a.window > u.first);
}

constexpr uint32_t FEW_BLOCKS = 592;             // at the most
static_assert(PAGED_COUNTERS >= FEW_BLOCKS * 4, "a counter per block");

// The rows warp + 4 k of a unit from its `parts` partial results, the first of them at `begin` (there the unit begins in the run), the others at `rest` and behind.
// What bounds it is the way to L2 and back, so loads are on their way together: all maxima and sums (a lane a part), and beside them the numerators of the
// first PARTS parts.
template <int W, int ROWS, typename T>
__device__ __forceinline__ void few_join_rows(const PagedParams& p, const FewUnit& u, uint32_t parts, const float* begin, const float* rest) {
    constexpr uint32_t ROW = W + 2, PARTS = 8 / ROWS;
    const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    // what is not there is read as the last of what is, so that no load has a condition
    auto part = [&](uint32_t i) {
        i = min(i, parts - 1);
        return i == 0 ? begin : rest + i * (2 * 16 * ROW);
    };
    uint32_t at[ROWS];
#pragma unroll
    for (int k = 0; k < ROWS; ++k) at[k] = min(warp + 4 * k, u.rows - 1) * ROW;
    float2 x[PARTS][ROWS][W / 64], v[ROWS][W / 64], st[ROWS];
    float top[ROWS], sum[ROWS], factor[ROWS];
    auto load = [&](uint32_t i) {
#pragma unroll
        for (uint32_t q = 0; q < PARTS; ++q)
#pragma unroll
            for (int k = 0; k < ROWS; ++k)
#pragma unroll
                for (int j = 0; j < W / 64; ++j) x[q][k][j] = __ldcg(reinterpret_cast<const float2*>(part(i + q) + at[k]) + j * 32 + lane);
    };
    auto load_st = [&](uint32_t i) {
#pragma unroll
        for (int k = 0; k < ROWS; ++k) st[k] = __ldcg(reinterpret_cast<const float2*>(part(i) + at[k] + W));
    };
    load_st(lane);
    load(0);
#pragma unroll
    for (int k = 0; k < ROWS; ++k) {
        top[k] = st[k].x;
        sum[k] = 0.0f;
#pragma unroll
        for (int j = 0; j < W / 64; ++j) v[k][j] = make_float2(0.0f, 0.0f);
    }
    for (uint32_t i = lane + 32; i < parts; i += 32)
#pragma unroll
        for (int k = 0; k < ROWS; ++k) top[k] = fmaxf(top[k], __ldcg(part(i) + at[k] + W));
#pragma unroll
    for (int d = 16; d > 0; d /= 2)
#pragma unroll
        for (int k = 0; k < ROWS; ++k) top[k] = fmaxf(top[k], __shfl_xor_sync(0xffffffffu, top[k], d));
    for (uint32_t i = 0; i < parts; i += PARTS) {
        if (i % 32 == 0) {
            if (i) load_st(i + lane);
#pragma unroll
            for (int k = 0; k < ROWS; ++k) {
                factor[k] = mx_ex2(st[k].x - (top[k] == -INFINITY ? 0.0f : top[k]));
                if (i + lane < parts) sum[k] = fmaf(factor[k], st[k].y, sum[k]);
            }
        }
        if (i) load(i);
#pragma unroll
        for (uint32_t q = 0; q < PARTS; ++q)
#pragma unroll
            for (int k = 0; k < ROWS; ++k) {
                const float f = __shfl_sync(0xffffffffu, factor[k], (i + q) & 31);
                if (i + q < parts)
#pragma unroll
                    for (int j = 0; j < W / 64; ++j) {
                        v[k][j].x = fmaf(f, x[q][k][j].x, v[k][j].x);
                        v[k][j].y = fmaf(f, x[q][k][j].y, v[k][j].y);
                    }
            }
    }
#pragma unroll
    for (int d = 16; d > 0; d /= 2)
#pragma unroll
        for (int k = 0; k < ROWS; ++k) sum[k] += __shfl_xor_sync(0xffffffffu, sum[k], d);
#pragma unroll
    for (int k = 0; k < ROWS; ++k) {
        const uint32_t r = warp + 4 * k;
        if (r >= u.rows) continue;
        const float inv = sum[k] == 0.0f ? 0.0f : 1.0f / sum[k];
        const uint32_t R = u.row0 + r, token = p.per.div(R), h = u.kvh * p.per.d + R - token * p.per.d;
        T* out = reinterpret_cast<T*>(p.a.out) + (uint64_t)(u.seq.start + token) * p.a.out_ld + (uint64_t)h * p.a.vdim;
#pragma unroll
        for (int j = 0; j < W / 64; ++j) {
            const uint32_t c = j * 64 + lane * 2;
            if (c < p.a.vdim) out[c] = from_f32<T>(v[k][j].x * inv);
            if (c + 1 < p.a.vdim) out[c + 1] = from_f32<T>(v[k][j].y * inv);
        }
    }
}

// Partial results of a unit joined by the block that comes last, in the order of the runs.  Layout [block][whether the unit begins in its run][16][W + 2].
template <int W, typename T>
__device__ __forceinline__ void few_join(const PagedParams& p, const FewUnit& u, uint64_t unit_at, const FewRun& run, const float* partial, uint32_t* done) {
    __shared__ uint32_t s_last;
    const uint32_t c0 = (uint32_t)few_div(unit_at, run.length), c1 = (uint32_t)few_div(unit_at + u.tiles - 1, run.length), parts = c1 - c0 + 1;
    few_sync();
    if (threadIdx.x == 0) {
        // releases what the block wrote (the barrier is before it) and acquires what the others did (a barrier is behind it)
        uint32_t before;
        asm volatile("atom.acq_rel.gpu.global.add.u32 %0, [%1], 1;" : "=r"(before) : "l"(done + c0) : "memory");
        s_last = before + 1 == parts;
        if (s_last) done[c0] = 0;
    }
    few_sync();
    if (!s_last) return;
    const float *rest = partial + (uint64_t)c0 * 2 * 16 * (W + 2), *begin = rest + 16 * (W + 2);
    if (u.rows <= 4) few_join_rows<W, 1, T>(p, u, parts, begin, rest);
    else if (u.rows <= 8) few_join_rows<W, 2, T>(p, u, parts, begin, rest);
    else few_join_rows<W, 4, T>(p, u, parts, begin, rest);
}

// Shared memory: STAGES tiles of keys and values, rows in parts of 128 bytes whose 16-byte pieces lie at (piece ^ row % 8), so that neither eight rows of a
// piece nor eight pieces of a row meet in a bank.  K and V of a tile are W * 128 bytes each: 64 keys in bf16, 32 in f32.
template <typename T, int W>
struct FewShape {
    static constexpr uint32_t KEYS = 128 / sizeof(T), PART = KEYS * 128, PARTS = W * sizeof(T) / 128, TILE = PART * PARTS;
    static constexpr uint32_t STAGES = W == 64 ? 4 : 3, RING = STAGES * 2 * TILE;
    __device__ static __forceinline__ uint32_t at(uint32_t row, uint32_t piece) { return (piece >> 3) * PART + row * 128 + (((piece ^ row) & 7) << 4); }
};
// Barriers of the ring, and what is behind them in shared memory.
template <typename T, int W>
struct FewRing {
    uint8_t* tiles;
    uint64_t *full, *empty;
    volatile int* abort_flag;
    __device__ __forceinline__ FewRing(uint8_t* raw) {
        tiles = raw + ((1024u - (smem_u32(raw) & 1023u)) & 1023u);
        full = reinterpret_cast<uint64_t*>(tiles + FewShape<T, W>::RING);
        empty = full + FewShape<T, W>::STAGES;
        abort_flag = reinterpret_cast<volatile int*>(empty + FewShape<T, W>::STAGES);
    }
};
constexpr uint32_t FEW_RING_EXTRA = 1024 + 128;      // alignment; barriers and the flag

// What the fifth warp does: tile after tile of the run into the ring.  TMA: pools are tensors {width, head, row, page}, a box is the largest power of two of rows
// that divides a page, and lane i asks for box i; a box that nobody sees, or whose page lies outside the pool, gets coordinates outside: zeros.  Else (pages
// whose rows are no multiple of 8) 16-byte copies, two or one rows a lane.
template <typename T, int W, bool TMA>
__device__ __forceinline__ void few_feed(const PagedParams& p, const CUtensorMap* map_k, const CUtensorMap* map_v, uint32_t box, const FewRun& run,
                                         FewCursor<FewShape<T, W>::KEYS> c, bool whole, const FewRing<T, W>& ring, uint64_t limit) {
    using S = FewShape<T, W>;
    const PagedAttention& a = p.a;
    const uint32_t lane = threadIdx.x & 31;
    for (uint32_t n = 0; whole ? c.at < run.end || c.tile : c.at < run.end; ++n) {
        const uint32_t stage = n % S::STAGES, key0 = c.key0();
        const uint32_t* entries = a.table + (uint64_t)c.u.s * a.table_ld;
        uint8_t* tile = ring.tiles + stage * 2 * S::TILE;
        if (TMA) {
            const uint32_t boxes = S::KEYS / box, key = key0 + lane * box;
            int32_t page = (int32_t)a.pool_pages, row = 0;
            const bool mine = lane < boxes;
            // the box's first key that may be seen, or its last
            if (mine && (int32_t)key <= c.u.last && (!a.window || key < a.sinks || (int64_t)key + box - 1 + a.window > c.u.first)) {
                const uint32_t i = p.page.div(key), entry = entries[i];
                row = (int32_t)(key - i * p.page.d);
                if (entry < a.pool_pages) page = (int32_t)entry;
                else report(a.d_status, DEV_BAD_PAGE);
            }
            if (!__all_sync(0xffffffffu, mbar_wait(ring.empty + stage, ((n / S::STAGES) & 1) ^ 1, ring.abort_flag, limit))) return;
            if (lane == 0) mbar_expect_tx(ring.full + stage, 2 * S::TILE);
            __syncwarp();
            if (mine)
#pragma unroll
                for (uint32_t part = 0; part < S::PARTS; ++part) {
                    const uint32_t dst = smem_u32(tile) + part * S::PART + lane * box * 128;
                    tma_load_4d(dst, map_k, (int32_t)(part * 128 / sizeof(T)), (int32_t)c.u.kvh, row, page, ring.full + stage);
                    tma_load_4d(dst + S::TILE, map_v, (int32_t)(part * 128 / sizeof(T)), (int32_t)c.u.kvh, row, page, ring.full + stage);
                }
        } else {
            constexpr uint32_t ROWS = S::KEYS / 32, PIECES = W * sizeof(T) / 16, PER = 16 / sizeof(T);
            const T *k[ROWS], *v[ROWS];
#pragma unroll
            for (uint32_t r = 0; r < ROWS; ++r) {
                const uint32_t key = key0 + r * 32 + lane;
                k[r] = v[r] = nullptr;
                if (!unit_sees(p, c.u, key)) continue;
                uint32_t page, row;
                if (paged_key(p, entries, key, page, row)) {
                    k[r] = reinterpret_cast<const T*>(a.k_pool) + a.k_page * page + a.k_row * row + a.k_head * c.u.kvh;
                    v[r] = reinterpret_cast<const T*>(a.v_pool) + a.v_page * page + a.v_row * row + a.v_head * c.u.kvh;
                } else {
                    report(a.d_status, DEV_BAD_PAGE);
                }
            }
            if (!__all_sync(0xffffffffu, mbar_wait(ring.empty + stage, ((n / S::STAGES) & 1) ^ 1, ring.abort_flag, limit))) return;
#pragma unroll
            for (uint32_t r = 0; r < ROWS; ++r)
#pragma unroll 8
                for (uint32_t i = 0; i < PIECES; ++i) {
                    const uint32_t dst = S::at(r * 32 + lane, i);
                    const bool k_there = k[r] && i * PER < a.dim, v_there = v[r] && i * PER < a.vdim;
                    mx_cp16(tile + dst, k_there ? k[r] + i * PER : reinterpret_cast<const T*>(a.k_pool), k_there);
                    mx_cp16(tile + S::TILE + dst, v_there ? v[r] + i * PER : reinterpret_cast<const T*>(a.v_pool), v_there);
                }
            asm volatile("cp.async.mbarrier.arrive.noinc.shared.b64 [%0];" ::"r"(smem_u32(ring.full + stage)) : "memory");
        }
        c.next(p);
    }
    if (!TMA) mx_wait<0>();
}

// The start of either kernel: barriers, the plan, the fifth warp's work.  False: nothing (more) to do for this thread.
template <typename T, int W, bool TMA>
__device__ __forceinline__ bool few_begin(const PagedParams& p, const CUtensorMap* map_k, const CUtensorMap* map_v, uint32_t box, bool whole, const FewRing<T, W>& ring,
                                          uint64_t limit, FewRun& run, FewCursor<FewShape<T, W>::KEYS>& c) {
    using S = FewShape<T, W>;
    if (threadIdx.x == 0) {
        for (uint32_t i = 0; i < S::STAGES; ++i) {
            mbar_init(ring.full + i, TMA ? 1 : 32);
            mbar_init(ring.empty + i, 4);
        }
        *ring.abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    pdl_wait();
    pdl_trigger();
    if (!few_plan<S::KEYS>(p, whole, run, c)) return false;      // with barriers of the whole block
    if (threadIdx.x < 128) return true;
    few_feed<T, W, TMA>(p, map_k, map_v, box, run, c, whole, ring, limit);
    return false;
}
// A wait that gave up: what was computed since is not to be used.  Copies that are still on their way get time to land.
__device__ __forceinline__ void few_end(const PagedParams& p, volatile int* abort_flag) {
    if (!*abort_flag) return;
    const uint64_t start = global_timer_ns();
    while (global_timer_ns() - start < 200000ull) __nanosleep(1000);
    if (threadIdx.x == 0) report(p.a.d_status, DEV_TIMEOUT);
}
// Values of a tile that some rows see and others do not: rows that nobody sees become zeros (their page may be somebody else's by now); whether one of the others
// holds infinities or NaN while the rows do not all see the same.
template <typename T, int W>
__device__ __forceinline__ bool few_odd_values(const PagedParams& p, const FewUnit& u, uint32_t key0, uint8_t* values) {
    using S = FewShape<T, W>;
    bool odd = false;
    for (uint32_t i = threadIdx.x; i < S::TILE / 16; i += 128) {
        const uint32_t row = i / (W * sizeof(T) / 16), piece = i % (W * sizeof(T) / 16);
        uint4* x = reinterpret_cast<uint4*>(values + S::at(row, piece));
        if (!unit_sees(p, u, key0 + row)) {
            *x = make_uint4(0u, 0u, 0u, 0u);
        } else if (u.first != u.last) {
            const uint4 v = *x;
            const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
            for (int e = 0; e < 4; ++e)
                odd |= sizeof(T) == 4 ? (w[e] & 0x7f800000u) == 0x7f800000u : ((((w[e] & 0x7f807f80u) + 0x00800080u) & 0x80008000u) != 0);
        }
    }
    return odd;
}

// bf16 on mma.sync: a tile is 64 keys.  Scores: a warp has 16 keys and all 16 rows; the value product: a warp has a quarter of the columns and all
// 64 keys, so that nothing is left to be added up between the warps but the sums of the weights.  Weights enter the value product as two bf16 pieces
// (16 bits): the kernel waits for memory, not for the tensor cores.  Values that are hidden from some rows of a tile may be infinities or NaN, which a weight
// of 0 does not keep out: such a tile's product is made key by key for each row.
// The rings keep 192 KB per SM on their way: four tiles at widths of 64 (three blocks per SM), three at 128 (two) and 256 (one).
constexpr uint32_t FEW_P_PITCH = 64 * 2 + 16, FEW_P_BYTES = 2 * 16 * FEW_P_PITCH;

template <int W, bool UPPER, bool TMA>
__global__ void __launch_bounds__(160, W == 64 ? 3 : W == 128 ? 2 : 1) paged_few_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
                                                        const __grid_constant__ PagedParams p, uint32_t box, float* partial, uint32_t* done, uint64_t limit) {
    using S = FewShape<bf16, W>;
    extern __shared__ uint8_t smem[];
    __shared__ __align__(16) uint8_t weights[FEW_P_BYTES];
    __shared__ float tops[64], sums[64];                                 // [4][16]
    const FewRing<bf16, W> ring(smem);
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g8 = lane >> 2, t4 = lane & 3;
    FewRun run;
    FewCursor<64> c;
    if (!few_begin<bf16, W, TMA>(p, &map_k, &map_v, box, partial == nullptr, ring, limit, run, c)) return;
    const PagedAttention& a = p.a;

    uint32_t qa[W / 16][4];
    float o[W / 32][4], m0, m1, l0, l1;
    int32_t at0, at1;                    // positions of rows g8 and g8 + 8
    uint64_t unit_at;
    auto begin_unit = [&]() {
        unit_at = c.at - c.tile;
        const int32_t base = (int32_t)c.u.seq.length - (int32_t)c.u.seq.count;
        auto place = [&](uint32_t r, uint32_t& token) {
            const uint32_t R = c.u.row0 + min(r, c.u.rows - 1);
            token = p.per.div(R);
            return c.u.kvh * p.per.d + R - token * p.per.d;
        };
        uint32_t token0, token1;
        const uint32_t h0 = place(g8, token0), h1 = place(g8 + 8, token1);
        at0 = base + (int32_t)token0;
        at1 = base + (int32_t)token1;
        const bf16* q0 = reinterpret_cast<const bf16*>(a.q) + (uint64_t)(c.u.seq.start + token0) * a.q_ld + (uint64_t)h0 * a.dim;
        const bf16* q1 = reinterpret_cast<const bf16*>(a.q) + (uint64_t)(c.u.seq.start + token1) * a.q_ld + (uint64_t)h1 * a.dim;
        auto pair = [&](const bf16* q, uint32_t col) { return col < a.dim ? *reinterpret_cast<const uint32_t*>(q + col) : 0u; };
#pragma unroll
        for (int k = 0; k < W / 16; ++k) {
            qa[k][0] = pair(q0, k * 16 + t4 * 2);
            qa[k][1] = UPPER ? pair(q1, k * 16 + t4 * 2) : 0u;
            qa[k][2] = pair(q0, k * 16 + 8 + t4 * 2);
            qa[k][3] = UPPER ? pair(q1, k * 16 + 8 + t4 * 2) : 0u;
        }
#pragma unroll
        for (int n = 0; n < W / 32; ++n) o[n][0] = o[n][1] = o[n][2] = o[n][3] = 0.0f;
        m0 = m1 = -INFINITY;
        l0 = l1 = 0.0f;
    };
    auto end_unit = [&]() {
        // sums of the weights over a row's four lanes and the four warps
        l0 += __shfl_xor_sync(0xffffffffu, l0, 1);
        l0 += __shfl_xor_sync(0xffffffffu, l0, 2);
        if (UPPER) {
            l1 += __shfl_xor_sync(0xffffffffu, l1, 1);
            l1 += __shfl_xor_sync(0xffffffffu, l1, 2);
        }
        if (t4 == 0) {
            sums[warp * 16 + g8] = l0;
            if (UPPER) sums[warp * 16 + g8 + 8] = l1;
        }
        few_sync();
        const bool all = unit_at >= run.begin && c.tile + 1 == c.u.tiles;      // c stands at the unit's last tile in this run
#pragma unroll
        for (int half = 0; half < (UPPER ? 2 : 1); ++half) {
            const uint32_t r = g8 + half * 8;
            if (r >= c.u.rows) continue;
            const float l = sums[r] + sums[16 + r] + sums[32 + r] + sums[48 + r];
            if (all) {
                const uint32_t R = c.u.row0 + r, token = p.per.div(R), h = c.u.kvh * p.per.d + R - token * p.per.d;
                const float inv = l == 0.0f ? 0.0f : 1.0f / l;
                bf16* out = reinterpret_cast<bf16*>(a.out) + (uint64_t)(c.u.seq.start + token) * a.out_ld + (uint64_t)h * a.vdim;
#pragma unroll
                for (int n = 0; n < W / 32; ++n) {
                    const uint32_t col = warp * (W / 4) + n * 8 + t4 * 2;
                    if (col < a.vdim) *reinterpret_cast<uint32_t*>(out + col) = pack_bf16x2(o[n][2 * half] * inv, o[n][2 * half + 1] * inv);
                }
            } else {
                float* dst = partial + (((uint64_t)blockIdx.x * 2 + (unit_at >= run.begin)) * 16 + r) * (W + 2);
#pragma unroll
                for (int n = 0; n < W / 32; ++n)
                    *reinterpret_cast<float2*>(dst + warp * (W / 4) + n * 8 + t4 * 2) = make_float2(o[n][2 * half], o[n][2 * half + 1]);
                if (warp == 0 && t4 == 0) {
                    dst[W] = half ? m1 : m0;
                    dst[W + 1] = l;
                }
            }
        }
        return all;
    };
    begin_unit();
    for (uint32_t n = 0;; ++n) {
        const uint32_t stage = n % S::STAGES, key0 = c.key0();
        uint8_t* tile = ring.tiles + stage * 2 * S::TILE;
        mbar_wait(ring.full + stage, (n / S::STAGES) & 1, ring.abort_flag, limit);      // given up: the run goes on without waiting
        const uint32_t sk = smem_u32(tile), sv = sk + S::TILE;
        float sc[2][4] = {}, odd[2][4] = {};
        {
            const uint32_t key = warp * 16 + (lane & 7) + (lane >> 4) * 8, piece = (lane >> 3) & 1;
#pragma unroll
            for (int k = 0; k < W / 16; k += 2) {
                uint32_t b[4], d[4];
                mx_ldsm(sk + S::at(key, k * 2 + piece), b);
                mx_ldsm(sk + S::at(key, k * 2 + 2 + piece), d);
                mx_mma(sc[0], qa[k], b[0], b[1]);
                mx_mma(sc[1], qa[k], b[2], b[3]);
                mx_mma(odd[0], qa[k + 1], d[0], d[1]);
                mx_mma(odd[1], qa[k + 1], d[2], d[3]);
            }
        }
        const bool partly = (int64_t)key0 + 63 > c.u.first || (a.window && (int64_t)key0 + a.window <= c.u.last);
        float top0 = -INFINITY, top1 = -INFINITY;
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
            for (int e = 0; e < (UPPER ? 4 : 2); ++e) {
                float v = (sc[n][e] + odd[n][e]) * p.scale_log2;
                if (partly && !row_sees(p, e < 2 ? at0 : at1, key0 + warp * 16 + n * 8 + t4 * 2 + (e & 1))) v = -INFINITY;
                sc[n][e] = v;
                if (e < 2) top0 = fmaxf(top0, v); else top1 = fmaxf(top1, v);
            }
        top0 = fmaxf(top0, __shfl_xor_sync(0xffffffffu, top0, 1));
        top0 = fmaxf(top0, __shfl_xor_sync(0xffffffffu, top0, 2));
        if (UPPER) {
            top1 = fmaxf(top1, __shfl_xor_sync(0xffffffffu, top1, 1));
            top1 = fmaxf(top1, __shfl_xor_sync(0xffffffffu, top1, 2));
        }
        if (t4 == 0) {
            tops[warp * 16 + g8] = top0;
            if (UPPER) tops[warp * 16 + g8 + 8] = top1;
        }
        few_sync();
        auto weigh = [&](int half, float& m, float& l) {
            const float* t = tops + half * 8 + g8;
            const float top = fmaxf(fmaxf(m, fmaxf(t[0], t[16])), fmaxf(t[32], t[48])), ms = top == -INFINITY ? 0.0f : top, f = mx_ex2(m - ms);
            m = top;
            float sum = 0.0f;
            uint8_t* dst = weights + (half * 8 + g8) * FEW_P_PITCH + (warp * 16 + t4 * 2) * 2;
#pragma unroll
            for (int n = 0; n < 2; ++n) {
                const float x = mx_ex2(sc[n][2 * half] - ms), y = mx_ex2(sc[n][2 * half + 1] - ms);
                sum += x + y;
                uint32_t hi, lo;
                split_bf16x2(x, y, hi, lo);
                *reinterpret_cast<uint32_t*>(dst + n * 16) = hi;
                *reinterpret_cast<uint32_t*>(dst + 16 * FEW_P_PITCH + n * 16) = lo;
            }
            l = l * f + sum;
#pragma unroll
            for (int n = 0; n < W / 32; ++n) {
                o[n][2 * half] *= f;
                o[n][2 * half + 1] *= f;
            }
        };
        weigh(0, m0, l0);
        if (UPPER) weigh(1, m1, l1);
        if (few_any(partly && few_odd_values<bf16, W>(p, c.u, key0, tile + S::TILE))) {
            for (uint32_t j = 0; j < 64; ++j) {
#pragma unroll
                for (int half = 0; half < (UPPER ? 2 : 1); ++half) {
                    if (!row_sees(p, half ? at1 : at0, key0 + j)) continue;
                    const uint8_t* w = weights + (half * 8 + g8) * FEW_P_PITCH + j * 2;
                    const float x = __bfloat162float(*reinterpret_cast<const bf16*>(w)) + __bfloat162float(*reinterpret_cast<const bf16*>(w + 16 * FEW_P_PITCH));
#pragma unroll
                    for (int n = 0; n < W / 32; ++n) {
                        const float2 v = bf16x2_to_f32(*reinterpret_cast<const uint32_t*>(tile + S::TILE + S::at(j, (warp * (W / 4) + n * 8) / 8) + t4 * 4));
                        o[n][2 * half] = fmaf(x, v.x, o[n][2 * half]);
                        o[n][2 * half + 1] = fmaf(x, v.y, o[n][2 * half + 1]);
                    }
                }
            }
        } else {
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                uint32_t hi[4], lo[4];
                const uint32_t wa = mx_smem(weights) + ((lane & 7) + ((lane >> 3) & 1) * 8) * FEW_P_PITCH + k * 32 + (lane >> 4) * 16;
                mx_ldsm(wa, hi);
                mx_ldsm(wa + 16 * FEW_P_PITCH, lo);
                if (!UPPER) hi[1] = hi[3] = lo[1] = lo[3] = 0;
#pragma unroll
                for (int n = 0; n < W / 64; ++n) {
                    uint32_t b[4];
                    mx_ldsm_t(sv + S::at(k * 16 + (lane & 7) + ((lane >> 3) & 1) * 8, (warp * (W / 4) + n * 16) / 8 + (lane >> 4)), b);
                    mx_mma(o[2 * n], hi, b[0], b[1]);
                    mx_mma(o[2 * n + 1], hi, b[2], b[3]);
                    mx_mma(o[2 * n], lo, b[0], b[1]);
                    mx_mma(o[2 * n + 1], lo, b[2], b[3]);
                }
            }
        }
        // the tile has been read (and, where rows became zeros, written: the copies that follow are another proxy's)
        if (partly) fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(ring.empty + stage);
        const bool unit_over = c.tile + 1 == c.u.tiles, run_over = partial ? c.at + 1 >= run.end : unit_over && c.at + 1 >= run.end;
        if (unit_over || run_over) {
            if (!end_unit()) few_join<W, bf16>(p, c.u, unit_at, run, partial, done);
            if (run_over) break;
        }
        c.next(p);
        if (unit_over) begin_unit();
    }
    few_end(p, ring.abort_flag);
}

// f32 on CUDA cores: a tile is 32 keys.  Scores: a thread has a key and the rows warp, warp + 4, ...; the value product: a thread has a column (two
// at widths of 256; half the keys at 64) and all rows.  RQ: rows of a warp.
// 32 sequences of up to 8192 keys, 16 / 4 heads of 128 (684 MB): 135 us = 5.1 TB/s; with 64 rows a sequence the CUDA cores bound it.
template <int W, int RQ, bool TMA>
__global__ void __launch_bounds__(160, W == 64 ? 3 : W == 128 ? 2 : 1) paged_few_f32_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
                                                            const __grid_constant__ PagedParams p, uint32_t box, float* partial, uint32_t* done, uint64_t limit) {
    using S = FewShape<float, W>;
    extern __shared__ uint8_t smem[];
    __shared__ __align__(16) float sq[RQ * 4 * W], weights[32 * 16], half_sums[W == 64 ? 64 * 16 : 1];      // weights: [32 keys][16 rows]; half_sums: [16][64]
    __shared__ float factors[16], sums[16], tops[16];
    __shared__ int32_t places[16];
    const FewRing<float, W> ring(smem);
    const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    FewRun run;
    FewCursor<32> c;
    if (!few_begin<float, W, TMA>(p, &map_k, &map_v, box, partial == nullptr, ring, limit, run, c)) return;
    const PagedAttention& a = p.a;

    constexpr int COLUMNS = W == 256 ? 2 : 1, KEYS = W == 64 ? 16 : 32;   // of a thread in the value product
    const uint32_t col = tid % W, key_first = W == 64 ? (tid / 64) * 16 : 0;
    float o[COLUMNS][RQ * 4], m[RQ], l[RQ];
    uint64_t unit_at;
    auto begin_unit = [&]() {
        unit_at = c.at - c.tile;
        few_sync();                     // the last unit's rows are done with
        const int32_t base = (int32_t)c.u.seq.length - (int32_t)c.u.seq.count;
        // all loads on their way together
        float q[RQ * 4 * W / 128];
#pragma unroll
        for (uint32_t n = 0; n < RQ * 4 * W / 128; ++n) {
            const uint32_t i = n * 128 + tid, r = i / W, x = i % W, R = c.u.row0 + min(r, c.u.rows - 1), token = p.per.div(R), h = c.u.kvh * p.per.d + R - token * p.per.d;
            q[n] = r < c.u.rows && x < a.dim ? reinterpret_cast<const float*>(a.q)[(uint64_t)(c.u.seq.start + token) * a.q_ld + (uint64_t)h * a.dim + x] : 0.0f;
            if (x == 0) places[r] = base + (int32_t)token;
        }
#pragma unroll
        for (uint32_t n = 0; n < RQ * 4 * W / 128; ++n) sq[n * 128 + tid] = q[n] * p.scale_log2;
#pragma unroll
        for (int i = 0; i < RQ * 4; ++i)
#pragma unroll
            for (int n = 0; n < COLUMNS; ++n) o[n][i] = 0.0f;
#pragma unroll
        for (int i = 0; i < RQ; ++i) {
            m[i] = -INFINITY;
            l[i] = 0.0f;
        }
    };
    auto end_unit = [&]() {
#pragma unroll
        for (int i = 0; i < RQ; ++i) {
            float sum = l[i];
#pragma unroll
            for (int d = 16; d > 0; d /= 2) sum += __shfl_xor_sync(0xffffffffu, sum, d);
            if (lane == 0) {
                sums[warp + 4 * i] = sum;
                tops[warp + 4 * i] = m[i];
            }
        }
        if (W == 64 && tid >= 64)
#pragma unroll
            for (int r = 0; r < RQ * 4; ++r) half_sums[r * 64 + col] = o[0][r];
        few_sync();
        const bool all = unit_at >= run.begin && c.tile + 1 == c.u.tiles;
        if (W != 64 || tid < 64) {
#pragma unroll
            for (int r = 0; r < RQ * 4; ++r) {
                if (r >= c.u.rows) continue;
                float* dst = partial + (((uint64_t)blockIdx.x * 2 + (unit_at >= run.begin)) * 16 + r) * (W + 2);
                float inv = 1.0f;
                if (all) {
                    const uint32_t R = c.u.row0 + r, token = p.per.div(R), h = c.u.kvh * p.per.d + R - token * p.per.d;
                    dst = reinterpret_cast<float*>(a.out) + (uint64_t)(c.u.seq.start + token) * a.out_ld + (uint64_t)h * a.vdim;
                    inv = sums[r] == 0.0f ? 0.0f : 1.0f / sums[r];
                }
#pragma unroll
                for (int n = 0; n < COLUMNS; ++n) {
                    const uint32_t x = col + n * 128;
                    const float v = W == 64 ? o[n][r] + half_sums[r * 64 + col] : o[n][r];
                    if (!all || x < a.vdim) dst[x] = v * inv;
                }
                if (!all && tid == 0) *reinterpret_cast<float2*>(dst + W) = make_float2(tops[r], sums[r]);
            }
        }
        return all;
    };
    begin_unit();
    for (uint32_t n = 0;; ++n) {
        const uint32_t stage = n % S::STAGES, key0 = c.key0();
        uint8_t* tile = ring.tiles + stage * 2 * S::TILE;
        mbar_wait(ring.full + stage, (n / S::STAGES) & 1, ring.abort_flag, limit);      // given up: the run goes on without waiting
        few_sync();                          // the rows of a new unit are there, the weights of the last tile have been read
        float dot[RQ] = {}, odd_dot[RQ] = {};
#pragma unroll 4
        for (uint32_t x = 0; x < a.dim / 4; ++x) {
            const float4 kv = *reinterpret_cast<const float4*>(tile + S::at(lane, x));
#pragma unroll
            for (int i = 0; i < RQ; ++i) {
                const float4 q = reinterpret_cast<const float4*>(sq + (warp + 4 * i) * W)[x];
                dot[i] = fmaf(q.x, kv.x, fmaf(q.y, kv.y, dot[i]));
                odd_dot[i] = fmaf(q.z, kv.z, fmaf(q.w, kv.w, odd_dot[i]));
            }
        }
#pragma unroll
        for (int i = 0; i < RQ; ++i) {
            const float x = row_sees(p, places[warp + 4 * i], key0 + lane) ? dot[i] + odd_dot[i] : -INFINITY;
            float top = fmaxf(m[i], x);
#pragma unroll
            for (int d = 16; d > 0; d /= 2) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
            const float ms = top == -INFINITY ? 0.0f : top, f = exp2f(m[i] - ms), w = exp2f(x - ms);
            m[i] = top;
            l[i] = l[i] * f + w;
            weights[lane * 16 + warp + 4 * i] = w;
            if (lane == 0) factors[warp + 4 * i] = f;
        }
        const bool partly = (int64_t)key0 + 31 > c.u.first || (a.window && (int64_t)key0 + a.window <= c.u.last);
        const bool careful = few_any(partly && few_odd_values<float, W>(p, c.u, key0, tile + S::TILE));
#pragma unroll
        for (int r = 0; r < RQ * 4; ++r)
#pragma unroll
            for (int n = 0; n < COLUMNS; ++n) o[n][r] *= factors[r];
        auto product = [&](int j, bool all) {
            float v[COLUMNS];
#pragma unroll
            for (int n = 0; n < COLUMNS; ++n) v[n] = *reinterpret_cast<const float*>(tile + S::TILE + S::at(key_first + j, (col + n * 128) / 4) + (col % 4) * 4);
            const float4* w = reinterpret_cast<const float4*>(weights + (key_first + j) * 16);
#pragma unroll
            for (int q = 0; q < RQ; ++q) {
                const float4 x = w[q];
                const float f[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (all || row_sees(p, places[4 * q + e], key0 + key_first + j))
#pragma unroll
                        for (int n = 0; n < COLUMNS; ++n) o[n][4 * q + e] = fmaf(f[e], v[n], o[n][4 * q + e]);
            }
        };
        if (careful) {
#pragma unroll 1
            for (int j = 0; j < KEYS; ++j) product(j, false);
        } else {
#pragma unroll
            for (int j = 0; j < KEYS; ++j) product(j, true);
        }
        // the tile has been read (and, where rows became zeros, written: the copies that follow are another proxy's)
        if (partly) fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(ring.empty + stage);
        const bool unit_over = c.tile + 1 == c.u.tiles, run_over = partial ? c.at + 1 >= run.end : unit_over && c.at + 1 >= run.end;
        if (unit_over || run_over) {
            if (!end_unit()) few_join<W, float>(p, c.u, unit_at, run, partial, done);
            if (run_over) break;
        }
        c.next(p);
        if (unit_over) begin_unit();
    }
    few_end(p, ring.abort_flag);
}

// ---- launch ------------------------------------------------------------------------------------------------------------------------
namespace {
// Rows (tokens x heads of a group) of a sequence up to which this kernel takes bf16 calls that the other one for many rows could take: a unit of 16 always, up to 64
// while all units find an SM each, for every unit reads the keys for itself.  us here / there, heads of 128, 4 per key/value head: one sequence of 4096 keys, 32 / 64 /
// 256 rows 19 / 31, 24 / 31, 50 / 37; 16 of 2048, 32 / 64 rows 42 / 38, 69 / 38; 64 of 1024, 64 rows 150 / 71.
// Rows are known by their bound, `chunk`: what a sequence brings stands on the device.
constexpr uint32_t FEW_ROWS = 64, FEW_UNITS = 148;

uint32_t few_width(uint32_t dim, uint32_t vdim) {
    const uint32_t w = std::max(dim, vdim);
    return w <= 64 ? 64 : w <= 128 ? 128 : 256;
}
// As many blocks as run at once: shared memory lets three (widths of 64), two or one of them on an SM.
uint32_t few_blocks(uint32_t width) { return 148 * (width == 64 ? 3 : width == 128 ? 2 : 1); }

struct FewLaunch {
    CUtensorMap k, v;
    uint32_t box, grid;      // box 0: no tensor maps
};

// Pools as tensors {width, head, row, page}; boxes of 128 bytes x `box` rows, pieces of 16 bytes exchanged as FewShape::at says.
bool few_map(CUtensorMap* map, const void* base, int dtype, uint32_t width, const PagedAttention& a, uint64_t head, uint64_t row, uint64_t page, uint32_t box) {
    const uint64_t size = dtype == TNSR_B200_F32 ? 4 : 2;
    const cuuint64_t dims[4] = {width, a.kv_heads, a.page_rows, a.pool_pages}, strides[3] = {head * size, row * size, page * size};
    const cuuint32_t boxes[4] = {(cuuint32_t)(128 / size), 1, box, 1}, ones[4] = {1, 1, 1, 1};
    return encode_fn()(map, dtype == TNSR_B200_F32 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, const_cast<void*>(base), dims, strides, boxes,
                       ones, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                       CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <typename T, int W, auto KERNEL>
int launch_few(const PagedParams& p, const FewLaunch& f, cudaStream_t stream) {
    constexpr uint32_t bytes = FewShape<T, W>::RING + FEW_RING_EXTRA;
    if (const int rc = allow_shared<KERNEL>(bytes, "paged_attention attribute")) return rc;
    float* partial = nullptr;
    uint32_t* done = nullptr;
    if (p.a.workspace) {
        done = reinterpret_cast<uint32_t*>(p.a.workspace);
        partial = reinterpret_cast<float*>(reinterpret_cast<uint8_t*>(p.a.workspace) + PAGED_COUNTERS);
    }
    launch_kernel(KERNEL, dim3(f.grid), dim3(160), bytes, stream, f.k, f.v, p, f.box, partial, done, g_wait_limit_ns.load(std::memory_order_relaxed));
    return TNSR_B200_OK;
}
template <int W, bool TMA>
int launch_few_width(const PagedParams& p, int dtype, uint32_t rows, const FewLaunch& f, cudaStream_t stream) {
    if (dtype == TNSR_B200_BF16)
        return rows > 8 ? launch_few<bf16, W, paged_few_kernel<W, true, TMA>>(p, f, stream) : launch_few<bf16, W, paged_few_kernel<W, false, TMA>>(p, f, stream);
    return rows > 8   ? launch_few<float, W, paged_few_f32_kernel<W, 4, TMA>>(p, f, stream)
           : rows > 4 ? launch_few<float, W, paged_few_f32_kernel<W, 2, TMA>>(p, f, stream)
                      : launch_few<float, W, paged_few_f32_kernel<W, 1, TMA>>(p, f, stream);
}
template <bool TMA>
int launch_few_any(const PagedParams& p, int dtype, uint32_t width, uint32_t rows, const FewLaunch& f, cudaStream_t stream) {
    return width == 64    ? launch_few_width<64, TMA>(p, dtype, rows, f, stream)
           : width == 128 ? launch_few_width<128, TMA>(p, dtype, rows, f, stream)
                          : launch_few_width<256, TMA>(p, dtype, rows, f, stream);
}
}  // namespace

uint64_t paged_attention_workspace_bytes(uint32_t dim, uint32_t vdim, int dtype) {
    const uint32_t w = few_width(dim, vdim);
    const uint64_t few = PAGED_COUNTERS + (uint64_t)few_blocks(w) * 2 * 16 * (w + 2) * 4;
    return dtype == TNSR_B200_BF16 ? std::max(few, paged_prompt_workspace_bytes(dim, vdim)) : few;
}

int launch_paged_attention(const PagedAttention& args, int dtype, cudaStream_t stream) {
    if (args.rows == 0 || args.sequences == 0) return TNSR_B200_OK;
    PagedAttention a = args;
    a.chunk = std::min(a.chunk, a.rows);             // no sequence has more
    PagedParams p;
    p.a = a;
    p.page = fast_div(a.page_rows);
    p.per = fast_div(a.heads / a.kv_heads);
    p.capacity = (uint32_t)std::min<uint64_t>((uint64_t)a.table_ld * a.page_rows, PAGED_MAX_KEYS);
    p.scale_log2 = a.scale * 1.4426950408889634f;
    if (a.window >= p.capacity) p.a.window = p.a.sinks = 0;          // as long as any sequence; smaller ones are positions, of 31 bits
    // the other kernels copy 16 bytes at a time, and write pairs of columns
    const uint32_t per = dtype == TNSR_B200_F32 ? 4 : 8;
    const uint64_t strides = (uint64_t)a.dim | a.vdim | a.k_page | a.k_row | a.k_head | a.v_page | a.v_row | a.v_head;
    const bool wide = strides % per == 0 && ((uintptr_t)a.k_pool | (uintptr_t)a.v_pool) % 16 == 0 &&
                      (a.q_ld | a.out_ld) % 2 == 0 && ((uintptr_t)a.q | (uintptr_t)a.out) % 8 == 0;
    const uint64_t rows = (uint64_t)a.chunk * p.per.d;
    int rc = TNSR_B200_OK;
    if (!wide || rows > 0x7fffffffu) {
        const dim3 grid((unsigned)ceil_div64((uint64_t)a.rows * a.heads, 4));
        if (dtype == TNSR_B200_F32) launch_kernel(paged_rows_kernel<float>, grid, dim3(128), 0, stream, p);
        else launch_kernel(paged_rows_kernel<bf16>, grid, dim3(128), 0, stream, p);
    } else if ((rows > FEW_ROWS || (rows > 16 && a.sequences * ceil_div64(rows, 16) * a.kv_heads > FEW_UNITS)) && paged_prompt_eligible(a, dtype)) {
        rc = launch_paged_prompt(p, stream);
    } else {
        const uint32_t w = few_width(a.dim, a.vdim), most = (uint32_t)std::min<uint64_t>(16, rows), keys = dtype == TNSR_B200_F32 ? 32u : 64u;
        // no more blocks than there can be tiles
        const uint64_t tiles = (uint64_t)a.sequences * a.kv_heads * ceil_div64(rows, 16) * (ceil_div(p.capacity, keys) + 1);
        FewLaunch f = {};
        f.grid = (uint32_t)std::min<uint64_t>(tiles, few_blocks(w));
        f.box = std::min(keys, a.page_rows & (0u - a.page_rows));
        const uint64_t largest = std::max({a.k_page, a.k_row, a.k_head, a.v_page, a.v_row, a.v_head}), smallest = std::min({a.k_page, a.k_row, a.k_head, a.v_page, a.v_row, a.v_head});
        // strides of a tensor map are less than 2^40 bytes, its coordinates 31 bits
        const bool tma = f.box >= 8 && smallest > 0 && largest < (1ull << 37) && a.pool_pages < 0x7fffffffu && encode_fn() != nullptr;
        if (tma) {
            if (!few_map(&f.k, a.k_pool, dtype, a.dim, a, a.k_head, a.k_row, a.k_page, f.box) ||
                !few_map(&f.v, a.v_pool, dtype, a.vdim, a, a.v_head, a.v_row, a.v_page, f.box)) {
                set_thread_error("paged_attention: tensor map encoding failed");
                return TNSR_B200_ERR_CUDA;
            }
            rc = launch_few_any<true>(p, dtype, w, most, f, stream);
        } else {
            rc = launch_few_any<false>(p, dtype, w, most, f, stream);
        }
    }
    if (rc) return rc;
    count_launch();
    return check_launch("paged_attention");
}

}  // namespace tb
