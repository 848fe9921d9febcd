// Attention over pages for many rows per sequence, on tcgen05: bf16, widths up to 128 (multiples of 8).
//
// A tile is 128 rows (as many tokens as fit, times the query heads that share a key/value head), one TMEM lane each; an item is two tiles
// of one sequence and key/value head that walk the same key blocks of 128 and take turns on the tensor cores: while one tile's
// scores are turned into weights, the other's products run.  Blocks that no row of a tile sees are left out for it, those that no row of the
// item sees are not read.
//
//   warp 0        TMA: per item the two query tiles, then blocks of keys and values into rings.  Pools are tensors {width, head, row, page}
//                 of any strides; a box is the largest power of two of rows that divides a page, lane i of the warp looks box i's page up and asks for
//                 it.  Boxes that are not wanted, or whose page lies outside the pool, get coordinates outside: zeros.
//   warp 1        one thread issues S = Q K^T (128 x 128) and O += P V (128 x W), per tile: P V of block j, then S of block j + 1.
//   warp 2        looks through the values of blocks that are seen in part, before any product has them (below).
//   warps 4-7, 8-11   softmax of tile 0 and 1, a thread per row: no exchange between threads.  The row's weights go back over its
//                 scores as bf16 (the A operand in TMEM).  O stays in TMEM through an item and is rescaled only when a row's maximum has
//                 grown by more than 2^8 since the last time (weights then are at most 2^8, sums f32); S of block j is complete only when
//                 P V of block j - 1 is, so the rescaling needs no barrier of its own.
//
// Items go round the grid, the last tokens of every sequence first (they have the most keys).  Those of the last round, fewer than blocks of the grid, are divided
// where that pays: their key blocks, one item behind the other, are cut into equal runs, a run per block of the grid.  An item whose blocks lie in several
// runs leaves per run what its rows have so far (maximum, sum, numerators in f32); the run whose part of a tile is written last joins them in the order of
// the runs.  Every block finds its items by itself from the lengths, so a captured call follows them.
//
// Values that some rows of an item see and others do not may hold infinities or NaN, which a weight of 0 does not keep out, and so may the
// rest of a last page: in blocks that are not seen by all, each row of values is looked through and such elements are zeroed before the
// product; rows that see one of them are computed once more key by key.  One warp does that for both tiles: it alone changes values, each block passes it on its way to
// the products, and its list of an item's keys is read when the item is complete.  It takes the time in which the block's scores become weights.
//
// Every wait is bounded as elsewhere: one that gives up raises the abort flag, the roles fall through and the status word is set.
//
// Bound by a tile's chain of scores, softmax and product: 4050 cycles for a pair of blocks, of which the special functions need 2050 and the products 2660.  6000 rows
// over 12000 keys, window 4096, 32 / 8 heads of 128 (404 GFLOP): 448 us = 902 TFLOP/s (485 among other work).
#include <algorithm>

#include "mixers.cuh"
#include "paged.cuh"
#include "tc_common.cuh"

namespace tb {

constexpr uint32_t PP_THREADS = 384;
constexpr uint32_t PP_ODD = 16;                      // keys with values of no finite number that an item's list holds
constexpr uint32_t PP_HALF = 128 * 128;              // 128 rows of 64 bf16

template <int W>
struct PromptShape {
    static constexpr uint32_t TILE = PP_HALF * (W / 64);                // 128 rows of W
    static constexpr uint32_t STAGES = W == 128 ? 2 : 4;
    static constexpr uint32_t PLAN = 2 * TILE + STAGES * 2 * TILE + 1024, BYTES = 1024 + PLAN;      // alignment; tiles, barriers; the plan behind them
};
constexpr uint32_t PP_BLOCKS = 148;                  // of the grid: one of an SM
constexpr uint32_t PP_ENTRIES = 4096;                // pairs of tiles (of all sequences) up to which the last round is divided: the list is in shared memory
constexpr uint32_t PP_PARTS = 4;                     // that the longest item of the last round is cut into, at the most (and one more where runs begin inside)
constexpr uint32_t PP_JOIN = 8;                      // key blocks that could be gone through in the time that a join takes
constexpr uint32_t PP_TMEM = 512;                    // scores 2 x 128, outputs 2 x W
constexpr uint32_t PP_O = 256;

constexpr uint32_t PP_IDESC_S = (1u << 4) | (1u << 7) | (1u << 10) | ((128u >> 3) << 17) | ((128u >> 4) << 24);
template <int W>
constexpr uint32_t PP_IDESC_O = (1u << 4) | (1u << 7) | (1u << 10) | (1u << 16) | (((uint32_t)W >> 3) << 17) | ((128u >> 4) << 24);

struct PromptParams {
    PagedParams p;
    uint32_t tokens;             // of a tile
    uint32_t pairs;              // items of a sequence and key/value head at the most
    uint32_t units, items;       // sequences x key/value heads; items if all are there
    uint32_t box;                // rows of a key box
    uint64_t wait_limit_ns;
    float* partial;              // divided: [block][whether the item begins in its run][2 tiles][W + 2][128 rows]; else null
    uint32_t* done;              // [block][2 tiles], zero between launches
};

// Matrix descriptors differ in their lower word only, by constants: one thread issues all products of the block, and what it computes
// between them is time that the tensor cores wait.
template <bool ACCUMULATE>
__device__ __forceinline__ void pp_mma(uint32_t d_tmem, uint32_t a_low, uint32_t b_low, uint32_t desc_high, uint32_t idesc) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t.reg .b64 a, b;\n\t"
        "mov.b64 a, {%1, %3};\n\tmov.b64 b, {%2, %3};\n\tsetp.ne.b32 p, %5, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %4, p;\n\t}"
        ::"r"(d_tmem), "r"(a_low), "r"(b_low), "r"(desc_high), "r"(idesc), "n"(ACCUMULATE ? 1 : 0)
        : "memory");
}
// The left operand in TMEM.
__device__ __forceinline__ void pp_mma_ta(uint32_t d_tmem, uint32_t a_tmem, uint32_t b_low, uint32_t desc_high, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t.reg .b64 b;\n\t"
        "mov.b64 b, {%2, %3};\n\tsetp.ne.b32 p, %5, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], b, %4, p;\n\t}"
        ::"r"(d_tmem), "r"(a_tmem), "r"(b_low), "r"(desc_high), "r"(idesc), "r"(accumulate)
        : "memory");
}
__device__ __forceinline__ void pp_st16(uint32_t taddr, const uint32_t* r) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};"
                 ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]),
                 "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]) : "memory");
}
// Behind this the values of earlier loads may be used (they pass through, so that no use of them moves ahead of the wait).
__device__ __forceinline__ void pp_ld_wait(float (&v)[128]) {
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
    for (int i = 0; i < 128; i += 16)
        asm volatile("" : "+f"(v[i]), "+f"(v[i + 1]), "+f"(v[i + 2]), "+f"(v[i + 3]), "+f"(v[i + 4]), "+f"(v[i + 5]), "+f"(v[i + 6]), "+f"(v[i + 7]),
                          "+f"(v[i + 8]), "+f"(v[i + 9]), "+f"(v[i + 10]), "+f"(v[i + 11]), "+f"(v[i + 12]), "+f"(v[i + 13]), "+f"(v[i + 14]), "+f"(v[i + 15]));
}
// 16 columns of a row, waited for.
__device__ __forceinline__ void pp_ld16(uint32_t taddr, float (&v)[16]) {
    uint32_t* r = reinterpret_cast<uint32_t*>(v);
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];\n\t"
        "tcgen05.wait::ld.sync.aligned;"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]),
          "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(taddr)
        : "memory");
}
__device__ __forceinline__ void pp_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void pp_load_3d(uint32_t dst, const CUtensorMap* map, int32_t x, int32_t y, int32_t z, uint64_t* bar) {
    asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];"
                 ::"r"(dst), "l"(map), "r"(smem_u32(bar)), "r"(x), "r"(y), "r"(z) : "memory");
}

// Two values at once.
__device__ __forceinline__ uint64_t pp_pair(float x, float y) {
    uint64_t d;
    asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "f"(x), "f"(y));
    return d;
}
__device__ __forceinline__ void pp_split(uint64_t v, float& x, float& y) { asm("mov.b64 {%0, %1}, %2;" : "=f"(x), "=f"(y) : "l"(v)); }
__device__ __forceinline__ uint64_t pp_fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
    return d;
}
__device__ __forceinline__ uint64_t pp_add2(uint64_t a, uint64_t b) {
    uint64_t d;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}
template <int N>
__device__ __forceinline__ void pp_more_registers() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N)); }
template <int N>
__device__ __forceinline__ void pp_fewer_registers() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N)); }

// Two tiles of a sequence and key/value head.
struct PromptItem {
    PagedSequence seq;
    uint32_t s, kvh, token0;             // first token of the first tile
    uint32_t tokens[2];                  // of each tile
    int32_t first[2], last[2];           // positions of a tile's first and last token
    int32_t from[2], whole[2];           // first key of the window of the tile's first row, and of its last
    int32_t high;                        // position of the item's last token
    uint32_t blocks, head_blocks, gap;   // blocks that somebody sees; those of the first keys; block of the window's first key
};
__device__ __forceinline__ uint32_t item_key0(const PromptItem& it, uint32_t j) { return (j < it.head_blocks ? j : it.gap + j - it.head_blocks) * 128; }
// Whether a row of the tile sees a key of the block; whether one of the rows of tiles t0 to t1 does not see one.
__device__ __forceinline__ bool tile_sees(const PagedParams& p, const PromptItem& it, int t, uint32_t key0) {
    return (int32_t)key0 <= it.last[t] && ((int32_t)key0 + 127 >= it.from[t] || key0 < p.a.sinks);
}
__device__ __forceinline__ bool partly_seen(const PagedParams& p, const PromptItem& it, int t0, int t1, uint32_t key0) {
    return (int32_t)key0 + 127 > it.first[t0] || ((int32_t)key0 < it.whole[t1] && key0 + 128 > p.a.sinks);
}

// Tiles 2 pair and 2 pair + 1 of a sequence and key/value head; false: there are no such rows.
__device__ __forceinline__ bool prompt_item(const PromptParams& prm, uint32_t s, uint32_t kvh, uint32_t pair, PromptItem& it) {
    const PagedParams& p = prm.p;
    it.s = s;
    it.kvh = kvh;
    it.seq = paged_sequence(p, it.s);
    it.token0 = pair * 2 * prm.tokens;
    if (it.token0 >= it.seq.count) return false;
    const uint32_t left = it.seq.count - it.token0;
    it.tokens[0] = min(left, prm.tokens);
    it.tokens[1] = min(left - it.tokens[0], prm.tokens);
    const int32_t base = (int32_t)it.seq.length - (int32_t)it.seq.count;
    it.first[0] = base + (int32_t)it.token0;
    it.last[0] = it.first[0] + (int32_t)it.tokens[0] - 1;
    it.first[1] = it.last[0] + 1;
    it.last[1] = it.high = it.last[0] + (int32_t)it.tokens[1];
    const int32_t window = (int32_t)min(p.a.window, 0x7fffffffu);
#pragma unroll
    for (int t = 0; t < 2; ++t) {
        it.from[t] = window && it.first[t] >= window ? it.first[t] - window + 1 : 0;
        it.whole[t] = window && it.last[t] >= window ? it.last[t] - window + 1 : 0;
    }
    if (it.tokens[1] == 0) it.last[1] = -1;          // sees nothing
    it.head_blocks = it.gap = it.blocks = 0;
    if (it.high < 0) return true;
    it.gap = (uint32_t)it.from[0] / 128;
    it.head_blocks = min((min(p.a.sinks, (uint32_t)it.high + 1) + 127) / 128, it.gap);
    it.blocks = it.head_blocks + (uint32_t)it.high / 128 - it.gap + 1;
    return true;
}
// The last block of [j0, j1) that a tile sees, + 1; 0: none.
__device__ __forceinline__ uint32_t last_seen(const PagedParams& p, const PromptItem& it, int t, uint32_t j0, uint32_t j1) {
    uint32_t j = it.last[t] < 0 ? 0u : it.head_blocks + (uint32_t)it.last[t] / 128 - it.gap + 1;
    if (j0 == 0 && j1 == it.blocks) return j;
    j = min(j, j1);
    while (j > j0 && !tile_sees(p, it, t, item_key0(it, j - 1))) --j;
    return j > j0 ? j : 0u;
}
// In shared memory: which items there are, and what becomes of the last round's.
struct PromptPlan {
    uint32_t whole;                  // items below this number are taken whole, every gridDim.x-th one
    uint32_t divided;                // number of the first item of the last round
    uint32_t first, length, end;     // the block's run: its first item (of the last round), key blocks of a run, where it ends
    uint32_t most;                   // key blocks of the longest of them
    uint32_t before[PP_BLOCKS];      // key blocks before an item of the last round
    uint32_t entries[PP_ENTRIES];    // pairs of tiles that are there: (pairs - 1 - pair) * sequences + sequence
};

// A block's way through the work.  Undivided: items by number, those that are not there passed over.
template <bool DIVIDED>
struct PromptWalk {
    uint32_t next;
    __device__ __forceinline__ PromptWalk(const PromptPlan&) : next(blockIdx.x) {}
    // key blocks of the item that are this block's
    __device__ __forceinline__ uint32_t begin() const { return 0; }
    __device__ __forceinline__ uint32_t end(const PromptItem& it) const { return it.blocks; }
    __device__ __forceinline__ bool more(const PromptParams& prm, const PromptPlan&) const { return next < prm.items; }
    __device__ __forceinline__ bool step(const PromptParams& prm, const PromptPlan&, PromptItem& it) {
        const uint32_t row = next / prm.units, rest = next - row * prm.units;
        next += gridDim.x;
        return prompt_item(prm, rest / prm.p.a.kv_heads, rest % prm.p.a.kv_heads, prm.pairs - 1 - row, it);
    }
};
// Divided: whole items by their number among those that are there, then the run.
template <>
struct PromptWalk<true> {
    uint32_t number, at;             // whole items: the next one; then the next key block of the run
    uint32_t j0, j1;
    __device__ __forceinline__ uint32_t begin() const { return j0; }
    __device__ __forceinline__ uint32_t end(const PromptItem& it) const { return it.blocks ? j1 : 0u; }
    __device__ __forceinline__ PromptWalk(const PromptPlan& plan) : number(blockIdx.x), at(plan.length * blockIdx.x), j0(0), j1(0) {}
    __device__ __forceinline__ bool more(const PromptParams&, const PromptPlan& plan) const { return number < plan.whole || at < plan.end; }
    // the next item; false: it is not there
    __device__ __forceinline__ bool step(const PromptParams& prm, const PromptPlan& plan, PromptItem& it) {
        const PagedParams& p = prm.p;
        if (number >= plan.whole) {
            if (at == plan.length * blockIdx.x) number = plan.divided + plan.first;
        }
        const uint32_t entry = number / p.a.kv_heads, e = plan.entries[entry], row = e / p.a.sequences;
        prompt_item(prm, e - row * p.a.sequences, number - entry * p.a.kv_heads, prm.pairs - 1 - row, it);
        j0 = 0;
        j1 = it.blocks;
        if (number < plan.whole) {
            number += gridDim.x;
            return true;
        }
        const uint32_t begin = plan.before[number - plan.divided];
        j0 = at - begin;
        j1 = min(max(it.blocks, 1u), plan.end - begin);
        at = begin + j1;
        ++number;
        return true;
    }
};

// Exclusive prefix sum over the block.
__device__ __forceinline__ uint32_t prompt_scan(uint32_t v, uint32_t* warps, uint32_t& total) {
    const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    uint32_t x = v;
#pragma unroll
    for (int d = 1; d < 32; d *= 2) {
        const uint32_t y = __shfl_up_sync(0xffffffffu, x, d);
        if (lane >= d) x += y;
    }
    if (lane == 31) warps[warp] = x;
    __syncthreads();
    uint32_t before = x - v;
    total = 0;
#pragma unroll
    for (uint32_t w = 0; w < PP_THREADS / 32; ++w) {
        if (w < warp) before += warps[w];
        total += warps[w];
    }
    __syncthreads();
    return before;
}

// Which items there are, and this block's run of those of the last round.
__device__ __forceinline__ void prompt_plan(const PromptParams& prm, PromptPlan& plan, uint32_t* warps) {
    const PagedParams& p = prm.p;
    const uint32_t all = p.a.sequences * prm.pairs, share = (all + PP_THREADS - 1) / PP_THREADS;
    const uint32_t e0 = min(all, threadIdx.x * share), e1 = min(all, e0 + share);
    PromptItem it;
    uint32_t total = all;
    if (p.a.row_starts) {
        uint32_t mine = 0;
        for (uint32_t e = e0; e < e1; ++e) mine += prompt_item(prm, e % p.a.sequences, 0, prm.pairs - 1 - e / p.a.sequences, it);
        uint32_t at = prompt_scan(mine, warps, total);
        for (uint32_t e = e0; e < e1; ++e)
            if (prompt_item(prm, e % p.a.sequences, 0, prm.pairs - 1 - e / p.a.sequences, it)) plan.entries[at++] = e;
    } else {
        for (uint32_t e = threadIdx.x; e < all; e += PP_THREADS) plan.entries[e] = e;
    }
    if (threadIdx.x == 0) plan.most = 0;
    __syncthreads();
    const uint32_t items = total * p.a.kv_heads, left = items % gridDim.x, divided = items - left;
    uint32_t weight = 0, blocks;
    if (threadIdx.x < left) {
        const uint32_t number = divided + threadIdx.x, e = plan.entries[number / p.a.kv_heads];
        prompt_item(prm, e % p.a.sequences, 0, prm.pairs - 1 - e / p.a.sequences, it);
        weight = max(it.blocks, 1u);                  // rows that see nothing become zeros
        atomicMax(&plan.most, weight);
    }
    const uint32_t before = prompt_scan(weight, warps, blocks);
    // a join reads all parts: no more than some of an item
    const uint32_t length = max((plan.most + PP_PARTS - 1) / PP_PARTS, (blocks + gridDim.x - 1) / gridDim.x), begin = length * blockIdx.x;
    const bool pays = plan.most > length + PP_JOIN;
    if (threadIdx.x < left) {
        plan.before[threadIdx.x] = before;
        if (begin >= before && begin < before + weight) plan.first = threadIdx.x;
    }
    if (threadIdx.x == 0) {
        plan.length = length;
        plan.divided = divided;
        plan.whole = pays ? divided : items;
        plan.end = pays ? min(begin + length, blocks) : 0u;
    }
    __syncthreads();
}

template <int W, bool DIVIDED>
__global__ void __launch_bounds__(PP_THREADS, 1)
paged_prompt_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
                    const __grid_constant__ PromptParams prm) {
    using S = PromptShape<W>;
    constexpr uint32_t STAGES = S::STAGES, HALVES = W / 64;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
    uint8_t* q_tiles = smem;                                   // [2]
    uint8_t* k_ring = smem + 2 * S::TILE;                      // [STAGES]
    uint8_t* v_ring = k_ring + STAGES * S::TILE;
    uint64_t* bars = reinterpret_cast<uint64_t*>(v_ring + STAGES * S::TILE);
    uint64_t *q_full = bars, *q_empty = bars + 2, *s_full = bars + 4, *p_full = bars + 6, *o_full = bars + 8;       // a tile each
    uint64_t *met = bars + 10;                                 // a tile each: its warps wait for one another when they join
    uint64_t *listed = bars + 12, *read = bars + 14;           // items of even and odd number: their list is complete; all have read it
    uint64_t *k_full = bars + 16, *k_empty = k_full + STAGES, *v_full = k_empty + STAGES, *v_empty = v_full + STAGES, *v_clean = v_empty + STAGES;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(v_clean + STAGES);
    volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
    uint32_t* odd_count = tmem_slot + 2;                       // [2]: of the lists
    uint32_t* odd_keys = odd_count + 2;                        // [2][PP_ODD]
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const PagedParams& p = prm.p;
    const uint64_t limit = prm.wait_limit_ns;

    if (threadIdx.x == 0) {
        for (int t = 0; t < 2; ++t) {
            mbar_init(q_full + t, 1);
            mbar_init(q_empty + t, 1);
            mbar_init(s_full + t, 1);
            mbar_init(p_full + t, 4);
            mbar_init(o_full + t, 1);
            mbar_init(met + t, 4);
            mbar_init(listed + t, 1);
            mbar_init(read + t, 8);
        }
        for (uint32_t i = 0; i < STAGES; ++i) {
            mbar_init(k_full + i, 1);
            mbar_init(k_empty + i, 1);
            mbar_init(v_full + i, 1);
            mbar_init(v_empty + i, 1);
            mbar_init(v_clean + i, 1);
        }
        *abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    pdl_wait();
    pdl_trigger();
    __shared__ volatile uint32_t join_now[2];
    PromptPlan& plan = *reinterpret_cast<PromptPlan*>(smem + S::PLAN);
    if constexpr (DIVIDED) {
        __shared__ uint32_t warps[PP_THREADS / 32];
        prompt_plan(prm, plan, warps);
    }
    PromptWalk<DIVIDED> walk(plan);
    if (warp == 1) {
        tmem_alloc(tmem_slot, PP_TMEM);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    PromptItem it;

    auto teardown = [&]() {
        tc_fence_before();
        __syncthreads();
        if (*abort_flag) {
            // copies that are still on their way get time to land before the shared memory is somebody else's
            const uint64_t start = global_timer_ns();
            while (global_timer_ns() - start < 200000ull) __nanosleep(1000);
            if (threadIdx.x == 0) report(p.a.d_status, DEV_TIMEOUT);
            __syncthreads();
        }
        if (warp == 1) {
            tc_fence_after();
            tmem_dealloc(tmem, PP_TMEM);
        }
    };
    // The softmax warps' registers come from the others: 4 x 32 x 104 + 8 x 32 x 200 (or 88 and 208) are no more than the 12 x 32 x 168 that the block starts with.
    // The two kinds of warps do not meet again, or all would be held to the smaller number.
    if (warp < 4) {
        pp_fewer_registers<W == 64 ? 88 : 104>();
    if (warp == 0) {
        // ---------------- copies ----------------
        uint32_t blocks = 0, used[2] = {0, 0};       // key blocks so far; items so far that had rows in a tile
        bool ok = true;
        while (ok && walk.more(prm, plan)) {
            if (!walk.step(prm, plan, it) || it.blocks == 0) continue;
            const uint32_t boxes = 128 / prm.box;
            const uint32_t j0 = walk.begin(), j1 = walk.end(it);
            for (uint32_t j = j0; ok && j < j1; ++j, ++blocks) {
                const uint32_t stage = blocks % STAGES, parity = ((blocks / STAGES) & 1) ^ 1;
                const uint32_t key = item_key0(it, j) + lane * prm.box;
                int32_t page = (int32_t)p.a.pool_pages, row = 0;          // outside: zeros
                if (lane < boxes && (int32_t)key <= it.high && (key < p.a.sinks || (int32_t)(key + prm.box) > it.from[0])) {
                    const uint32_t i = p.page.div(key), entry = p.a.table[(uint64_t)it.s * p.a.table_ld + i];
                    row = (int32_t)(key - i * p.page.d);
                    if (entry < p.a.pool_pages) page = (int32_t)entry;
                    else report(p.a.d_status, DEV_BAD_PAGE);
                }
                ok = mbar_wait(k_empty + stage, parity, abort_flag, limit);
                ok = __all_sync(0xffffffffu, ok);
                if (!ok) break;
                if (lane == 0) mbar_expect_tx(k_full + stage, S::TILE);
                __syncwarp();
                if (lane < boxes)
#pragma unroll
                    for (uint32_t h = 0; h < HALVES; ++h)
                        tma_load_4d(smem_u32(k_ring) + stage * S::TILE + h * PP_HALF + lane * prm.box * 128, &map_k, (int32_t)(h * 64), (int32_t)it.kvh, row, page,
                                   k_full + stage);
                if (j == j0) {
                    for (int t = 0; t < 2 && ok; ++t) {
                        if (!it.tokens[t]) continue;
                        ok = used[t] == 0 || mbar_wait(q_empty + t, (used[t] - 1) & 1, abort_flag, limit);
                        ++used[t];
                        ok = __all_sync(0xffffffffu, ok);
                        if (ok && lane == 0) {
                            mbar_expect_tx(q_full + t, HALVES * prm.tokens * p.per.d * 128);
                            for (uint32_t h = 0; h < HALVES; ++h)
                                pp_load_3d(smem_u32(q_tiles) + t * S::TILE + h * PP_HALF, &map_q, (int32_t)(h * 64), (int32_t)(it.kvh * p.per.d),
                                           (int32_t)(it.seq.start + it.token0 + t * prm.tokens), q_full + t);
                        }
                    }
                    if (!ok) break;
                }
                ok = mbar_wait(v_empty + stage, parity, abort_flag, limit);
                ok = __all_sync(0xffffffffu, ok);
                if (!ok) break;
                if (lane == 0) mbar_expect_tx(v_full + stage, S::TILE);
                __syncwarp();
                if (lane < boxes)
#pragma unroll
                    for (uint32_t h = 0; h < HALVES; ++h)
                        tma_load_4d(smem_u32(v_ring) + stage * S::TILE + h * PP_HALF + lane * prm.box * 128, &map_v, (int32_t)(h * 64), (int32_t)it.kvh, row, page,
                                   v_full + stage);
            }
        }
    } else if (warp == 1) {
        // ---------------- products ----------------
        if (lane == 0) {
            uint32_t blocks = 0, used[2] = {0, 0}, seen[2] = {0, 0};     // key blocks; items; blocks of a tile so far
            const uint64_t kmajor = make_kmajor_sw128_desc(0), mnmajor = make_mnmajor_sw128_desc(0, PP_HALF, 1024);
            const uint32_t k_high = (uint32_t)(kmajor >> 32), v_high = (uint32_t)(mnmajor >> 32);
            const uint32_t q_low = (uint32_t)kmajor + (smem_u32(q_tiles) >> 4), k_low = (uint32_t)kmajor + (smem_u32(k_ring) >> 4),
                           v_low = (uint32_t)mnmajor + (smem_u32(v_ring) >> 4);
            auto issue_s = [&](int t, uint32_t stage) {
                const uint32_t a = q_low + t * (S::TILE >> 4), b = k_low + stage * (S::TILE >> 4);
#pragma unroll
                for (uint32_t h = 0; h < HALVES; ++h)
#pragma unroll
                    for (uint32_t kk = 0; kk < 4; ++kk) {
                        if (h == 0 && kk == 0) pp_mma<false>(tmem + t * 128, a, b, k_high, PP_IDESC_S);
                        else pp_mma<true>(tmem + t * 128, a + h * (PP_HALF >> 4) + kk * 2, b + h * (PP_HALF >> 4) + kk * 2, k_high, PP_IDESC_S);
                    }
                umma_commit(s_full + t);
            };
            bool ok = true;
            while (ok && walk.more(prm, plan)) {
                if (!walk.step(prm, plan, it) || it.blocks == 0) continue;
                const uint32_t j0 = walk.begin(), j1 = walk.end(it);
                // behind the scores of the last block that a tile sees its queries may change, behind its product the output is complete; a tile
                // that sees nothing gives its queries back with the item's first block
                const uint32_t last[2] = {last_seen(p, it, 0, j0, j1), last_seen(p, it, 1, j0, j1)};
                uint32_t accumulate[2] = {0, 0};
                for (int t = 0; t < 2 && ok; ++t)
                    if (it.tokens[t]) {
                        ok = mbar_wait(q_full + t, used[t] & 1, abort_flag, limit);
                        ++used[t];
                    }
                if (!ok) break;
                auto scores = [&](uint32_t j, int t, bool sees, uint32_t stage) {
                    if (sees) issue_s(t, stage);
                    if (it.tokens[t] && j + 1 == max(last[t], j0 + 1)) umma_commit(q_empty + t);
                };
                uint32_t stage = blocks % STAGES, parity = (blocks / STAGES) & 1, key0 = item_key0(it, j0);
                bool sees[2] = {tile_sees(p, it, 0, key0), tile_sees(p, it, 1, key0)};
                if (!mbar_wait(k_full + stage, parity, abort_flag, limit)) break;
                tc_fence_after();
                scores(j0, 0, sees[0], stage);
                scores(j0, 1, sees[1], stage);
                umma_commit(k_empty + stage);
                for (uint32_t j = j0; j < j1; ++j) {
                    const bool more = j + 1 < j1;
                    const uint32_t next = stage + 1 == STAGES ? 0 : stage + 1, next_parity = next ? parity : parity ^ 1;
                    bool then[2] = {false, false};
                    if (more) {
                        key0 = item_key0(it, j + 1);
                        then[0] = tile_sees(p, it, 0, key0);
                        then[1] = tile_sees(p, it, 1, key0);
                        ok = mbar_wait(k_full + next, next_parity, abort_flag, limit);
                    }
                    ok = ok && mbar_wait(v_full + stage, parity, abort_flag, limit) && mbar_wait(v_clean + stage, parity, abort_flag, limit);
                    if (!ok) break;
                    const uint32_t v = v_low + stage * (S::TILE >> 4);
#pragma unroll
                    for (int t = 0; t < 2; ++t) {
                        if (sees[t]) {
                            ok = ok && mbar_wait(p_full + t, seen[t] & 1, abort_flag, limit);
                            if (!ok) break;
                            ++seen[t];
                            tc_fence_after();
                            pp_mma_ta(tmem + PP_O + t * W, tmem + t * 128, v, v_high, PP_IDESC_O<W>, accumulate[t]);
#pragma unroll
                            for (uint32_t kk = 1; kk < 8; ++kk)
                                pp_mma_ta(tmem + PP_O + t * W, tmem + t * 128 + kk * 8, v + kk * 128, v_high, PP_IDESC_O<W>, 1);
                            accumulate[t] = 1;
                            if (j + 1 == last[t]) umma_commit(o_full + t);
                        }
                        if (more) scores(j + 1, t, then[t], next);
                    }
                    if (!ok) break;
                    umma_commit(v_empty + stage);
                    if (more) umma_commit(k_empty + next);
                    sees[0] = then[0];
                    sees[1] = then[1];
                    stage = next;
                    parity = next_parity;
                }
                blocks += j1 - j0;
            }
        }
    } else if (warp == 2) {
        // ---------------- values of no finite number ----------------
        uint32_t blocks = 0, number = 0;             // key blocks; items so far
        auto wait = [&](uint64_t* bar, uint32_t parity) { return __all_sync(0xffffffffu, mbar_wait(bar, parity, abort_flag, limit)); };
        bool ok = true;
        while (ok && walk.more(prm, plan)) {
            if (!walk.step(prm, plan, it) || it.blocks == 0) continue;
            const uint32_t j0 = walk.begin(), j1 = walk.end(it), slot = number & 1;
            // the list was that of the item before the last one
            if (number >= 2 && !wait(read + slot, ((number >> 1) - 1) & 1)) break;
            uint32_t count = 0;
            bool sees[2] = {false, false};
            for (uint32_t j = j0; j < j1; ++j, ++blocks) {
                const uint32_t stage = blocks % STAGES, key0 = item_key0(it, j);
                sees[0] |= tile_sees(p, it, 0, key0);
                sees[1] |= tile_sees(p, it, 1, key0);
                ok = wait(v_full + stage, (blocks / STAGES) & 1);
                if (!ok) break;
                if (partly_seen(p, it, 0, it.tokens[1] ? 1 : 0, key0)) {
                    // a row a lane, four times
                    for (uint32_t row = lane; row < 128; row += 32) {
                        uint8_t* v_row = v_ring + stage * S::TILE + row * 128;
                        // the order of the pieces by lane: neighbours read other banks.  An exponent of ones carries into the sign's place.
                        uint32_t ones = 0;
#pragma unroll
                        for (uint32_t i = 0; i < 8 * HALVES; ++i) {
                            const uint4 x = *reinterpret_cast<const uint4*>(v_row + (i / 8) * PP_HALF + ((i + lane) & 7) * 16);
                            ones |= ((x.x & 0x7f807f80u) + 0x00800080u) | ((x.y & 0x7f807f80u) + 0x00800080u) | ((x.z & 0x7f807f80u) + 0x00800080u) |
                                    ((x.w & 0x7f807f80u) + 0x00800080u);
                        }
                        const bool found = ones & 0x80008000u;
                        if (found) {
#pragma unroll 1
                            for (uint32_t i = 0; i < 32 * HALVES; ++i) {
                                uint32_t* x = reinterpret_cast<uint32_t*>(v_row + (i / 32) * PP_HALF) + i % 32;
                                const uint32_t v = *x, odd = ((v & 0x7f807f80u) + 0x00800080u) & 0x80008000u;
                                if (odd) *x = v & ~((odd & 0x8000u ? 0xffffu : 0u) | (odd & 0x80000000u ? 0xffff0000u : 0u));
                            }
                        }
                        __syncwarp();
                        const uint32_t key = key0 + row;
                        const bool note = found && (int32_t)key <= it.high && ((int32_t)key >= it.from[0] || key < p.a.sinks);
                        const uint32_t notes = __ballot_sync(0xffffffffu, note), place = count + __popc(notes & ((1u << lane) - 1));
                        if (note && place < PP_ODD) odd_keys[slot * PP_ODD + place] = key;
                        count += __popc(notes);
                    }
                    fence_proxy_async_smem();
                }
                __syncwarp();
                if (lane == 0) mbar_arrive(v_clean + stage);
            }
            if (!ok) break;
            if (lane == 0) odd_count[slot] = count;
            __syncwarp();
            if (lane == 0) {
                mbar_arrive(listed + slot);
                // for the warps of a tile that sees nothing here, which pass the item over
                for (int n = (sees[0] ? 0 : 4) + (sees[1] ? 0 : 4); n > 0; --n) mbar_arrive(read + slot);
            }
            ++number;
        }
    }
    teardown();
    return;
    }
    pp_more_registers<W == 64 ? 208 : 200>();
    {
        // ---------------- softmax ----------------
        const int t = (int)(warp - 4) >> 2;
        const uint32_t quarter = warp & 3, row = quarter * 32 + lane;
        const uint32_t s_addr = tmem + t * 128 + ((quarter * 32u) << 16), o_addr = tmem + PP_O + t * W + ((quarter * 32u) << 16);
        const uint32_t my_token = p.per.div(row), my_head = row - my_token * p.per.d;
        uint32_t seen = 0, outputs = 0, number = 0, meets = 0;      // blocks of the tile; its outputs; items with keys; turns of `met` so far
        bool ok = true;
        // a warp gives up as a whole
        auto wait = [&](uint64_t* bar, uint32_t parity) { return __all_sync(0xffffffffu, mbar_wait(bar, parity, abort_flag, limit)); };
        while (ok && walk.more(prm, plan)) {
            if (!walk.step(prm, plan, it)) continue;
            const uint32_t j0 = walk.begin(), j1 = walk.end(it);
            if (!it.tokens[t]) {
                if (it.blocks) ++number;
                continue;
            }
            // Whether the row (`mine`) sees a key whose values must not be multiplied by 0: by the item's list, once it is complete.  For warps that have waited for
            // products of this item, so that no earlier turn of the barrier is taken for this one.
            auto odd_in_sight = [&](bool mine, int32_t at) {
                const uint32_t slot = number & 1;
                if (!wait(listed + slot, (number >> 1) & 1)) ok = false;
                const uint32_t count = *(volatile uint32_t*)(odd_count + slot);
                bool odd = count > PP_ODD;
                if (mine)
                    for (uint32_t i = 0; i < min(count, PP_ODD); ++i) {
                        const uint32_t key = *(volatile uint32_t*)(odd_keys + slot * PP_ODD + i);
                        odd |= (int32_t)key <= at && (!p.a.window || key < p.a.sinks || (int64_t)key + p.a.window > at);
                    }
                __syncwarp();
                if (lane == 0) mbar_arrive(read + slot);
                return odd && mine;
            };
            const int32_t at = it.first[t] + (int32_t)min(my_token, it.tokens[t] - 1);
            const int32_t lowest = p.a.window ? at - (int32_t)min(p.a.window, 0x7fffffffu) + 1 : 0;
            float m = -INFINITY, l = 0.0f;
            bool any = false;
            for (uint32_t j = j0; j < j1; ++j) {
                const uint32_t key0 = item_key0(it, j);
                if (!tile_sees(p, it, t, key0)) continue;
                any = true;
                if (!wait(s_full + t, seen & 1)) { ok = false; break; }
                ++seen;
                tc_fence_after();
                __syncwarp();
                float v[128];
#pragma unroll
                for (int c = 0; c < 4; ++c) tmem_ld32(s_addr + c * 32, v + c * 32);
                pp_ld_wait(v);
                if (partly_seen(p, it, t, t, key0)) {
                    // one edge or the other; both and the first keys only where they meet in a block
                    const int32_t high = at - (int32_t)key0, low = lowest - (int32_t)key0, head = (int32_t)min(p.a.sinks, 0x7fffffffu) - (int32_t)key0;
                    if ((int32_t)key0 >= it.whole[t]) {
#pragma unroll
                        for (int i = 0; i < 128; ++i)
                            if (i > high) v[i] = -INFINITY;
                    } else if ((int32_t)key0 + 127 <= it.first[t] && head <= 0) {
#pragma unroll
                        for (int i = 0; i < 128; ++i)
                            if (i < low) v[i] = -INFINITY;
                    } else {
#pragma unroll
                        for (int i = 0; i < 128; ++i)
                            if (i > high || (i < low && i >= head)) v[i] = -INFINITY;
                    }
                }
                float top4[4] = {m, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                for (int i = 0; i < 128; i += 8)
#pragma unroll
                    for (int k = 0; k < 4; ++k) top4[k] = fmaxf(fmaxf(top4[k], v[i + 2 * k]), v[i + 2 * k + 1]);
                const float top = fmaxf(fmaxf(top4[0], top4[1]), fmaxf(top4[2], top4[3]));
                // `m` stays while weights do not grow past 2^8
                float f = 1.0f;
                if (m == -INFINITY) {
                    m = top;
                } else if ((top - m) * p.scale_log2 > 8.0f) {
                    f = mx_ex2((m - top) * p.scale_log2);
                    m = top;
                }
                if (__any_sync(0xffffffffu, f != 1.0f)) {
                    l *= f;
#pragma unroll
                    for (int c = 0; c < W / 16; ++c) {
                        float o[16];
                        pp_ld16(o_addr + c * 16, o);
#pragma unroll
                        for (int i = 0; i < 16; ++i) o[i] *= f;
                        pp_st16(o_addr + c * 16, reinterpret_cast<const uint32_t*>(o));
                    }
                }
                const float neg = m == -INFINITY ? 0.0f : -m * p.scale_log2;
                const uint64_t scale2 = pp_pair(p.scale_log2, p.scale_log2), neg2 = pp_pair(neg, neg);
                uint64_t sums[2] = {0, 0};
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    uint32_t packed[16];
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        float x, y;
                        pp_split(pp_fma2(pp_pair(v[c * 32 + 2 * i], v[c * 32 + 2 * i + 1]), scale2, neg2), x, y);
                        x = mx_ex2(x);
                        y = mx_ex2(y);
                        sums[i & 1] = pp_add2(sums[i & 1], pp_pair(x, y));
                        packed[i] = pack_bf16x2(x, y);
                    }
                    pp_st16(s_addr + c * 16, packed);
                }
                float sum_x, sum_y;
                pp_split(pp_add2(sums[0], sums[1]), sum_x, sum_y);
                l += sum_x + sum_y;
                pp_st_wait();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(p_full + t);
            }
            if (!ok) break;
            if (any) {
                if (!wait(o_full + t, outputs & 1)) { ok = false; break; }
                ++outputs;
                tc_fence_after();
            }
            bool mine = my_token < it.tokens[t], odd = any && odd_in_sight(mine, at);
            if (!ok) break;
            if (it.blocks) ++number;
            mine &= !odd;
            bf16* out = reinterpret_cast<bf16*>(p.a.out) + (uint64_t)(it.seq.start + it.token0 + t * prm.tokens + my_token) * p.a.out_ld +
                        (uint64_t)(it.kvh * p.per.d + my_head) * p.a.vdim;
            bool joined = false;                     // or left to be
            if constexpr (DIVIDED) {
                joined = j0 != 0 || j1 < it.blocks;
                if (joined) {
                    // in part: the row's maximum (+inf: to be computed once more), sum and numerators
                    float* dst = prm.partial + (((uint64_t)blockIdx.x * 2 + (j0 == 0)) * 2 + t) * 128 * (W + 2) + row;
#pragma unroll
                    for (int c = 0; c < W / 16; ++c) {
                        float o[16];
                        if (!any) break;
                        pp_ld16(o_addr + c * 16, o);
#pragma unroll
                        for (int i = 0; i < 16; ++i) dst[(c * 16 + i) * 128] = o[i];
                    }
                    dst[W * 128] = odd ? INFINITY : m * p.scale_log2;
                    dst[(W + 1) * 128] = l;
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(met + t);
                    if (!wait(met + t, meets++ & 1)) { ok = false; break; }
                    const uint32_t item_at = plan.before[walk.number - 1 - plan.divided], c0 = item_at / plan.length,
                                   parts = (item_at + it.blocks - 1) / plan.length - c0 + 1;
                    if (row == 0) {
                        __threadfence();             // with the barriers before and behind it, for all of the tile
                        const bool last = atomicAdd(prm.done + c0 * 2 + t, 1u) + 1 == parts;
                        if (last) prm.done[c0 * 2 + t] = 0;
                        __threadfence();
                        join_now[t] = last;
                    }
                    __syncwarp();
                    if (lane == 0) mbar_arrive(met + t);
                    if (!wait(met + t, meets++ & 1)) { ok = false; break; }
                    if (!join_now[t]) continue;
                    const bool there = my_token < it.tokens[t];
                    const float* tile = prm.partial + ((uint64_t)c0 * 4 + t) * 128 * (W + 2) + row;
                    auto part = [&](uint32_t i) {
                        i = min(i, parts - 1);
                        return tile + ((uint64_t)i * 2 + (i == 0)) * 2 * 128 * (W + 2);
                    };
                    float factor[PP_PARTS + 1], top = -INFINITY, sum = 0.0f;
                    bool known[PP_PARTS + 1];                 // the row saw something in the part: else there is no more of it than its maximum
#pragma unroll
                    for (uint32_t i = 0; i <= PP_PARTS; ++i) {
                        factor[i] = __ldcg(part(i) + W * 128);
                        top = fmaxf(top, factor[i]);
                    }
                    odd = there && top == INFINITY;
                    const float ms = top == -INFINITY ? 0.0f : top;
#pragma unroll
                    for (uint32_t i = 0; i <= PP_PARTS; ++i) {
                        known[i] = i < parts && factor[i] != -INFINITY;
                        factor[i] = mx_ex2(factor[i] - ms);
                        if (i < parts) sum = fmaf(factor[i], __ldcg(part(i) + (W + 1) * 128), sum);
                    }
                    const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
                    for (uint32_t c = 0; c < p.a.vdim; c += 8) {
                        float x[PP_PARTS + 1][8], acc[8] = {};
#pragma unroll
                        for (uint32_t i = 0; i <= PP_PARTS; ++i)
#pragma unroll
                            for (uint32_t k = 0; k < 8; ++k) x[i][k] = __ldcg(part(i) + (c + k) * 128);
#pragma unroll
                        for (uint32_t i = 0; i <= PP_PARTS; ++i)
                            if (known[i])
#pragma unroll
                                for (uint32_t k = 0; k < 8; ++k) acc[k] = fmaf(factor[i], x[i][k], acc[k]);
                        if (there && !odd)
                            *reinterpret_cast<uint4*>(out + c) = make_uint4(pack_bf16x2(acc[0] * inv, acc[1] * inv), pack_bf16x2(acc[2] * inv, acc[3] * inv),
                                                                            pack_bf16x2(acc[4] * inv, acc[5] * inv), pack_bf16x2(acc[6] * inv, acc[7] * inv));
                    }
                }
            }
            if (!joined) {
                const float inv = l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll
                for (int c = 0; c < W / 16; ++c) {
                    float o[16];
                    if (any) pp_ld16(o_addr + c * 16, o);
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        if (!mine || (uint32_t)(c * 16 + i * 8) >= p.a.vdim) continue;
                        uint4 w = make_uint4(0u, 0u, 0u, 0u);
                        if (l != 0.0f) {
                            w.x = pack_bf16x2(o[8 * i] * inv, o[8 * i + 1] * inv);
                            w.y = pack_bf16x2(o[8 * i + 2] * inv, o[8 * i + 3] * inv);
                            w.z = pack_bf16x2(o[8 * i + 4] * inv, o[8 * i + 5] * inv);
                            w.w = pack_bf16x2(o[8 * i + 6] * inv, o[8 * i + 7] * inv);
                        }
                        *reinterpret_cast<uint4*>(out + c * 16 + i * 8) = w;
                    }
                }
                tc_fence_before();
            }
            // rows key by key, by the whole warp
            for (uint32_t rows = __ballot_sync(0xffffffffu, odd); rows; rows &= rows - 1) {
                const uint32_t r = quarter * 32 + __ffs(rows) - 1, token = p.per.div(r);
                paged_row<bf16>(p, it.s, it.seq, it.seq.start + it.token0 + t * prm.tokens + token, it.kvh * p.per.d + r - token * p.per.d, lane);
            }
        }
    }
    teardown();
}

// ---- launch ------------------------------------------------------------------------------------------------------------------------
static bool pp_map(CUtensorMap* map, const void* base, uint32_t rank, const uint64_t* dims, const uint64_t* strides, const uint32_t* box) {
    cuuint64_t d[4], st[3];
    cuuint32_t b[4], e[4] = {1, 1, 1, 1};
    for (uint32_t i = 0; i < rank; ++i) {
        d[i] = dims[i];
        b[i] = box[i];
        if (i) st[i - 1] = strides[i - 1] * 2;
    }
    return encode_fn()(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, rank, const_cast<void*>(base), d, st, b, e, CU_TENSOR_MAP_INTERLEAVE_NONE,
                       CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

uint64_t paged_prompt_workspace_bytes(uint32_t dim, uint32_t vdim) {
    const uint32_t w = std::max(dim, vdim) <= 64 ? 64 : 128;
    return std::max(dim, vdim) > 128 ? 0 : PAGED_COUNTERS + (uint64_t)PP_BLOCKS * 2 * 2 * 128 * (w + 2) * 4;
}

bool paged_prompt_eligible(const PagedAttention& a, int dtype) {
    const uint64_t strides = (uint64_t)a.dim | a.vdim | a.k_page | a.k_row | a.k_head | a.v_page | a.v_row | a.v_head | a.q_ld | a.out_ld | a.page_rows;
    const uintptr_t at = (uintptr_t)a.q | (uintptr_t)a.k_pool | (uintptr_t)a.v_pool | (uintptr_t)a.out;
    const uint64_t most = std::max({a.k_page, a.k_row, a.k_head, a.v_page, a.v_row, a.v_head});
    const uint64_t least = std::min({a.k_page, a.k_row, a.k_head, a.v_page, a.v_row, a.v_head});
    return dtype == TNSR_B200_BF16 && a.dim <= 128 && a.vdim <= 128 && strides % 8 == 0 && at % 16 == 0 && a.scale > 0.0f && a.heads / a.kv_heads <= 128 &&
           (uint64_t)a.sequences * a.kv_heads * ceil_div(a.chunk, 2 * (128 / (a.heads / a.kv_heads))) < 0x7fffff00u && least > 0 && most < (1ull << 38) && a.pool_pages < 0x7fffffffu && g_gemm_engine != 1 && encode_fn() != nullptr;
}

template <int W, bool DIVIDED>
static int launch_prompt_width(const PromptParams& prm, const CUtensorMap& mq, const CUtensorMap& mk, const CUtensorMap& mv, cudaStream_t stream) {
    constexpr uint32_t bytes = PromptShape<W>::BYTES + (DIVIDED ? sizeof(PromptPlan) : 0);
    if (const int rc = allow_shared<paged_prompt_kernel<W, DIVIDED>>(bytes, "paged_attention attribute")) return rc;
    int dev = 0, sms = 0;
    cudaGetDevice(&dev);
    cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
    const uint32_t most = std::min<uint32_t>(sms > 0 ? sms : PP_BLOCKS, PP_BLOCKS), grid = DIVIDED ? most : std::min(prm.items, most);
    launch_kernel(paged_prompt_kernel<W, DIVIDED>, dim3(grid), dim3(PP_THREADS), (size_t)bytes, stream, mq, mk, mv, prm);
    return TNSR_B200_OK;
}

int launch_paged_prompt(const PagedParams& p, cudaStream_t stream) {
    const PagedAttention& a = p.a;
    PromptParams prm;
    prm.p = p;
    prm.tokens = 128 / p.per.d;
    prm.pairs = ceil_div(a.chunk, 2 * prm.tokens);
    prm.units = a.sequences * a.kv_heads;
    prm.items = prm.units * prm.pairs;           // fewer than 2^31: paged_prompt_eligible
    prm.box = std::min(128u, a.page_rows & (0u - a.page_rows));
    prm.wait_limit_ns = g_wait_limit_ns.load(std::memory_order_relaxed);
    // The last round is divided where it can pay: items of more key blocks than the joins cost, and (as far as can be told here) a round that leaves a quarter of
    // the grid idle.  One prompt of 6000 rows over 12000 keys, window 4096, 32 / 8 heads: 472 -> 447 us; 3 x 100 rows over up to 4000 keys: 70 -> 47; where nothing
    // pays the plan alone costs 2 to 4 us.
    const uint64_t entries = (uint64_t)a.sequences * prm.pairs;
    const uint32_t span = a.window ? (uint32_t)std::min<uint64_t>(p.capacity, (uint64_t)a.window + 2 * prm.tokens + std::min(a.sinks, p.capacity) + 256) : p.capacity;
    const uint32_t most = ceil_div(span, 128u), left = prm.items % PP_BLOCKS;
    const bool divided = a.workspace && entries <= PP_ENTRIES && most - most / PP_PARTS > PP_JOIN &&
                         (a.row_starts || (left > 0 && left < PP_BLOCKS * 3 / 4));
    prm.done = divided ? reinterpret_cast<uint32_t*>(a.workspace) : nullptr;
    prm.partial = divided ? reinterpret_cast<float*>(reinterpret_cast<uint8_t*>(a.workspace) + PAGED_COUNTERS) : nullptr;
    CUtensorMap mq, mk, mv;
    const uint64_t q_dims[3] = {a.dim, a.heads, a.rows}, q_strides[2] = {a.dim, a.q_ld};
    const uint32_t q_box[3] = {64, p.per.d, prm.tokens}, kv_box[4] = {64, 1, prm.box, 1};
    const uint64_t k_dims[4] = {a.dim, a.kv_heads, a.page_rows, a.pool_pages}, v_dims[4] = {a.vdim, a.kv_heads, a.page_rows, a.pool_pages};
    const uint64_t k_strides[3] = {a.k_head, a.k_row, a.k_page}, v_strides[3] = {a.v_head, a.v_row, a.v_page};
    if (!pp_map(&mq, a.q, 3, q_dims, q_strides, q_box) || !pp_map(&mk, a.k_pool, 4, k_dims, k_strides, kv_box) ||
        !pp_map(&mv, a.v_pool, 4, v_dims, v_strides, kv_box)) {
        set_thread_error("paged_attention: tensor map encoding failed");
        return TNSR_B200_ERR_CUDA;
    }
    if (std::max(a.dim, a.vdim) <= 64)
        return divided ? launch_prompt_width<64, true>(prm, mq, mk, mv, stream) : launch_prompt_width<64, false>(prm, mq, mk, mv, stream);
    return divided ? launch_prompt_width<128, true>(prm, mq, mk, mv, stream) : launch_prompt_width<128, false>(prm, mq, mk, mv, stream);
}

}  // namespace tb
