// Beam search's selection: of a group's beams x vocabulary candidates the `keep` best by
//
//   score(beam, token) = c_beam + (x_token - log sum_j exp x_j)
//
// in this order: score in 64 bits, larger first; of equal scores the earlier beam; within a beam the larger logit, then the smaller token.
// A finished beam has one candidate with its own score, the end token; its other tokens, and all of a beam whose sum or score is no finite
// number (a NaN or +inf logit, nothing but -inf, a score of -inf), count as -inf.
//
// beam_scan_kernel reads every logit once: a block has a run of a row, a thread's values pass through its registers, 16 at a time, and leave their maximum and their
// sum of exponentials.  The largest of the warps' threads bound the keep-th best value from below; threads that have one at or above the bound have
// their values read again, and what is at or above it is gathered and ranked by counting: keep and a few more.  Keys are (value, index) pairs, so no
// two are equal.  Where equal values (masked tokens, say) let too many in, the run is gone through once more by keys alone.  The block that comes last
// of a group's joins its runs in the same way.
//
// Sums: 16 terms in f32, the rest in f64.  A block's order of terms does not depend on the row, so that equal rows have equal sums to the last bit.
// Bound by HBM (each logit once) for large groups, else by the chain of barriers behind the reading: 48 groups x 6 beams x 50021 logits, keep 12, 22.8 us =
// 2.53 TB/s (one wave of blocks: reading is half of it); one group x 4 beams x 32000, keep 4, 9.8 us.
#include <algorithm>
#include <cmath>

#include "beam.cuh"
#include "paged.cuh"
#include "tc_common.cuh"

namespace tb {

constexpr uint32_t BS_THREADS = 256, BS_WARPS = BS_THREADS / 32;
constexpr uint32_t BS_RUNS = 32;              // runs of a row at the most
constexpr uint32_t BS_BLOCKS = 296;           // two of an SM
constexpr uint32_t BS_LEAST_RUN = 2048;       // values of a run at the least, if the row has them
constexpr uint32_t BS_GATHER = 4096;         // room for what is gathered: more than BEAM_MAX_KEEP * (32 + 1)

// Order of floats as of integers; -0 is 0.
__device__ __forceinline__ uint32_t bs_ordered(float x) {
    const uint32_t bits = __float_as_uint(x + 0.0f);
    return bits & 0x80000000u ? ~bits : bits | 0x80000000u;
}
__device__ __forceinline__ float bs_value(uint32_t key) { return __uint_as_float(key & 0x80000000u ? key & 0x7fffffffu : ~key); }
// Larger is better: value, then the smaller index.  0 is below every key.
__device__ __forceinline__ uint64_t bs_key(float x, uint32_t index) { return (uint64_t)bs_ordered(x) << 32 | (uint32_t)~index; }

__device__ __forceinline__ float bs_ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// sum_j exp x_j of a run is sum * exp(base); base is the largest x.
struct BeamRun {
    double sum, base;
};
constexpr float BS_LOG2E = 1.4426950408889634f;
// exp(x - base) for x <= base, or NaN for a base of +inf: the difference first, so that logits of any finite size have terms of at most 1 (a base times log2(e) would
// overflow, or be rounded by more than an exponent holds, for the large negative numbers that mask tokens).
__device__ __forceinline__ float bs_term(float x, float base) { return bs_ex2((x - base) * BS_LOG2E); }

// ---- a group's runs joined ----------------------------------------------------------------------------------------------------
// Larger is better: score, then beam, logit and token in one word.
struct BeamCandidate {
    uint64_t score, rest;
};
__device__ __forceinline__ bool bs_better(const BeamCandidate& a, const BeamCandidate& b) {
    return (a.score > b.score) | ((a.score == b.score) & (a.rest > b.rest));      // no branches: comparisons of many candidates run side by side
}
__device__ __forceinline__ BeamCandidate bs_candidate(double score, uint32_t beam, uint32_t logit_key, uint32_t token) {
    const uint64_t bits = (uint64_t)__double_as_longlong(score + 0.0);
    BeamCandidate c;
    c.score = bits >> 63 ? ~bits : bits | 0x8000000000000000ull;
    // a score of -inf has no logit: the smaller token is the better one
    c.rest = (uint64_t)(63 - beam) << 58 | (uint64_t)(score == -INFINITY ? 0u : logit_key) << 26 | (BEAM_MAX_VOCAB - 1 - token);
    return c;
}

constexpr uint32_t BS_FEW_LISTS = 64;
constexpr uint32_t BS_STAGED = 32768;         // bytes of lists up to which the joining block has them in shared memory
struct MergeShape {
    uint32_t lists, place, bounds;       // lists of a group; at which place of every list the bound is looked for, and the how-many-th largest it is
};
static MergeShape merge_shape(uint32_t beams, uint32_t runs, uint32_t keep) {
    MergeShape m;
    m.lists = beams * runs;
    m.place = ceil_div(keep, m.lists) - 1;
    m.bounds = ceil_div(keep, m.place + 1);
    return m;
}
// What can be at or above the bound: `bounds` lists with all of theirs, the others with less than `place + 1`.
static uint32_t merge_room(const MergeShape& m, uint32_t keep) { return m.bounds * keep + (m.lists - m.bounds) * m.place; }

// By one block.  `space`: [lists] at the place of the bound, what is gathered, and (`staged`) the lists.
__device__ void beam_merge(const BeamSelect& b, uint32_t group, uint32_t runs, const MergeShape& shape, uint32_t room, bool staged, const BeamRun* parts,
                           const uint64_t* lists, BeamCandidate* space) {
    __shared__ double base_of[BEAM_MAX], log_sum[BEAM_MAX], score_of[BEAM_MAX];     // a beam's largest logit, log sum exp(x - largest) (NaN: all of its candidates are -inf), score
    __shared__ uint8_t ended[BEAM_MAX], was[BEAM_MAX];
    __shared__ BeamCandidate bound;
    __shared__ uint32_t places[BS_WARPS];
    __shared__ uint32_t count;
    const uint32_t tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, first = group * b.beams;
    // what the sums do not wait for first
    const uint64_t* entries = lists + (uint64_t)first * runs * b.keep;
    uint64_t* copy = reinterpret_cast<uint64_t*>(space + shape.lists + room);
    if (staged)
        for (uint32_t x = tid; x < shape.lists * b.keep; x += BS_THREADS) copy[x] = __ldcg(entries + x);
    for (uint32_t beam = warp; beam < b.beams; beam += BS_WARPS) {
        const BeamRun* run = parts + (uint64_t)(first + beam) * runs;
        const float c = b.scores[first + beam];
        const bool over = b.finished && b.finished[first + beam];
        double base = -INFINITY, sum = 0.0;
        if (lane < runs) { base = __ldcg(&run[lane].base); sum = __ldcg(&run[lane].sum); }
        double top = base;
#pragma unroll
        for (int d = 16; d > 0; d /= 2) top = fmax(top, __shfl_xor_sync(0xffffffffu, top, d));
        // a run of nothing but -inf has a sum of 0, or of NaN; factors are off by 2^-22 of themselves, as terms are
        if (base != -INFINITY) sum *= bs_ex2((float)((base - top) * 1.4426950408889634));
#pragma unroll
        for (int d = 16; d > 0; d /= 2) sum += __shfl_xor_sync(0xffffffffu, sum, d);
        if (lane == 0) {
            was[beam] = over;
            ended[beam] = over && b.end_token < b.vocab && isfinite(c);
            const double total = log(sum);
            base_of[beam] = top;
            log_sum[beam] = !over && isfinite(top) && isfinite(total) && isfinite(c) ? total : nan("");
            score_of[beam] = c;
        }
    }
    if (tid == 0) count = 0;
    __syncthreads();
    // entry `i` of list `l` (run l % runs of beam l / runs); a beam without sums has one list that counts
    auto entry = [&](uint32_t l, uint32_t i) -> BeamCandidate {
        const uint32_t beam = l / runs;
        if (isnan(log_sum[beam])) {
            if (l % runs) return {0, 0};
            uint32_t token = i;
            if (ended[beam]) {
                if (i == 0) return bs_candidate(b.scores[first + beam], beam, 0, b.end_token);
                token = i - 1 + (i - 1 >= b.end_token);
            }
            return token < b.vocab ? bs_candidate(-INFINITY, beam, 0, token) : BeamCandidate{0, 0};
        }
        const uint64_t key = staged ? copy[l * b.keep + i] : __ldcg(entries + (uint64_t)l * b.keep + i);
        if (key == 0) return {0, 0};
        // the largest logit goes first: beside one of 10^20 the sum's logarithm would be lost
        return bs_candidate(score_of[beam] + (((double)bs_value((uint32_t)(key >> 32)) - base_of[beam]) - log_sum[beam]), beam, (uint32_t)(key >> 32), ~(uint32_t)key);
    };
    // The bound.  If the q-th largest of the lists' entries at place p has (p + 1) q >= keep, so many entries are at or above it.  Few lists: by scores rounded
    // down to f32, a warp each for places 0, 1, 3, 7, ..., and the largest of what they find (heads alone let all of a good beam's lists in where the beams
    // lie far apart).  Many lists, or too many equal scores: by one place, exactly.
    auto single = [&](const BeamCandidate& c) -> uint32_t {      // 0: no candidate
        if (!c.score) return 0u;
        const uint64_t bits = c.score >> 63 ? c.score & 0x7fffffffffffffffull : ~c.score;
        return bs_ordered(__double2float_rd(__longlong_as_double((long long)bits)));
    };
    BeamCandidate* gathered = space + shape.lists;
    uint32_t n = room + 1;
    if (shape.lists <= BS_FEW_LISTS) {
        const uint32_t place = (1u << warp) - 1, nth = (b.keep + place) / (place + 1);
        uint32_t found = 0;
        if (place < b.keep && (uint64_t)shape.lists * (place + 1) >= b.keep) {
            const uint32_t key[2] = {lane < shape.lists ? single(entry(lane, place)) : 0u, lane + 32 < shape.lists ? single(entry(lane + 32, place)) : 0u};
            uint32_t rank[2] = {0, 0};
#pragma unroll
            for (int i = 0; i < 32; ++i) {
                const uint32_t x = __shfl_sync(0xffffffffu, key[0], i), y = __shfl_sync(0xffffffffu, key[1], i);
                rank[0] += (x > key[0]) + ((x == key[0]) & (i < lane)) + (y > key[0]);
                rank[1] += (x >= key[1]) + (y > key[1]) + ((y == key[1]) & (i < lane));
            }
            found = __reduce_max_sync(0xffffffffu, rank[0] == nth - 1 ? key[0] : rank[1] == nth - 1 ? key[1] : 0u);
        }
        if (lane == 0) places[warp] = found;
        __syncthreads();
        uint32_t low = places[0];
#pragma unroll
        for (int w = 1; w < (int)BS_WARPS; ++w) low = max(low, places[w]);
        for (uint32_t x = tid; x < shape.lists * b.keep; x += BS_THREADS) {
            const BeamCandidate c = entry(x / b.keep, x % b.keep);
            if (c.score && single(c) >= low) {
                const uint32_t at = atomicAdd(&count, 1u);
                if (at < room) gathered[at] = c;
            }
        }
        __syncthreads();
        n = count;
        __syncthreads();
    }
    if (n > room) {
        if (tid == 0) count = 0;
        for (uint32_t l = tid; l < shape.lists; l += BS_THREADS) space[l] = entry(l, shape.place);
        __syncthreads();
        for (uint32_t l = tid; l < shape.lists; l += BS_THREADS) {
            const BeamCandidate c = space[l];
            uint32_t rank = 0;
#pragma unroll 4
            for (uint32_t i = 0; i < shape.lists; ++i) rank += bs_better(space[i], c) | ((space[i].rest == c.rest) & (space[i].score == c.score) & (i < l));
            if (rank == shape.bounds - 1) bound = c;
        }
        __syncthreads();
        const BeamCandidate low = bound;
        for (uint32_t x = tid; x < shape.lists * b.keep; x += BS_THREADS) {
            const BeamCandidate c = entry(x / b.keep, x % b.keep);
            if (c.score && !bs_better(low, c)) gathered[atomicAdd(&count, 1u)] = c;
        }
        __syncthreads();
        n = count;
    }
    // ranks, eight threads a candidate
    for (uint32_t x0 = 0; x0 < n; x0 += BS_THREADS / 8) {
        const uint32_t x = x0 + tid / 8;
        const BeamCandidate c = gathered[min(x, n - 1)];
        uint32_t rank = 0;
        for (uint32_t i = tid % 8; i < n; i += 8) rank += bs_better(gathered[i], c);
#pragma unroll
        for (int d = 1; d < 8; d *= 2) rank += __shfl_xor_sync(0xffffffffu, rank, d);
        if (tid % 8 || x >= n || rank >= b.keep) continue;
        const uint32_t beam = 63 - (uint32_t)(c.rest >> 58), token = BEAM_MAX_VOCAB - 1 - (uint32_t)(c.rest & (BEAM_MAX_VOCAB - 1));
        const uint64_t at = (uint64_t)group * b.keep + rank, bits = c.score >> 63 ? c.score & 0x7fffffffffffffffull : ~c.score;
        b.next_scores[at] = (float)__longlong_as_double((long long)bits);
        b.tokens[at] = token;
        b.parents[at] = first + beam;
        if (b.next_finished) b.next_finished[at] = was[beam] || token == b.end_token;
    }
}

__global__ void __launch_bounds__(BS_THREADS) beam_merge_kernel(BeamSelect b, uint32_t runs, MergeShape shape, uint32_t room, bool staged, const BeamRun* parts,
                                                                const uint64_t* lists) {
    extern __shared__ __align__(16) uint8_t space[];
    pdl_wait();
    pdl_trigger();
    beam_merge(b, blockIdx.x, runs, shape, room, staged, parts, lists, reinterpret_cast<BeamCandidate*>(space));
}

// Descending order over the lanes.
__device__ __forceinline__ float bs_sort_warp(float v, uint32_t lane) {
#pragma unroll
    for (uint32_t size = 2; size <= 32; size *= 2)
#pragma unroll
        for (uint32_t d = size / 2; d > 0; d /= 2) {
            const float w = __shfl_xor_sync(0xffffffffu, v, d);
            v = ((lane & d) == 0) == ((lane & size) == 0) ? fmaxf(v, w) : fminf(v, w);
        }
    return v;
}

// best[0 .. min(n, keep)) <- the best of gathered[0 .. n), best first.
__device__ __forceinline__ void bs_rank(uint64_t* gathered, uint32_t n, uint32_t keep, uint64_t* best) {
    const uint32_t tid = threadIdx.x;
    if (n <= 2 * BS_THREADS) {
        // eight threads a key
        for (uint32_t x0 = 0; x0 < n; x0 += BS_THREADS / 8) {
            const uint32_t x = x0 + tid / 8;
            const uint64_t mine = gathered[min(x, n - 1)];
            uint32_t rank = 0;
            for (uint32_t i = tid % 8; i < n; i += 8) rank += gathered[i] > mine;
#pragma unroll
            for (int d = 1; d < 8; d *= 2) rank += __shfl_xor_sync(0xffffffffu, rank, d);
            if (tid % 8 == 0 && x < n && rank < keep) best[rank] = mine;
        }
    } else {                     // something unusual: by sorting
        uint32_t size = 2 * BS_THREADS;
        while (size < n) size *= 2;
        for (uint32_t i = n + tid; i < size; i += BS_THREADS) gathered[i] = 0;
        __syncthreads();
        for (uint32_t width = 2; width <= size; width *= 2)
            for (uint32_t d = width / 2; d > 0; d /= 2) {
                for (uint32_t i = tid; i < size / 2; i += BS_THREADS) {
                    const uint32_t x = 2 * d * (i / d) + i % d, y = x + d;
                    const uint64_t gx = gathered[x], gy = gathered[y];
                    if ((gx < gy) == ((x & width) == 0)) {
                        gathered[x] = gy;
                        gathered[y] = gx;
                    }
                }
                __syncthreads();
            }
        if (tid < keep) best[tid] = gathered[tid];
    }
    __syncthreads();
}

// The `keep` best keys of row[first .. end), however many values are equal: by pieces of 32 values a thread, of which those are gathered that are at or above the
// keep-th largest of the threads' best keys, at most keep x 32, beside the best of the pieces before.  Returns how many there are.
template <typename T>
__device__ uint32_t bs_select_exactly(const T* row, uint32_t first, uint32_t end, uint32_t keep, uint64_t* gathered, uint64_t* best, uint64_t* tops, uint64_t* bound,
                                      uint32_t* count) {
    const uint32_t tid = threadIdx.x;
    uint32_t kept = 0;
    for (uint32_t base = first; base < end; base += 32 * BS_THREADS) {
        const uint32_t stop = min(end, base + 32 * BS_THREADS);
        uint64_t mine = 0;
        for (uint32_t at = base + tid; at < stop; at += BS_THREADS) mine = max(mine, bs_key(to_f32(row[at]), at));
        __syncthreads();
        tops[tid] = mine;
        if (tid < kept) gathered[tid] = best[tid];
        if (tid == 0) *count = kept;
        __syncthreads();
        uint32_t rank = 0;
        for (uint32_t i = 0; i < BS_THREADS; ++i) rank += (tops[i] > mine) | ((tops[i] == mine) & (i < tid));
        if (rank == keep - 1) *bound = mine;
        __syncthreads();
        const uint64_t low = *bound;
        for (uint32_t at = base + tid; at < stop; at += BS_THREADS) {
            const uint64_t key = bs_key(to_f32(row[at]), at);
            if (key >= low) {
                const uint32_t place = atomicAdd(count, 1u);
                if (place < BS_GATHER) gathered[place] = key;       // NaN may be more: the row does not count then
            }
        }
        __syncthreads();
        const uint32_t n = min(*count, BS_GATHER);
        __syncthreads();
        bs_rank(gathered, n, keep, best);
        kept = min(keep, n);
    }
    return kept;
}

// A piece of a run is 16 values a thread; three of them are on their way to shared memory by bulk copies.
constexpr uint32_t BS_PIECE = 16 * BS_THREADS, BS_STAGES = 3;
template <typename T>
struct BeamStage {
    static constexpr uint32_t BYTES = BS_PIECE * sizeof(T) + 16;
    static constexpr uint32_t SPACE = BS_STAGES * BYTES > BS_GATHER * 8 ? BS_STAGES * BYTES : BS_GATHER * 8;
};

// Per value: a load from shared memory, a maximum, a multiplication-addition, an exponential and an addition.  The few threads with a value at or above the bound
// have their values read once more, from L2.  Rows start anywhere: a copy takes the 16-byte units that its values lie in, and so what is beside them in the
// array; what would lie outside the array is read value by value.
template <typename T>
__global__ void __launch_bounds__(BS_THREADS, 4) beam_scan_kernel(BeamSelect b, uint32_t run, uint32_t row_runs, BeamRun* runs, uint64_t* lists, MergeShape shape, uint32_t room,
                                                                  bool staged, uint32_t* tickets, uint64_t wait_limit_ns) {
    constexpr int W = 4 / sizeof(T);                     // neighbours that a thread has together
    constexpr int TOPS = BEAM_MAX_KEEP / BS_WARPS;       // of a warp, for the bound
    extern __shared__ __align__(16) uint8_t space[];     // BeamStage<T>::SPACE
    __shared__ uint64_t best[BEAM_MAX_KEEP], tops[BS_THREADS], exact_bound, full[BS_STAGES];
    __shared__ float warp_tops[BS_WARPS][TOPS];
    __shared__ double sums[BS_WARPS];
    __shared__ uint32_t count, threads;
    __shared__ uint8_t listed[BS_THREADS];
    __shared__ int gave_up;
    const uint32_t tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    if (tid == 0) {
        for (uint32_t i = 0; i < BS_STAGES; ++i) mbar_init(full + i, 1);
        gave_up = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    __syncthreads();
    pdl_wait();
    pdl_trigger();
    // runs of a row, rows of a group behind one another: a group is complete before the last blocks of the launch begin
    const uint32_t row_number = blockIdx.x / row_runs, keep = b.keep;
    const T* row = reinterpret_cast<const T*>(b.logits) + (uint64_t)row_number * b.logits_ld;
    const uint32_t first = blockIdx.x % row_runs * run, end = min(b.vocab, first + run), pieces = (end - first + BS_PIECE - 1) / BS_PIECE;
    // the array in whole units
    const uintptr_t inside = ((uintptr_t)b.logits + 15) & ~(uintptr_t)15,
                    outside = (uintptr_t)(reinterpret_cast<const T*>(b.logits) + ((uint64_t)b.groups * b.beams - 1) * b.logits_ld + b.vocab) & ~(uintptr_t)15;
    const uint32_t skew = (uint32_t)((uintptr_t)(row + first) & 15);      // bytes before a piece's first value in its first unit: pieces are whole units
    auto fetch = [&](uint32_t i) {                                        // by one thread
        const uintptr_t begin = (uintptr_t)(row + first + i * BS_PIECE) - skew, stop = (uintptr_t)(row + min(end, first + (i + 1) * BS_PIECE));
        const uintptr_t from = max(begin, inside), to = min((stop + 15) & ~(uintptr_t)15, outside);
        const uint32_t stage = i % BS_STAGES, bytes = to > from ? (uint32_t)(to - from) : 0u;
        mbar_expect_tx(full + stage, bytes);
        if (bytes)
            asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
                         ::"r"(smem_u32(space + stage * BeamStage<T>::BYTES) + (uint32_t)(from - begin)), "l"(from), "r"(bytes), "r"(smem_u32(full + stage))
                         : "memory");
    };
    if (tid == 0)
        for (uint32_t i = 0; i < min(pieces, BS_STAGES); ++i) fetch(i);

    // The thread's largest value and its sum of exponentials of what the others are below it.
    float mine = -INFINITY;
    double sum = 0.0;
    for (uint32_t i = 0; i < pieces; ++i) {
        const uint32_t stage = i % BS_STAGES, base = first + i * BS_PIECE, here = min(end - base, BS_PIECE);
        if (!mbar_wait(full + stage, (i / BS_STAGES) & 1, &gave_up, wait_limit_ns)) {                    // the row does not count then
            sum = nan("");
            report(b.d_status, DEV_TIMEOUT);
        }
        // value j * W + e of the thread is number (j * BS_THREADS + tid) * W + e of the piece; what is not there is -inf
        float v[16];
        const uint8_t* src = space + stage * BeamStage<T>::BYTES + skew;
        const uintptr_t at = (uintptr_t)(row + base);
        if (here == BS_PIECE && at >= inside && at + BS_PIECE * sizeof(T) <= outside) {
#pragma unroll
            for (int j = 0; j < 16 / W; ++j) {
                const uint8_t* x = src + (j * BS_THREADS + tid) * 4;
                if (W == 1) {
                    v[j] = *reinterpret_cast<const float*>(x);
                } else if (skew % 4 == 0) {
                    const float2 f = bf16x2_to_f32(*reinterpret_cast<const uint32_t*>(x));
                    v[j * W] = f.x;
                    v[j * W + W - 1] = f.y;
                } else {
#pragma unroll
                    for (int e = 0; e < W; ++e) v[j * W + e] = to_f32(reinterpret_cast<const T*>(x)[e]);
                }
            }
        } else {
#pragma unroll
            for (int j = 0; j < 16; ++j) {
                const uint32_t k = (j / W * BS_THREADS + tid) * W + j % W;
                v[j] = -INFINITY;
                if (k < here) {
                    const bool copied = (at + k * sizeof(T)) >= inside && (at + (k + 1) * sizeof(T)) <= outside;
                    v[j] = to_f32(copied ? reinterpret_cast<const T*>(src)[k] : row[base + k]);
                }
            }
        }
        if (pieces > BS_STAGES) {
            __syncthreads();             // the stage may be overwritten
            if (tid == 0 && i + BS_STAGES < pieces) {
                fence_proxy_async_smem();
                fetch(i + BS_STAGES);
            }
        }
        float largest = v[0];
#pragma unroll
        for (int j = 1; j < 16; ++j) largest = fmaxf(largest, v[j]);
        if (largest > mine) {
            if (mine != -INFINITY) sum *= bs_term(mine, largest);
            mine = largest;
        }
        const float base_value = mine == -INFINITY ? 0.0f : mine;       // -inf alone: terms of 0
        float part[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int j = 0; j < 16; ++j) part[j & 3] += bs_term(v[j], base_value);
        sum += (double)((part[0] + part[1]) + (part[2] + part[3]));
    }
    if (gave_up) {                       // copies that are still on their way get time to land
        const uint64_t start = global_timer_ns();
        while (global_timer_ns() - start < 200000ull) __nanosleep(1000);
    }
    uint64_t* gathered = reinterpret_cast<uint64_t*>(space);        // behind the barrier below
    // the largest of the warp's threads, one after the other (equal ones count once: the bound may be lower then, and is one still)
    {
        uint32_t left = bs_ordered(mine);
        const int places = keep <= 32 ? 4 : TOPS;
#pragma unroll
        for (int i = 0; i < TOPS; ++i) {
            if (i >= places) break;
            const uint32_t largest = __reduce_max_sync(0xffffffffu, left);
            if (lane == 0) warp_tops[warp][i] = bs_value(largest);
            if (left == largest) left = 0x007fffffu;      // -inf
        }
    }
    if (tid == 0) count = threads = 0;
    __syncthreads();
    // The bound: the keep-th largest of the four largest of every warp's threads, or (more than 32) the smallest of the warps' eighth ones.
    float low, top;
    if (keep <= 32) {
        const float all = bs_sort_warp(warp_tops[lane >> 2][lane & 3], lane);
        low = __shfl_sync(0xffffffffu, all, keep - 1);
        top = __shfl_sync(0xffffffffu, all, 0);
    } else {
        low = warp_tops[0][TOPS - 1];
        top = warp_tops[0][0];
#pragma unroll
        for (int w = 1; w < (int)BS_WARPS; ++w) {
            low = fminf(low, warp_tops[w][TOPS - 1]);
            top = fmaxf(top, warp_tops[w][0]);
        }
    }
    // Threads with a value at or above the bound, a list of which is divided among the warps, have their values read again, a value a lane, four (of two threads
    // eight) on their way at a time.  Where the bound is -inf, which is also what stands for values behind the end, and where equal values let too many in, all
    // is done exactly.
    if (mine >= low && low != -INFINITY) listed[atomicAdd(&threads, 1u)] = (uint8_t)tid;
    // the sums at one base
    if (mine != -INFINITY) sum *= bs_term(mine, top);               // what had no finite number has a sum of 0, or of NaN
#pragma unroll
    for (int d = 16; d > 0; d /= 2) sum += __shfl_xor_sync(0xffffffffu, sum, d);
    if (lane == 0) sums[warp] = sum;
    __syncthreads();
    const uint32_t values = (end - first + BS_THREADS * W - 1) / (BS_THREADS * W) * W;       // of a thread at the most
    for (uint32_t x = warp; x < threads; x += 2 * BS_WARPS) {
        const uint32_t other[2] = {listed[x], x + BS_WARPS < threads ? listed[x + BS_WARPS] : BS_THREADS};
        for (uint32_t i0 = 0; i0 < values; i0 += 128) {
            float again[8];
            uint32_t index[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                const uint32_t i = i0 + (k & 3) * 32 + lane;
                index[k] = first + ((i / W) * BS_THREADS + other[k >> 2]) * W + i % W;
                again[k] = i < values && other[k >> 2] < BS_THREADS && index[k] < end ? to_f32(row[index[k]]) : -INFINITY;
            }
#pragma unroll
            for (int k = 0; k < 8; ++k)
                if (again[k] >= low) {
                    const uint32_t at = atomicAdd(&count, 1u);
                    if (at < 2 * BS_THREADS) gathered[at] = bs_key(again[k], index[k]);
                }
        }
    }
    __syncthreads();
    uint32_t kept = count;
    __syncthreads();
    if (low == -INFINITY || kept > 2 * BS_THREADS) {
        kept = bs_select_exactly(row, first, end, keep, gathered, best, tops, &exact_bound, &count);
    } else {
        bs_rank(gathered, kept, keep, best);
        kept = min(kept, keep);
    }
    double total = 0.0;
#pragma unroll
    for (int w = 0; w < (int)BS_WARPS; ++w) total += sums[w];
    if (tid == 0) runs[blockIdx.x] = {total, (double)top};
    if (tid < keep) lists[(uint64_t)blockIdx.x * keep + tid] = tid < kept ? best[tid] : 0;
    if (!tickets) return;
    // the block that comes last joins the group's runs
    __syncthreads();
    const uint32_t group = row_number / b.beams;
    if (tid == 0) {
        __threadfence();             // with the barriers before and behind it, for all of the block
        count = atomicAdd(tickets + group, 1u) + 1 == shape.lists;
        if (count) tickets[group] = 0;
        __threadfence();
    }
    __syncthreads();
    if (!count) return;
    beam_merge(b, group, row_runs, shape, room, staged, runs, lists, reinterpret_cast<BeamCandidate*>(gathered));
}

// ---- launch --------------------------------------------------------------------------------------------------------------------
struct BeamPlan {
    uint32_t run, runs;      // values of a run; runs of a row
};
// Runs so long that about two blocks per SM cover all rows: what comes behind the reading is paid per run.  Multiples of 16 values, so that a piece is whole
// 16-byte units behind its first value.
static BeamPlan beam_plan(uint64_t rows, uint32_t vocab) {
    const uint64_t wanted = std::min<uint64_t>(BS_RUNS, std::max<uint64_t>(1, BS_BLOCKS / std::max<uint64_t>(1, rows)));
    BeamPlan p;
    p.runs = (uint32_t)std::min<uint64_t>(wanted, ceil_div(vocab, BS_LEAST_RUN));
    p.run = ceil_div(ceil_div(vocab, p.runs), 16u) * 16;
    p.runs = ceil_div(vocab, p.run);
    return p;
}

uint64_t beam_select_workspace_bytes(uint32_t groups, uint32_t beams, uint32_t vocab, uint32_t keep) {
    // rows x runs of beam_plan at the most, for this call and for all with no more groups, beams, vocabulary and candidates: fewer rows have more runs each
    const uint64_t rows = (uint64_t)groups * beams, most = std::min<uint64_t>(BS_RUNS, ceil_div(std::max(vocab, 1u), BS_LEAST_RUN));
    return BEAM_COUNTERS + std::max(rows, std::min<uint64_t>(BS_BLOCKS, rows * most)) * (sizeof(BeamRun) + 8ull * keep);
}

template <typename T>
static int launch_scan(const BeamSelect& b, const BeamPlan& p, BeamRun* runs, uint64_t* lists, const MergeShape& shape, uint32_t room, bool staged,
                        uint32_t* tickets, cudaStream_t stream) {
    if (int rc = allow_shared<beam_scan_kernel<T>>(BeamStage<T>::SPACE, "beam_select attribute")) return rc;
    launch_kernel(beam_scan_kernel<T>, dim3(b.groups * b.beams * p.runs), dim3(BS_THREADS), BeamStage<T>::SPACE, stream, b, p.run, p.runs, runs, lists, shape, room, staged, tickets,
                  g_wait_limit_ns.load(std::memory_order_relaxed));
    return TNSR_B200_OK;
}

int launch_beam_select(const BeamSelect& b, int dtype, cudaStream_t stream) {
    if (b.groups == 0) return TNSR_B200_OK;
    const BeamPlan p = beam_plan((uint64_t)b.groups * b.beams, b.vocab);
    uint32_t* tickets = reinterpret_cast<uint32_t*>(b.workspace);
    uint64_t* lists = reinterpret_cast<uint64_t*>(reinterpret_cast<uint8_t*>(b.workspace) + BEAM_COUNTERS);
    BeamRun* runs = reinterpret_cast<BeamRun*>(lists + (uint64_t)b.groups * b.beams * p.runs * b.keep);
    const MergeShape shape = merge_shape(b.beams, p.runs, b.keep);
    const uint32_t room = merge_room(shape, b.keep), bytes = (uint32_t)sizeof(BeamCandidate) * (shape.lists + room), list_bytes = shape.lists * b.keep * 8;
    // joined by a group's last block where that has the shared memory for it and the group a ticket, else by a launch of its own (2 us of the 40 or more that over a
    // thousand groups take)
    const bool joined = bytes + list_bytes <= BS_GATHER * 8 && b.groups <= BEAM_COUNTERS / 4, staged = joined || list_bytes <= BS_STAGED;
    int rc = dtype == TNSR_B200_F32 ? launch_scan<float>(b, p, runs, lists, shape, room, staged, joined ? tickets : nullptr, stream)
                                    : launch_scan<bf16>(b, p, runs, lists, shape, room, staged, joined ? tickets : nullptr, stream);
    if (rc) return rc;
    count_launch();
    if ((rc = check_launch("beam_select"))) return rc;
    if (joined) return TNSR_B200_OK;
    if ((rc = allow_shared<beam_merge_kernel>(16 * (BEAM_MAX * BS_RUNS + BEAM_MAX_KEEP * (BEAM_MAX_KEEP + 1)) + BS_STAGED, "beam_select attribute"))) return rc;
    launch_kernel(beam_merge_kernel, dim3(b.groups), dim3(BS_THREADS), bytes + (staged ? list_bytes : 0), stream, b, p.runs, shape, room, staged, runs, lists);
    count_launch();
    return check_launch("beam_select");
}

}  // namespace tb
