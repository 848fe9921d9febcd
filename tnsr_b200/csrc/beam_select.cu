// Beam search's selection: of a group's beams x vocabulary candidates the `keep` best by
//
//   score(beam, token) = c_beam + (x_token - log sum_j exp x_j)
//
// in this order: score in 64 bits, larger first; of equal scores the earlier beam; within a beam the larger logit, then the smaller token.
// A finished beam has one candidate with its own score, the end token; its other tokens, and all of a beam whose sum or score is no finite
// number (a NaN or +inf logit, nothing but -inf, a score of -inf), count as -inf.
//
// Two launches.  beam_scan_kernel reads every logit once: a block has a run of a row in registers (32 values a thread), so it needs no
// second pass over memory.  It gives the run's maximum, its sum of exponentials and its `keep` best: the largest values of its threads,
// sorted by warp, bound the keep-th best from below (if each of eight warps has keep / 8 values at or above a bound, so has the block keep);
// what is at or above the bound is gathered and ranked by counting.  Keys are (value, index) pairs, so no two are equal and runs of equal
// values, of masked tokens say, cannot crowd the gathering: where the warps' bound lets too many in, the keep-th of all threads' maxima lets
// at most keep x 32 in.  beam_merge_kernel joins a group's runs the same way, a block per group.
//
// Sums: 32 terms in f32, the rest in f64.  A block's order of terms does not depend on the row, so that equal rows have equal sums to the last bit.
// Bound by HBM (each logit once) for large groups, else by two launches and their chains of barriers.
#include <algorithm>
#include <cmath>

#include "beam.cuh"

namespace tb {

constexpr uint32_t BS_THREADS = 256, BS_WARPS = BS_THREADS / 32;
constexpr uint32_t BS_RUNS = 32;              // runs of a row at the most
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

struct BeamRun {
    double sum;
    float max;
    uint32_t pad;
};

__device__ __forceinline__ uint64_t bs_shfl_xor(uint64_t v, int d) {
    return (uint64_t)__shfl_xor_sync(0xffffffffu, (uint32_t)(v >> 32), d) << 32 | __shfl_xor_sync(0xffffffffu, (uint32_t)v, d);
}
// Descending order over the lanes.
__device__ __forceinline__ uint64_t bs_sort_warp(uint64_t v, uint32_t lane) {
#pragma unroll
    for (uint32_t size = 2; size <= 32; size *= 2)
#pragma unroll
        for (uint32_t d = size / 2; d > 0; d /= 2) {
            const uint64_t w = bs_shfl_xor(v, d);
            const bool larger = ((lane & d) == 0) == ((lane & size) == 0);
            v = (v > w) == larger ? v : w;
        }
    return v;
}

// `PER` values a thread at a time.  VEC: 16-byte loads.
template <typename T, int PER, bool VEC>
__global__ void __launch_bounds__(BS_THREADS, 3) beam_scan_kernel(const T* logits, uint64_t ld, uint32_t vocab, uint32_t run, uint32_t keep, BeamRun* runs,
                                                               uint64_t* lists) {
    constexpr int W = VEC ? 16 / sizeof(T) : 1;
    __shared__ uint64_t gathered[BS_GATHER], best[BEAM_MAX_KEEP], tops[BS_THREADS], bound[BS_WARPS];
    __shared__ double sums[BS_WARPS];
    __shared__ uint32_t count;
    const uint32_t tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    pdl_wait();
    pdl_trigger();
    const T* row = logits + (uint64_t)blockIdx.x * ld;
    const uint32_t first = blockIdx.y * run, end = min(vocab, first + run);
    uint32_t kept = 0;          // entries of `best`
    float top = -INFINITY;
    double total = 0.0;
    for (uint32_t base = first; base < end; base += PER * BS_THREADS) {
        float v[PER];
#pragma unroll
        for (int j = 0; j < PER / W; ++j) {
            const uint32_t at = base + (j * BS_THREADS + tid) * W;
            if (VEC && at + W <= end) {
                const uint4 u = *reinterpret_cast<const uint4*>(row + at);
                if (sizeof(T) == 4) {
                    v[j * W] = __uint_as_float(u.x); v[j * W + 1] = __uint_as_float(u.y); v[j * W + 2] = __uint_as_float(u.z); v[j * W + 3] = __uint_as_float(u.w);
                } else {
                    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
                    for (int e = 0; e < W / 2; ++e) {
                        const float2 f = bf16x2_to_f32(w[e]);
                        v[j * W + 2 * e] = f.x;
                        v[j * W + 2 * e + 1] = f.y;
                    }
                }
            } else {
#pragma unroll
                for (int e = 0; e < W; ++e) v[j * W + e] = at + e < end ? to_f32(row[at + e]) : -INFINITY;
            }
        }
        // the thread's largest value (of equal ones the first)
        uint64_t mine = 0;
        {
            float m = -INFINITY;
            uint32_t index = base + tid * W;
#pragma unroll
            for (int i = 0; i < PER; ++i)
                if (v[i] > m) { m = v[i]; index = base + ((i / W) * BS_THREADS + tid) * W + i % W; }
            if (index < end) mine = bs_key(m, index);
        }
        const uint64_t sorted = bs_sort_warp(mine, lane);
        const uint32_t place = (keep + BS_WARPS - 1) / BS_WARPS - 1;
        if (lane == place) bound[warp] = sorted;
        if (lane == 0) tops[warp] = sorted;
        if (tid == 0) count = kept;
        __syncthreads();
        uint64_t low = bound[0], high = tops[0];
#pragma unroll
        for (int w = 1; w < (int)BS_WARPS; ++w) {
            low = min(low, bound[w]);
            high = max(high, tops[w]);
        }
        if (kept == keep) low = max(low, best[keep - 1]);
        const float m = fmaxf(top, bs_value((uint32_t)(high >> 32)));
        const float ms = m == -INFINITY ? 0.0f : m;
        float part = 0.0f;
        auto gather = [&](uint64_t from) {
#pragma unroll
            for (int i = 0; i < PER; ++i) {
                const uint32_t index = base + ((i / W) * BS_THREADS + tid) * W + i % W;
                if (bs_ordered(v[i]) >= (uint32_t)(from >> 32) && index < end) {
                    const uint64_t key = bs_key(v[i], index);
                    if (key >= from) {
                        const uint32_t at = atomicAdd(&count, 1u);
                        if (at < BS_GATHER) gathered[at] = key;
                    }
                }
            }
        };
#pragma unroll
        for (int i = 0; i < PER; ++i) part += bs_ex2((v[i] - ms) * 1.4426950408889634f);
        if (tid < kept) gathered[tid] = best[tid];
        gather(low);
        double sum = part;
#pragma unroll
        for (int d = 16; d > 0; d /= 2) sum += __shfl_xor_sync(0xffffffffu, sum, d);
        if (lane == 0) sums[warp] = sum;
        __syncthreads();
        if (count > BS_GATHER) {
            // one bound for the block: the keep-th of the threads' largest values
            __syncthreads();
            tops[tid] = mine;
            if (tid == 0) count = kept;
            __syncthreads();
            uint32_t rank = 0;
            for (uint32_t i = 0; i < BS_THREADS; ++i) rank += tops[i] > mine || (tops[i] == mine && i < tid);
            if (rank == keep - 1) bound[0] = mine;
            __syncthreads();
            gather(bound[0]);
            __syncthreads();
        }
        const uint32_t n = min(count, BS_GATHER);
        double all = 0.0;
#pragma unroll
        for (int w = 0; w < (int)BS_WARPS; ++w) all += sums[w];
        total = total * (top == -INFINITY ? 0.0 : exp((double)top - ms)) + all;
        top = m;
        // ranks by counting, unless something unusual was gathered: then by sorting
        if (n <= 2 * BS_THREADS) {
            uint64_t a = tid < n ? gathered[tid] : 0, b = tid + BS_THREADS < n ? gathered[tid + BS_THREADS] : 0;
            uint32_t ra = 0, rb = 0;
            for (uint32_t i = 0; i < n; ++i) {
                const uint64_t g = gathered[i];
                ra += g > a;
                rb += g > b;
            }
            if (a && ra < keep) best[ra] = a;
            if (b && rb < keep) best[rb] = b;
        } else {
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
        kept = min(keep, n);
        __syncthreads();
    }
    const uint64_t slot = (uint64_t)blockIdx.x * gridDim.y + blockIdx.y;
    if (tid == 0) runs[slot] = {total, top, 0u};
    if (tid < keep) lists[slot * keep + tid] = tid < kept ? best[tid] : 0;
}

// ---- a group's runs joined ----------------------------------------------------------------------------------------------------
// Larger is better: score, then beam, logit and token in one word.
struct BeamCandidate {
    uint64_t score, rest;
};
__device__ __forceinline__ bool bs_better(const BeamCandidate& a, const BeamCandidate& b) {
    return a.score > b.score || (a.score == b.score && a.rest > b.rest);
}
__device__ __forceinline__ BeamCandidate bs_candidate(double score, uint32_t beam, uint32_t logit_key, uint32_t token) {
    const uint64_t bits = (uint64_t)__double_as_longlong(score + 0.0);
    BeamCandidate c;
    c.score = bits >> 63 ? ~bits : bits | 0x8000000000000000ull;
    // a score of -inf has no logit: the smaller token is the better one
    c.rest = (uint64_t)(63 - beam) << 58 | (uint64_t)(score == -INFINITY ? 0u : logit_key) << 26 | (BEAM_MAX_VOCAB - 1 - token);
    return c;
}

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
// What is at or above the bound: `bounds` lists with all of theirs, the others with less than `place + 1`.
static uint32_t merge_room(const MergeShape& m, uint32_t keep) { return m.bounds * keep + (m.lists - m.bounds) * m.place; }

__global__ void __launch_bounds__(BS_THREADS) beam_merge_kernel(BeamSelect b, uint32_t runs, MergeShape shape, const BeamRun* parts, const uint64_t* lists) {
    extern __shared__ BeamCandidate space[];      // [lists] at the place of the bound, then what was gathered
    __shared__ double offset[BEAM_MAX];           // of a beam's logits; NaN: all of its candidates are -inf
    __shared__ uint8_t ended[BEAM_MAX];
    __shared__ BeamCandidate bound;
    __shared__ uint32_t count;
    pdl_wait();
    pdl_trigger();
    const uint32_t tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, first = blockIdx.x * b.beams;
    for (uint32_t beam = warp; beam < b.beams; beam += BS_WARPS) {
        const BeamRun* run = parts + (uint64_t)(first + beam) * runs;
        float m = -INFINITY;
        double s = 0.0;
        if (lane < runs) { m = run[lane].max; s = run[lane].sum; }
        float top = m;
#pragma unroll
        for (int d = 16; d > 0; d /= 2) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
        s = m == -INFINITY ? s : s * exp((double)m - top);      // a run of nothing but -inf has a sum of 0, or of NaN
#pragma unroll
        for (int d = 16; d > 0; d /= 2) s += __shfl_xor_sync(0xffffffffu, s, d);
        if (lane == 0) {
            const float c = b.scores[first + beam];
            const bool over = b.finished && b.finished[first + beam];
            ended[beam] = over && b.end_token < b.vocab && isfinite(c);
            const double total = top + log(s);
            offset[beam] = !over && isfinite(total) && isfinite(c) ? (double)c - total : nan("");
        }
    }
    if (tid == 0) count = 0;
    __syncthreads();
    // entry `i` of list `l` (run l % runs of beam l / runs); a beam without sums has one list that counts
    auto entry = [&](uint32_t l, uint32_t i) -> BeamCandidate {
        const uint32_t beam = l / runs;
        const double o = offset[beam];
        if (isnan(o)) {
            if (l % runs) return {0, 0};
            uint32_t token = i;
            if (ended[beam]) {
                if (i == 0) return bs_candidate(b.scores[first + beam], beam, 0, b.end_token);
                token = i - 1 + (i - 1 >= b.end_token);
            }
            return token < b.vocab ? bs_candidate(-INFINITY, beam, 0, token) : BeamCandidate{0, 0};
        }
        const uint64_t key = lists[((uint64_t)first * runs + l) * b.keep + i];
        if (key == 0) return {0, 0};
        return bs_candidate(o + bs_value((uint32_t)(key >> 32)), beam, (uint32_t)(key >> 32), ~(uint32_t)key);
    };
    for (uint32_t l = tid; l < shape.lists; l += BS_THREADS) space[l] = entry(l, shape.place);
    __syncthreads();
    for (uint32_t l = tid; l < shape.lists; l += BS_THREADS) {
        const BeamCandidate c = space[l];
        uint32_t rank = 0;
        for (uint32_t i = 0; i < shape.lists; ++i) rank += bs_better(space[i], c) || (space[i].rest == c.rest && space[i].score == c.score && i < l);
        if (rank == shape.bounds - 1) bound = c;
    }
    __syncthreads();
    const BeamCandidate low = bound;
    BeamCandidate* gathered = space + shape.lists;
    for (uint32_t x = tid; x < shape.lists * b.keep; x += BS_THREADS) {
        const BeamCandidate c = entry(x / b.keep, x % b.keep);
        if (c.score && !bs_better(low, c)) gathered[atomicAdd(&count, 1u)] = c;
    }
    __syncthreads();
    const uint32_t n = count;
    for (uint32_t x = tid; x < n; x += BS_THREADS) {
        const BeamCandidate c = gathered[x];
        uint32_t rank = 0;
        for (uint32_t i = 0; i < n && rank < b.keep; ++i) rank += bs_better(gathered[i], c);
        if (rank >= b.keep) continue;
        const uint32_t beam = 63 - (uint32_t)(c.rest >> 58), token = BEAM_MAX_VOCAB - 1 - (uint32_t)(c.rest & (BEAM_MAX_VOCAB - 1));
        const uint64_t at = (uint64_t)blockIdx.x * b.keep + rank, bits = c.score >> 63 ? c.score & 0x7fffffffffffffffull : ~c.score;
        b.next_scores[at] = (float)__longlong_as_double((long long)bits);
        b.tokens[at] = token;
        b.parents[at] = first + beam;
        if (b.next_finished) b.next_finished[at] = (b.finished && b.finished[first + beam]) || token == b.end_token;
    }
}

// ---- launch --------------------------------------------------------------------------------------------------------------------
struct BeamPlan {
    uint32_t per, run, runs;      // values of a thread at a time; values of a run; runs of a row
};
// The longest runs that still give two blocks per SM; they are a row's parts, multiples of 16 values.
static BeamPlan beam_plan(uint64_t rows, uint32_t vocab) {
    BeamPlan p{32, 0, 0};
    while (p.per > 8 && rows * ceil_div(vocab, p.per * BS_THREADS) < 296) p.per /= 2;
    p.runs = std::min(BS_RUNS, ceil_div(vocab, p.per * BS_THREADS));
    p.run = ceil_div(ceil_div(vocab, p.runs), 16u) * 16;
    p.runs = ceil_div(vocab, p.run);
    return p;
}

uint64_t beam_select_workspace_bytes(uint32_t groups, uint32_t beams, uint32_t vocab, uint32_t keep) {
    const uint64_t rows = (uint64_t)groups * beams;
    return rows * beam_plan(rows, std::max(vocab, 1u)).runs * (sizeof(BeamRun) + 8ull * keep);
}

template <typename T>
static void launch_scan(const BeamSelect& b, const BeamPlan& p, BeamRun* runs, uint64_t* lists, cudaStream_t stream) {
    const dim3 grid((unsigned)(b.groups * b.beams), p.runs);
    const bool vec = (uintptr_t)b.logits % 16 == 0 && b.logits_ld * sizeof(T) % 16 == 0;
    auto go = [&](auto kernel) { launch_kernel(kernel, grid, dim3(BS_THREADS), 0, stream, (const T*)b.logits, b.logits_ld, b.vocab, p.run, b.keep, runs, lists); };
    if (p.per == 32) vec ? go(beam_scan_kernel<T, 32, true>) : go(beam_scan_kernel<T, 32, false>);
    else if (p.per == 16) vec ? go(beam_scan_kernel<T, 16, true>) : go(beam_scan_kernel<T, 16, false>);
    else vec ? go(beam_scan_kernel<T, 8, true>) : go(beam_scan_kernel<T, 8, false>);
}

int launch_beam_select(const BeamSelect& b, int dtype, cudaStream_t stream) {
    if (b.groups == 0) return TNSR_B200_OK;
    const BeamPlan p = beam_plan((uint64_t)b.groups * b.beams, b.vocab);
    uint64_t* lists = reinterpret_cast<uint64_t*>(b.workspace);
    BeamRun* runs = reinterpret_cast<BeamRun*>(lists + (uint64_t)b.groups * b.beams * p.runs * b.keep);
    if (dtype == TNSR_B200_F32) launch_scan<float>(b, p, runs, lists, stream);
    else launch_scan<bf16>(b, p, runs, lists, stream);
    count_launch();
    if (int rc = check_launch("beam_select")) return rc;
    const MergeShape shape = merge_shape(b.beams, p.runs, b.keep);
    const uint32_t bytes = (uint32_t)sizeof(BeamCandidate) * (shape.lists + merge_room(shape, b.keep));
    if (int rc = allow_shared<beam_merge_kernel>(16 * (BEAM_MAX * BS_RUNS + BEAM_MAX_KEEP * (BEAM_MAX_KEEP + 1)), "beam_select attribute")) return rc;
    launch_kernel(beam_merge_kernel, dim3(b.groups), dim3(BS_THREADS), bytes, stream, b, p.runs, shape, runs, lists);
    count_launch();
    return check_launch("beam_select");
}

}  // namespace tb
