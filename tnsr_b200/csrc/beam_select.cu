// Beam search's selection: of a group's beams x vocabulary candidates the `keep` best by
//
//   score(beam, token) = c_beam + (x_token - log sum_j exp x_j)
//
// in this order: score in 64 bits, larger first; of equal scores the earlier beam; within a beam the larger logit, then the smaller token.
// A finished beam has one candidate with its own score, the end token; its other tokens, and all of a beam whose sum or score is no finite
// number (a NaN or +inf logit, nothing but -inf, a score of -inf), count as -inf.
//
// beam_scan_kernel reads every logit once: a block has a run of a row, a thread's values pass through its registers, 32 at a time, and leave their maximum and their
// sum of exponentials.  The largest of the warps' threads bound the keep-th best value from below; threads that have one at or above the bound have
// their values read again, and what is at or above it is gathered and ranked by counting: keep and a few more.  Keys are (value, index) pairs, so no
// two are equal.  Where equal values (masked tokens, say) let too many in, the run is gone through once more by keys alone.  The block that comes last
// of a group's joins its runs in the same way.
//
// Sums: 32 terms in f32, the rest in f64.  A block's order of terms does not depend on the row, so that equal rows have equal sums to the last bit.
// Bound by HBM (each logit once) for large groups, else by the chain of barriers behind the reading.
#include <algorithm>
#include <cmath>

#include "beam.cuh"

namespace tb {

constexpr uint32_t BS_THREADS = 256, BS_WARPS = BS_THREADS / 32;
constexpr uint32_t BS_RUNS = 32;              // runs of a row at the most
constexpr uint32_t BS_BLOCKS = 592;           // four of an SM
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

// sum_j exp x_j of a run is sum * exp(base); base is about the largest x.
struct BeamRun {
    double sum, base;
};
constexpr float BS_LOG2E = 1.4426950408889634f;

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
// What can be at or above the bound: `bounds` lists with all of theirs, the others with less than `place + 1`; of several bounds the one that lets the fewest in.
static uint32_t merge_room(const MergeShape& m, uint32_t keep) {
    auto room = [&](uint32_t place) {
        const uint32_t nth = ceil_div(keep, place + 1);
        return nth * keep + (m.lists - nth) * place;
    };
    if (m.lists > BS_FEW_LISTS) return room(m.place);
    uint32_t least = 0xffffffffu;
    for (uint32_t w = 0; w < BS_WARPS; ++w) {
        const uint32_t place = (1u << w) - 1;
        if (place < keep && m.lists * (place + 1) >= keep) least = std::min(least, room(place));
    }
    return least;
}

// By one block.  `space`: [lists] at the place of the bound, what is gathered, and (`staged`) the lists.
__device__ void beam_merge(const BeamSelect& b, uint32_t group, uint32_t runs, const MergeShape& shape, uint32_t room, bool staged, const BeamRun* parts,
                           const uint64_t* lists, BeamCandidate* space) {
    __shared__ double offset[BEAM_MAX];           // of a beam's logits; NaN: all of its candidates are -inf
    __shared__ uint8_t ended[BEAM_MAX];
    __shared__ BeamCandidate bound, bounds[BS_WARPS];
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
            ended[beam] = over && b.end_token < b.vocab && isfinite(c);
            const double total = top + log(sum);
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
        const uint64_t key = staged ? copy[l * b.keep + i] : __ldcg(entries + (uint64_t)l * b.keep + i);
        if (key == 0) return {0, 0};
        return bs_candidate(o + bs_value((uint32_t)(key >> 32)), beam, (uint32_t)(key >> 32), ~(uint32_t)key);
    };
    // The bound.  If the q-th largest of the lists' entries at place p has (p + 1) q >= keep, so many entries are at or above it.  Few lists: a warp each for
    // places 0, 1, 3, 7, ..., and the largest of what they find (heads alone let all of a good beam's lists in where the beams lie far apart).
    if (shape.lists <= BS_FEW_LISTS) {
        const uint32_t place = (1u << warp) - 1;
        const bool there = place < b.keep && (uint64_t)shape.lists * (place + 1) >= b.keep;
        const uint32_t nth = (b.keep + place) / (place + 1);
        if (tid < BS_WARPS) bounds[tid] = {0, 0};
        __syncthreads();
        if (there) {
            BeamCandidate mine[BS_FEW_LISTS / 32];
            uint32_t rank[BS_FEW_LISTS / 32] = {};
#pragma unroll
            for (int k = 0; k < (int)BS_FEW_LISTS / 32; ++k) mine[k] = k * 32 + lane < shape.lists ? entry(k * 32 + lane, place) : BeamCandidate{0, 0};
#pragma unroll
            for (int k = 0; k < (int)BS_FEW_LISTS / 32; ++k) {
                if (k * 32 >= shape.lists) break;
#pragma unroll 8
                for (int i = 0; i < 32; ++i) {
                    BeamCandidate other;
                    other.score = __shfl_sync(0xffffffffu, mine[k].score, i);
                    other.rest = __shfl_sync(0xffffffffu, mine[k].rest, i);
#pragma unroll
                    for (int m = 0; m < (int)BS_FEW_LISTS / 32; ++m) rank[m] += bs_better(other, mine[m]);
                }
            }
            // only what is missing is equal, and below everything
#pragma unroll
            for (int k = 0; k < (int)BS_FEW_LISTS / 32; ++k)
                if (rank[k] == nth - 1 && mine[k].score) bounds[warp] = mine[k];
        }
        __syncthreads();
        if (tid == 0) {
            BeamCandidate best = bounds[0];
            for (uint32_t w = 1; w < BS_WARPS; ++w)
                if (bs_better(bounds[w], best)) best = bounds[w];
            bound = best;
        }
        __syncthreads();
    } else {
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
    }
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
        for (uint32_t i0 = 0; i0 < n && rank < b.keep; i0 += 8)
#pragma unroll
            for (uint32_t i = i0; i < i0 + 8; ++i) rank += i < n && bs_better(gathered[min(i, n - 1)], c);
        if (rank >= b.keep) continue;
        const uint32_t beam = 63 - (uint32_t)(c.rest >> 58), token = BEAM_MAX_VOCAB - 1 - (uint32_t)(c.rest & (BEAM_MAX_VOCAB - 1));
        const uint64_t at = (uint64_t)group * b.keep + rank, bits = c.score >> 63 ? c.score & 0x7fffffffffffffffull : ~c.score;
        b.next_scores[at] = (float)__longlong_as_double((long long)bits);
        b.tokens[at] = token;
        b.parents[at] = first + beam;
        if (b.next_finished) b.next_finished[at] = (b.finished && b.finished[first + beam]) || token == b.end_token;
    }
}

__global__ void __launch_bounds__(BS_THREADS) beam_merge_kernel(BeamSelect b, uint32_t runs, MergeShape shape, uint32_t room, bool staged, const BeamRun* parts,
                                                                const uint64_t* lists) {
    extern __shared__ BeamCandidate merge_space[];
    pdl_wait();
    pdl_trigger();
    beam_merge(b, blockIdx.x, runs, shape, room, staged, parts, lists, merge_space);
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
        for (uint32_t x = tid; x < n; x += BS_THREADS) {
            const uint64_t mine = gathered[x];
            uint32_t rank = 0;
#pragma unroll 8
            for (uint32_t i = 0; i < n; ++i) rank += gathered[i] > mine;
            if (rank < keep) best[rank] = mine;
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

// `PER` values a thread at a time.  VEC: 16-byte loads.
// Per value: a load, a maximum, a multiplication-addition, an exponential and an addition.  The few threads with a value at or above the bound have their values
// read once more, from L2.
template <typename T, int PER, bool VEC>
__global__ void __launch_bounds__(BS_THREADS, 4) beam_scan_kernel(BeamSelect b, uint32_t run, uint32_t row_runs, BeamRun* runs, uint64_t* lists, MergeShape shape, uint32_t room,
                                                                  bool staged, uint32_t* tickets) {
    constexpr int W = VEC ? 16 / sizeof(T) : 1;
    constexpr int TOPS = BEAM_MAX_KEEP / BS_WARPS;       // of a warp, for the bound
    __shared__ __align__(16) uint64_t gathered[BS_GATHER];
    __shared__ uint64_t best[BEAM_MAX_KEEP], tops[BS_THREADS], exact_bound;
    __shared__ float warp_tops[BS_WARPS][TOPS];
    __shared__ double sums[BS_WARPS];
    __shared__ uint32_t count;
    const uint32_t tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    pdl_wait();
    pdl_trigger();
    // runs of a row, rows of a group behind one another: a group is complete before the last blocks of the launch begin
    const uint32_t row_number = blockIdx.x / row_runs, keep = b.keep;
    const T* row = reinterpret_cast<const T*>(b.logits) + (uint64_t)row_number * b.logits_ld;
    const uint32_t first = blockIdx.x % row_runs * run, end = min(b.vocab, first + run);

    // The thread's largest value and its sum of exponentials.  A term is 2^(x L + shift) with L the float nearest to log2(e): the base of the sum is what the
    // rounded shift stands for and not the maximum it was made from, or all terms would be off by the same factor.
    float mine = -INFINITY, shift = 0.0f;
    double sum = 0.0;
    for (uint32_t base = first; base < end; base += PER * BS_THREADS) {
        // value j * W + e of the thread is number (j * BS_THREADS + tid) * W + e of the piece; what is not there is -inf
        float v[PER];
        const uint32_t here = min(end - base, (uint32_t)PER * BS_THREADS), whole = here / (BS_THREADS * W);
        const T* src = row + base + tid * W;
        auto load = [&](int j, bool check) {
            if (VEC && !check) {
                const uint4 u = *reinterpret_cast<const uint4*>(src + j * BS_THREADS * W);
                const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    if (sizeof(T) == 4) {
                        v[j * W + e] = __uint_as_float(w[e]);
                    } else {
                        const float2 f = bf16x2_to_f32(w[e]);
                        v[j * W + 2 * e] = f.x;
                        v[j * W + (W > 1 ? 2 * e + 1 : 0)] = f.y;
                    }
                }
            } else {
#pragma unroll
                for (int e = 0; e < W; ++e)
                    v[j * W + e] = !check || (j * BS_THREADS + tid) * W + e < here ? to_f32(src[j * BS_THREADS * W + e]) : -INFINITY;
            }
        };
        if (whole == PER / W) {
#pragma unroll
            for (int j = 0; j < PER / W; ++j) load(j, false);
        } else {
#pragma unroll
            for (int j = 0; j < PER / W; ++j) {
                if (j * BS_THREADS * W < here) {
                    load(j, true);
                } else {
#pragma unroll
                    for (int e = 0; e < W; ++e) v[j * W + e] = -INFINITY;
                }
            }
        }
        float largest = v[0];
#pragma unroll
        for (int i = 1; i < PER; ++i) largest = fmaxf(largest, v[i]);
        if (largest > mine) {
            const float now = -largest * BS_LOG2E;
            if (mine != -INFINITY) sum *= bs_ex2(now - shift);
            mine = largest;
            shift = now;
        }
        float part[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int i = 0; i < PER; ++i) part[i & 3] += bs_ex2(fmaf(v[i], BS_LOG2E, shift));
        sum += (double)((part[0] + part[1]) + (part[2] + part[3]));
    }
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
    if (tid == 0) count = 0;
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
    // Threads with a value at or above the bound: the warp reads such a thread's values again, a value a lane.  Where the bound is -inf, which is also what
    // stands for values behind the end, and where equal values let too many in, all is done exactly.
    if (low != -INFINITY)
        for (uint32_t who = __ballot_sync(0xffffffffu, mine >= low); who; who &= who - 1) {
            const uint32_t other = tid - lane + __ffs(who) - 1;
#pragma unroll 4
            for (uint32_t i = lane;; i += 32) {
                const uint32_t index = first + ((i / W) * BS_THREADS + other) * W + i % W;
                if (!__any_sync(0xffffffffu, index < end)) break;
                const float x = index < end ? to_f32(row[index]) : -INFINITY;
                if (x >= low) {
                    const uint32_t at = atomicAdd(&count, 1u);
                    if (at < 2 * BS_THREADS) gathered[at] = bs_key(x, index);
                }
            }
        }
    // the sums at one base
    const float block_shift = top == -INFINITY ? 0.0f : -top * BS_LOG2E;
    if (mine != -INFINITY) sum *= bs_ex2(block_shift - shift);      // what had no finite number has a sum of 0, or of NaN
#pragma unroll
    for (int d = 16; d > 0; d /= 2) sum += __shfl_xor_sync(0xffffffffu, sum, d);
    if (lane == 0) sums[warp] = sum;
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
    const double old_base = top == -INFINITY ? -INFINITY : -(double)block_shift / BS_LOG2E;
    if (tid == 0) runs[blockIdx.x] = {total, old_base};
    if (tid < keep) lists[(uint64_t)blockIdx.x * keep + tid] = tid < kept ? best[tid] : 0;
    if (!tickets) return;
    // the block that comes last joins the group's runs
    __threadfence();
    __syncthreads();
    const uint32_t group = row_number / b.beams;
    if (tid == 0) count = atomicAdd(tickets + group, 1u) + 1 == shape.lists;
    __syncthreads();
    if (!count) return;
    __threadfence();
    if (tid == 0) tickets[group] = 0;
    __syncthreads();
    beam_merge(b, group, row_runs, shape, room, staged, runs, lists, reinterpret_cast<BeamCandidate*>(gathered));
}

// ---- launch --------------------------------------------------------------------------------------------------------------------
struct BeamPlan {
    uint32_t per, run, runs;      // values of a thread at a time; values of a run; runs of a row
};
// Runs so long that about four blocks per SM cover all rows (what comes behind the reading is paid per run), but no longer than a few pieces of 32 values a
// thread; few rows: pieces of 16 or 8 values.  Multiples of 16 values, so that 16-byte loads stay whole.
static BeamPlan beam_plan(uint64_t rows, uint32_t vocab) {
    BeamPlan p{32, 0, 0};
    const uint64_t wanted = std::min<uint64_t>(BS_RUNS, std::max<uint64_t>(1, BS_BLOCKS / std::max<uint64_t>(1, rows)));
    while (p.per > 8 && ceil_div(vocab, p.per * BS_THREADS) < wanted) p.per /= 2;
    p.runs = (uint32_t)std::min<uint64_t>(wanted, ceil_div(vocab, p.per * BS_THREADS));
    p.run = ceil_div(ceil_div(vocab, p.runs), 16u) * 16;
    p.runs = ceil_div(vocab, p.run);
    return p;
}

uint64_t beam_select_workspace_bytes(uint32_t groups, uint32_t beams, uint32_t vocab, uint32_t keep) {
    const uint64_t rows = (uint64_t)groups * beams;
    return rows * beam_plan(rows, std::max(vocab, 1u)).runs * (sizeof(BeamRun) + 8ull * keep) + 4ull * groups;
}

template <typename T>
static void launch_scan(const BeamSelect& b, const BeamPlan& p, BeamRun* runs, uint64_t* lists, const MergeShape& shape, uint32_t room, bool staged,
                        uint32_t* tickets, cudaStream_t stream) {
    const dim3 grid(b.groups * b.beams * p.runs);
    const bool vec = (uintptr_t)b.logits % 16 == 0 && b.logits_ld * sizeof(T) % 16 == 0;
    auto go = [&](auto kernel) { launch_kernel(kernel, grid, dim3(BS_THREADS), 0, stream, b, p.run, p.runs, runs, lists, shape, room, staged, tickets); };
    if (p.per == 32) vec ? go(beam_scan_kernel<T, 32, true>) : go(beam_scan_kernel<T, 32, false>);
    else if (p.per == 16) vec ? go(beam_scan_kernel<T, 16, true>) : go(beam_scan_kernel<T, 16, false>);
    else vec ? go(beam_scan_kernel<T, 8, true>) : go(beam_scan_kernel<T, 8, false>);
}

int launch_beam_select(const BeamSelect& b, int dtype, cudaStream_t stream) {
    if (b.groups == 0) return TNSR_B200_OK;
    const BeamPlan p = beam_plan((uint64_t)b.groups * b.beams, b.vocab);
    uint64_t* lists = reinterpret_cast<uint64_t*>(b.workspace);
    BeamRun* runs = reinterpret_cast<BeamRun*>(lists + (uint64_t)b.groups * b.beams * p.runs * b.keep);
    uint32_t* tickets = reinterpret_cast<uint32_t*>(runs + (uint64_t)b.groups * b.beams * p.runs);
    const MergeShape shape = merge_shape(b.beams, p.runs, b.keep);
    const uint32_t room = merge_room(shape, b.keep), bytes = (uint32_t)sizeof(BeamCandidate) * (shape.lists + room), list_bytes = shape.lists * b.keep * 8;
    // joined by a group's last block where that has the shared memory for it, else by a launch of its own
    const bool joined = bytes + list_bytes <= BS_GATHER * 8, staged = joined || list_bytes <= BS_STAGED;
    if (dtype == TNSR_B200_F32) launch_scan<float>(b, p, runs, lists, shape, room, staged, joined ? tickets : nullptr, stream);
    else launch_scan<bf16>(b, p, runs, lists, shape, room, staged, joined ? tickets : nullptr, stream);
    count_launch();
    if (int rc = check_launch("beam_select")) return rc;
    if (joined) return TNSR_B200_OK;
    if (int rc = allow_shared<beam_merge_kernel>(16 * (BEAM_MAX * BS_RUNS + BEAM_MAX_KEEP * (BEAM_MAX_KEEP + 1)) + BS_STAGED, "beam_select attribute")) return rc;
    launch_kernel(beam_merge_kernel, dim3(b.groups), dim3(BS_THREADS), bytes + (staged ? list_bytes : 0), stream, b, p.runs, shape, room, staged, runs, lists);
    count_launch();
    return check_launch("beam_select");
}

}  // namespace tb
