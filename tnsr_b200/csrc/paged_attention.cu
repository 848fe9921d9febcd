// Attention over key-value caches in pages, rows of any number per sequence: out = softmax(scale q . k) v over the keys a row sees.  A row at
// position p sees keys j <= p with j > p - window, and the first `sinks` ones beside the window; window 0: all of them.  The rows of a
// sequence are the last of its keys; a row before its first key sees nothing and gives zeros.
#include <algorithm>

#include "mixers.cuh"
#include "paged.cuh"

namespace tb {

constexpr uint32_t PA_NONE = 0xffffffffu;

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

// ---- any widths, strides and alignment: a warp per row and head, keys one by one ------------------------------------------------
template <typename T>
__device__ __forceinline__ void paged_row(const PagedParams& p, uint32_t s, const PagedSequence& seq, uint32_t row, uint32_t h, uint32_t lane) {
    const PagedAttention& a = p.a;
    constexpr int N = 8;                         // 32 x 8 columns
    const T* q = reinterpret_cast<const T*>(a.q) + (uint64_t)row * a.q_ld + (uint64_t)h * a.dim;
    const uint32_t kvh = p.per.div(h), i = row - seq.start;
    float qv[N], acc[N] = {};
#pragma unroll
    for (int n = 0; n < N; ++n) qv[n] = n * 32 + lane < a.dim ? to_f32(q[n * 32 + lane]) : 0.0f;
    float m = -INFINITY, l = 0.0f;
    const int64_t at = (int64_t)seq.length - seq.count + i;
    const uint32_t* entries = a.table + (uint64_t)s * a.table_ld;
    const uint32_t keys = at < 0 ? 0u : (uint32_t)at + 1, first = a.window && keys > a.window ? keys - a.window : 0u;
    for (uint32_t j = 0; j < keys; ++j) {
        if (j < first && j >= a.sinks) {
            j = first;                           // first <= at < keys
        }
        uint32_t page, r;
        const bool real = paged_key(p, entries, j, page, r);
        if (!real && lane == 0) report(a.d_status, DEV_BAD_PAGE);
        const T* k = reinterpret_cast<const T*>(a.k_pool) + a.k_page * (real ? page : 0) + a.k_row * r + a.k_head * kvh;
        const T* v = reinterpret_cast<const T*>(a.v_pool) + a.v_page * (real ? page : 0) + a.v_row * r + a.v_head * kvh;
        float dot = 0.0f;
#pragma unroll
        for (int n = 0; n < N; ++n)
            if (real && n * 32 + lane < a.dim) dot = fmaf(qv[n], to_f32(k[n * 32 + lane]), dot);
#pragma unroll
        for (int d = 16; d > 0; d /= 2) dot += __shfl_xor_sync(0xffffffffu, dot, d);
        const float x = dot * p.scale_log2, top = fmaxf(m, x), ms = top == -INFINITY ? 0.0f : top;
        const float w = exp2f(x - ms), c = exp2f(m - ms);
        m = top;
        l = l * c + w;
#pragma unroll
        for (int n = 0; n < N; ++n) {
            const float y = real && n * 32 + lane < a.vdim ? to_f32(v[n * 32 + lane]) : 0.0f;
            acc[n] = fmaf(w, y, acc[n] * c);
        }
    }
    T* out = reinterpret_cast<T*>(a.out) + (uint64_t)row * a.out_ld + (uint64_t)h * a.vdim;
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll
    for (int n = 0; n < N; ++n)
        if (n * 32 + lane < a.vdim) out[n * 32 + lane] = from_f32<T>(l == 0.0f ? 0.0f : acc[n] * inv);
}

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

uint64_t paged_attention_workspace_bytes(uint32_t dim, uint32_t vdim, int dtype) { return 256; }

int launch_paged_attention(const PagedAttention& a, int dtype, cudaStream_t stream) {
    if (a.rows == 0 || a.sequences == 0) return TNSR_B200_OK;
    PagedParams p;
    p.a = a;
    p.page = fast_div(a.page_rows);
    p.per = fast_div(a.heads / a.kv_heads);
    p.capacity = (uint32_t)std::min<uint64_t>((uint64_t)a.table_ld * a.page_rows, PAGED_MAX_KEYS);
    p.scale_log2 = a.scale * 1.4426950408889634f;
    const dim3 grid((unsigned)ceil_div64((uint64_t)a.rows * a.heads, 4));
    if (dtype == TNSR_B200_F32) launch_kernel(paged_rows_kernel<float>, grid, dim3(128), 0, stream, p);
    else launch_kernel(paged_rows_kernel<bf16>, grid, dim3(128), 0, stream, p);
    count_launch();
    return check_launch("paged_attention");
}

}  // namespace tb
