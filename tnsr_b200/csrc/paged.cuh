// Key-value caches in pages as operators see them: where a key lies, which rows a call brings, what a row sees.  Shared by the attention
// kernels over pages (paged_attention.cu, paged_prompt.cu) and the operators that manage pages (pages.cu).
#pragma once

#include "common.cuh"

namespace tb {

// More values of the device status word (common.cuh): what a call that must not be trusted with memory says of its tables.
enum : int {
    DEV_BAD_PAGE = 4,        // a live table entry names a page outside the pool
    DEV_NO_PAGES = 5,        // more pages wanted than are free: nothing was changed
    DEV_BAD_PARENT = 6       // a parent outside its group: the row keeps what it has
};

// n / d for n < 2^31 by a multiplication: d is a parameter of the launch.
struct FastDiv {
    uint32_t d, mul, shift;
#ifdef __CUDACC__
    __device__ __forceinline__ uint32_t div(uint32_t n) const { return (__umulhi(n, mul) + n) >> shift; }
#endif
};
inline FastDiv fast_div(uint32_t d) {
    FastDiv f{d, 0, 0};
    while (f.shift < 31 && (1ull << f.shift) < d) ++f.shift;
    f.mul = (uint32_t)(((1ull << 32) * ((1ull << f.shift) - d)) / d + 1);
    return f;
}

constexpr uint64_t PAGED_MAX_KEYS = 0x7fffff00ull;      // keys a sequence can hold: positions are 31 bits

struct PagedAttention {
    const void *q, *k_pool, *v_pool;
    const uint32_t *table, *lengths, *row_starts;       // row_starts: [sequences + 1] or null (chunk rows each)
    void* out;
    void* workspace;
    int* d_status;
    uint64_t workspace_bytes;
    uint64_t k_page, k_row, k_head, v_page, v_row, v_head;   // elements between pages, rows of a page, heads of a row
    uint32_t sequences, chunk, rows, q_ld, out_ld, heads, kv_heads, dim, vdim, table_ld, page_rows, pool_pages;
    uint32_t window, sinks;                             // window 0: every earlier key
    float scale;
};

// What kernels get: the call and what follows from it.
struct PagedParams {
    PagedAttention a;
    FastDiv page, per;          // rows of a page; query heads per key/value head
    uint32_t capacity;          // keys that a table row can name
    float scale_log2;
};

int launch_paged_attention(const PagedAttention& a, int dtype, cudaStream_t stream);
uint64_t paged_attention_workspace_bytes(uint32_t dim, uint32_t vdim, int dtype);
constexpr uint32_t PAGED_COUNTERS = 4096;           // bytes of a workspace before its partial results
// Many rows, on the tensor cores of the fifth generation (paged_prompt.cu).
uint64_t paged_prompt_workspace_bytes(uint32_t dim, uint32_t vdim);
bool paged_prompt_eligible(const PagedAttention& a, int dtype);
int launch_paged_prompt(const PagedParams& p, cudaStream_t stream);

#ifdef __CUDACC__
__device__ __forceinline__ void report(int* d_status, int what) {
    if (d_status) atomicCAS(d_status, DEV_OK, what);
}

// The rows a sequence brings: first row in q, how many, and its keys (new ones included).
struct PagedSequence {
    uint32_t start, count, length;
};
__device__ __forceinline__ PagedSequence paged_sequence(const PagedParams& p, uint32_t s) {
    PagedSequence q;
    q.length = p.a.lengths[s];
    if (q.length > p.capacity) {
        q.length = p.capacity;
        report(p.a.d_status, DEV_BAD_LENGTH);
    }
    if (!p.a.row_starts) {
        q.start = s * p.a.chunk;
        q.count = p.a.chunk;
        return q;
    }
    q.start = min(p.a.row_starts[s], p.a.rows);
    const uint32_t end = min(p.a.row_starts[s + 1], p.a.rows);
    q.count = end > q.start ? end - q.start : 0u;
    if (q.count > p.a.chunk) {          // rows that the launch has no room for stay as they are
        q.count = p.a.chunk;
        report(p.a.d_status, DEV_BAD_LENGTH);
    }
    return q;
}
// Page of key `key` and its row there; false: no page of the pool.
__device__ __forceinline__ bool paged_key(const PagedParams& p, const uint32_t* entries, uint32_t key, uint32_t& page, uint32_t& row) {
    const uint32_t i = p.page.div(key);
    row = key - i * p.page.d;
    page = entries[i];
    return page < p.a.pool_pages;
}
// One row and head by a warp, keys one by one: any widths, strides and alignment.
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
#endif

}  // namespace tb
