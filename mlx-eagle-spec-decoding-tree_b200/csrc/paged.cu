// Attention over a paged cache behind a prefix that all requests of the pass share.
//
//   o = softmax(scale * q [Kp; Kb]^T + mask) [Vp; Vb]:  prefix rows Kp, Vp and the rows Kb, Vb of the token's own request
//
// One warp per (token, query head) goes through all its keys, dims across the lanes, with the running maximum and sum of the softmax in fp32.
#include "paged.cuh"
#include "pipeline.cuh"

namespace b200 {
namespace {

struct PagedParams {
    const void *q, *k_pages, *v_pages;
    void* out;
    const int *table, *lengths, *row_starts, *prefix_pages;
    const unsigned long long* mask;
    long long q_token, q_head, out_token, out_head, page_stride, head_stride, row_stride, table_stride;
    int requests, tokens, heads, kv_heads, pages, page_size, table_width, prefix;
    float scale;
};

template <typename T, int HD>
__global__ void __launch_bounds__(128) paged_attention_kernel(const PagedParams p) {
    pdl_wait();
    pdl_launch_dependents();
    constexpr int N = HD / 32;
    const int lane = threadIdx.x & 31, head = blockIdx.y * 4 + (threadIdx.x >> 5), t = blockIdx.x;
    if (head >= p.heads || t < p.row_starts[0] || t >= p.row_starts[p.requests]) return;
    int req = 0;
    while (req + 1 < p.requests && p.row_starts[req + 1] <= t) req++;
    const int kh = head / (p.heads / p.kv_heads), length = min(max(p.lengths[req], 0), p.table_width * p.page_size);
    const int old = p.lengths[req] - (p.row_starts[req + 1] - p.row_starts[req]), index = t - p.row_starts[req];
    float q[N], o[N] = {}, m = -INFINITY, l = 0.f;
    for (int e = 0; e < N; e++) q[e] = to_f32(static_cast<const T*>(p.q)[t * p.q_token + head * p.q_head + lane * N + e]) * p.scale;
    for (int k = 0; k < p.prefix + length; k++) {
        const int own = k - p.prefix;
        if (own >= old) {
            const int j = own - old;
            if (p.mask == nullptr ? j > index : (j > 63 || !((p.mask[t] >> j) & 1))) continue;
        }
        const int row = own < 0 ? k : own, page = own < 0 ? p.prefix_pages[row / p.page_size] : p.table[req * p.table_stride + row / p.page_size];
        const bool there = page >= 0 && page < p.pages;
        const long long at = page * p.page_stride + kh * p.head_stride + row % p.page_size * p.row_stride + lane * N;
        float s = 0.f;
        if (there)
            for (int e = 0; e < N; e++) s += q[e] * to_f32(static_cast<const T*>(p.k_pages)[at + e]);
        for (int x = 16; x > 0; x >>= 1) s += __shfl_xor_sync(0xffffffffu, s, x);
        const float top = fmaxf(m, s);
        if (top == -INFINITY) continue;
        const float a = __expf(m - top), w = __expf(s - top);
        for (int e = 0; e < N; e++) o[e] = o[e] * a + (there ? w * to_f32(static_cast<const T*>(p.v_pages)[at + e]) : 0.f);
        l = l * a + w;
        m = top;
    }
    for (int e = 0; e < N; e++) static_cast<T*>(p.out)[t * p.out_token + head * p.out_head + lane * N + e] = from_f32<T>(l > 0.f ? o[e] / l : 0.f);
}

}  // namespace
}  // namespace b200

extern "C" {

size_t b200_paged_attention_workspace_bytes(const b200_paged* c) {
    if (b200::check_paged(c) != B200_OK) return 0;
    return 16;
}

int b200_paged_attention(const b200_paged* c, const void* q, long long q_token, long long q_head, void* out, long long out_token, long long out_head,
                         const int* prefix_pages, int prefix_length, const unsigned long long* mask, float scale, void* workspace,
                         size_t workspace_bytes, int* error, void* stream) {
    const int bad = b200::check_paged(c);
    if (bad != B200_OK) return bad;
    if ((c->head_dim != 64 && c->head_dim != 128) || prefix_length < 0 || (prefix_length > 0 && !prefix_pages)) return B200_EINVAL;
    if ((c->page_size < 128 && (c->page_size < 8 || (c->page_size & (c->page_size - 1)))) || (c->page_size > 128 && c->page_size % 128)) return B200_EINVAL;
    if (c->requests > 1024) return B200_ELIMIT;
    if (c->tokens == 0 || c->requests == 0) return B200_OK;
    if (!q || !out || !workspace || !error) return B200_EINVAL;
    if (workspace_bytes < b200_paged_attention_workspace_bytes(c)) return B200_EWORKSPACE;
    if (!b200::aligned16(q) || !b200::aligned16(out) || !b200::aligned16(c->k_pages) || !b200::aligned16(c->v_pages) || !b200::aligned16(workspace))
        return B200_EALIGN;
    if (q_token % 8 || q_head % 8 || out_token % 8 || out_head % 8 || c->page_stride % 8 || c->head_stride % 8 || c->row_stride % 8) return B200_EALIGN;
    b200::PagedParams p{q, c->k_pages, c->v_pages, out, c->page_table, c->lengths, c->row_starts, prefix_pages, mask, q_token, q_head, out_token, out_head,
                        c->page_stride, c->head_stride, c->row_stride, c->table_stride, c->requests, c->tokens, c->heads, c->kv_heads, c->pages,
                        c->page_size, c->table_width, prefix_length, scale};
    const dim3 grid(c->tokens, (c->heads + 3) / 4);
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    auto go = [&](auto kern) { b200::launch_kernel(kern, grid, dim3(128), 0, st, p); };
    if (c->dtype == B200_DTYPE_BF16) {
        if (c->head_dim == 128) go(b200::paged_attention_kernel<__nv_bfloat16, 128>);
        else go(b200::paged_attention_kernel<__nv_bfloat16, 64>);
    } else if (c->head_dim == 128) {
        go(b200::paged_attention_kernel<__half, 128>);
    } else {
        go(b200::paged_attention_kernel<__half, 64>);
    }
    return b200::check_launch();
}

}  // extern "C"
