// Rotary positions in general form, and the append of a pass's keys and values to a paged cache with the rotation on the way.
//
//   theta = position * scaling * inv_freq[i];  (a, b) -> magnitude * (a cos - b sin, a sin + b cos)
//
// for the pairs (x[i], x[i + R/2]) or, interleaved, (x[2i], x[2i + 1]) of the first R dims; the dims behind them pass through.
//
// The angle is reduced in whole numbers: scaling * inv_freq / 2 pi as a 64-bit fraction of a turn, times the position modulo 2^64, is the
// fraction of a turn of the product.  The fraction comes from a product in two doubles each and is off by 2^-64 at most, so the angle by 2^-24
// radians, fp32's own step, at 2^37 rows (2^-44 at 131072, where a product in single precision is off by 2^-9; one double's 53 bits left 2.4e-7 radians at
// 2^31 and 1.2e-4 at 2^40).  Products and sums of a pair are fp32, rounded once to the result's type.
//
// A CTA has a token or two: its threads turn the angles once (the only costly arithmetic), then all go over the heads, 16 bytes an item, two in
// flight.  What bounds it: the wait for loads and angles, a third of an SM's warps being there to pass it (80 registers), and instructions; 4099 tokens of 32 x 128 16-bit elements 13.3 us (5.0 TB/s, 77 %
// of a copy's rate; 13.2 with the fraction from one double), ragged prompts 49.4 (4.3 TB/s, 65 %; 49.3), one token 3.9 (the launch).
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "paged.cuh"
#include "typed.cuh"

namespace b200 {
namespace {

constexpr int kRotThreads = 256;
constexpr int kRotTokens = 2;                    // of a CTA, at most
static_assert(kRotTokens == 2, "which token an angle is for is a comparison");
constexpr int kRotSweeps = 2;                    // of its threads over the heads, whose loads are in flight together

// One block of heads that share addresses: head h of token t at base + t * token + h * head (elements).
struct Heads {
    char* base;
    long long token, head;
};

struct RotParams {
    Heads in, out;                               // queries of the append
    Heads k, v;                                  // the append's new rows
    char *k_pages, *v_pages;
    long long page_stride, page_head, page_row;  // elements
    const void* positions;                       // or NULL: row in the request, behind the prefix
    int pos64;
    const float* inv_freqs;
    double turns, turns_low;                     // scaling / 2 pi, and what its rounding left
    float magnitude;
    int inverse;
    int tokens, heads, kv_heads, dim, half;      // half: pairs that are rotated
    int per_cta;                                 // tokens of a CTA
    // append
    const int *table, *lengths, *row_starts;
    long long table_stride;
    int requests, pages, page_size, table_width, prefix;
};

// Largest r with starts[r] <= t, by the lanes of a warp (starts ascending, starts[0] <= t).
__device__ __forceinline__ int find_request(const int* starts, int requests, int t, int lane) {
    int lo = 0, hi = requests;
    while (hi - lo > 1) {
        const int step = (hi - lo + 31) / 32, at = lo + (lane + 1) * step;
        const int n = __popc(__ballot_sync(0xffffffffu, at < hi && starts[at] <= t));
        lo += n * step;
        hi = min(hi, lo + step);
    }
    return lo;
}

// magnitude * (cos, sin) of frequency i at a position.
__device__ __forceinline__ float2 turn_of(const RotParams& p, int i, long long pos) {
    const double f = p.inv_freqs[i], high = f * p.turns, low = fma(f, p.turns_low, fma(f, p.turns, -high));
    const unsigned long long fraction = (unsigned long long)__double2ll_rn((high - rint(high)) * 0x1p64) + (unsigned long long)__double2ll_rn(low * 0x1p64);
    const unsigned long long phase = fraction * (unsigned long long)pos;
    const unsigned quarter = (unsigned)((phase + (1ull << 61)) >> 62);                       // the nearest quarter of a turn, what is left to either side
    float s, c;
    sincospif((float)(long long)(phase - ((unsigned long long)quarter << 62)) * 0x1p-63f, &s, &c);
    if (quarter & 1) {
        const float x = s;
        s = c;
        c = -x;
    }
    if (quarter & 2) {
        s = -s;
        c = -c;
    }
    return make_float2(c * p.magnitude, (p.inverse ? -s : s) * p.magnitude);
}

// An item is VE dims of one head (interleaved: VE / 2 pairs), or the VE pairs of two times VE dims.  WHOLE: all loads are of 16 bytes; else element
// by element, for any strides and sizes.  What bounds it: launch latency up to a few MB, then HBM.
template <typename T, int VE, bool WHOLE, bool INTERLEAVED, bool APPEND>
__global__ void __launch_bounds__(kRotThreads, INTERLEAVED ? 4 : 3) rotary_kernel(const RotParams p) {
    pdl_wait();
    pdl_launch_dependents();
    extern __shared__ __align__(16) float2 turned[];                                   // [token][half]: magnitude * (cos, sin)
    __shared__ long long s_row[kRotTokens];                              // cache offset, -1: nowhere, -2: no request's token
    const int t0 = blockIdx.x * p.per_cta, toks = min(p.per_cta, p.tokens - t0);
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int rot = p.half * 2, pair_items = (INTERLEAVED ? rot + VE - 1 : p.half + VE - 1) / VE;
    const int head_items = pair_items + (p.dim - rot + VE - 1) / VE, heads = APPEND ? p.heads + 2 * p.kv_heads : p.heads;
    // A thread keeps its place in the head and goes through the heads, `sweep` of them at a time: no division but one at the start.
    const int cols = min(head_items, kRotThreads), sweep = kRotThreads / cols, mine = threadIdx.x / cols;
    const int h0 = blockIdx.y * (sweep * kRotSweeps) + mine, step = sweep * kRotSweeps * gridDim.y;
    Vec<T, VE> a[kRotTokens][kRotSweeps], b[kRotTokens][kRotSweeps];
    int it = mine < sweep ? threadIdx.x - mine * cols : head_items;
    bool pairs;
    int c, n;                                                            // the place: first dim, elements of a side
    auto place = [&]() {
        pairs = it < pair_items;
        c = pairs ? it * VE : rot + (it - pair_items) * VE;
        n = min((pairs ? (INTERLEAVED ? rot : p.half) : p.dim) - c, VE);
    };
    auto load = [&](int first) {
#pragma unroll
        for (int s = 0; s < kRotSweeps; s++) {
            int h = first + s * sweep;
            if (h >= heads) break;
            const T* src;
            long long token = p.in.token;
            if (!APPEND || h < p.heads) {
                src = reinterpret_cast<const T*>(p.in.base) + h * p.in.head;
            } else {
                const bool is_k = h < p.heads + p.kv_heads;
                src = reinterpret_cast<const T*>(is_k ? p.k.base : p.v.base) + (h - (is_k ? p.heads : p.heads + p.kv_heads)) * p.k.head;
                token = p.k.token;
            }
            src += t0 * token + c;
#pragma unroll
            for (int k = 0; k < kRotTokens; k++)
                if (k < toks) {
                    load_vec<WHOLE>(a[k][s], src + k * token, n);
                    if (!INTERLEAVED && pairs) load_vec<WHOLE>(b[k][s], src + k * token + p.half, n);
                }
        }
    };
    // Loads first: places and angles take as long as they do.
    place();
    if (it < head_items) load(h0);
    auto given = [&](int t) { return p.pos64 ? static_cast<const long long*>(p.positions)[t] : (long long)static_cast<const int*>(p.positions)[t]; };
    if constexpr (!APPEND) {
        for (int i = threadIdx.x; i < toks * p.half; i += kRotThreads) {
            const int k = i >= p.half;                                   // (two tokens at most)
            turned[i] = turn_of(p, i - k * p.half, given(t0 + k));
        }
    } else {
        // Four warps a token (all, if there is one), each of which looks for the token's place itself, so that nothing waits in between.
        const int per = kRotThreads / 32 / p.per_cta, k = warp / per, sub = warp - k * per, t = t0 + k;
        if (k < toks) {
            long long row = 0, at = -2;
            if (t >= p.row_starts[0] && t < p.row_starts[p.requests]) {
                const int r = find_request(p.row_starts, p.requests, t, lane);
                row = (long long)p.lengths[r] - p.row_starts[r + 1] + t;
                at = -1;
                if (sub == 0 && row >= 0 && row < (long long)p.table_width * p.page_size) {
                    const int index = (int)row / p.page_size, page = p.table[r * p.table_stride + index];
                    if (page >= 0 && page < p.pages) at = page * p.page_stride + ((int)row - index * p.page_size) * p.page_row;
                }
            }
            if (sub == 0 && lane == 0) s_row[k] = at;
            const long long pos = p.positions == nullptr ? row + p.prefix : given(t);
            for (int i = sub * 32 + lane; i < p.half; i += per * 32) turned[k * p.half + i] = turn_of(p, i, pos);
        }
    }
    __syncthreads();
    auto store = [&](int first) {
        constexpr int PAIRS = INTERLEAVED ? VE / 2 : VE;
#pragma unroll
        for (int k = 0; k < kRotTokens; k++) {
            if (k >= toks) break;
            Vec<float2, PAIRS> w;                                        // of the place, for all heads
            if (pairs) {
                const float2* cs = turned + k * p.half + (INTERLEAVED ? c / 2 : c);
                if constexpr (WHOLE) {
#pragma unroll
                    for (int e = 0; e < PAIRS; e += 2) *reinterpret_cast<float4*>(w.v + e) = *reinterpret_cast<const float4*>(cs + e);
                } else {
#pragma unroll
                    for (int e = 0; e < PAIRS; e++) w.v[e] = e < n ? cs[e] : make_float2(0.f, 0.f);
                }
            }
            const long long row = APPEND ? s_row[k] : 0;
#pragma unroll
            for (int s = 0; s < kRotSweeps; s++) {
                const int h = first + s * sweep;
                if (h >= heads) break;
                T* dst;
                bool turn = pairs;
                if (!APPEND || h < p.heads) {
                    if (APPEND && row == -2) continue;
                    dst = reinterpret_cast<T*>(p.out.base) + (t0 + k) * p.out.token + h * p.out.head + c;
                } else {
                    if (row < 0) continue;
                    const bool is_k = h < p.heads + p.kv_heads;
                    turn = turn && is_k;
                    dst = reinterpret_cast<T*>(is_k ? p.k_pages : p.v_pages) + row + (h - (is_k ? p.heads : p.heads + p.kv_heads)) * p.page_head + c;
                }
                if (turn) {
                    T *x = a[k][s].v, *y = b[k][s].v;
                    if (INTERLEAVED) {
#pragma unroll
                        for (int e = 0; e < PAIRS; e++) {
                            const float2 z = pair_of(x + 2 * e);
                            set_pair(x + 2 * e, z.x * w.v[e].x - z.y * w.v[e].y, z.x * w.v[e].y + z.y * w.v[e].x);
                        }
                    } else {
#pragma unroll
                        for (int e = 0; e < PAIRS; e += 2) {             // (neighbours are rounded together)
                            const float2 lo = pair_of(x + e), hi = pair_of(y + e), u = w.v[e], v = w.v[e + 1];
                            set_pair(x + e, lo.x * u.x - hi.x * u.y, lo.y * v.x - hi.y * v.y);
                            set_pair(y + e, lo.x * u.y + hi.x * u.x, lo.y * v.y + hi.y * v.x);
                        }
                    }
                }
                store_vec<WHOLE>(dst, a[k][s], n);
                if (!INTERLEAVED && pairs) store_vec<WHOLE>(dst + p.half, b[k][s], n);
            }
        }
    };
    while (it < head_items) {                                            // (once, but for heads of more places than there are threads)
        for (int h = h0; h < heads;) {
            store(h);
            h += step;
            if (h < heads) load(h);
        }
        it += cols;
        if (it >= head_items) break;
        place();
        load(h0);
    }
}

// Whether all rows start at 16 bytes and their pieces are whole loads.
bool whole(const RotParams& p, const Heads& h, int ve) { return aligned16(h.base) && h.token % ve == 0 && h.head % ve == 0; }

template <typename T, bool APPEND>
int launch_rotary(RotParams& p, bool interleaved, cudaStream_t stream) {
    constexpr int VE = 16 / sizeof(T);
    const int rot = 2 * p.half;
    bool vec = p.dim % VE == 0 && (interleaved ? rot : p.half) % VE == 0 && whole(p, p.in, VE) && whole(p, p.out, VE);
    if (APPEND)
        vec = vec && whole(p, p.k, VE) && whole(p, p.v, VE) && aligned16(p.k_pages) && aligned16(p.v_pages) && p.page_stride % VE == 0 &&
              p.page_head % VE == 0 && p.page_row % VE == 0;
    const int ve = vec ? VE : 2, heads = APPEND ? p.heads + 2 * p.kv_heads : p.heads;
    const int items = ((interleaved ? rot : p.half) + ve - 1) / ve + (p.dim - rot + ve - 1) / ve, sweep = std::max(kRotThreads / items, 1);
    // Two tokens a CTA where there are CTAs enough (4099 tokens in L2 9.2 us, 13.1 by one token a CTA; 600 tokens 3.2 and 3.5); where there are few, the
    // heads of one go to several (16 tokens appended 3.6 us, 4.1 by two tokens a CTA).
    p.per_cta = p.tokens >= 4 * 148 ? kRotTokens : 1;
    const int gy = p.tokens >= 2 * 148 ? 1 : std::min((heads + sweep * kRotSweeps - 1) / (sweep * kRotSweeps), 65535);
    const dim3 grid((p.tokens + p.per_cta - 1) / p.per_cta, gy);
    const size_t smem = sizeof(float2) * p.half * p.per_cta;
    auto go = [&](auto kern) { launch_kernel(kern, grid, dim3(kRotThreads), smem, stream, p); };
    if (vec) {
        if (interleaved) go(rotary_kernel<T, VE, true, true, APPEND>);
        else go(rotary_kernel<T, VE, true, false, APPEND>);
    } else if (interleaved) {
        go(rotary_kernel<T, 2, false, true, APPEND>);
    } else {
        go(rotary_kernel<T, 2, false, false, APPEND>);
    }
    return check_launch();
}

// 1 / 2 pi, and what its rounding left.
constexpr double kTurn = 0x1.45f306dc9c883p-3, kTurnLow = -0x1.6b01ec5417056p-57;
void set_turns(RotParams& p, double scaling) {
    p.turns = scaling * kTurn;
    p.turns_low = std::fma(scaling, kTurn, -p.turns) + scaling * kTurnLow;
}

}  // namespace
}  // namespace b200

extern "C" {

int b200_rotate(const b200_rotary* r, const void* x, long long x_token, long long x_head, void* out, long long out_token, long long out_head,
                int dtype, int tokens, int heads, int dim, void* stream) {
    if (!r || tokens < 0 || heads < 0 || dim < 1 || dim > 2048) return B200_EINVAL;
    if (r->rotary_dim < 2 || (r->rotary_dim & 1) || r->rotary_dim > dim) return B200_EINVAL;
    if (b200::dtype_size(dtype) == 0) return B200_EUNSUPPORTED;
    if (tokens == 0 || heads == 0) return B200_OK;
    if (!x || !out || !r->positions || !r->inv_freqs || heads > 65535) return B200_EINVAL;
    b200::RotParams p{};
    p.in = {static_cast<char*>(const_cast<void*>(x)), x_token, x_head};
    p.out = {static_cast<char*>(out), out_token, out_head};
    p.positions = r->positions; p.pos64 = r->positions_64; p.inv_freqs = r->inv_freqs; b200::set_turns(p, r->scaling);
    p.magnitude = r->magnitude; p.inverse = r->inverse; p.tokens = tokens; p.heads = heads; p.dim = dim; p.half = r->rotary_dim / 2;
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (dtype == B200_DTYPE_F32) return b200::launch_rotary<float, false>(p, r->interleaved, st);
    if (dtype == B200_DTYPE_BF16) return b200::launch_rotary<__nv_bfloat16, false>(p, r->interleaved, st);
    return b200::launch_rotary<__half, false>(p, r->interleaved, st);
}

int b200_paged_append(const b200_paged* c, const b200_rotary* r, const void* q, long long q_token, long long q_head, const void* k, const void* v,
                      long long kv_token, long long kv_head, void* q_out, long long out_token, long long out_head, int prefix_length, void* stream) {
    const int bad = b200::check_paged(c);
    if (bad != B200_OK) return bad;
    if (!r || r->rotary_dim < 2 || (r->rotary_dim & 1) || r->rotary_dim > c->head_dim || prefix_length < 0 || r->inverse) return B200_EINVAL;
    if (c->tokens == 0 || c->requests == 0) return B200_OK;
    if (!q || !k || !v || !q_out || !r->inv_freqs) return B200_EINVAL;
    b200::RotParams p{};
    p.in = {static_cast<char*>(const_cast<void*>(q)), q_token, q_head};
    p.k = {static_cast<char*>(const_cast<void*>(k)), kv_token, kv_head};
    p.v = {static_cast<char*>(const_cast<void*>(v)), kv_token, kv_head};
    p.out = {static_cast<char*>(q_out), out_token, out_head};
    p.k_pages = static_cast<char*>(c->k_pages); p.v_pages = static_cast<char*>(c->v_pages);
    p.page_stride = c->page_stride; p.page_head = c->head_stride; p.page_row = c->row_stride;
    p.positions = r->positions; p.pos64 = r->positions_64; p.inv_freqs = r->inv_freqs; b200::set_turns(p, r->scaling);
    p.magnitude = r->magnitude;
    p.tokens = c->tokens; p.heads = c->heads; p.kv_heads = c->kv_heads; p.dim = c->head_dim; p.half = r->rotary_dim / 2;
    p.table = c->page_table; p.lengths = c->lengths; p.row_starts = c->row_starts; p.table_stride = c->table_stride;
    p.requests = c->requests; p.pages = c->pages; p.page_size = c->page_size; p.table_width = c->table_width; p.prefix = prefix_length;
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (c->dtype == B200_DTYPE_BF16) return b200::launch_rotary<__nv_bfloat16, true>(p, r->interleaved, st);
    return b200::launch_rotary<__half, true>(p, r->interleaved, st);
}

}  // extern "C"
