// Attention over a paged cache behind a prefix that all requests of the pass share, on the fifth-generation tensor cores.
//
//   o = softmax(scale * q [Kp; Kb]^T + mask) [Vp; Vb]:  prefix rows Kp, Vp and the rows Kb, Vb of the token's own request
//
// The softmax is split over its keys: a piece of them gives its maximum m, l = sum exp(s - m) and O = sum exp(s - m) v, and pieces are joined by
// weights exp(m - max m) / sum.  A segment is the prefix with a tile of 128 query rows (token, head of the group) of any requests, or a request's
// own rows with a tile of its tokens; its work is counted in blocks of 128 keys.  All blocks of all segments stand in one line, and every worker takes
// an equal stretch of it, whatever the lengths: at most one piece a worker begins inside a segment, so a segment's first piece has its place by
// (token, head) and the others theirs by worker.  A second kernel joins them.
//
// One CTA an SM, two workers (streams) a CTA: four warps each, a query row a thread, its scores and output in tensor memory (128 + 128 columns).  The
// streams' blocks alternate, so that one's products run while the other's softmax does.  Where the prefix has two tiles of queries or more, the
// CTA takes them in pairs, a tile a stream, over the same blocks: keys and values are then copied once for 256 rows.  Keys and values come page
// by page (TMA, boxes of a page or 128 rows) into one ring in the order in which they are used.
//
// Probabilities are at most one and rounded to the type of V for the second product; scores, statistics, sums and outputs are fp32.
// Every wait is bounded; one that runs out sets the error word and goes on.  No copy uses cluster multicast.
#include <algorithm>
#include <atomic>
#include <type_traits>

#include "paged.cuh"
#include "pipeline.cuh"
#include "tensor_map.cuh"
#include "umma.cuh"

namespace b200 {
namespace {

constexpr int kKeys = 128;                       // of a block
constexpr int kRows = 128;                       // query rows of a tile
constexpr int kPgThreads = 384;                  // 2 x 4 softmax warps, keys and values, products, queries of either stream
constexpr int kPgMaxRequests = 1024;
constexpr int kLoader = 8, kIssuer = 9, kQueries = 10;

template <int HD>
struct PGeo {
    static constexpr int QTILE = kRows * HD * 2, SLOT = kKeys * HD * 2, SLOTS = HD == 128 ? 4 : 8;
    static constexpr int KV0 = 2 * QTILE, END = KV0 + SLOTS * SLOT;
    static constexpr int SMEM = END + 1024;
};

struct PagedParams {
    CUtensorMap qmap, q1map, kmap, vmap;         // queries by tile and by token, pages
    const int *table, *lengths, *row_starts, *prefix_pages;
    const unsigned long long* mask;
    void* out;
    float *first_prefix, *first_own, *more_pair, *more;      // pieces [..][HD]
    float2* ml;                                  // (m, l) in the order of the pieces
    int* plan;                                   // sums of the own blocks, by request
    long long table_stride, out_token, out_head;
    int requests, tokens, heads, kv_heads, group, tile_heads, tile_tokens, head_sets;
    int page_size, box_rows, table_width, prefix;
    float scale_log2;                            // positive
    bool negative;                               // ... of a negative scale
    int* err;
    int polls;
};

// The line of blocks.
struct Line {
    int nbp;                                     // blocks of the prefix
    int tiles, pairs;                            // query tiles of the prefix, per kv head
    int odd;                                     // blocks of prefix segments without a partner
    long long pair_total, total;                 // blocks for pairs; for single streams: odd ones, then own ones
};
__device__ __forceinline__ Line line_of(const PagedParams& p, long long own) {
    Line l;
    l.nbp = (p.prefix + kKeys - 1) / kKeys;
    l.tiles = (p.tokens + p.tile_tokens - 1) / p.tile_tokens * p.head_sets;
    l.pairs = l.tiles / 2;
    l.odd = l.tiles & 1 ? p.kv_heads * l.nbp : 0;
    l.pair_total = (long long)p.kv_heads * l.pairs * l.nbp;
    l.total = l.odd + own;
    return l;
}
// Stretch of worker i of n.
__device__ __forceinline__ long long stretch(long long total, int i, int n) { return total * i / n; }
// The worker of n whose stretch holds block w.
__device__ __forceinline__ int worker_of(long long total, long long w, int n) { return (int)(((w + 1) * n - 1) / total); }

struct Request {
    int start, count, length, blocks, tiles;
};
__device__ __forceinline__ Request request_of(const PagedParams& p, int b) {
    Request r;
    const int s0 = p.row_starts[b], s1 = p.row_starts[b + 1], len = p.lengths[b];
    r.start = min(max(s0, 0), p.tokens);
    r.count = min(max(s1 - r.start, 0), p.tokens - r.start);
    r.length = (int)min((long long)max(len, 0), (long long)p.table_width * p.page_size);
    r.blocks = (r.length + kKeys - 1) / kKeys;
    r.tiles = (r.count + p.tile_tokens - 1) / p.tile_tokens * p.head_sets;
    return r;
}

struct Piece {
    int req;                                     // -1: the prefix
    int tok0, toks, hs, hk;
    int kb0, kb1, length;
    int old;                                     // rows ahead of the pass's (own segments)
};
// The piece of block w of the line of single streams, up to `end`; cum: own blocks ahead of each request.
__device__ __forceinline__ void tile_tokens(const PagedParams& p, int tile, int start, int count, Piece& c) {
    const int ts = tile / p.head_sets;
    c.hs = tile - ts * p.head_sets;
    c.tok0 = start + ts * p.tile_tokens;
    c.toks = min(p.tile_tokens, count - ts * p.tile_tokens);
}
__device__ __forceinline__ Piece piece_of_pair(const PagedParams& p, const Line& l, int w, int end, int s) {
    Piece c;
    const int seg = w / l.nbp;
    c.req = -1;
    c.kb0 = w - seg * l.nbp;
    c.kb1 = min(l.nbp, c.kb0 + end - w);
    c.hk = seg / l.pairs;
    c.length = p.prefix;
    c.old = p.prefix;
    tile_tokens(p, 2 * (seg - c.hk * l.pairs) + s, 0, p.tokens, c);
    return c;
}
__device__ __forceinline__ Piece piece_of(const PagedParams& p, const Line& l, const int* cum, int w, int end) {
    Piece c;
    if (w < l.odd) {
        c.req = -1;
        c.hk = w / l.nbp;
        c.kb0 = w - c.hk * l.nbp;
        c.kb1 = min(l.nbp, c.kb0 + end - w);
        c.length = p.prefix;
        c.old = p.prefix;
        tile_tokens(p, l.tiles - 1, 0, p.tokens, c);
        return c;
    }
    const int v = w - l.odd;
    int lo = 0, hi = p.requests;                 // the last request that begins at v or before
    while (hi - lo > 1) {
        const int mid = (lo + hi) / 2;
        if (cum[mid] <= v) lo = mid;
        else hi = mid;
    }
    const Request r = request_of(p, lo);
    const int in = v - cum[lo], seg = in / r.blocks, tile = seg / p.kv_heads;
    c.req = lo;
    c.hk = seg - tile * p.kv_heads;
    c.kb0 = in - seg * r.blocks;
    c.kb1 = min(r.blocks, c.kb0 + end - w);
    c.length = r.length;
    c.old = p.lengths[lo] - (p.row_starts[lo + 1] - p.row_starts[lo]);
    tile_tokens(p, tile, r.start, r.count, c);
    return c;
}

__device__ __forceinline__ uint64_t sw128_desc_n_major(uint32_t saddr, uint32_t box) {      // V: keys by dims, the next 64 dims `box` bytes on
    return (uint64_t)((saddr & 0x3ffffu) >> 4) | ((uint64_t)(box >> 4) << 16) | ((uint64_t)(1024 >> 4) << 32) | ((uint64_t)1 << 46) |
           ((uint64_t)2 << 61);
}
__device__ __forceinline__ void tma_box3(uint32_t dst, const void* tmap, int x, int y, int z, uint32_t bar) {
    asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];\n"
                 ::"r"(dst), "l"(tmap), "r"(x), "r"(y), "r"(z), "r"(bar) : "memory");
}
__device__ __forceinline__ void tma_box4(uint32_t dst, const void* tmap, int x, int y, int z, int w, uint32_t bar) {
    asm volatile("cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];\n"
                 ::"r"(dst), "l"(tmap), "r"(x), "r"(y), "r"(z), "r"(w), "r"(bar) : "memory");
}
__device__ __forceinline__ float exp2_approx(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ void tmem_ld32(uint32_t* r, uint32_t addr) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,"
                 "%28,%29,%30,%31}, [%32];\n"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]),
                   "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]),
                   "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]),
                   "=r"(r[31]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void tmem_st32(uint32_t addr, const uint32_t* r) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,"
                 "%28,%29,%30,%31,%32};\n" ::"r"(addr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]),
                 "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]),
                 "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]),
                 "r"(r[31]) : "memory");
}
__device__ __forceinline__ void tmem_st8(uint32_t addr, const uint32_t* r) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};\n" ::"r"(addr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]),
                 "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]) : "memory");
}
__device__ __forceinline__ uint32_t pack2(float lo, float hi, __half*) { return h2_as_u32(__floats2half2_rn(lo, hi)); }
__device__ __forceinline__ uint32_t pack2(float lo, float hi, __nv_bfloat16*) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
}

template <typename T, int HD>
__global__ void __launch_bounds__(kPgThreads, 1) paged_kernel(const __grid_constant__ PagedParams p) {
    using G = PGeo<HD>;
    constexpr int ST = G::SLOTS, NB = HD / 64;
    extern __shared__ unsigned char smem_raw[];
    unsigned char* smem = smem_raw + ((0u - smem_u32(smem_raw)) & 1023u);
    __shared__ uint64_t full[ST], freed[ST], qfull[2], qfree[2], sfull[2], pready[2], pvdone[2];
    __shared__ uint32_t s_tmem;
    __shared__ int s_cum[kPgMaxRequests + 1];
    __shared__ long long s_warp[kPgThreads / 32], s_total;
    const uint32_t sbase = smem_u32(smem);
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, ctas = gridDim.x, cta = blockIdx.x;

    if (threadIdx.x == 0) {
        asm volatile("prefetch.tensormap [%0];\n" ::"l"(&p.kmap) : "memory");
        asm volatile("prefetch.tensormap [%0];\n" ::"l"(&p.vmap) : "memory");
        asm volatile("prefetch.tensormap [%0];\n" ::"l"(&p.qmap) : "memory");
        asm volatile("prefetch.tensormap [%0];\n" ::"l"(&p.q1map) : "memory");
        for (int s = 0; s < ST; s++) {
            mbar_init(smem_u32(full + s), 1);
            mbar_init(smem_u32(freed + s), 1);
        }
        for (int s = 0; s < 2; s++) {
            mbar_init(smem_u32(qfull + s), 1);
            mbar_init(smem_u32(qfree + s), 1);
            mbar_init(smem_u32(sfull + s), 1);
            mbar_init(smem_u32(pready + s), 4);
            mbar_init(smem_u32(pvdone + s), 1);
        }
        asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
    }
    if (warp == kIssuer) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;\n" ::"r"(smem_u32(&s_tmem)) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;\n" ::: "memory");
    }
    asm volatile("tcgen05.fence::before_thread_sync;\n" ::: "memory");
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory");
    const uint32_t tmem = s_tmem;
    pdl_launch_dependents();
    pdl_wait();

    // ---- own blocks ahead of each request: consecutive requests a thread, then a scan (a line beyond 2^30 blocks is cut there)
    {
        const int per = (p.requests + kPgThreads - 1) / kPgThreads, b0 = min((int)threadIdx.x * per, p.requests), b1 = min(b0 + per, p.requests);
        long long mine = 0, before;
        for (int b = b0; b < b1; b++) {
            const Request r = request_of(p, b);
            mine += (long long)r.blocks * r.tiles * p.kv_heads;
        }
        long long scan = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const long long other = __shfl_up_sync(0xffffffffu, scan, o);
            if (lane >= o) scan += other;
        }
        if (lane == 31) s_warp[warp] = scan;
        __syncthreads();
        before = scan - mine;
        for (int w = 0; w < warp; w++) before += s_warp[w];
        for (int b = b0; b < b1; b++) {
            s_cum[b] = (int)min(before, 1ll << 30);
            const Request r = request_of(p, b);
            before += (long long)r.blocks * r.tiles * p.kv_heads;
        }
        if (threadIdx.x == kPgThreads - 1) {
            s_cum[p.requests] = (int)min(before, 1ll << 30);
            s_total = s_cum[p.requests];
        }
        __syncthreads();
    }
    if (cta == 0)
        for (int b = threadIdx.x; b <= p.requests; b += kPgThreads) p.plan[b] = s_cum[b];
    const Line l = line_of(p, s_total);
    // This CTA's stretch of the pairs, and its streams' of the rest.
    const int a0 = (int)stretch(l.pair_total, cta, ctas), a1 = (int)stretch(l.pair_total, cta + 1, ctas);
    const int w0 = (int)stretch(l.total, 2 * cta, 2 * ctas), w1 = (int)stretch(l.total, 2 * cta + 1, 2 * ctas), w2 = (int)stretch(l.total, 2 * cta + 2, 2 * ctas);
    const int from[2] = {w0, w1}, to[2] = {w1, w2};

    if (warp == kLoader) {
        // ------------------------------------------------------------------ keys and values, in the order of their use
        asm volatile("fence.proxy.async;\n" ::: "memory");               // (appended by ordinary stores of an earlier kernel)
        int ring = 0;
        struct At {
            int w, end, hk, kb, kb1, req, length, page, row, boxes;
        } at[2];
        auto open = [&](At& x, const Piece& c) {
            x.hk = c.hk; x.kb = c.kb0; x.kb1 = c.kb1; x.req = c.req; x.length = c.length;
        };
        // pages of the cursor's block: a lane each, or the one that holds all of it
        auto pages = [&](At& x) {
            const int key0 = x.kb * kKeys, rows = min(kKeys, x.length - key0);
            x.boxes = (rows + p.box_rows - 1) / p.box_rows;
            x.row = p.page_size > kKeys ? key0 % p.page_size : 0;
            const int index = key0 / p.page_size + lane;
            if (lane < x.boxes) x.page = x.req < 0 ? p.prefix_pages[index] : p.table[x.req * p.table_stride + index];
        };
        auto load = [&](const At& x, const CUtensorMap* map) {
            const int slot = ring % ST;
            if (ring >= ST) mbar_wait_reported(smem_u32(freed + slot), (ring / ST - 1) & 1, p.polls, p.err, 31);
            __syncwarp();
            const uint32_t bar = smem_u32(full + slot), dst = sbase + G::KV0 + slot * G::SLOT;
            if (elect_one()) mbar_expect_tx(bar, x.boxes * p.box_rows * HD * 2);
            __syncwarp();
            if (lane < x.boxes) {
#pragma unroll
                for (int h = 0; h < NB; h++)
                    tma_box4(dst + h * (kKeys * 128) + lane * p.box_rows * 128, map, h * 64, x.row, x.hk, x.page, bar);
            }
            __syncwarp();
            ring++;
        };
        // pairs
        {
            At& x = at[0];
            for (int w = a0; w < a1;) {
                const Piece c = piece_of_pair(p, l, w, a1, 0);
                open(x, c);
                for (; x.kb < x.kb1; x.kb++) {
                    pages(x);
                    load(x, &p.kmap);
                    load(x, &p.vmap);
                }
                w += c.kb1 - c.kb0;
            }
        }
        // single streams: K a block ahead of V
        auto next = [&](At& x) {                                         // the cursor's block, its pages
            if (x.kb == x.kb1) open(x, piece_of(p, l, s_cum, x.w, x.end));
            pages(x);
            load(x, &p.kmap);
            x.w++;
            x.kb++;
        };
#pragma unroll
        for (int s = 0; s < 2; s++) {
            at[s].w = from[s];
            at[s].end = to[s];
            at[s].kb = at[s].kb1 = 0;
            if (at[s].w < at[s].end) next(at[s]);
        }
        for (int i = 0; i < max(w1 - w0, w2 - w1); i++) {
#pragma unroll
            for (int s = 0; s < 2; s++) {
                if (i >= to[s] - from[s]) continue;
                load(at[s], &p.vmap);
                if (at[s].w < at[s].end) next(at[s]);
            }
        }
    } else if (warp == kIssuer) {
        // ------------------------------------------------------------------ products
        constexpr bool BF = std::is_same<T, __nv_bfloat16>::value;
        constexpr uint32_t base = (1u << 4) | ((uint32_t)(kRows >> 4) << 24) | (BF ? (1u << 7) | (1u << 10) : 0u);
        constexpr uint32_t idesc_o = base | (1u << 16) | ((uint32_t)(HD >> 3) << 17);
        const uint64_t qdesc = sw128_desc(sbase), kdesc = sw128_desc(sbase + G::KV0), vdesc = sw128_desc_n_major(sbase + G::KV0, kKeys * 128);
        int ring = 0;
        int blocks[2] = {0, 0}, pieces[2] = {0, 0};                      // scores asked for, pieces begun
        struct At {
            int w, end, kb, kb1, length;
            int keys;                                                    // of the block whose scores were asked for last
            bool first, last;                                            // ... of its piece
        } at[2];
        // Scores of the cursor's block of stream s.
        auto scores = [&](int s, At& x, bool take, bool give) {
            const int slot = ring % ST;
            if (take) {
                mbar_wait_reported(smem_u32(full + slot), (ring / ST) & 1, p.polls, p.err, 31);
            }
            if (x.first) {
                mbar_wait_reported(smem_u32(qfull + s), pieces[s] & 1, p.polls, p.err, 31);
                pieces[s]++;
            }
            if (blocks[s] > 0) mbar_wait_reported(smem_u32(pvdone + s), (blocks[s] - 1) & 1, p.polls, p.err, 31);      // (probabilities where the scores go)
            asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory");
            __syncwarp();
            if (elect_one()) {
                const uint32_t d = tmem + s * kKeys, idesc = base | ((uint32_t)((x.keys + 15) / 16 * 2) << 17);
                const uint64_t q0 = qdesc + s * (G::QTILE / 16), k0 = kdesc + slot * (G::SLOT / 16);
#pragma unroll
                for (int ks = 0; ks < HD / 16; ks++)
                    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(d),
                                 "l"(q0 + (ks >> 2) * (kRows * 128 / 16) + (ks & 3) * 2), "l"(k0 + (ks >> 2) * (kKeys * 128 / 16) + (ks & 3) * 2), "r"(idesc),
                                 "r"(ks) : "memory");
                commit_to(smem_u32(sfull + s));
                if (give) commit_to(smem_u32(freed + slot));
                if (x.last) commit_to(smem_u32(qfree + s));
            }
            __syncwarp();
            blocks[s]++;
            if (give) ring++;
        };
        // Output of the block whose scores stream s asked for last.
        auto output = [&](int s, const At& x, bool take, bool give) {
            const int slot = ring % ST;
            const int steps = (x.keys + 15) / 16;
            if (take) {
                mbar_wait_reported(smem_u32(full + slot), (ring / ST) & 1, p.polls, p.err, 31);
                if (x.keys & 15) {
                    // Rows behind the last, up to the step of the product: whatever is there has probability 0, and 0 x Inf or NaN would be NaN.
                    const uint32_t v = sbase + G::KV0 + slot * G::SLOT;
                    for (int k = x.keys * 8 + lane; k < steps * 16 * 8; k += 32)
#pragma unroll
                        for (int h = 0; h < NB; h++)
                            asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};\n" ::"r"(v + h * (kKeys * 128) + k * 16), "r"(0) : "memory");
                    fence_proxy_async();
                    __syncwarp();
                }
            }
            mbar_wait_reported(smem_u32(pready + s), (blocks[s] - 1) & 1, p.polls, p.err, 31);
            asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory");
            __syncwarp();
            if (elect_one()) {
                const uint64_t v0 = vdesc + slot * (G::SLOT / 16);
                const uint32_t d = tmem + 2 * kKeys + s * HD, a0 = tmem + s * kKeys;
                for (int ks = 0; ks < steps; ks++)
                    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}\n" ::"r"(d),
                                 "r"(a0 + ks * 8), "l"(v0 + ks * (2048 / 16)), "r"(idesc_o), "r"((x.first ? 0 : 1) + ks) : "memory");
                if (give) commit_to(smem_u32(freed + slot));
                commit_to(smem_u32(pvdone + s));                         // (the last thing that a CTA's end waits for)
            }
            __syncwarp();
            if (give) ring++;
        };
        auto enter = [&](At& x) {
            x.first = x.kb == x.kb1;
        };
        auto block = [&](At& x, int kb) {                                // the cursor stands before block kb
            x.keys = min(kKeys, x.length - kb * kKeys);
            x.last = kb + 1 == x.kb1;
            x.kb = kb + 1;
            x.w++;
        };
        auto pair_next = [&](At& x) {
            enter(x);
            if (x.first) {
                const Piece c = piece_of_pair(p, l, x.w, a1, 0);
                x.kb = c.kb0;
                x.kb1 = c.kb1;
                x.length = c.length;
            }
            block(x, x.kb);
        };
        auto next = [&](At& x) {
            enter(x);
            if (x.first) {
                const Piece c = piece_of(p, l, s_cum, x.w, x.end);
                x.kb = c.kb0;
                x.kb1 = c.kb1;
                x.length = c.length;
            }
            block(x, x.kb);
        };
        if (a0 < a1) {
            At x, y;                                                     // the block whose output is next; the one whose scores are
            x.w = a0;
            x.kb = x.kb1 = 0;
            pair_next(x);
            scores(0, x, true, false);
            scores(1, x, false, true);
            for (int i = a0; i < a1; i++) {
                // (V of this block stands ahead of the next block's K in the ring: `ring` is V's)
                y = x;
                const bool more = i + 1 < a1;
                if (more) pair_next(y);
                output(0, x, true, false);
                if (more) {
                    ring++;
                    scores(0, y, true, false);
                    ring--;
                }
                output(1, x, false, true);
                if (more) scores(1, y, false, true);
                x = y;
            }
        }
#pragma unroll
        for (int s = 0; s < 2; s++) {
            at[s].w = from[s];
            at[s].end = to[s];
            at[s].kb = at[s].kb1 = 0;
            if (at[s].w < at[s].end) {
                next(at[s]);
                scores(s, at[s], true, true);
            }
        }
        for (int i = 0; i < max(w1 - w0, w2 - w1); i++) {
#pragma unroll
            for (int s = 0; s < 2; s++) {
                if (i >= to[s] - from[s]) continue;
                output(s, at[s], true, true);
                if (at[s].w < at[s].end) {
                    next(at[s]);
                    scores(s, at[s], true, true);
                }
            }
        }
    } else if (warp >= kQueries) {
        // ------------------------------------------------------------------ queries of stream s, a piece ahead of nobody: once the last piece's scores are done
        asm volatile("fence.proxy.async;\n" ::: "memory");
        const int s = warp - kQueries;
        int piece = 0;
        auto load = [&](const Piece& c) {
            if (piece > 0) mbar_wait_reported(smem_u32(qfree + s), (piece - 1) & 1, p.polls, p.err, 31);
            __syncwarp();
            if (elect_one()) {
                const uint32_t bar = smem_u32(qfull + s), dst = sbase + s * G::QTILE;
                const int head = c.hk * p.group + c.hs * p.tile_heads;
                if (c.toks <= 4) {                                       // (a box of the whole tile would bring 128 rows)
                    mbar_expect_tx(bar, c.toks * p.tile_heads * HD * 2);
                    for (int t = 0; t < c.toks; t++)
#pragma unroll
                        for (int h = 0; h < NB; h++)
                            tma_box3(dst + h * (kRows * 128) + t * p.tile_heads * 128, &p.q1map, h * 64, head, c.tok0 + t, bar);
                } else {
                    mbar_expect_tx(bar, p.tile_tokens * p.tile_heads * HD * 2);
#pragma unroll
                    for (int h = 0; h < NB; h++) tma_box3(dst + h * (kRows * 128), &p.qmap, h * 64, head, c.tok0, bar);
                }
            }
            __syncwarp();
            piece++;
        };
        for (int w = a0; w < a1;) {
            const Piece c = piece_of_pair(p, l, w, a1, s);
            load(c);
            w += c.kb1 - c.kb0;
        }
        for (int w = from[s]; w < to[s];) {
            const Piece c = piece_of(p, l, s_cum, w, to[s]);
            load(c);
            w += c.kb1 - c.kb0;
        }
    } else {
        // ------------------------------------------------------------------ softmax: a query row a thread
        const int s = warp >> 2, r = (warp & 3) * 32 + lane;
        const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16, tS = tmem + s * kKeys + lanes, tO = tmem + 2 * kKeys + s * HD + lanes;
        const int dt = r / p.tile_heads;
        int blocks = 0;
        auto run = [&](const Piece& c, bool pair, int worker) {
            const int rows = c.toks * p.tile_heads, g = c.hs * p.tile_heads + r - dt * p.tile_heads, t = c.tok0 + dt;
            const bool valid = dt < c.toks && g < p.group, busy = (warp & 3) * 32 < rows;      // (busy: some row of the warp may be)
            // The first key that this row does not see by its place; the new rows it sees by mask.
            const bool masked = c.req >= 0 && p.mask != nullptr;
            int limit = c.length;
            unsigned long long bits = 0;
            if (c.req >= 0) {
                limit = min(limit, masked ? c.old : c.old + (t - p.row_starts[c.req]) + 1);
                if (masked && valid) bits = p.mask[t];
            }
            const int sure = c.req < 0 ? c.length : c.old;               // keys up to here are seen by all rows
            float m = -INFINITY, sum = 0.f;
#pragma unroll 1
            for (int kb = c.kb0; kb < c.kb1; kb++, blocks++) {
                mbar_wait_reported(smem_u32(sfull + s), blocks & 1, p.polls, p.err, 31);
                __syncwarp();
                asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory");
                if (busy) {
                    uint32_t raw[kKeys];
#pragma unroll
                    for (int j = 0; j < kKeys; j += 32) tmem_ld32(raw + j, tS + j);
                    asm volatile("tcgen05.wait::ld.sync.aligned;\n" ::: "memory");
                    const int key0 = kb * kKeys;
                    if (p.negative) {
#pragma unroll
                        for (int j = 0; j < kKeys; j++) raw[j] ^= 0x80000000u;
                    }
                    if (key0 + kKeys > sure || key0 + kKeys > c.length) {
#pragma unroll
                        for (int w = 0; w < kKeys / 32; w++) {
                            const int n = limit - key0 - 32 * w, o = key0 + 32 * w - c.old;      // keys of the word ahead of the limit; first key's new row
                            uint32_t seen = n >= 32 ? 0xffffffffu : (n <= 0 ? 0u : (1u << n) - 1u);
                            if (masked && o > -32 && o < 64) {
                                uint32_t x = (uint32_t)(o >= 0 ? bits >> o : bits << -o);
                                const int there = c.length - key0 - 32 * w;
                                if (there < 32) x &= there <= 0 ? 0u : (1u << there) - 1u;
                                seen |= x;
                            }
#pragma unroll
                            for (int j = 0; j < 32; j++)
                                if (!((seen >> j) & 1u)) raw[32 * w + j] = 0xff800000u;
                        }
                    }
                    float x[4];
#pragma unroll
                    for (int j = 0; j < 4; j++) x[j] = fmaxf(__uint_as_float(raw[j]), __uint_as_float(raw[4 + j]));
#pragma unroll
                    for (int j = 8; j < kKeys; j++) x[j & 3] = fmaxf(x[j & 3], __uint_as_float(raw[j]));
                    const float top = fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])) * p.scale_log2;
                    const bool grown = top > m;
                    const float al = !grown ? 1.f : (m == -INFINITY ? 0.f : exp2_approx(m - top));
                    if (grown) m = top;
                    const float ref = m == -INFINITY ? 0.f : -m;
                    if (__any_sync(0xffffffffu, grown && valid) && kb > c.kb0) {
                        // (the block before has been added: its product was waited for ahead of these scores)
#pragma unroll
                        for (int d = 0; d < HD; d += 16) {               // (few at a time: the scores stand in 128 registers)
                            uint32_t o[16];
                            tmem_ld<16>(o, tO + d);
                            asm volatile("tcgen05.wait::ld.sync.aligned;\n" ::: "memory");
#pragma unroll
                            for (int j = 0; j < 16; j++) o[j] = __float_as_uint(__uint_as_float(o[j]) * al);
                            tmem_st8(tO + d, o);
                            tmem_st8(tO + d + 8, o + 8);
                        }
                    }
                    float part[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int j = 0; j < kKeys; j += 2) {
                        const float e0 = exp2_approx(fmaf(__uint_as_float(raw[j]), p.scale_log2, ref)), e1 = exp2_approx(fmaf(__uint_as_float(raw[j + 1]), p.scale_log2, ref));
                        part[j & 2] += e0;
                        part[(j & 2) + 1] += e1;
                        raw[j / 2] = pack2(e0, e1, (T*)nullptr);
                    }
                    tmem_st32(tS, raw);
                    tmem_st32(tS + 32, raw + 32);
                    sum = sum * al + ((part[0] + part[1]) + (part[2] + part[3]));
                    asm volatile("tcgen05.wait::st.sync.aligned;\n" ::: "memory");
                }
                asm volatile("tcgen05.fence::before_thread_sync;\n" ::: "memory");
                __syncwarp();
                if (lane == 0) mbar_arrive(smem_u32(pready + s));
            }
            // ---- the piece's state -> its place
            mbar_wait_reported(smem_u32(pvdone + s), (blocks - 1) & 1, p.polls, p.err, 31);
            __syncwarp();
            asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory");
            if (busy) {
                const long long row = (long long)t * p.heads + c.hk * p.group + g, all = (long long)p.tokens * p.heads;
                float* dst;
                long long at;
                if (c.kb0 == 0) {
                    dst = (c.req < 0 ? p.first_prefix : p.first_own) + row * HD;
                    at = (c.req < 0 ? 0 : all) + row;
                } else if (pair) {
                    dst = p.more_pair + ((long long)worker * 2 * kRows + s * kRows + r) * HD;
                    at = 2 * all + (long long)worker * 2 * kRows + s * kRows + r;
                } else {
                    dst = p.more + ((long long)worker * kRows + r) * HD;
                    at = 2 * all + (long long)ctas * 2 * kRows + (long long)worker * kRows + r;
                }
                if (valid) p.ml[at] = make_float2(m, sum);
#pragma unroll
                for (int d = 0; d < HD; d += 32) {
                    uint32_t o[32];
                    tmem_ld32(o, tO + d);
                    asm volatile("tcgen05.wait::ld.sync.aligned;\n" ::: "memory");
                    if (valid) {
#pragma unroll
                        for (int j = 0; j < 32; j += 4) *reinterpret_cast<uint4*>(dst + d + j) = make_uint4(o[j], o[j + 1], o[j + 2], o[j + 3]);
                    }
                }
                asm volatile("tcgen05.fence::before_thread_sync;\n" ::: "memory");
            }
        };
        for (int w = a0; w < a1;) {
            const Piece c = piece_of_pair(p, l, w, a1, s);
            run(c, true, cta);
            w += c.kb1 - c.kb0;
        }
        for (int w = from[s]; w < to[s];) {
            const Piece c = piece_of(p, l, s_cum, w, to[s]);
            run(c, false, 2 * cta + s);
            w += c.kb1 - c.kb0;
        }
    }
    asm volatile("tcgen05.fence::before_thread_sync;\n" ::: "memory");
    __syncthreads();
    if (warp == kIssuer) {
        asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory");
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;\n" ::"r"(tmem) : "memory");
    }
}

// A warp joins the pieces of one query row.  `ctas` is the grid of the kernel above.
template <typename T, int HD>
__global__ void __launch_bounds__(128) paged_join_kernel(const __grid_constant__ PagedParams p, int ctas) {
    pdl_launch_dependents();
    pdl_wait();
    constexpr int N = HD / 32;
    const int lane = threadIdx.x & 31, head = blockIdx.y * 4 + (threadIdx.x >> 5), t = blockIdx.x;
    if (head >= p.heads) return;
    if (t < p.row_starts[0] || t >= p.row_starts[p.requests]) return;
    int lo = 0, hi = p.requests;
    while (hi - lo > 1) {
        const int step = (hi - lo + 31) / 32, at = lo + (lane + 1) * step;
        const int n = __popc(__ballot_sync(0xffffffffu, at < hi && p.row_starts[at] <= t));
        lo += n * step;
        hi = min(hi, lo + step);
    }
    const Request q = request_of(p, lo);
    const Line l = line_of(p, p.plan[p.requests]);
    const int hk = head / p.group, g = head - hk * p.group, hs = g / p.tile_heads, in = g - hs * p.tile_heads;
    const long long row = (long long)t * p.heads + head, all = (long long)p.tokens * p.heads;
    float m = -INFINITY, sum = 0.f, o[N] = {};
    auto add = [&](const float* src, float2 x) {
        if (x.x == -INFINITY) return;
        const float top = fmaxf(m, x.x), a = exp2_approx(m - top), b = exp2_approx(x.x - top);
        sum = sum * a + x.y * b;
#pragma unroll
        for (int e = 0; e < N; e++) o[e] = o[e] * a + src[lane * N + e] * b;
        m = top;
    };
    auto pieces = [&](long long total, long long start, int blocks, int workers, const float* first, long long first_ml, const float* more, long long more_ml,
                      int rows, int r) {
        if (blocks == 0) return;
        add(first + row * HD, p.ml[first_ml + row]);
        const int last = worker_of(total, start + blocks - 1, workers);
        for (int w = worker_of(total, start, workers) + 1; w <= last; w++)
            if (stretch(total, w, workers) < stretch(total, w + 1, workers)) {
                const long long at = (long long)w * rows + r;
                add(more + at * HD, p.ml[more_ml + at]);
            }
    };
    {
        const int ts = t / p.tile_tokens, tile = ts * p.head_sets + hs, r = (t - ts * p.tile_tokens) * p.tile_heads + in;
        if (tile < 2 * l.pairs)
            pieces(l.pair_total, ((long long)hk * l.pairs + tile / 2) * l.nbp, l.nbp, ctas, p.first_prefix, 0, p.more_pair, 2 * all, 2 * kRows, (tile & 1) * kRows + r);
        else
            pieces(l.total, (long long)hk * l.nbp, l.nbp, 2 * ctas, p.first_prefix, 0, p.more, 2 * all + (long long)ctas * 2 * kRows, kRows, r);
    }
    {
        const int dt = t - q.start, ts = dt / p.tile_tokens, tile = ts * p.head_sets + hs, r = (dt - ts * p.tile_tokens) * p.tile_heads + in;
        pieces(l.total, l.odd + p.plan[lo] + ((long long)tile * p.kv_heads + hk) * q.blocks, q.blocks, 2 * ctas, p.first_own, all, p.more,
               2 * all + (long long)ctas * 2 * kRows, kRows, r);
    }
    const float inv = sum > 0.f ? 1.f / sum : 0.f;
    T* dst = static_cast<T*>(p.out) + t * p.out_token + head * p.out_head + lane * N;
#pragma unroll
    for (int e = 0; e < N; e++) dst[e] = from_f32<T>(sum == 0.f ? 0.f : o[e] * inv);
}

struct Room {
    size_t prefix, own, pair, more, ml, plan, total;                     // byte offsets
    int ctas;
};
Room room_of(const b200_paged* c, int ctas) {
    Room r{};
    const size_t all = (size_t)c->tokens * c->heads, row = (size_t)c->head_dim * 4, pair = (size_t)ctas * 2 * kRows, more = (size_t)2 * ctas * kRows;
    r.ctas = ctas;
    r.own = all * row;
    r.pair = r.own + all * row;
    r.more = r.pair + pair * row;
    r.ml = r.more + more * row;
    r.plan = r.ml + (2 * all + pair + more) * sizeof(float2);
    r.total = r.plan + (c->requests + 1) * sizeof(int);
    r.total = (r.total + 15) / 16 * 16;
    return r;
}
int grid_ctas() {
    static std::atomic<int> known[64];
    int dev = 0, n = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 0;
    n = known[dev].load(std::memory_order_relaxed);
    if (n == 0 && cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) == cudaSuccess) known[dev].store(n, std::memory_order_relaxed);
    return n;
}

template <typename T, int HD>
int launch_paged(const PagedParams& p, int ctas, cudaStream_t stream) {
    auto kern = paged_kernel<T, HD>;
    static std::atomic<uint64_t> done{0};
    if (!allow_smem(kern, PGeo<HD>::SMEM, done)) return check_launch();
    const int rc = launch_chain(kern, dim3(ctas), kPgThreads, PGeo<HD>::SMEM, 1, stream, p);
    if (rc != B200_OK) return rc;
    launch_kernel(paged_join_kernel<T, HD>, dim3(p.tokens, (p.heads + 3) / 4), dim3(128), 0, stream, p, ctas);
    return check_launch();
}

// Strides of a dimension of one element are of no consequence, and not always such as a tensor map takes.
uint64_t stride_bytes(long long elements, long long size, int row) { return (uint64_t)(size > 1 ? elements : row) * 2; }

}  // namespace
}  // namespace b200

extern "C" {

size_t b200_paged_attention_workspace_bytes(const b200_paged* c) {
    if (b200::check_paged(c) != B200_OK) return 0;
    return b200::room_of(c, 148).total;
}

int b200_paged_attention(const b200_paged* c, const void* q, long long q_token, long long q_head, void* out, long long out_token, long long out_head,
                         const int* prefix_pages, int prefix_length, const unsigned long long* mask, float scale, void* workspace,
                         size_t workspace_bytes, int* error, void* stream) {
    using namespace b200;
    const int bad = check_paged(c);
    if (bad != B200_OK) return bad;
    if ((c->head_dim != 64 && c->head_dim != 128) || prefix_length < 0 || (prefix_length > 0 && !prefix_pages)) return B200_EINVAL;
    if ((c->page_size < 128 && (c->page_size < 8 || (c->page_size & (c->page_size - 1)))) || (c->page_size > 128 && c->page_size % 128)) return B200_EINVAL;
    if (c->requests > kPgMaxRequests) return B200_ELIMIT;
    if (c->tokens == 0 || c->requests == 0) return B200_OK;
    if (!q || !out || !workspace || !error) return B200_EINVAL;
    if (workspace_bytes < b200_paged_attention_workspace_bytes(c)) return B200_EWORKSPACE;
    if (!aligned16(q) || !aligned16(out) || !aligned16(c->k_pages) || !aligned16(c->v_pages) || !aligned16(workspace)) return B200_EALIGN;
    if (q_token % 8 || q_head % 8 || out_token % 8 || out_head % 8 || c->page_stride % 8 || c->head_stride % 8 || c->row_stride % 8) return B200_EALIGN;

    PagedParams p{};
    p.group = c->heads / c->kv_heads;
    p.tile_heads = std::min(p.group, kRows);
    p.tile_tokens = kRows / p.tile_heads;
    p.head_sets = (p.group + p.tile_heads - 1) / p.tile_heads;
    const int ctas = std::min(grid_ctas(), 148);
    if (ctas < 1) {
        (void)check_launch();
        return B200_ECUDA;
    }
    // The line of blocks is counted in 32 bits.
    const double tiles = ((double)c->tokens / p.tile_tokens + c->requests + 1) * p.head_sets * c->kv_heads;
    if (tiles * ((double)c->table_width * c->page_size / kKeys + prefix_length / kKeys + 2) > (double)(1 << 30)) return B200_ELIMIT;
    const int hd = c->head_dim, box = std::min(c->page_size, kKeys);
    const bool bf = c->dtype == B200_DTYPE_BF16;
    const CUtensorMapDataType type = bf ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
    for (int one = 0; one < 2; one++) {
        const int rc = make_map_3d(one ? &p.q1map : &p.qmap, type, q, hd, c->heads, c->tokens, stride_bytes(q_head, c->heads, hd),
                                   stride_bytes(q_token, c->tokens, hd), 64, p.tile_heads, one ? 1 : p.tile_tokens, CU_TENSOR_MAP_SWIZZLE_128B,
                                   CU_TENSOR_MAP_L2_PROMOTION_L2_128B);
        if (rc != B200_OK) return rc;
    }
    for (int v = 0; v < 2; v++) {
        const cuuint64_t dims[4] = {(cuuint64_t)hd, (cuuint64_t)c->page_size, (cuuint64_t)c->kv_heads, (cuuint64_t)c->pages};
        const cuuint64_t strides[3] = {stride_bytes(c->row_stride, c->page_size, hd), stride_bytes(c->head_stride, c->kv_heads, hd),
                                       stride_bytes(c->page_stride, c->pages, hd)};
        const cuuint32_t boxes[4] = {64, (cuuint32_t)box, 1, 1};
        const int rc = make_map(v ? &p.vmap : &p.kmap, type, 4, v ? c->v_pages : c->k_pages, dims, strides, boxes, CU_TENSOR_MAP_SWIZZLE_128B,
                                CU_TENSOR_MAP_L2_PROMOTION_L2_256B);
        if (rc != B200_OK) return rc;
    }
    const Room r = room_of(c, 148);
    char* ws = static_cast<char*>(workspace);
    p.first_prefix = reinterpret_cast<float*>(ws + r.prefix); p.first_own = reinterpret_cast<float*>(ws + r.own);
    p.more_pair = reinterpret_cast<float*>(ws + r.pair); p.more = reinterpret_cast<float*>(ws + r.more);
    p.ml = reinterpret_cast<float2*>(ws + r.ml); p.plan = reinterpret_cast<int*>(ws + r.plan);
    p.table = c->page_table; p.lengths = c->lengths; p.row_starts = c->row_starts; p.prefix_pages = prefix_pages; p.mask = mask; p.out = out;
    p.table_stride = c->table_stride; p.out_token = out_token; p.out_head = out_head;
    p.requests = c->requests; p.tokens = c->tokens; p.heads = c->heads; p.kv_heads = c->kv_heads;
    p.page_size = c->page_size; p.box_rows = box; p.table_width = c->table_width; p.prefix = prefix_length;
    // (of a scale of nothing, weights are equal; a positive one, however small, keeps hidden scores at minus infinity)
    p.negative = scale < 0.f;
    p.scale_log2 = std::max(std::abs(scale) * 1.4426950408889634f, 1e-30f);
    p.err = error;
    p.polls = wait_polls(kWaitPolls, kFirmPolls / 2);
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (bf) return hd == 128 ? launch_paged<__nv_bfloat16, 128>(p, ctas, st) : launch_paged<__nv_bfloat16, 64>(p, ctas, st);
    return hd == 128 ? launch_paged<__half, 128>(p, ctas, st) : launch_paged<__half, 64>(p, ctas, st);
}

}  // extern "C"
