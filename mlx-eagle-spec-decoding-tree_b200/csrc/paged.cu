// Attention over a paged cache behind a prefix that all requests of the pass share, on the fifth-generation tensor cores.
//
//   o = softmax(scale * q [Kp; Kb]^T + mask) [Vp; Vb]:  prefix rows Kp, Vp and the rows Kb, Vb of the token's own request
//
// The softmax is split over its keys: a piece of them gives its maximum m, l = sum exp(s - m) and O = sum exp(s - m) v, and pieces are joined by
// weights exp(m - max m) / sum.  A segment is the prefix with a tile of 128 query rows (token, head of the group) of any requests, or a request's
// own rows with a tile of its tokens; its work is counted in blocks of 128 keys.  All blocks of all segments stand in one line, and every worker
// takes an equal stretch of it, whatever the lengths: at most one piece a worker begins inside a segment, so a segment's first piece has its place by
// (token, head) and the others theirs by worker.  A second kernel joins them.
//
// One CTA an SM, two workers (streams) a CTA: eight warps each, two threads a query row, its scores and output in tensor memory (128 +
// 128 columns); one warp issues the products of both in turn, so that one's run while the other's softmax does.  (A warp for each let both
// streams wait for the tensor cores and for the exponentials at the same time: 4800 cycles a block of 256 rows in place of 4300.)  Where the prefix has two
// tiles of queries or more, the CTA takes them in pairs, a tile a stream, over the same blocks: keys and values are then copied once for 256
// rows.  Keys and values come page by page (TMA, boxes of a page or 128 rows) into one ring, blocks of the streams in turn.
//
// Weights are at most 2^kLag and rounded to the type of V for the second product; scores, statistics, sums and outputs are fp32.
// Every wait is bounded; one that runs out sets the error word and goes on.  No copy uses cluster multicast.
//
// What bounds it: for pairs the chain of products, softmax and waits (4240 cycles a block of 256 rows, 2144 of them products: 16 x 64 tokens of 32
// heads behind 32768 rows 505 us, 1.1 PFLOP/s, and 576 at the power limit); for single streams the copies (64 x 1 tokens behind 16384 rows, 1024 rows
// each: 65 us, 3.2 TB/s), and where they are short the start and the join, some 10 us.
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
constexpr int kParts = 2;                        // threads of a query row
constexpr int kPgThreads = 608;                  // 2 x 8 softmax warps, keys and queries, products, values
constexpr int kPgMaxRequests = 1024;
constexpr int kKeyLoader = 16, kIssuer = 17, kValueLoader = 18;
constexpr float kLag = 8.f;                      // a row's maximum may exceed its reference by 2^8

template <int HD>
struct PGeo {
    static constexpr int QTILE = kRows * HD * 2, SLOT = kKeys * HD * 2, SLOTS = HD == 128 ? 2 : 4;      // of keys, and of values
    static constexpr int KV0 = 2 * QTILE, END = KV0 + 2 * SLOTS * SLOT;
    static constexpr int SMEM = END + 1024;
};

// A line of blocks dealt out to workers in equal stretches, none of them empty: n of them, the first r of q + 1 blocks, the others of q.
struct Share {
    int total, n, q, r;
    __device__ __forceinline__ Share(int total, int workers) : total(total), n(min(workers, total)), q(n ? total / n : 0), r(total - q * n) {}
    __device__ __forceinline__ int start(int w) const { return w < n ? q * w + min(w, r) : total; }
    __device__ __forceinline__ int owner(int b) const { return b < r * (q + 1) ? b / (q + 1) : r + (b - r * (q + 1)) / q; }
};
// Blocks of the prefix, its query tiles (per kv head) and pairs of them, blocks for pairs; blocks for tiles without a partner, which head the
// line of single streams.
struct Line {
    int nbp, tiles, pairs, pair_total, odd;
};
// Blocks of a pair's segment that come first, for all pairs of a head, then what is left of them: a worker's stretch, so that all that work on a head
// at a time stand at the same keys and find them in L2.  (Segment by segment, stretches of 222 blocks begin anywhere in the 256 of a prefix of
// 32768 rows: 1.87 GB of its 134 MB were read from HBM for 16 pairs.)  Only where a stretch is more than half a segment.
__device__ __forceinline__ int first_blocks(const Line& l, int workers) {
    if (l.pairs < 2 || workers < 1) return l.nbp;
    const int stretch = (l.pair_total + workers - 1) / workers;
    return stretch < l.nbp && l.nbp <= 2 * stretch ? stretch : l.nbp;
}
// CTAs for single streams, of `ctas`: each has either pairs or single streams, so that a CTA leaves two pieces, not four, and never changes from
// the one to the other (12000 cycles).  By the time they take, in units of 2100 cycles: 2 a block of a pair, 1 a block of single streams, which
// run side by side, and 2 more a segment of theirs.
__device__ __forceinline__ int single_ctas(const Line& l, int own, int segments, int kv_heads, int ctas) {
    const int single = l.odd + own;
    if (l.pair_total == 0) return ctas;
    if (single == 0) return 0;
    const float a = 2.f * l.pair_total, b = (float)single + 2.f * (segments + (l.odd ? kv_heads : 0));
    return min(max((int)(b / (a + b) * ctas + 0.5f), 1), ctas - 1);
}

struct PagedParams {
    CUtensorMap qmap, qhmap, q1map, kmap, vmap;  // queries by tile, half a tile and token; pages
    const int *table, *lengths, *row_starts, *prefix_pages;
    const unsigned long long* mask;
    void* out;
    float *first_prefix, *first_own, *first_behind, *more_pair, *more;      // pieces [..][HD]
    float2* ml;                                  // (m, l) in the order of the pieces
    const void *q, *k_pages, *v_pages;           // as memory, for what comes seldom
    long long q_token, q_head, page_stride, head_stride, row_stride;
    int pages;
    int* plan;                                   // sums of the own blocks, by request; CTAs for single streams
    long long table_stride, out_token, out_head;
    int requests, tokens, heads, kv_heads, group, tile_heads, tile_tokens, half_tokens, head_sets;
    int page_size, page_shift, page_blocks;      // a page's rows; their logarithm, or the page's blocks if it is more than one
    int box_rows, table_width, prefix;
    Line line;
    float scale_log2;                            // positive
    int* err;
    int polls;
};

struct Request {
    int start, count, length, old;               // first token, tokens, rows, rows ahead of the pass's (as the lengths say, whatever the table holds)
    int blocks, tiles;
};
__device__ __forceinline__ Request request_of(const PagedParams& p, int b) {
    Request r;
    const int s0 = __ldcg(p.row_starts + b), s1 = __ldcg(p.row_starts + b + 1), len = __ldcg(p.lengths + b);
    r.start = min(max(s0, 0), p.tokens);
    r.count = min(max(s1 - r.start, 0), p.tokens - r.start);
    r.length = (int)min((long long)max(len, 0), (long long)p.table_width * p.page_size);
    r.old = len - (s1 - s0);
    r.blocks = (r.length + kKeys - 1) / kKeys;
    r.tiles = (r.count <= p.tile_tokens ? min(r.count, 1) : (r.count + p.tile_tokens - 1) / p.tile_tokens) * p.head_sets;
    return r;
}

// A worker's place in the line: block kb of a segment that ends before `blocks`.
struct Cursor {
    int w, end;                                  // in the line
    int kb, blocks;
    int head;                                    // where the segment begins: 0, or behind the blocks of a pair that came first
    int req;                                     // -1: the prefix
    int hk, tile;
    Request r;                                   // of the prefix: all tokens, its rows
    __device__ __forceinline__ int last() const { return min(blocks, kb + end - w); }      // where its piece of the segment ends
};
__device__ __forceinline__ void enter(Cursor& c, const Request* reqs, int req) {
    c.req = req;
    c.r = reqs[req];
    c.blocks = c.r.blocks;
    c.tile = c.hk = c.kb = c.head = 0;
}
// The cursor of block w of the line of pairs (its tile is the first stream's) or of single streams; cum: own blocks ahead of each request.
// `ahead`: blocks of a pair's segment that come first.
__device__ __forceinline__ Cursor cursor_at(const PagedParams& p, const int* cum, const Request* reqs, bool pair, int ahead, int w, int end) {
    const Line& l = p.line;
    Cursor c{};
    c.w = w;
    c.end = end;
    if (w >= end) return c;
    if (pair || w < l.odd) {
        c.req = -1;
        c.r = {0, p.tokens, p.prefix, p.prefix, l.nbp, l.tiles};
        int blocks = l.nbp, in = w;
        if (pair) {
            c.hk = w / (l.pairs * l.nbp);
            in = w - c.hk * l.pairs * l.nbp;
            const bool behind = in >= l.pairs * ahead;
            if (behind) in -= l.pairs * ahead;
            c.head = behind ? ahead : 0;
            blocks = behind ? l.nbp - ahead : ahead;
        }
        const int seg = in / blocks;
        c.kb = c.head + in - seg * blocks;
        c.blocks = c.head + blocks;
        if (pair) c.tile = 2 * seg;
        else c.hk = seg, c.tile = l.tiles - 1;
        return c;
    }
    const int v = w - l.odd;
    int lo = 0, hi = p.requests;                 // the last request that begins at v or before
    while (hi - lo > 1) {
        const int mid = (lo + hi) / 2;
        if (cum[mid] <= v) lo = mid;
        else hi = mid;
    }
    enter(c, reqs, lo);
    const int in = v - cum[lo], seg = in / c.blocks;
    c.kb = in - seg * c.blocks;
    c.tile = seg / p.kv_heads;
    c.hk = seg - c.tile * p.kv_heads;
    return c;
}
// Past its piece.
__device__ __forceinline__ void advance(Cursor& c, const PagedParams& p, const Request* reqs, bool pair, int ahead) {
    const int n = c.last() - c.kb;
    c.w += n;
    c.kb += n;
    if (c.kb < c.blocks || c.w >= c.end) return;
    c.kb = c.head;
    if (pair) {
        c.tile += 2;
        if (c.tile < 2 * p.line.pairs) return;
        c.tile = 0;
        const bool behind = c.head == 0 && ahead < p.line.nbp;           // what is left of the head's segments, or the next head
        if (!behind) c.hk++;
        c.kb = c.head = behind ? ahead : 0;
        c.blocks = behind ? p.line.nbp : ahead;
        return;
    }
    if (++c.hk < p.kv_heads) return;
    c.hk = 0;
    if (c.req >= 0 && ++c.tile < c.r.tiles) return;
    int b = c.req + 1;
    while (b + 1 < p.requests && reqs[b].blocks * reqs[b].tiles == 0) b++;
    enter(c, reqs, b);
}
// The tile's tokens and heads.
struct Tile {
    int tok0, toks, hs;
};
__device__ __forceinline__ Tile tile_of(const PagedParams& p, const Request& r, int tile) {
    Tile x;
    const int ts = p.head_sets == 1 ? tile : tile / p.head_sets;
    x.hs = tile - ts * p.head_sets;
    x.tok0 = r.start + ts * p.tile_tokens;
    x.toks = min(p.tile_tokens, r.count - ts * p.tile_tokens);
    return x;
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
__device__ __forceinline__ void tmem_st16(uint32_t addr, const uint32_t* r) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};\n" ::"r"(addr), "r"(r[0]), "r"(r[1]),
                 "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]),
                 "r"(r[14]), "r"(r[15]) : "memory");
}
__device__ __forceinline__ uint32_t pack2(float lo, float hi, __half*) { return h2_as_u32(__floats2half2_rn(lo, hi)); }
__device__ __forceinline__ uint32_t pack2(float lo, float hi, __nv_bfloat16*) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
}

// A value that is the same in all lanes, as one that the compiler knows to be: operands of products and copies then stay in uniform registers.
__device__ __forceinline__ int uniform(int x) { return __shfl_sync(0xffffffffu, x, 0); }

// Maxima that are NaN where a value is.
__device__ __forceinline__ float max3(float a, float b, float c) {
    float d;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}
__device__ __forceinline__ float max2(float a, float b) {
    float d;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
    return d;
}
template <typename T, int HD>
__global__ void __launch_bounds__(kPgThreads, 1) paged_kernel(const __grid_constant__ PagedParams p) {
    using G = PGeo<HD>;
    constexpr int ST = G::SLOTS, NB = HD / 64;
    extern __shared__ unsigned char smem_raw[];
    unsigned char* smem = smem_raw + ((0u - smem_u32(smem_raw)) & 1023u);
    __shared__ uint64_t kfull[ST], kfree[ST], vfull[ST], vfree[ST], qfull[2][2], qfree[2][2], sfull[2], pready[2], pvdone[2];
    __shared__ uint32_t s_tmem;
    __shared__ int s_cum[kPgMaxRequests + 1];
    __shared__ Request s_req[kPgMaxRequests];
    __shared__ long long s_warp[kPgThreads / 32];
    __shared__ Cursor s_from[2];                                         // of either stream; the first's for both of a pair
    __shared__ int s_segments;
    __shared__ float s_part[2][2][kParts][kRows];                        // [stream][in turn]: the maxima that a row's threads tell one another
    __shared__ float s_sum[2][kRows];                                    // of a piece, from the row's second thread to its first
    const uint32_t sbase = smem_u32(smem);
    const int lane = threadIdx.x & 31, warp = uniform(threadIdx.x >> 5), ctas = gridDim.x, cta = blockIdx.x;

    if (threadIdx.x == 0) {
        s_segments = 0;
        asm volatile("prefetch.tensormap [%0];\n" ::"l"(&p.kmap) : "memory");
        asm volatile("prefetch.tensormap [%0];\n" ::"l"(&p.vmap) : "memory");
        asm volatile("prefetch.tensormap [%0];\n" ::"l"(&p.qmap) : "memory");
        asm volatile("prefetch.tensormap [%0];\n" ::"l"(&p.q1map) : "memory");
        for (int s = 0; s < ST; s++) {
            mbar_init(smem_u32(kfull + s), 1);
            mbar_init(smem_u32(kfree + s), 1);
            mbar_init(smem_u32(vfull + s), 1);
            mbar_init(smem_u32(vfree + s), 1);
        }
        for (int s = 0; s < 2; s++) {
            for (int u = 0; u < 2; u++) {
                mbar_init(smem_u32(&qfull[s][u]), 1);
                mbar_init(smem_u32(&qfree[s][u]), 1);
            }
            mbar_init(smem_u32(sfull + s), 1);
            mbar_init(smem_u32(pready + s), 4 * kParts);
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
    pdl_wait();
    pdl_launch_dependents();                                             // (behind the wait: the join reads row_starts and lengths before it waits itself)
    // (what earlier kernels wrote by ordinary stores, rows and queries: 2000 cycles, of which all but a few pass behind the scan below)
    if (warp == kKeyLoader || warp == kValueLoader) asm volatile("fence.proxy.async;\n" ::: "memory");

    // ---- own blocks ahead of each request: consecutive requests a thread, then a scan (a line beyond 2^28 blocks is cut there)
    {
        const int per = (p.requests + kPgThreads - 1) / kPgThreads, b0 = min((int)threadIdx.x * per, p.requests), b1 = min(b0 + per, p.requests);
        long long mine = 0, before;
        int segments = 0;
        for (int b = b0; b < b1; b++) {
            const Request r = request_of(p, b);
            s_req[b] = r;
            mine += (long long)r.blocks * r.tiles * p.kv_heads;
            if (r.blocks > 0) segments += r.tiles * p.kv_heads;
        }
        segments = __reduce_add_sync(0xffffffffu, segments);
        if (lane == 0 && segments > 0) atomicAdd(&s_segments, segments);
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
            s_cum[b] = (int)min(before, 1ll << 28);
            before += (long long)s_req[b].blocks * s_req[b].tiles * p.kv_heads;
        }
        if (threadIdx.x == kPgThreads - 1) s_cum[p.requests] = (int)min(before, 1ll << 28);
        __syncthreads();
    }
    const int singles = uniform(single_ctas(p.line, s_cum[p.requests], s_segments, p.kv_heads, ctas));
    const bool pair = cta < ctas - singles;
    const int ahead = uniform(first_blocks(p.line, ctas - singles));
    if (warp < 2 && lane == 0) {
        // (the streams' workers: first one of every CTA, then the other)
        const Share share = pair ? Share(p.line.pair_total, ctas - singles) : Share(p.line.odd + s_cum[p.requests], 2 * singles);
        const int w = pair ? cta : cta - (ctas - singles) + warp * singles;
        s_from[warp] = cursor_at(p, s_cum, s_req, pair, ahead, share.start(w), share.start(w + 1));
    } else if (cta == 0 && warp >= 2) {
        for (int b = threadIdx.x - 64; b <= p.requests; b += kPgThreads - 64) p.plan[b] = s_cum[b];
        if (threadIdx.x == 64) p.plan[p.requests + 1] = singles;
    }
    __syncthreads();
    // Blocks of either stream (a pair's are the same).
    const int n0 = uniform(s_from[0].end - s_from[0].w), n1 = uniform(s_from[1].end - s_from[1].w);

    if (warp == kKeyLoader || warp == kValueLoader) {
        // ------------------------------------------------------------------ keys and queries, or values, in the order of their use
        // (both by one warp: 73 us in place of 64 for the 64 requests of the benchmark in pages of 16, eight boxes a tile and 64 dims)
        const bool values = warp == kValueLoader;
        const CUtensorMap* map = values ? &p.vmap : &p.kmap;
        uint64_t *const full = values ? vfull : kfull, *const free = values ? vfree : kfree;
        const uint32_t slots = sbase + G::KV0 + (values ? ST * G::SLOT : 0);
        int ring = 0;
        int asked[4] = {0, 0, 0, 0}, half = 3;                           // uses of the streams' halves of queries; the halves last taken, a bit a stream
        // A tile of queries, or, of 64 rows at most, one of its halves in turn, so that the next piece's come while this one's are in use.
        auto ask = [&](int s, const Cursor& c, int tile) {
            const Tile x = tile_of(p, c.r, tile);
            const int toks = uniform(x.toks), tok0 = uniform(x.tok0), head = uniform(c.hk * p.group + x.hs * p.tile_heads);
            const bool small = toks * p.tile_heads <= kRows / 2;
            if (small) half ^= 1 << s;
            const int u = small ? (half >> s) & 1 : 0;
#pragma unroll
            for (int k = 0; k < 4; k++)
                if (k == 2 * s + u || (!small && k == 2 * s + 1)) {
                    if (asked[k] > 0) mbar_wait_reported(smem_u32(&qfree[s][k & 1]), (asked[k] - 1) & 1, p.polls, p.err, 31);
                    asked[k]++;
                }
            __syncwarp();
            if (elect_one()) {
                const uint32_t bar = smem_u32(&qfull[s][u]), dst = sbase + s * G::QTILE + u * (kRows / 2 * 128);
                if (small && toks <= 4) {                                // (a box of half the tile would bring 64 rows)
                    mbar_expect_tx(bar, toks * p.tile_heads * HD * 2);
                    for (int t = 0; t < toks; t++)
#pragma unroll
                        for (int h = 0; h < NB; h++)
                            tma_box3(dst + h * (kRows * 128) + t * p.tile_heads * 128, &p.q1map, h * 64, head, tok0 + t, bar);
                } else {
                    mbar_expect_tx(bar, (small ? p.half_tokens : p.tile_tokens) * p.tile_heads * HD * 2);
#pragma unroll
                    for (int h = 0; h < NB; h++) tma_box3(dst + h * (kRows * 128), small ? &p.qhmap : &p.qmap, h * 64, head, tok0, bar);
                }
            }
            __syncwarp();
        };
        struct At {
            Cursor c;
            int kb, kb1;                                                 // of the piece
            int ahead;                                                   // a page of the next block a lane
        };
        auto page_at = [&](const At& x, int kb) {
            const int key = kb * kKeys + (lane & 15) * p.box_rows;
            int page = 0;
            if ((lane & 15) * p.box_rows < kKeys && key < x.c.r.length && kb < x.kb1) {
                const int index = p.page_blocks > 1 ? kb / p.page_blocks : key >> p.page_shift;
                page = x.c.req < 0 ? p.prefix_pages[index] : p.table[x.c.req * p.table_stride + index];
            }
            return page;
        };
        auto start = [&](At& x, int which) {
            x.c = s_from[which];
            x.kb = x.c.kb;
            x.kb1 = x.c.last();
            x.ahead = page_at(x, x.kb);
        };
        // The cursor's next block; s: the stream that uses it, 2: both.
        auto next = [&](At& x, int s) {
            const bool first = x.kb == x.c.kb;
            const int page = x.ahead, key0 = x.kb * kKeys, slot = ring % ST, row = p.page_blocks > 1 ? x.kb % p.page_blocks * kKeys : 0;
            const int boxes = (min(kKeys, x.c.r.length - key0) + p.box_rows - 1) / p.box_rows;
            x.ahead = page_at(x, x.kb + 1);
            if (ring >= ST) mbar_wait_reported(smem_u32(free + slot), (ring / ST - 1) & 1, p.polls, p.err, 31);
            __syncwarp();
            const uint32_t bar = smem_u32(full + slot), dst = slots + slot * G::SLOT;
            if (elect_one()) mbar_expect_tx(bar, boxes * p.box_rows * HD * 2);
            __syncwarp();
            // (a box a lane, a page's next 64 dims in the lanes behind: from one thread, one after the other, they took half as long again)
            if ((lane & 15) < boxes && lane >> 4 < NB)
                tma_box4(dst + (lane >> 4) * (kKeys * 128) + (lane & 15) * p.box_rows * 128, map, (lane >> 4) * 64, row, x.c.hk, page, bar);
            __syncwarp();
            ring++;
            if (first && !values) {                                      // (behind the keys: their slot is free earlier)
                if (s != 1) ask(0, x.c, x.c.tile);
                if (s != 0) ask(1, x.c, x.c.tile + (s == 2));
            }
            if (++x.kb == x.kb1) {
                advance(x.c, p, s_req, s == 2, ahead);
                x.kb = x.c.kb;
                x.kb1 = x.c.last();
                x.ahead = page_at(x, x.kb);
            }
        };
        At x, y;
        if (n0 > 0) start(x, 0);
        if (!pair && n1 > 0) start(y, 1);
#pragma unroll 1
        for (int i = 0; i < max(n0, n1); i++) {
            if (i < n0) next(x, pair ? 2 : 0);
            if (!pair && i < n1) next(y, 1);
        }
    } else if (warp == kIssuer) {
        // ------------------------------------------------------------------ products
        constexpr bool BF = std::is_same<T, __nv_bfloat16>::value;
        constexpr uint32_t base = (1u << 4) | ((uint32_t)(kRows >> 4) << 24) | (BF ? (1u << 7) | (1u << 10) : 0u);
        constexpr uint32_t idesc_s = base | ((uint32_t)(kKeys >> 3) << 17), idesc_o = base | (1u << 16) | ((uint32_t)(HD >> 3) << 17);
        const uint64_t qdesc = sw128_desc(sbase), kdesc = sw128_desc(sbase + G::KV0), vdesc = sw128_desc_n_major(sbase + G::KV0 + ST * G::SLOT, kKeys * 128);
        struct At {
            Cursor c;
            int left;                                                    // blocks whose scores have not been asked for
            int kb, kb1;                                                 // of the piece
            int keys;                                                    // of the block whose scores were asked for last
            bool first, small;                                           // ... of its piece; its queries take half a tile
            int blocks, came0, came1, half;                              // scores asked for; arrivals of queries, the half last used
        } at[2];
        int kring = 0, vring = 0;
        // Scores of the next block of stream s.  take: wait for its keys, give: hand them back (a pair's second stream does).
        auto scores = [&](int s, At& x, bool take, bool give) {
            const int slot = kring % ST;
            x.first = x.kb == x.kb1;
            if (x.first) {
                x.kb = uniform(x.c.kb);
                x.kb1 = uniform(x.c.last());
                x.small = uniform(tile_of(p, x.c.r, x.c.tile + (pair ? s : 0)).toks) * p.tile_heads <= kRows / 2;
                if (x.small) x.half ^= 1;
                const int q = x.small ? x.half : 0;
                mbar_wait_reported(smem_u32(&qfull[s][q]), (q ? x.came1 : x.came0) & 1, p.polls, p.err, 31);
                if (q) x.came1++;
                else x.came0++;
            }
            x.keys = uniform(min(kKeys, x.c.r.length - x.kb * kKeys));
            x.kb++;
            x.left--;
            const bool last = x.kb == x.kb1;
            if (take) mbar_wait_reported(smem_u32(kfull + slot), (kring / ST) & 1, p.polls, p.err, 31);
            if (x.blocks > 0) mbar_wait_reported(smem_u32(pvdone + s), (x.blocks - 1) & 1, p.polls, p.err, 31);      // (probabilities stand where the scores go)
            asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory");
            __syncwarp();
            if (elect_one()) {
                const int q = x.small ? x.half : 0;
                const uint64_t q0 = qdesc + s * (G::QTILE / 16) + q * (kRows / 2 * 128 / 16), k0 = kdesc + slot * (G::SLOT / 16);
#pragma unroll
                for (int ks = 0; ks < HD / 16; ks++)
                    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}\n" ::"r"(tmem + s * kKeys),
                                 "l"(q0 + (ks >> 2) * (kRows * 128 / 16) + (ks & 3) * 2), "l"(k0 + (ks >> 2) * (kKeys * 128 / 16) + (ks & 3) * 2), "r"(idesc_s),
                                 "r"(ks) : "memory");
                commit_to(smem_u32(sfull + s));
                if (give) commit_to(smem_u32(kfree + slot));
                if (last) {
                    commit_to(smem_u32(&qfree[s][q]));
                    if (!x.small) commit_to(smem_u32(&qfree[s][1]));
                }
            }
            __syncwarp();
            x.blocks++;
            if (give) kring++;
            if (last) advance(x.c, p, s_req, pair, ahead);
        };
        // Output of the block whose scores stream s asked for last.
        auto output = [&](int s, const At& x, bool take, bool give) {
            const int slot = vring % ST, steps = (x.keys + 15) / 16;
            if (take) {
                mbar_wait_reported(smem_u32(vfull + slot), (vring / ST) & 1, p.polls, p.err, 31);
                if (x.keys & 15) {
                    // Rows behind the last, up to the step of the product: whatever is there has probability 0, and 0 x Inf or NaN would be NaN.
                    const uint32_t v = sbase + G::KV0 + (ST + slot) * G::SLOT;
                    for (int k = x.keys * 8 + lane; k < steps * 16 * 8; k += 32)
#pragma unroll
                        for (int h = 0; h < NB; h++)
                            asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};\n" ::"r"(v + h * (kKeys * 128) + k * 16), "r"(0) : "memory");
                    fence_proxy_async();
                    __syncwarp();
                }
            }
            mbar_wait_reported(smem_u32(pready + s), (x.blocks - 1) & 1, p.polls, p.err, 31);
            asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory");
            __syncwarp();
            if (elect_one()) {
                const uint64_t v0 = vdesc + slot * (G::SLOT / 16);
#pragma unroll
                for (int ks = 0; ks < kKeys / 16; ks++)                  // (each part's probabilities stand at the beginning of its scores)
                    if (ks < steps)
                        asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}\n" ::"r"(tmem + 2 * kKeys + s * HD),
                                     "r"(tmem + s * kKeys + ks / 4 * (kKeys / kParts) + ks % 4 * 8), "l"(v0 + ks * (2048 / 16)), "r"(idesc_o),
                                     "r"((x.first ? 0 : 1) + ks) : "memory");
                if (give) commit_to(smem_u32(vfree + slot));
                commit_to(smem_u32(pvdone + s));                         // (the last thing that a CTA's end waits for)
            }
            __syncwarp();
            if (give) vring++;
        };
#pragma unroll
        for (int s = 0; s < 2; s++) {
            at[s].blocks = at[s].came0 = at[s].came1 = 0;
            at[s].half = 1;
            at[s].c = s_from[pair ? 0 : s];
            at[s].left = s ? n1 : n0;
            at[s].kb = at[s].kb1 = 0;
        }
#pragma unroll 1
        for (int i = -1; i < max(n0, n1); i++)
#pragma unroll
            for (int s = 0; s < 2; s++) {
                if (i >= (s ? n1 : n0)) continue;
                if (i >= 0) output(s, at[s], !pair || s == 0, !pair || s == 1);
                if (at[s].left > 0) scores(s, at[s], !pair || s == 0, !pair || s == 1);
            }
    } else {
        // ------------------------------------------------------------------ softmax: 64 keys of a block of a query row a thread
        constexpr int KEYS = kKeys / kParts, DIMS = HD / kParts;
        static_assert(KEYS == 64, "a row's thread has a word of keys");
        const int s = warp >> 3, part = (warp >> 2) & 1, r = (warp & 3) * 32 + lane;
        const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16, tS = tmem + s * kKeys + part * KEYS + lanes, tO = tmem + 2 * kKeys + s * HD + part * DIMS + lanes;
        const int dt = r / p.tile_heads;
        auto row_sync = [&]() { asm volatile("bar.sync %0, %1;\n" ::"r"(1 + s * 4 + (warp & 3)), "n"(kParts * 32) : "memory"); };      // the warps of these rows
        int blocks = 0;
        auto run = [&](const Cursor& c) {
            const Tile tile = tile_of(p, c.r, c.tile + (pair ? s : 0));
            const int rows = tile.toks * p.tile_heads, g = tile.hs * p.tile_heads + r - dt * p.tile_heads, t = tile.tok0 + dt, kb1 = c.last();
            const bool valid = dt < tile.toks && g < p.group, busy = (warp & 3) * 32 < rows;      // (busy: some row of the warp may be)
            // The first key that this row does not see by its place; the new rows it sees by mask.
            const bool masked = c.req >= 0 && p.mask != nullptr;
            const int length = c.r.length, old = c.r.old, sure = min(old, length);      // (sure: keys up to here are seen by all rows)
            int limit = length;
            unsigned long long bits = 0;
            if (c.req >= 0) {
                limit = min(limit, masked ? old : old + (t - c.r.start) + 1);
                if (masked && valid) bits = p.mask[t];
            }
            float m = -INFINITY, sum = 0.f;                    // the reference of the row's weights, no more than 2^kLag below its maximum
#pragma unroll 1
            for (int kb = c.kb; kb < kb1; kb++, blocks++) {
                mbar_wait_reported(smem_u32(sfull + s), blocks & 1, p.polls, p.err, 31);
                __syncwarp();
                asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory");
                if (busy) {
                    const int key0 = kb * kKeys + part * KEYS;
                    float a[KEYS];
                    {
                        uint32_t raw[KEYS];
                        tmem_ld32(raw, tS);
                        tmem_ld32(raw + 32, tS + 32);
                        asm volatile("tcgen05.wait::ld.sync.aligned;\n" ::: "memory");
#pragma unroll
                        for (int j = 0; j < KEYS; j++) a[j] = __uint_as_float(raw[j]);
                    }
                    if (key0 + KEYS > sure) {                            // what the row does not see is minus infinity
                        const int o = key0 - old, there = length - key0, n = limit - key0;      // the first key among the new rows; keys there are; keys seen
                        unsigned long long seen = n >= KEYS ? ~0ull : (n <= 0 ? 0ull : (1ull << n) - 1);
                        if (masked && o > -KEYS && o < 64) seen |= (o >= 0 ? bits >> o : bits << -o) & (there >= KEYS ? ~0ull : (there <= 0 ? 0ull : (1ull << there) - 1));
#pragma unroll
                        for (int j = 0; j < KEYS; j++)
                            if (!((seen >> j) & 1)) a[j] = -INFINITY;
                    }
                    float x[4];
#pragma unroll
                    for (int e = 0; e < 4; e++) x[e] = max3(a[e], a[e + 4], a[e + 8]);
#pragma unroll
                    for (int j = 12; j + 8 <= KEYS; j += 8) {
#pragma unroll
                        for (int e = 0; e < 4; e++) x[e] = max3(x[e], a[j + e], a[j + 4 + e]);
                    }
#pragma unroll
                    for (int e = 0; e < 4; e++) x[e] = max2(x[e], a[KEYS - 4 + e]);
                    float top = max2(max2(x[0], x[1]), max2(x[2], x[3])) * p.scale_log2;
                    s_part[s][blocks & 1][part][r] = top;
                    row_sync();
                    top = max2(top, s_part[s][blocks & 1][part ^ 1][r]);
                    const bool grown = !(top <= m + kLag);               // (of no key so far: m is minus infinity; NaN stays)
                    const float al = !grown || m != m ? 1.f : (m == -INFINITY ? 0.f : exp2_approx(m - top));
                    if (grown) m = top;
                    const float ref = m == -INFINITY ? 0.f : -m;
                    const bool rescale = __any_sync(0xffffffffu, grown && valid) && kb > c.kb;      // (the same in the rows' other warp)
                    float more[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int h = 0; h < KEYS; h += 32) {
                        uint32_t pk[16];
#pragma unroll
                        for (int j = 0; j < 32; j += 2) {
                            const float e0 = exp2_approx(fmaf(a[h + j], p.scale_log2, ref)), e1 = exp2_approx(fmaf(a[h + j + 1], p.scale_log2, ref));
                            more[j & 2] += e0;
                            more[(j & 2) + 1] += e1;
                            pk[j / 2] = pack2(e0, e1, (T*)nullptr);
                        }
                        tmem_st16(tS + h / 2, pk);
                    }
                    const float m0 = more[0] + more[1], m1 = more[2] + more[3];
                    sum = sum * al + (m0 + m1);
                    if (rescale) {
                        // (the block before has been added: its product was waited for ahead of these scores)
#pragma unroll
                        for (int d = 0; d < DIMS; d += 32) {
                            uint32_t o[32];
                            tmem_ld32(o, tO + d);
                            asm volatile("tcgen05.wait::ld.sync.aligned;\n" ::: "memory");
#pragma unroll
                            for (int j = 0; j < 32; j++) o[j] = __float_as_uint(__uint_as_float(o[j]) * al);
                            tmem_st32(tO + d, o);
                        }
                    }
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
                // (in a place of their own: a partner held up behind this barrier reads while the next piece's first maxima are written, and its next
                // sum is written behind their barrier)
                if (part == 1) s_sum[s][r] = sum;
                row_sync();
                const float l = sum + s_sum[s][r];                       // (used by the first)
                const long long row = (long long)t * p.heads + c.hk * p.group + g, all = (long long)p.tokens * p.heads;
                float* dst;
                long long at;
                if (c.kb == c.head) {
                    dst = (c.head > 0 ? p.first_behind : (c.req < 0 ? p.first_prefix : p.first_own)) + row * HD;
                    at = (c.head > 0 ? 2 * all : (c.req < 0 ? 0 : all)) + row;
                } else {
                    // (pairs: 256 rows a CTA; single streams: 128 a stream, behind them)
                    const int w = cta - (ctas - singles) + s * singles;          // (of single streams)
                    const long long slot = pair ? (long long)cta * 2 * kRows + s * kRows + r : (long long)w * kRows + r;
                    dst = (pair ? p.more_pair : p.more) + slot * HD;
                    at = 3 * all + (pair ? 0 : (long long)ctas * 2 * kRows) + slot;
                }
                if (valid && part == 0) p.ml[at] = make_float2(l == l ? m : INFINITY, l);      // (scores of NaN alone leave no maximum, but the row is NaN)
                const unsigned long long mine = reinterpret_cast<unsigned long long>(dst + part * DIMS);      // (used where the row is valid)
                const bool many = rows > 16;
#pragma unroll
                for (int d = 0; d < DIMS; d += 32) {
                    uint32_t o[32];
                    tmem_ld32(o, tO + d);
                    asm volatile("tcgen05.wait::ld.sync.aligned;\n" ::: "memory");
                    if (many) {
                        // Rows of four lanes at a time: each takes a quarter of the 32 dims of all four, so that a store covers whole lines of memory.  (A row
                        // a lane: 3300 cycles, 7000 with both streams at it.)
#pragma unroll
                        for (int x = 1; x < 4; x *= 2) {
#pragma unroll
                            for (int a = 0; a < 4; a++) {
                                if (a & x) continue;
#pragma unroll
                                for (int j = 0; j < 8; j++) {
                                    uint32_t &lo = o[a * 8 + j], &hi = o[(a | x) * 8 + j];
                                    const uint32_t other = __shfl_xor_sync(0xffffffffu, lane & x ? lo : hi, x);
                                    if (lane & x) lo = other;
                                    else hi = other;
                                }
                            }
                        }
                    }
#pragma unroll
                    for (int a = 0; a < 4; a++) {                        // unit `lane & 3` of the row of lane a of the four; or unit a of the own row
                        unsigned long long to = mine + a * 32;
                        bool there = valid;
                        if (many) {
                            to = __shfl_sync(0xffffffffu, mine, (lane & ~3) | a) + (lane & 3) * 32;
                            there = __shfl_sync(0xffffffffu, (int)valid, (lane & ~3) | a);
                        }
                        const uint32_t* v = o + a * 8;
                        if (there)
                            asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};\n" ::"l"(to + d * 4), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]),
                                         "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]) : "memory");
                    }
                }
                asm volatile("tcgen05.fence::before_thread_sync;\n" ::: "memory");
            }
        };
        Cursor c = s_from[pair ? 0 : s];
#pragma unroll 1
        while (c.w < c.end) {
            run(c);
            advance(c, p, s_req, pair, ahead);
        }
    }
    asm volatile("tcgen05.fence::before_thread_sync;\n" ::: "memory");
    __syncthreads();
    if (warp == kIssuer) {
        asm volatile("tcgen05.fence::after_thread_sync;\n" ::: "memory");
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;\n" ::"r"(tmem) : "memory");
    }
}

// A warp joins the pieces of one query row: a lane looks at a piece's statistics, then all lanes add its output, four dims (two) each.  With WAYS
// of 4 a row has the four warps of a CTA, every fourth piece each: where there are few rows, they have many pieces, and too few warps to have
// their loads in flight.  (512 rows of 16 requests behind 16384 rows: attention in 34.7 us, by one warp a row 38.2; 2048 rows of 64: 86 and
// 81; the two meet at some 1300.)
// True: something of the row is not finite, and it has to be looked at AGAIN, from the start, so that what that needs is not held in registers meanwhile (4 x 1000
// tokens of 32 heads 271 us, in one loop 302; by a call of a function 277).
template <typename T, int HD, int WAYS, bool AGAIN>
__device__ __forceinline__ bool join_row(const PagedParams& p, int ctas) {
    constexpr int N = HD / 32, BATCH = 4;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, t = blockIdx.x;
    const int head = WAYS == 1 ? blockIdx.y * 4 + warp : blockIdx.y, way = WAYS == 1 ? 0 : warp;
    // Whose token it is does not depend on the attention, which starts this kernel only once all ahead of it is there: these reads pass while its
    // last CTAs work (64 requests behind 16384 rows 58.2 -> 56.6 us, 4 short ones 11.3 -> 10.7, though 557 -> 566 where the join has 32768 rows: measured when this was moved).  Who
    // has nothing to do waits all the same: a kernel behind this one must not start ahead of the attention's end.
    if (!AGAIN && (head >= p.heads || t < __ldcg(p.row_starts) || t >= __ldcg(p.row_starts + p.requests))) {
        pdl_wait();
        return false;
    }
    int lo = 0, hi = p.requests;
    while (hi - lo > 1) {
        const int step = (hi - lo + 31) / 32, at = lo + (lane + 1) * step;
        const int n = __popc(__ballot_sync(0xffffffffu, at < hi && __ldcg(p.row_starts + at) <= t));
        lo += n * step;
        hi = min(hi, lo + step);
    }
    const Request q = request_of(p, lo);
    if (!AGAIN) pdl_wait();
    const Line& l = p.line;
    const int singles = p.plan[p.requests + 1];
    const Share single(l.odd + p.plan[p.requests], 2 * singles);
    const int hk = head / p.group, g = head - hk * p.group, hs = g / p.tile_heads, in = g - hs * p.tile_heads;
    const long long row = (long long)t * p.heads + head, all = (long long)p.tokens * p.heads;
    // The row's segments, of the prefix, its own, of the prefix again: their first pieces by row, the others by worker (`more`: of which array, rows of a worker, row in them).
    struct Segment {
        int from, to;                            // pieces: the first, then workers from + 1 .. to
        const float *first, *more;
        long long first_ml, more_ml;
        int rows, r;
    } seg[3];
    {
        const int ts = t / p.tile_tokens, tile = ts * p.head_sets + hs, r = (t - ts * p.tile_tokens) * p.tile_heads + in;
        const bool pair = tile < 2 * l.pairs;
        const Share share = pair ? Share(l.pair_total, ctas - singles) : single;
        const int ahead = pair ? first_blocks(l, ctas - singles) : l.nbp;
#pragma unroll
        for (int part = 0; part < 2; part++) {
            Segment& x = seg[2 * part];
            const int blocks = part ? l.nbp - ahead : ahead;
            const int start = pair ? hk * l.pairs * l.nbp + part * l.pairs * ahead + tile / 2 * blocks : hk * l.nbp;
            x.from = x.to = -1;
            if (blocks > 0) {
                x.from = share.owner(start);
                x.to = share.owner(start + blocks - 1);
            }
            x.first = part ? p.first_behind : p.first_prefix;
            x.first_ml = part ? 2 * all : 0;
            x.more = pair ? p.more_pair : p.more;
            x.more_ml = 3 * all + (pair ? 0 : (long long)ctas * 2 * kRows);
            x.rows = pair ? 2 * kRows : kRows;
            x.r = pair ? (tile & 1) * kRows + r : r;
        }
    }
    {
        const int dt = t - q.start, ts = dt / p.tile_tokens, tile = ts * p.head_sets + hs, r = (dt - ts * p.tile_tokens) * p.tile_heads + in;
        Segment& x = seg[1];
        const Share& share = single;
        const int start = l.odd + p.plan[lo] + (tile * p.kv_heads + hk) * q.blocks;
        x.from = x.to = -1;
        if (q.blocks > 0) {
            x.from = share.owner(start);
            x.to = share.owner(start + q.blocks - 1);
        }
        x.first = p.first_own;
        x.first_ml = all;
        x.more = p.more;
        x.more_ml = 3 * all + (long long)ctas * 2 * kRows;
        x.rows = kRows;
        x.r = r;
    }
    auto count = [](const Segment& s) { return s.from < 0 ? 0 : s.to - s.from + 1; };
    const int n0 = count(seg[0]), n1 = n0 + count(seg[1]), n = n1 + count(seg[2]);
    // Again: the own pieces; then, if they are not finite, the others and the own rows one by one, or else all.
    enum { kOthers = 1, kOwn = 2, kAll = 3 };
    for (int turn = AGAIN ? kOwn : kAll;;) {
        float m = -INFINITY, sum = 0.f, o[N] = {};
#pragma unroll 1
        for (int base = 0; base < n; base += 32 * WAYS) {
            // a piece a lane
            const int k = base + lane * WAYS + way;
            const float* src = nullptr;
            float2 x = make_float2(-INFINITY, 0.f);
            if (k < n && (k >= n0 && k < n1 ? turn & kOwn : turn & kOthers)) {
                auto pick = [&](auto a, auto b, auto c) { return k < n0 ? a : (k < n1 ? b : c); };      // (by value: the segments stay in registers)
                const int j = k - pick(0, n0, n1), w = pick(seg[0].from, seg[1].from, seg[2].from) + j;
                if (j == 0) {
                    src = pick(seg[0].first, seg[1].first, seg[2].first) + row * HD;
                    x = p.ml[pick(seg[0].first_ml, seg[1].first_ml, seg[2].first_ml) + row];
                } else {
                    const long long at = (long long)w * pick(seg[0].rows, seg[1].rows, seg[2].rows) + pick(seg[0].r, seg[1].r, seg[2].r);
                    src = pick(seg[0].more, seg[1].more, seg[2].more) + at * HD;
                    x = p.ml[pick(seg[0].more_ml, seg[1].more_ml, seg[2].more_ml) + at];
                }
            }
            // (all of them, those of weight 0 too: 0 x Inf or NaN is NaN, wherever the line was cut)
            unsigned left = __ballot_sync(0xffffffffu, src != nullptr);
            if (left == 0) continue;
            float top = x.x;
#pragma unroll
            for (int d = 16; d > 0; d >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
            const float high = fmaxf(m, top), before = m == high ? 1.f : exp2_approx(m - high), weight = x.x == -INFINITY ? 0.f : exp2_approx(x.x - high);
            float l2 = weight * x.y;
#pragma unroll
            for (int d = 16; d > 0; d >>= 1) l2 += __shfl_xor_sync(0xffffffffu, l2, d);
            sum = sum * before + l2;
            m = high;
#pragma unroll
            for (int e = 0; e < N; e++) o[e] *= before;
            while (left) {
                float w[BATCH];
                Vec<float, N> v[BATCH];
#pragma unroll
                for (int b = 0; b < BATCH; b++) {                            // (loads of several pieces in flight)
                    const int j = left ? __ffs(left) - 1 : 0;
                    const float* from = reinterpret_cast<const float*>(__shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(src), j));
                    w[b] = __shfl_sync(0xffffffffu, weight, j);
                    if (left) load_vec<true>(v[b], from + lane * N, N);
                    else w[b] = -1.f;
                    if (w[b] < 0.f)                                          // (none; by a test on `left` the code came out 0.4 us a call slower)
#pragma unroll
                        for (int e = 0; e < N; e++) v[b].v[e] = 0.f;
                    left &= left - 1;
                }
#pragma unroll
                for (int b = 0; b < BATCH; b++)
#pragma unroll
                    for (int e = 0; e < N; e++) o[e] += w[b] * v[b].v[e];
            }
        }
        if constexpr (WAYS > 1) {
            __shared__ float s_m[WAYS], s_sum[WAYS], s_o[WAYS][HD];
            if (AGAIN && turn != kOwn) __syncthreads();
            if (lane == 0) {
                s_m[way] = m;
                s_sum[way] = sum;
            }
#pragma unroll
            for (int e = 0; e < N; e++) s_o[way][lane * N + e] = o[e];
            __syncthreads();
            m = fmaxf(fmaxf(s_m[0], s_m[1]), fmaxf(s_m[2], s_m[3]));
            sum = 0.f;
#pragma unroll
            for (int e = 0; e < N; e++) o[e] = 0.f;
#pragma unroll
            for (int w = 0; w < WAYS; w++) {                                 // (in order: the same bits every time)
                const float a = s_m[w] == m ? 1.f : exp2_approx(s_m[w] - m);
                sum += a * s_sum[w];
#pragma unroll
                for (int e = 0; e < N; e++) o[e] += a * s_o[w][lane * N + e];
            }
        }
        // Inf and NaN in the values of new rows that this row does not see have come in as 0 x Inf or NaN.  That is seldom: where anything of its own rows is
        // not finite, they are gone through one by one, and those that it does not see are left out.  (Not for what the prefix holds, which all see.)
        if (!AGAIN || turn == kOwn) {
            bool bad = !(fabsf(sum) < INFINITY);
#pragma unroll
            for (int e = 0; e < N; e++) bad = bad || !(fabsf(o[e]) < INFINITY);
            bad = __any_sync(0xffffffffu, bad);                              // (of four warps, all)
            if (AGAIN) {
                turn = bad ? kOthers : kAll;
                continue;
            }
            if (bad) return true;
        }
        if (AGAIN && turn == kOthers) {
            if (way > 0) return false;
            const T* mine = static_cast<const T*>(p.q) + t * p.q_token + head * p.q_head + lane * N;
            float x[N];
#pragma unroll
            for (int e = 0; e < N; e++) x[e] = to_f32(mine[e]) * p.scale_log2;
#pragma unroll 1
            for (int key = 0; key < q.length; key++) {
                const int j = key - q.old;                                   // which new row
                if (p.mask != nullptr ? j >= 0 && (j > 63 || !((p.mask[t] >> j) & 1)) : j > t - q.start) continue;
                const int page = p.table[lo * p.table_stride + key / p.page_size];
                const bool there = page >= 0 && page < p.pages;
                const long long at = page * p.page_stride + hk * p.head_stride + key % p.page_size * p.row_stride + lane * N;
                float s = 0.f;
                if (there)
#pragma unroll
                    for (int e = 0; e < N; e++) s += x[e] * to_f32(static_cast<const T*>(p.k_pages)[at + e]);
#pragma unroll
                for (int d = 16; d > 0; d >>= 1) s += __shfl_xor_sync(0xffffffffu, s, d);
                const float high = s == s ? fmaxf(m, s) : s, a = m == high ? 1.f : exp2_approx(m - high), w = s == -INFINITY ? 0.f : exp2_approx(s - high);
                sum = sum * a + w;
#pragma unroll
                for (int e = 0; e < N; e++) o[e] = o[e] * a + (there ? w * to_f32(static_cast<const T*>(p.v_pages)[at + e]) : 0.f);
                m = high;
            }
        }
        if (WAYS > 1 && way > 0) return false;
        const float inv = sum == 0.f ? 0.f : 1.f / sum;
        Vec<T, N> y;
#pragma unroll
        for (int e = 0; e < N; e++) y.v[e] = from_f32<T>(o[e] * inv);
        store_vec<true>(static_cast<T*>(p.out) + t * p.out_token + head * p.out_head + lane * N, y, N);
        return false;
    }
}
template <typename T, int HD, int WAYS>
__global__ void __launch_bounds__(128, 8) paged_join_kernel(const __grid_constant__ PagedParams p, int ctas) {
    pdl_launch_dependents();
    if (join_row<T, HD, WAYS, false>(p, ctas)) join_row<T, HD, WAYS, true>(p, ctas);
}

struct Room {
    size_t prefix, own, behind, pair, more, ml, plan, total;             // byte offsets from the workspace's first place for them
    int ctas;
};
// Pieces are stored 32 bytes at a time; a workspace begins at a multiple of 16.
constexpr size_t kWorkAlign = 32, kGivenAlign = 16;
Room room_of(const b200_paged* c, int ctas) {
    Room r{};
    const size_t all = (size_t)c->tokens * c->heads, row = (size_t)c->head_dim * 4, pair = (size_t)ctas * 2 * kRows, more = (size_t)2 * ctas * kRows;
    r.ctas = ctas;
    r.own = all * row;
    r.behind = r.own + all * row;
    r.pair = r.behind + all * row;
    r.more = r.pair + pair * row;
    r.ml = r.more + more * row;
    r.plan = r.ml + (3 * all + pair + more) * sizeof(float2);
    r.total = r.plan + (c->requests + 2) * sizeof(int);
    r.total = (r.total + 15) / 16 * 16 + (kWorkAlign - kGivenAlign);
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
    // (a row a CTA as long as its warps find room at once)
    if ((long long)p.tokens * p.heads <= 8 * ctas) launch_kernel(paged_join_kernel<T, HD, 4>, dim3(p.tokens, p.heads), dim3(128), 0, stream, p, ctas);
    else launch_kernel(paged_join_kernel<T, HD, 1>, dim3(p.tokens, (p.heads + 3) / 4), dim3(128), 0, stream, p, ctas);
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
    if ((c->head_dim != 64 && c->head_dim != 128) || !(scale >= 0.f && scale <= 3e38f) || prefix_length < 0 || (prefix_length > 0 && !prefix_pages)) return B200_EINVAL;
    if ((c->page_size < 128 && (c->page_size < 8 || (c->page_size & (c->page_size - 1)))) || (c->page_size > 128 && c->page_size % 128)) return B200_EINVAL;
    constexpr int kMaxRows = 1 << 30;                                   // (rows and what is added to them stay in 32 bits)
    if (c->requests > kPgMaxRequests || prefix_length > kMaxRows || c->page_size > kMaxRows || (long long)c->table_width * c->page_size > kMaxRows) return B200_ELIMIT;
    if (c->tokens == 0 || c->requests == 0) return B200_OK;
    if (!q || !out || !workspace || !error) return B200_EINVAL;
    if (workspace_bytes < b200_paged_attention_workspace_bytes(c)) return B200_EWORKSPACE;
    if (!aligned16(q) || !aligned16(out) || !aligned16(c->k_pages) || !aligned16(c->v_pages) || !aligned16(workspace)) return B200_EALIGN;
    if (q_token % 8 || q_head % 8 || out_token % 8 || out_head % 8 || c->page_stride % 8 || c->head_stride % 8 || c->row_stride % 8) return B200_EALIGN;

    // (a tensor map has no strides of 0)
    if ((c->tokens > 1 && q_token <= 0) || (c->heads > 1 && q_head <= 0) || (c->page_size > 1 && c->row_stride <= 0) || (c->kv_heads > 1 && c->head_stride <= 0) ||
        (c->pages > 1 && c->page_stride <= 0))
        return B200_EINVAL;

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
    if (tiles * ((double)c->table_width * c->page_size / kKeys + prefix_length / kKeys + 2) > (double)(1 << 28)) return B200_ELIMIT;
    const int hd = c->head_dim, box = std::min(c->page_size, kKeys);
    const bool bf = c->dtype == B200_DTYPE_BF16;
    const CUtensorMapDataType type = bf ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
    p.half_tokens = std::max(kRows / 2 / p.tile_heads, 1);              // (a head set of more than 64 rows is never half a tile)
    for (int k = 0; k < 3; k++) {
        const int rc = make_map_3d(k == 0 ? &p.qmap : (k == 1 ? &p.qhmap : &p.q1map), type, q, hd, c->heads, c->tokens, stride_bytes(q_head, c->heads, hd),
                                   stride_bytes(q_token, c->tokens, hd), 64, p.tile_heads, k == 0 ? p.tile_tokens : (k == 1 ? p.half_tokens : 1),
                                   CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_128B);
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
    char* ws = reinterpret_cast<char*>((reinterpret_cast<uintptr_t>(workspace) + kWorkAlign - 1) / kWorkAlign * kWorkAlign);
    p.first_prefix = reinterpret_cast<float*>(ws + r.prefix); p.first_own = reinterpret_cast<float*>(ws + r.own);
    p.first_behind = reinterpret_cast<float*>(ws + r.behind);
    p.more_pair = reinterpret_cast<float*>(ws + r.pair); p.more = reinterpret_cast<float*>(ws + r.more);
    p.ml = reinterpret_cast<float2*>(ws + r.ml); p.plan = reinterpret_cast<int*>(ws + r.plan);
    p.table = c->page_table; p.lengths = c->lengths; p.row_starts = c->row_starts; p.prefix_pages = prefix_pages; p.mask = mask; p.out = out;
    p.q = q; p.k_pages = c->k_pages; p.v_pages = c->v_pages; p.q_token = q_token; p.q_head = q_head;
    p.page_stride = c->page_stride; p.head_stride = c->head_stride; p.row_stride = c->row_stride; p.pages = c->pages;
    p.table_stride = c->table_stride; p.out_token = out_token; p.out_head = out_head;
    p.requests = c->requests; p.tokens = c->tokens; p.heads = c->heads; p.kv_heads = c->kv_heads;
    p.page_size = c->page_size; p.page_blocks = c->page_size / kKeys; p.box_rows = box;
    while (1 << p.page_shift < c->page_size) p.page_shift++;
    p.line.nbp = (prefix_length + kKeys - 1) / kKeys;
    p.line.tiles = (c->tokens + p.tile_tokens - 1) / p.tile_tokens * p.head_sets;
    p.line.pairs = p.line.tiles / 2;
    p.line.odd = p.line.tiles & 1 ? c->kv_heads * p.line.nbp : 0;
    p.line.pair_total = c->kv_heads * p.line.pairs * p.line.nbp;
    p.table_width = c->table_width; p.prefix = prefix_length;
    // (of a scale of nothing, weights are equal; a positive one, however small, keeps hidden scores at minus infinity)
    p.scale_log2 = std::max(scale * 1.4426950408889634f, 1e-30f);
    p.err = error;
    p.polls = wait_polls(kWaitPolls, kFirmPolls / 2);
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (bf) return hd == 128 ? launch_paged<__nv_bfloat16, 128>(p, ctas, st) : launch_paged<__nv_bfloat16, 64>(p, ctas, st);
    return hd == 128 ? launch_paged<__half, 128>(p, ctas, st) : launch_paged<__half, 64>(p, ctas, st);
}

}  // extern "C"
