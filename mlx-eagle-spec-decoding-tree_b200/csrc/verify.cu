// Verification of drafted tokens against the target's probabilities, from given random numbers.
//
// Drafted token x_i (drawn from q_i) stands while u_i q_i(x_i) < p_i(x_i).  The token behind the last that stands, n of them, is drawn by
// u_K from max(p_n - q_n, 0) if x_n was refused and from p_n if all stand: the lowest j whose sum of weights 0..j exceeds u_K times the sum
// of all.  What comes out is then distributed as tokens drawn from p, for p and q that sum to one.  Without q the drafts are taken as certain: x_i stands while
// u_i < p_i(x_i), and p_n without x_n is what a refusal leaves.
//
// Products, differences and sums are in 64 bits: u q is exact there, and a border between two tokens lies where exact sums would put it to within
// 2^-45 of the total.  Sums run in a fixed order (lanes of a warp, warps in the row's order), so a call repeated gives the same tokens.
//
// A cluster of CTAs takes one request: each sums its part of the row, a contiguous piece a warp, the sums go round through the
// CTAs' shared memory, and the CTA that holds the border looks through the one piece it lies in.  One row of the target and one of the
// draft are read per request, whatever the number of drafts.  What bounds it: HBM beyond about 16 requests, the chain of scattered reads,
// row and exchange (latency) below.  Measured: 64 requests of 7 drafts, 152064 entries in fp32, 15.2 us in a graph with their rows partly in L2, 18.6 from HBM (3.4 TB/s,
// half of a copy's rate: the chain ahead of and behind the one sweep); one request 7.2.
#include <algorithm>

#include "pipeline.cuh"
#include "typed.cuh"

namespace b200 {
namespace {

constexpr int kVerThreads = 512, kVerWarps = kVerThreads / 32;
constexpr int kVerMaxCluster = 8;

struct VerParams {
    const int* tokens;
    const void *target, *draft;
    const float* uniforms;
    const int* lengths;
    int *out, *accepted;
    long long tokens_stride, target_request, target_row, draft_request, draft_row, uniforms_stride;
    int drafts, vocab;
};

template <typename T>
__device__ __forceinline__ double weight(T p, T q, bool less) {
    const double w = less ? (double)to_f32(p) - (double)to_f32(q) : (double)to_f32(p);
    return w > 0.0 ? w : 0.0;                    // (NaN weighs nothing)
}
// Sum of the weights of elements lo .. hi of a row by a warp, per lane; lo is a multiple of VE.
template <typename T, int VE, bool LESS>
__device__ __forceinline__ double lane_sum(const T* a, const T* b, int lo, int hi, int lane) {
    constexpr int N = LESS ? 4 : 8;                                      // loads in flight, of either row
    double sum[2] = {0.0, 0.0};
    auto add = [&](const Vec<T, VE>& x, const Vec<T, VE>& y) {
#pragma unroll
        for (int e = 0; e < VE; e++) sum[e & 1] += weight(x.v[e], LESS ? y.v[e] : x.v[e], LESS);
    };
    int k = lo + lane * VE;
#pragma unroll 1
    for (; k + ((N - 1) * 32 + 1) * VE <= hi; k += N * 32 * VE) {
        Vec<T, VE> x[N], y[N];
#pragma unroll
        for (int j = 0; j < N; j++) {
            load_vec<true>(x[j], a + k + j * 32 * VE, VE);
            if (LESS) load_vec<true>(y[j], b + k + j * 32 * VE, VE);
        }
#pragma unroll
        for (int j = 0; j < N; j++) add(x[j], y[j]);
    }
#pragma unroll 2
    for (; k + VE <= hi; k += 32 * VE) {
        Vec<T, VE> x, y;
        load_vec<true>(x, a + k, VE);
        if (LESS) load_vec<true>(y, b + k, VE);
        add(x, y);
    }
    if (VE > 1) {                                                        // the last elements of the row
        k = max(hi / VE * VE, lo) + lane;
        if (k < hi) sum[0] += weight(a[k], LESS ? b[k] : a[k], LESS);
    }
    return sum[0] + sum[1];
}

// VE: elements of a load, of 16 bytes where every row starts at such, else one.
template <typename T, int VE>
__global__ void __launch_bounds__(kVerThreads, 2) verify_kernel(const VerParams p) {
    pdl_wait();
    pdl_launch_dependents();
    __shared__ double s_sums[kVerMaxCluster * kVerWarps];                // of all pieces of the row, in its order
    __shared__ int s_stand;
    __shared__ double s_scan[kVerWarps];
    __shared__ int s_found, s_last;
    cluster_arrive_relaxed();                                            // (waited for ahead of the first store to another CTA)
    const int rank = (int)cluster_rank(), cs = (int)cluster_size(), req = blockIdx.y;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int K = p.drafts, len = p.lengths == nullptr ? K : min(max(p.lengths[req], 0), K);
    const T* target = static_cast<const T*>(p.target) + req * p.target_request;
    const T* draft = static_cast<const T*>(p.draft) + req * p.draft_request;
    const int* tokens = p.tokens + req * p.tokens_stride;
    const float* u = p.uniforms + req * p.uniforms_stride;
    if (warp == 0) {
        int n = len;
        for (int i0 = 0; i0 < len && n == len; i0 += 32) {
            const int i = i0 + lane;
            bool stands = true;
            if (i < len) {
                const int x = tokens[i];
                stands = false;
                if (x >= 0 && x < p.vocab) {
                    const double q = p.draft == nullptr ? 1.0 : (double)to_f32(draft[i * p.draft_row + x]);
                    stands = (double)u[i] * q < (double)to_f32(target[i * p.target_row + x]);
                }
            }
            const unsigned refused = __ballot_sync(0xffffffffu, !stands);
            if (refused) n = i0 + __ffs(refused) - 1;
        }
        if (lane == 0) s_stand = n;
    }
    __syncthreads();
    const int n = s_stand, pieces = cs * kVerWarps;
    bool less = n < len && p.draft != nullptr;
    const int refused = n < len ? tokens[n] : -1;
    int skip = p.draft == nullptr ? refused : -1;                        // weighs nothing
    const T* a = target + n * p.target_row;
    const T* b = less ? draft + n * p.draft_row : a;
    const int per = ((p.vocab + pieces - 1) / pieces + VE - 1) / VE * VE;                     // elements of a piece
    // ---- sums of the pieces
    int found = -1;
    double before = 0.0, border = 0.0;
    for (int round = 0; round < 2; round++) {
        const int mine = rank * kVerWarps + warp, lo = min(mine * per, p.vocab), hi = min(lo + per, p.vocab);
        double sum;
        if (less) {
            sum = lane_sum<T, VE, true>(a, b, lo, hi, lane);
        } else if (skip >= lo && skip < hi) {                            // what lies around the load that holds the token, then that
            const int from = skip / VE * VE, to = min(from + VE, hi);
            sum = lane_sum<T, VE, false>(a, a, lo, from, lane) + lane_sum<T, VE, false>(a, a, to, hi, lane);
            if (from + lane < to && from + lane != skip) sum += weight(a[from + lane], a[from + lane], false);
        } else {
            sum = lane_sum<T, VE, false>(a, a, lo, hi, lane);
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        if (round == 0) cluster_wait();                                  // (the peers have started)
        if (lane < cs) {
            const uint32_t to = peer_addr(smem_u32(s_sums + mine), lane);
            asm volatile("st.shared::cluster.f64 [%0], %1;\n" ::"r"(to), "d"(sum) : "memory");
        }
        cluster_arrive();
        cluster_wait();
        // Every warp of every CTA by itself, the same sums in the same order: four pieces a lane, then a scan.
        constexpr int PER = kVerMaxCluster * kVerWarps / 32;
        double s[PER], own = 0.0;
#pragma unroll
        for (int j = 0; j < PER; j++) {
            s[j] = lane * PER + j < pieces ? s_sums[lane * PER + j] : 0.0;
            own += s[j];
        }
        double scan = own;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const double other = __shfl_up_sync(0xffffffffu, scan, o);
            if (lane >= o) scan += other;
        }
        const double total = __shfl_sync(0xffffffffu, scan, 31);
        if (total > 0.0) {
            border = (double)u[K] * total;
            double c = __shfl_up_sync(0xffffffffu, scan, 1);             // up to this lane's pieces
            if (lane == 0) c = 0.0;
            int hit = -1, last = -1;                                     // the first that exceeds the border, the last that has weight
            double hit_at = 0.0, last_at = 0.0;
#pragma unroll
            for (int j = 0; j < PER; j++) {
                if (s[j] > 0.0) {
                    last = lane * PER + j;
                    last_at = c;
                    if (hit < 0 && c + s[j] > border) {
                        hit = last;
                        hit_at = c;
                    }
                }
                c += s[j];
            }
            const unsigned hits = __ballot_sync(0xffffffffu, hit >= 0), some = __ballot_sync(0xffffffffu, last >= 0);
            const int from = hits ? __ffs(hits) - 1 : 31 - __clz(some);
            found = __shfl_sync(0xffffffffu, hits ? hit : last, from);
            before = __shfl_sync(0xffffffffu, hits ? hit_at : last_at, from);
            break;
        }
        // Nothing left of p - q: the target's own row; and where that is empty too, token 0.
        less = false;
        skip = -1;
        b = a;
        cluster_arrive();                                                // (the sums have been read)
        cluster_wait();
    }
    const int owner = found < 0 ? 0 : found / kVerWarps;
    if (rank == owner) {
        int token = 0;
        if (found >= 0) {
            // ---- the border's piece, in the row's order: `run` elements a thread
            const int lo = min(found * per, p.vocab), hi = min(lo + per, p.vocab);
            const int run = (hi - lo + kVerThreads - 1) / kVerThreads, first = min(lo + (int)threadIdx.x * run, hi), end = min(first + run, hi);
            double sum = 0.0;
            for (int k = first; k < end; k++)
                if (k != skip) sum += weight(a[k], b[k], less);
            double scan = sum;                                           // of the threads up to this one
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const double other = __shfl_up_sync(0xffffffffu, scan, o);
                if (lane >= o) scan += other;
            }
            if (lane == 31) s_scan[warp] = scan;
            if (threadIdx.x == 0) {
                s_found = 0x7fffffff;
                s_last = lo;
            }
            __syncthreads();
            double c = before;
            for (int j = 0; j < warp; j++) c += s_scan[j];
            c += scan - sum;
            int hit = 0x7fffffff, last = -1;
            for (int k = first; k < end; k++) {
                if (k == skip) continue;
                const double w = weight(a[k], b[k], less);
                c += w;
                if (w > 0.0) {
                    last = k;
                    if (c > border && hit == 0x7fffffff) hit = k;
                }
            }
            if (hit != 0x7fffffff) atomicMin(&s_found, hit);
            if (last >= 0) atomicMax(&s_last, last);
            __syncthreads();
            token = s_found != 0x7fffffff ? s_found : s_last;            // (sums of another order may end a hair below the border)
        }
        for (int i = threadIdx.x; i <= K; i += kVerThreads) p.out[(long long)req * (K + 1) + i] = i < n ? tokens[i] : (i == n ? token : -1);
        if (threadIdx.x == 0) p.accepted[req] = n;
    }
}

template <typename T, int VE>
void launch_verify(const VerParams& p, int requests, int cluster, cudaStream_t stream) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(cluster, requests);
    cfg.blockDim = dim3(kVerThreads);
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = cluster;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = g_use_pdl ? 2 : 1;
    cudaLaunchKernelEx(&cfg, verify_kernel<T, VE>, p);
}

}  // namespace
}  // namespace b200

extern "C" int b200_verify_tokens(const int* draft_tokens, long long tokens_stride, const void* target, long long target_request, long long target_row,
                                  const void* draft, long long draft_request, long long draft_row, const float* uniforms, long long uniforms_stride,
                                  const int* draft_lengths, int dtype, int requests, int drafts, int vocab, int* tokens_out, int* accepted, void* stream) {
    if (requests < 0 || drafts < 0 || drafts > 1024 || vocab < 1) return B200_EINVAL;
    const size_t size = b200::dtype_size(dtype);
    if (size == 0) return B200_EUNSUPPORTED;
    if (vocab > (1 << 30) || requests > 65535) return B200_ELIMIT;
    if (requests == 0) return B200_OK;
    if (!target || !uniforms || !tokens_out || !accepted || (drafts > 0 && !draft_tokens)) return B200_EINVAL;
    if (drafts == 0) draft = nullptr;
    b200::VerParams p{draft_tokens, target, draft, uniforms, draft_lengths, tokens_out, accepted, tokens_stride, target_request, target_row,
                      draft_request, draft_row, uniforms_stride, drafts, vocab};
    const int ve = (int)(16 / size);
    bool vec = b200::aligned16(target) && target_request % ve == 0 && target_row % ve == 0;
    if (draft) vec = vec && b200::aligned16(draft) && draft_request % ve == 0 && draft_row % ve == 0;
    // As many CTAs a request as still run at once, two to an SM (64 requests of 152064 entries: 15.2 us in clusters of 4, 20.0 in clusters of 8; of 128: 26.3 and 38.8).
    int cluster = b200::kVerMaxCluster;
    while (cluster > 1 && requests * cluster > 2 * 148) cluster /= 2;
    const cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (dtype == B200_DTYPE_F32) {
        if (vec) b200::launch_verify<float, 4>(p, requests, cluster, st);
        else b200::launch_verify<float, 1>(p, requests, cluster, st);
    } else if (dtype == B200_DTYPE_F16) {
        if (vec) b200::launch_verify<__half, 8>(p, requests, cluster, st);
        else b200::launch_verify<__half, 1>(p, requests, cluster, st);
    } else {
        if (vec) b200::launch_verify<__nv_bfloat16, 8>(p, requests, cluster, st);
        else b200::launch_verify<__nv_bfloat16, 1>(p, requests, cluster, st);
    }
    return b200::check_launch();
}
