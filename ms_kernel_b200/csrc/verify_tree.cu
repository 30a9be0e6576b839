// Verification of a drafted tree against the target's probabilities from given random numbers (recursive rejection sampling).
//
// cur is the root, r = p_cur and Z = 1; the nodes are looked at in index order, and one whose parent is cur is a candidate.  Its
// token x is accepted if  u_j q(x) Z < r(x),  q the distribution it was drawn from (the draft's row of cur; 1 where the drafts
// were not drawn).  Accepted: cur = the node, r = p_cur, Z = 1.  Rejected: r = max(r - Z q, 0), Z = sum(r) (not drawn: r(x) = 0,
// Z -= r(x)).  In the end the token behind the accepted ones is the first t with  cum r(t) > u_0 sum(r).  What leaves this has
// the target's distribution whatever the draft's.
//
// Decisions and tokens are whole numbers that hang on sums over the vocabulary, so everything is summed in 64 bits: two
// orders of a sum then part at a border about once in 10^10 draws (in 32 bits once in a few hundred).
//
// What bounds it: latency.  Only rows of visited nodes are read -- p (and q) of a node that rejects a child, and of the last one --
// a megabyte per pass over a row of 128256.  A cluster of eight thread blocks takes one sequence.  Every block walks
// the tree by itself on the p(x), q(x) of all candidates, fetched in one round trip; a pass over the vocabulary is shared: a warp
// sums a piece of neighbours, the sums of all warps go into every block's shared memory, and the sum of the last pass is
// also the table in which the token is looked up, so the search reads one warp's piece.  The residual is not stored: an
// element's value after n rejections follows from p, q and the n factors Z.  The code is kept small: unrolled further, with a loop
// over the rejections around each element, the kernel spent most of its time fetching instructions (one sequence, 8 nodes, 32000
// entries, no draft: 27 us, now 8.0 of which 5.2 on the device; 16 sequences, 64 nodes, 128256 entries, up to five
// rejections in a row: 75 us, now 35 to 61 by the draw).
#include "msaq_common.cuh"
#include "sm100_ptx.cuh"

namespace msaq {
namespace {

constexpr int VF_CLUSTER = 8, VF_WARPS = 16, VF_PIECES = VF_CLUSTER * VF_WARPS, VF_MAX_T = 64;
constexpr int VF_UNROLL = 4;                 // runs of 128 elements that a warp has in flight

struct VerifyArgs {
    const void* p;                           // target probabilities [B][T][V], strides in elements
    const void* q;                           // draft probabilities or null
    int64_t p_sb, p_st, q_sb, q_st;
    const int32_t* tokens;                   // [B][T]
    const int32_t* parents;                  // [B][T], or [T] (stride 0)
    int64_t parents_sb;
    const float* u;                          // [B][T]
    int32_t* path;                           // [B][T]
    int32_t* count;                          // [B]
    int32_t* token;                          // [B]
    int T, V, piece;                         // piece: elements per warp, a multiple of 128
    bool p_vec, q_vec;                       // rows can be read four elements at a time
};

__device__ __forceinline__ float vf_load(const float* p) { return *p; }
__device__ __forceinline__ float vf_load(const __nv_bfloat16* p) { return __bfloat162float(*p); }
__device__ __forceinline__ void vf_load4(const float* p, float (&v)[4]) {
    const float4 t = *reinterpret_cast<const float4*>(p);
    v[0] = t.x; v[1] = t.y; v[2] = t.z; v[3] = t.w;
}
__device__ __forceinline__ void vf_load4(const __nv_bfloat16* p, float (&v)[4]) {
    const uint2 t = *reinterpret_cast<const uint2*>(p);
    v[0] = bf16_lo(t.x); v[1] = bf16_hi(t.x); v[2] = bf16_lo(t.y); v[3] = bf16_hi(t.y);
}
// Entries that are not positive and finite count as nothing.
__device__ __forceinline__ float vf_clean(float x) { return x > 0.0f && x < INFINITY ? x : 0.0f; }

// Elements i .. i + 3 of a row, those at or beyond V as 0.
template <typename P>
__device__ __forceinline__ void vf_four(const P* row, int i, int V, bool vec, float (&v)[4]) {
    if (vec && i + 4 <= V) vf_load4(row + i, v);
    else
#pragma unroll
        for (int k = 0; k < 4; ++k) v[k] = i + k < V ? vf_load(row + i + k) : 0.0f;
}

__device__ __forceinline__ uint32_t vf_rank() { uint32_t r; asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(r)); return r; }
__device__ __forceinline__ void vf_store_at(uint32_t addr, uint32_t rank, double v) {
    asm volatile("{\n\t.reg .b32 a;\n\tmapa.shared::cluster.u32 a, %0, %1;\n\tst.shared::cluster.f64 [a], %2;\n\t}" ::"r"(addr), "r"(rank), "d"(v) : "memory");
}
__device__ __forceinline__ void vf_cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// What is left of p after the rejections at the current node.
struct Residual {
    const double* Z;                         // factors of the rejections (draft given)
    const int32_t* gone;                     // rejected tokens (no draft)
    int n;
};

// Elements i + 128 k .. i + 128 k + 3 of the row behind `res`, k < N, those at or beyond i1 as 0.
template <int N, typename P, bool DRAFT>
__device__ __forceinline__ void vf_residual(const VerifyArgs& a, const Residual& res, const P* prow, const P* qrow, int i, int i1,
                                            double (&r)[4 * N]) {
    float p[N][4], q[N][4];
#pragma unroll
    for (int k = 0; k < N; ++k) vf_four(prow, i + 128 * k, i1, a.p_vec, p[k]);
    if (DRAFT && res.n)
#pragma unroll
        for (int k = 0; k < N; ++k) vf_four(qrow, i + 128 * k, i1, a.q_vec, q[k]);
#pragma unroll
    for (int e = 0; e < 4 * N; ++e) r[e] = (double)vf_clean(p[e >> 2][e & 3]);
    if (DRAFT && res.n) {
        double d[4 * N];
#pragma unroll
        for (int e = 0; e < 4 * N; ++e) d[e] = (double)vf_clean(q[e >> 2][e & 3]);
#pragma unroll 1
        for (int n = 0; n < res.n; ++n) {
            const double z = res.Z[n];
#pragma unroll
            for (int e = 0; e < 4 * N; ++e) {
                r[e] = __dsub_rn(r[e], __dmul_rn(z, d[e]));
                if (!(r[e] > 0.0)) r[e] = 0.0;
            }
        }
    }
    if (!DRAFT)
#pragma unroll 1
        for (int n = 0; n < res.n; ++n) {
            const int at = res.gone[n] - i;
#pragma unroll
            for (int e = 0; e < 4 * N; ++e)
                if (at == 128 * (e >> 2) + (e & 3)) r[e] = 0.0;
        }
}

template <typename P, bool DRAFT>
__global__ void __launch_bounds__(VF_WARPS * 32)
verify_tree_kernel(const VerifyArgs a) {
    chain_release();
    chain_wait();
    __shared__ int32_t tok[VF_MAX_T], par[VF_MAX_T], path[VF_MAX_T], gone[VF_MAX_T];
    __shared__ float un[VF_MAX_T], pt[VF_MAX_T], qd[VF_MAX_T];
    __shared__ double Zs[VF_MAX_T], sums[2][VF_PIECES];
    __shared__ int s_cur, s_n, s_more;                            // the node, its rejections, whether the walk goes on after the pass
    __shared__ int s_left, s_count;                               // rejections that count for the token, nodes on the path
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int b = blockIdx.x / VF_CLUSTER;
    const uint32_t rank = vf_rank();
    const P* prow0 = static_cast<const P*>(a.p) + (int64_t)b * a.p_sb;
    const P* qrow0 = DRAFT ? static_cast<const P*>(a.q) + (int64_t)b * a.q_sb : nullptr;

    if (tid < a.T) {
        const int x = a.tokens[(int64_t)b * a.T + tid], pr = a.parents[(int64_t)b * a.parents_sb + tid];
        const bool ok = tid > 0 && pr >= 0 && pr < tid && x >= 0 && x < a.V;      // anything else is no candidate
        tok[tid] = x;
        par[tid] = ok ? pr : -1;
        un[tid] = a.u[(int64_t)b * a.T + tid];
        pt[tid] = ok ? vf_clean(vf_load(prow0 + pr * a.p_st + x)) : 0.0f;
        if (DRAFT) qd[tid] = ok ? vf_clean(vf_load(qrow0 + pr * a.q_st + x)) : 0.0f;
    }
    __syncwarp();
    vf_cluster_sync();                                            // this block's memory is written; the others' blocks run

    // thread 0's state of the walk
    int j = 1, cur = 0, n = 0, accepted = 1;
    double Z = 1.0;
    int parity = 0;
    double mine[4] = {0.0, 0.0, 0.0, 0.0}, total = 0.0;           // warp 0: sums of pieces 4 lane .. 4 lane + 3, and of all
    for (;;) {
        if (tid == 0) {
            bool pass = false;
            for (; j < a.T && !pass; ++j) {
                if (par[j] != cur) continue;
                double r = (double)pt[j];
                if (DRAFT) {
                    for (int k = 0; k < n; ++k) r = fmax(__dsub_rn(r, __dmul_rn(Zs[k], (double)qd[j])), 0.0);
                } else {
                    for (int k = 0; k < n; ++k)
                        if (gone[k] == tok[j]) r = 0.0;
                }
                const double limit = DRAFT ? (double)un[j] * (double)qd[j] * Z : (double)un[j] * Z;
                if (limit < r) {
                    cur = j;
                    n = 0;
                    Z = 1.0;
                    path[accepted++] = j;
                } else if (DRAFT) {
                    Zs[n++] = Z;
                    pass = true;                                  // the next factor is the sum of what is left
                } else {
                    gone[n++] = tok[j];
                    Z -= r;
                }
            }
            s_cur = cur;
            s_n = n;
            int more = 0;                                         // another candidate waits for this pass's sum
            for (int k = j; k < a.T && pass; ++k) more |= par[k] == cur;
            s_more = more;
        }
        __syncthreads();
        const int more = s_more;
        // ---- one pass over the vocabulary: the sum of each warp's piece ----
        Residual res{Zs, gone, s_n};
        const P* prow = prow0 + s_cur * a.p_st;
        const P* qrow = DRAFT ? qrow0 + s_cur * a.q_st : nullptr;
        for (;;) {
            const int i0 = (int)(rank * VF_WARPS + warp) * a.piece, i1 = min(i0 + a.piece, a.V);
            double s = 0.0;
#pragma unroll 1
            for (int i = i0 + 4 * lane; i < i1; i += 128 * VF_UNROLL) {
                double r[4 * VF_UNROLL];
                vf_residual<VF_UNROLL, P, DRAFT>(a, res, prow, qrow, i, i1, r);
#pragma unroll
                for (int k = 0; k < 4 * VF_UNROLL; k += 4) s += (r[k] + r[k + 1]) + (r[k + 2] + r[k + 3]);
            }
#pragma unroll
            for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
            if (lane < VF_CLUSTER) vf_store_at(smem_u32(&sums[parity][rank * VF_WARPS + warp]), (uint32_t)lane, s);
            __syncwarp();
            vf_cluster_sync();
            if (warp == 0) {                                      // the same order in every block: the same sum
#pragma unroll
                for (int k = 0; k < 4; ++k) mine[k] = sums[parity][4 * lane + k];
                total = (mine[0] + mine[1]) + (mine[2] + mine[3]);
#pragma unroll
                for (int o = 16; o; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
            }
            parity ^= 1;
            if (more || res.n == 0) break;
            // the walk is over: where the rejections left nothing, the token comes from p itself
            if (tid == 0) s_left = total > 0.0 ? res.n : 0;
            __syncthreads();
            if (s_left == res.n) break;
            res.n = 0;
        }
        Z = total;
        if (!more) {
            // ---- the token: warp 0 of the block that owns the piece ----
            if (warp == 0) {
                const double limit = (double)fminf(fmaxf(un[0], 0.0f), 1.0f) * total;
                const double four = (mine[0] + mine[1]) + (mine[2] + mine[3]);
                double upto = four;
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const double t = __shfl_up_sync(0xffffffffu, upto, o);
                    if (lane >= o) upto += t;
                }
                double before = __shfl_up_sync(0xffffffffu, upto, 1);
                if (lane == 0) before = 0.0;
                // the first piece whose cumulative sum exceeds the limit; where rounding leaves none, the last with anything in it
                int hit = -1, last = -1;
                double hit_before = 0.0, run = before;
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    if (mine[k] > 0.0) last = 4 * lane + k;
                    if (hit < 0 && mine[k] > 0.0 && run + mine[k] > limit) { hit = 4 * lane + k; hit_before = run; }
                    run += mine[k];
                }
                const unsigned hits = __ballot_sync(0xffffffffu, hit >= 0), any = __ballot_sync(0xffffffffu, last >= 0);
                int piece = -1;
                double cum = 0.0;
                if (hits) {
                    const int src = __ffs(hits) - 1;
                    piece = __shfl_sync(0xffffffffu, hit, src);
                    cum = __shfl_sync(0xffffffffu, hit_before, src);
                } else if (any) {
                    piece = __shfl_sync(0xffffffffu, last, 31 - __clz(any));
                    cum = -INFINITY;                              // nothing exceeds the limit: the piece's last token
                }
                int token = -1;
                const bool owner = piece >= 0 ? (uint32_t)(piece / VF_WARPS) == rank : rank == 0;
                if (owner && piece >= 0) {
                    const int i0 = piece * a.piece, i1 = min(i0 + a.piece, a.V);
                    int lastpos = -1;
#pragma unroll 1
                    for (int i = i0 + 4 * lane; i - 4 * lane < i1 && token < 0; i += 128) {
                        double r[4];
                        vf_residual<1, P, DRAFT>(a, res, prow, qrow, i, i1, r);
                        double incl = (r[0] + r[1]) + (r[2] + r[3]);
                        int pos = -1, found = -1;
#pragma unroll
                        for (int o = 1; o < 32; o <<= 1) {
                            const double t = __shfl_up_sync(0xffffffffu, incl, o);
                            if (lane >= o) incl += t;
                        }
                        double c = __shfl_up_sync(0xffffffffu, incl, 1);
                        c = cum + (lane ? c : 0.0);
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            c += r[e];
                            if (r[e] > 0.0) pos = i + e;
                            if (found < 0 && r[e] > 0.0 && c > limit) found = i + e;
                        }
                        const unsigned f = __ballot_sync(0xffffffffu, found >= 0), l = __ballot_sync(0xffffffffu, pos >= 0);
                        if (f) token = __shfl_sync(0xffffffffu, found, __ffs(f) - 1);
                        if (l) lastpos = __shfl_sync(0xffffffffu, pos, 31 - __clz(l));
                        cum += __shfl_sync(0xffffffffu, incl, 31);
                    }
                    if (token < 0) token = lastpos;
                }
                if (owner && lane == 0) a.token[b] = token;
            }
            break;
        }
    }
    if (rank == 0 && tid == 0) {
        path[0] = 0;
        a.count[b] = accepted;
        s_count = accepted;
    }
    __syncthreads();
    if (rank == 0 && tid < a.T) a.path[(int64_t)b * a.T + tid] = tid < s_count ? path[tid] : -1;
}

template <typename P>
void launch_verify(const VerifyArgs& a, int B, cudaStream_t st) {
    const dim3 grid((unsigned)B * VF_CLUSTER), block(VF_WARPS * 32);
    if (a.q) launch_chained_cluster(verify_tree_kernel<P, true>, grid, block, 0, VF_CLUSTER, st, a);
    else launch_chained_cluster(verify_tree_kernel<P, false>, grid, block, 0, VF_CLUSTER, st, a);
}

}  // namespace
}  // namespace msaq

using namespace msaq;

extern "C" int msaq_verify_tree(const void* target_probs, int64_t target_stride_b, int64_t target_stride_t, const void* draft_probs,
                                int64_t draft_stride_b, int64_t draft_stride_t, int probs_are_f32, const int32_t* tokens,
                                const int32_t* parents, int64_t parents_stride_b, const float* uniforms, int32_t* path,
                                int32_t* count, int32_t* token, int64_t B, int64_t T, int64_t V, void* stream) {
    const DeviceScope device;
    if (!target_probs || !tokens || !parents || !uniforms || !path || !count || !token) return fail(MSAQ_ERR_ARG, "null pointer");
    if (B <= 0 || V <= 0) return fail(MSAQ_ERR_ARG, "B and V must be positive");
    if (T <= 0 || T > VF_MAX_T) return fail(MSAQ_ERR_ARG, "a tree has 1 to %d nodes", VF_MAX_T);
    if (V > (1 << 30) || B > INT32_MAX / VF_CLUSTER) return fail(MSAQ_ERR_ARG, "size exceeds the supported range");
    if (target_stride_b < 0 || target_stride_t < 0 || parents_stride_b < 0 || (draft_probs && (draft_stride_b < 0 || draft_stride_t < 0)))
        return fail(MSAQ_ERR_ARG, "negative stride");
    const uintptr_t es = probs_are_f32 ? 4 : 2;
    if (reinterpret_cast<uintptr_t>(target_probs) % es || reinterpret_cast<uintptr_t>(draft_probs) % es)
        return fail(MSAQ_ERR_ARG, "probabilities must be aligned to their type");
    if (int rc = require_sm100()) return rc;
    VerifyArgs a{};
    a.p = target_probs; a.q = draft_probs;
    a.p_sb = target_stride_b; a.p_st = target_stride_t; a.q_sb = draft_stride_b; a.q_st = draft_stride_t;
    a.tokens = tokens; a.parents = parents; a.parents_sb = parents_stride_b; a.u = uniforms;
    a.path = path; a.count = count; a.token = token;
    a.T = (int)T; a.V = (int)V;
    a.piece = (int)(((V + VF_PIECES - 1) / VF_PIECES + 127) / 128 * 128);
    a.p_vec = reinterpret_cast<uintptr_t>(target_probs) % (4 * es) == 0 && target_stride_b % 4 == 0 && target_stride_t % 4 == 0;
    a.q_vec = draft_probs && reinterpret_cast<uintptr_t>(draft_probs) % (4 * es) == 0 && draft_stride_b % 4 == 0 && draft_stride_t % 4 == 0;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (probs_are_f32) launch_verify<float>(a, (int)B, st);
    else launch_verify<__nv_bfloat16>(a, (int)B, st);
    count_launch();
    return check_launch("verify_tree");
}
