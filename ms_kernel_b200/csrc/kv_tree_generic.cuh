// Attention for a tree of drafted tokens over a packed cache, any u, gs and head_dim in {32, 64, 128, 256}: the path behind the tuned
// kernel in kv_tree_umma.cuh.
//
// For query row r (node i, one of the G heads of a kv head) over the keys S = [0, len) and { len + j : bit j of mask[i] }:
//   out_r = sum_S p_k v_k / sum_S p_k,  p_k = exp(q_r . k / sqrt(D) - m),  an empty S gives 0.
// A thread block takes 32 query rows (all nodes and heads of one kv head, in row groups) and one piece of the keys.  Tiles of 32
// keys are dequantised into shared memory once for the 32 rows; eight neighbouring lanes share a row: four scores each, then D / 8
// channels each.  Running maximum and sum per row, in the exp2 domain.
#pragma once

#include "kv_planes.cuh"
#include "sm100_ptx.cuh"

namespace msaq {

constexpr int KT_MAX_T = 64;                  // nodes of a tree: one mask word
constexpr int KTG_THREADS = 256, KTG_ROWS = 32, KTG_KEYS = 32;

// Row r of (sequence b, kv head hk) is node r / G, head hk * G + r % G.  Partial results: [B][Hkv][T * G][S][D + 2]: acc, m, l.
struct KvTreeArgs {
    const __nv_bfloat16* q;      // [B][T][Hq][D]
    KvPlanes k, v;
    float* partial;
    const int32_t* lens;         // [B] keys in front of the tree, or null: Lk - T for every sequence
    const uint64_t* mask;        // [B][T] or [T]
    int64_t mask_stride;         // 0: one tree for all
    int T, Hq, Hkv, Lk, Lcap, D, NB, key_tile, S, qrot;
    float sm_scale_log2;         // log2(e) / sqrt(D)
    int* sticky;
    uint32_t max_polls;
    int skip_stage;
    Fmt fmt;
};

__device__ __forceinline__ int kt_len(const KvTreeArgs& a, int b) {
    return a.lens ? min(max(a.lens[b], 0), a.Lk - a.T) : a.Lk - a.T;
}

__host__ __device__ inline size_t ktg_smem_bytes(int D) {
    return (size_t)(KTG_ROWS * (D + 1) + KTG_KEYS * (D + 1) + KTG_KEYS * D + KTG_ROWS * (KTG_KEYS + 1)) * sizeof(float);
}

template <int EPL>
__global__ void __launch_bounds__(KTG_THREADS)
kv_tree_generic_kernel(const KvTreeArgs a) {
    chain_wait();
    constexpr int D = 32 * EPL;
    extern __shared__ float ktg_smem[];
    float* const qs = ktg_smem;                               // [32][D + 1]
    float* const ks = qs + KTG_ROWS * (D + 1);                // [32][D + 1]
    float* const vs = ks + KTG_KEYS * (D + 1);                // [32][D]
    float* const ps = vs + KTG_KEYS * D;                      // [32][33]
    __shared__ uint64_t mask_s[KT_MAX_T];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int groups = gridDim.y / a.Hkv, hk = blockIdx.y / groups, grp = blockIdx.y % groups, b = blockIdx.z;
    const int G = a.Hq / a.Hkv, R = a.T * G, r0 = grp * KTG_ROWS;
    const int len = kt_len(a, b);
    const int j0 = blockIdx.x * a.key_tile, j1 = min(j0 + a.key_tile, len + a.T);

    if (tid < a.T) mask_s[tid] = a.mask[b * a.mask_stride + tid];
    for (int rr = warp; rr < KTG_ROWS; rr += KTG_THREADS / 32) {
        float v[EPL];
        const int r = r0 + rr;
        const __nv_bfloat16* qp = a.q + (((int64_t)b * a.T + r / G) * a.Hq + hk * G + r % G) * D + lane * EPL;
#pragma unroll
        for (int i = 0; i < EPL; ++i) v[i] = r < R ? __bfloat162float(qp[i]) : 0.0f;
        if (a.qrot) {
            fwht_warp<EPL>(v, lane);
            const float inv = (float)(1.0 / sqrt((double)D));
#pragma unroll
            for (int i = 0; i < EPL; ++i) v[i] *= inv;
        }
#pragma unroll
        for (int i = 0; i < EPL; ++i) qs[rr * (D + 1) + lane * EPL + i] = v[i];
    }
    const int row = tid >> 3, sub = tid & 7;
    const int node = min((r0 + row) / G, a.T - 1);
    float m = -INFINITY, l = 0.0f, acc[D / 8];
#pragma unroll
    for (int i = 0; i < D / 8; ++i) acc[i] = 0.0f;
    const int64_t head_base = ((int64_t)b * a.Hkv + hk) * a.NB;
    const float lift = (float)(33 - __clz(a.Lk));             // probabilities below 1 / (2 Lk): the sum over all keys stays finite where the average does

    for (int c0 = j0; c0 < j1; c0 += KTG_KEYS) {
        __syncthreads();                                      // the tile before is read
        for (int i = tid; i < KTG_KEYS * D; i += KTG_THREADS) {
            const int blk = i / (KTG_KEYS * BLOCK), key = (i / BLOCK) % KTG_KEYS, k = i % BLOCK;
            float kv = 0.0f, vv = 0.0f;
            if (c0 + key < j1) {
                const int64_t slot = (head_base + blk) * a.Lcap + c0 + key;
                kv = kv_element(a.k, slot, k, a.fmt);
                vv = kv_element(a.v, slot, k, a.fmt);
            }
            ks[key * (D + 1) + blk * BLOCK + k] = kv;
            vs[key * D + blk * BLOCK + k] = vv;
        }
        __syncthreads();
        float s[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        for (int d = 0; d < D; ++d) {
            const float qd = qs[row * (D + 1) + d];
#pragma unroll
            for (int k = 0; k < 4; ++k) s[k] = fmaf(qd, ks[(sub + 8 * k) * (D + 1) + d], s[k]);
        }
        bool seen[4];
        float mx = -INFINITY;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const int j = c0 + sub + 8 * k - len;             // below 0: in front of the tree
            seen[k] = j < 0 || (j < a.T && (mask_s[node] >> j & 1));
            s[k] *= a.sm_scale_log2;
            if (seen[k]) mx = fmaxf(mx, s[k]);
        }
#pragma unroll
        for (int o = 1; o < 8; o <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
        const float m_new = fmaxf(m, mx), base = m_new == -INFINITY ? 0.0f : m_new + lift;
        const float alpha = m == -INFINITY ? 0.0f : exp2f(m - m_new);
        float sum = 0.0f;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const float p = seen[k] ? exp2f(s[k] - base) : 0.0f;
            ps[row * (KTG_KEYS + 1) + sub + 8 * k] = p;
            sum += p;
        }
#pragma unroll
        for (int o = 1; o < 8; o <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        l = fmaf(l, alpha, sum);
        m = m_new;
        __syncwarp();
#pragma unroll
        for (int i = 0; i < D / 8; ++i) acc[i] *= alpha;
        for (int k = 0; k < KTG_KEYS; ++k) {
            const float p = ps[row * (KTG_KEYS + 1) + k];
            if (p == 0.0f) continue;                          // what a row does not see is not multiplied by 0: it may be infinite
#pragma unroll
            for (int i = 0; i < D / 8; ++i) acc[i] = fmaf(p, vs[k * D + sub + 8 * i], acc[i]);
        }
    }
    if (r0 + row < R) {
        float* out = a.partial + ((((int64_t)b * a.Hkv + hk) * R + r0 + row) * a.S + blockIdx.x) * (D + 2);
#pragma unroll
        for (int i = 0; i < D / 8; ++i) out[sub + 8 * i] = acc[i];
        if (sub == 0) { out[D] = m; out[D + 1] = l; }
    }
}

// Merge of the key pieces of a row: weights 2^(m_s - max m).  Scores that were not numbers come through l and acc.
__global__ void __launch_bounds__(128)
kv_tree_combine_kernel(const float* __restrict__ partial, __nv_bfloat16* __restrict__ out, float* __restrict__ out_f32, int T, int Hq,
                       int Hkv, int D, int S) {
    chain_release();
    chain_wait();
    const int G = Hq / Hkv, R = T * G;
    const int r = blockIdx.x, hk = blockIdx.y, b = blockIdx.z;
    const float* base = partial + (((int64_t)b * Hkv + hk) * R + r) * S * (int64_t)(D + 2);
    float mg = -INFINITY;
    for (int s = 0; s < S; ++s) mg = fmaxf(mg, base[(int64_t)s * (D + 2) + D]);
    for (int d = threadIdx.x; d < D; d += blockDim.x) {
        float num = 0.0f, den = 0.0f;
        for (int s = 0; s < S; ++s) {
            const float* p = base + (int64_t)s * (D + 2);
            if (p[D] == -INFINITY && p[D + 1] == 0.0f) continue;      // a piece of which the row attends nothing
            const float w = exp2f(p[D] - mg);
            num = fmaf(p[d], w, num);
            den = fmaf(p[D + 1], w, den);
        }
        const float v = den == 0.0f ? 0.0f : num / den;
        const int64_t o = (((int64_t)b * T + r / G) * Hq + hk * G + r % G) * D + d;
        out[o] = __float2bfloat16_rn(v);
        if (out_f32) out_f32[o] = v;
    }
}

}  // namespace msaq
