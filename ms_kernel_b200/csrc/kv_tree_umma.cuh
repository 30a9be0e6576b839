// Tuned attention for a tree of drafted tokens over a packed cache: gs = 2, head_dim 128, any u, any Hq / Hkv, any capacity.
//
// A thread block takes up to 64 query rows (nodes x the heads of one kv head) against one piece of the keys, 128 at a time, with the
// KEYS on the tensor cores' wide side:
//     S^T[128 keys x rows] = K[128 x 128] . Q^T          P^T = 2^(S^T - m)          O^T[128 channels x rows] += V^T . P^T
// so that the tensor and exponential work follow the number of rows, every thread of the softmax owns one key (its scale is one
// register) and all warps have the same work whatever the number of rows.
//   * Codes go from global memory to registers one tile ahead, thread = (key, two 32-blocks).  Keys become fp16 operands
//     q 2^(e - e_max) relative to the largest exponent of THEIR row (exact down to 2^-24, 2^-31 of the row's largest value below) and
//     go to tensor memory as operand A; the factor 2^e_max is applied to the scores.  The block's codes are 8-bit integers
//     offset to bytes: a byte permute drops two of them into the mantissas of 1024.0, one fused multiply-add takes the offset out
//     and the scale in.  Values become fp16 operands q 2^(e + 2) in shared memory, [key][channel] with the channel as the
//     contiguous (M) dimension.
//   * A tile that holds a value block outside the exponents -26 .. 3 (2^-20 to 2^10 in magnitude) is done in bf16 instead, values and
//     probabilities: the range of fp32 at eight digits, so that a row is not touched by the range of a key it does not see.
//   * Queries are staged once, rotated in fp32, each row scaled by a power of two into fp16 (11 digits; the bf16 query has 8, its
//     rotation more).  Probabilities are fp16 (11 digits), 2^7 above the running maximum's scale so that they reach down to 2^-31.
//   * The maximum is lazy: a row's reference moves only when a score exceeds it by more than 2^8 -- one vote per tile -- and then
//     the accumulators of those rows are rescaled in tensor memory.  Sums and accumulators are fp32.
//   * Two thread blocks share an SM: one's conversions run under the other's MMAs and waits.
#pragma once

#include <cuda_fp16.h>

#include <type_traits>

#include "tcgen05.cuh"
#include "kv_tree_generic.cuh"

namespace msaq {

constexpr int KTU_THREADS = 256, KTU_KEYS = 128, KTU_ROWS = 64;
constexpr int KTU_COL_O = 0, KTU_COL_S = 64, KTU_COL_K = 128, KTU_COLS = 256;      // tensor memory columns
constexpr int KTU_V = 0, KTU_P = 32768, KTU_Q = KTU_P + 16384;                      // shared memory: values, probabilities, queries
__host__ __device__ constexpr int ktu_smem_bytes(int nr) { return KTU_Q + nr * 256 + 1024; }
constexpr int KTU_V_BITS = 2;                                                       // values are held times 2^2
constexpr float KTU_P_BITS = 7.0f, KTU_MOVE = 15.0f;                                // 2^7 at the reference, which moves at 2^15

// Upper half of a shared-memory matrix descriptor with 128-byte swizzle; the lower half is umma_desc_lo(address, lbo).
// MN-major: rows of 64 elements (128 bytes), 8 of them (K) to a 1024-byte atom, atoms `sbo` bytes apart in K and `lbo` in M or N.
// K-major: rows of 64 K elements, 8 rows to an atom, atoms `sbo` bytes apart.
__device__ __forceinline__ uint32_t ktu_desc_hi(uint32_t sbo) { return ((sbo >> 4) & 0x3FFFu) | (1u << 14) | (2u << 29); }
// Instruction descriptor of kind::f16, fp32 accumulator, M = 128: bf16 or fp16 operands, MN-major (1) or K-major (0).
__device__ __forceinline__ uint32_t ktu_idesc(int n, uint32_t bf16, uint32_t mn) {
    return (1u << 4) | (bf16 << 7) | (bf16 << 10) | (mn << 15) | (mn << 16) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(128 >> 4) << 24);
}
__device__ __forceinline__ void ktu_mma_ss(uint32_t d, uint32_t a_lo, uint32_t a_hi, uint32_t b_lo, uint32_t b_hi, uint32_t idesc, uint32_t acc) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t.reg .b64 da, db;\n\tsetp.ne.b32 p, %6, 0;\n\tmov.b64 da, {%1, %2};\n\tmov.b64 db, {%3, %4};\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %5, p;\n\t}" ::"r"(d), "r"(a_lo), "r"(a_hi), "r"(b_lo), "r"(b_hi), "r"(idesc), "r"(acc)
        : "memory");
}
__device__ __forceinline__ void ktu_mma_ts(uint32_t d, uint32_t a_tmem, uint32_t b_lo, uint32_t b_hi, uint32_t idesc, uint32_t acc) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t.reg .b64 db;\n\tsetp.ne.b32 p, %5, 0;\n\tmov.b64 db, {%2, %3};\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], db, %4, p;\n\t}" ::"r"(d), "r"(a_tmem), "r"(b_lo), "r"(b_hi), "r"(idesc), "r"(acc)
        : "memory");
}
__device__ __forceinline__ void ktu_st16(uint32_t taddr, const uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(taddr), "r"(r[0]),
        "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]),
        "r"(r[13]), "r"(r[14]), "r"(r[15])
        : "memory");
}
// Eight accumulator columns of this warp's lanes; ktu_ld_wait() before they are used.
__device__ __forceinline__ void ktu_ld8(uint32_t taddr, float* v) {
    uint32_t r[8];
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
                 : "r"(taddr)
                 : "memory");
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = __uint_as_float(r[i]);
}
__device__ __forceinline__ void ktu_st8(uint32_t taddr, const float* v) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(taddr), "r"(__float_as_uint(v[0])),
                 "r"(__float_as_uint(v[1])), "r"(__float_as_uint(v[2])), "r"(__float_as_uint(v[3])), "r"(__float_as_uint(v[4])),
                 "r"(__float_as_uint(v[5])), "r"(__float_as_uint(v[6])), "r"(__float_as_uint(v[7]))
                 : "memory");
}
__device__ __forceinline__ void ktu_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

__device__ __forceinline__ uint32_t hfma2(uint32_t a, uint32_t b, uint32_t c) {
    uint32_t r;
    asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(r) : "r"(a), "r"(b), "r"(c));
    return r;
}
__device__ __forceinline__ uint32_t hmul2(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
}
__device__ __forceinline__ float ktu_exp2(float x) {       // 2^x, x <= 15; -inf gives 0
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}

// 2^d, d <= 15, in both halves; below the smallest fp16 number 0.
__device__ __forceinline__ uint32_t ktu_pow2_h2(int d) {
    const uint32_t h = d >= -14 ? (uint32_t)(d + 15) << 10 : d >= -24 ? 1u << (d + 24) : 0u;
    return h * 0x00010001u;
}

// The packed bytes of one (key, 32-block).
template <int U> struct KtuRaw;
template <> struct KtuRaw<4> { uint4 u; uint2 s; };
template <> struct KtuRaw<3> { uint32_t u[5]; uint32_t s0, s1; };
template <> struct KtuRaw<2> { uint2 u[3]; uint32_t s; };

__device__ __forceinline__ uint4 ldg128(const void* p) {
    uint4 v;
    asm volatile("ld.global.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
    return v;
}
__device__ __forceinline__ uint2 ldg64(const void* p) {
    uint2 v;
    asm volatile("ld.global.v2.u32 {%0,%1}, [%2];" : "=r"(v.x), "=r"(v.y) : "l"(p));
    return v;
}
__device__ __forceinline__ uint32_t ldg32(const void* p) {
    uint32_t v;
    asm volatile("ld.global.u32 %0, [%1];" : "=r"(v) : "l"(p));
    return v;
}
__device__ __forceinline__ uint32_t ldg16(const void* p) {
    uint16_t v;
    asm volatile("ld.global.u16 %0, [%1];" : "=h"(v) : "l"(p));
    return v;
}
__device__ __forceinline__ int ldg_s8(const void* p) {
    int v;
    asm volatile("ld.global.s8 %0, [%1];" : "=r"(v) : "l"(p));
    return v;
}

__device__ __forceinline__ void ktu_load(KtuRaw<4>& r, const KvPlanes& p, int64_t slot) {
    r.u = ldg128(p.u + slot * 16);
    r.s = ldg64(p.h + slot * 8);
}
__device__ __forceinline__ void ktu_load(KtuRaw<3>& r, const KvPlanes& p, int64_t slot) {
#pragma unroll
    for (int i = 0; i < 5; ++i) r.u[i] = ldg32(p.u + slot * 20 + 4 * i);
    r.s0 = ldg16(p.h + slot * 6) | ldg16(p.h + slot * 6 + 2) << 16;
    r.s1 = ldg16(p.h + slot * 6 + 4);
}
__device__ __forceinline__ void ktu_load(KtuRaw<2>& r, const KvPlanes& p, int64_t slot) {
#pragma unroll
    for (int i = 0; i < 3; ++i) r.u[i] = ldg64(p.u + slot * 24 + 8 * i);
    r.s = ldg32(p.h + slot * 4);
}
__device__ __forceinline__ void ktu_clear(KtuRaw<4>& r) { r.u = make_uint4(0u, 0u, 0u, 0u); r.s = make_uint2(0u, 0u); }
__device__ __forceinline__ void ktu_clear(KtuRaw<3>& r) {
#pragma unroll
    for (int i = 0; i < 5; ++i) r.u[i] = 0u;
    r.s0 = r.s1 = 0u;
}
__device__ __forceinline__ void ktu_clear(KtuRaw<2>& r) { r.u[0] = r.u[1] = r.u[2] = make_uint2(0u, 0u); r.s = 0u; }
__device__ __forceinline__ bool ktu_zero(const KtuRaw<4>& r) { return (r.u.x | r.u.y | r.u.z | r.u.w | r.s.x | r.s.y) == 0u; }
__device__ __forceinline__ bool ktu_zero(const KtuRaw<3>& r) { return (r.u[0] | r.u[1] | r.u[2] | r.u[3] | r.u[4] | r.s0 | r.s1) == 0u; }
__device__ __forceinline__ bool ktu_zero(const KtuRaw<2>& r) {
    return (r.u[0].x | r.u[0].y | r.u[1].x | r.u[1].y | r.u[2].x | r.u[2].y | r.s) == 0u;
}

// Codes 8i .. 8i + 7 of a block as offset integers q + 128 + 2^(U-1), bytes 0 and 2 of the words of w: the mantissas of the fp16
// numbers 1024 + ...  Order inside the eight: U = 4: 0 2, 4 6, 1 3, 5 7 (ktu_place), else as they are.
template <int U> __device__ __forceinline__ void ktu_codes(const KtuRaw<U>& r, int i, uint32_t (&w)[4]);
template <> __device__ __forceinline__ void ktu_codes<4>(const KtuRaw<4>& r, int i, uint32_t (&w)[4]) {
    const uint32_t x = i == 0 ? r.u.x : i == 1 ? r.u.y : i == 2 ? r.u.z : r.u.w, s = i < 2 ? r.s.x : r.s.y;
    // the four shared codes of these elements (two elements each), one per byte; the sign bits of both codes flipped on the way
    const uint32_t t = prmt(s, 0u, (i & 1) ? 0x3322u : 0x1100u);
    const uint32_t lo = and_xor(t >> 4, 0x0F000F00u, and_xor(t, 0x000F000Fu, 0x88888888u));
    const uint32_t e = and_xor(x << 4, 0xF0F0F0F0u, lo), o = and_xor(x, 0xF0F0F0F0u, lo);
    w[0] = prmt(e, 0x64646464u, 0x4140u);
    w[1] = prmt(e, 0x64646464u, 0x4342u);
    w[2] = prmt(o, 0x64646464u, 0x4140u);
    w[3] = prmt(o, 0x64646464u, 0x4342u);
}
template <int U> __device__ __forceinline__ void ktu_codes_fields(const uint32_t* up, uint32_t s0, uint32_t s1, int i, uint32_t (&w)[4]) {
    constexpr int WB = 8 - U;
    constexpr uint32_t SM = (1u << U) - 1u, UM = ((1u << WB) - 1u) << U;
#pragma unroll
    for (int b = 0; b < 4; ++b) {
        const int g = 4 * i + b, ps = g * U;
        const uint32_t sf = (ps + U <= 32 ? s0 >> ps : ps >= 32 ? s1 >> (ps - 32) : __funnelshift_r(s0, s1, ps)) & SM;
        uint32_t f[2];
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            const int pk = (2 * g + t) * WB, wi = pk >> 5, po = pk & 31;
            const uint32_t v = po + WB <= 32 ? up[wi] >> po : __funnelshift_r(up[wi], up[wi + 1], po);
            f[t] = (v << U) & UM;
        }
        w[b] = prmt(f[0], f[1], 0x5410u) | ((sf | 0x6400u) * 0x00010001u);
    }
}
template <> __device__ __forceinline__ void ktu_codes<3>(const KtuRaw<3>& r, int i, uint32_t (&w)[4]) {
    uint32_t up[6];
#pragma unroll
    for (int k = 0; k < 5; ++k) up[k] = r.u[k] ^ field_signs(5, k);
    up[5] = 0u;
    ktu_codes_fields<3>(up, r.s0 ^ field_signs(3, 0), r.s1 ^ (field_signs(3, 1) & 0xFFFFu), i, w);
}
template <> __device__ __forceinline__ void ktu_codes<2>(const KtuRaw<2>& r, int i, uint32_t (&w)[4]) {
    uint32_t up[7];
#pragma unroll
    for (int k = 0; k < 3; ++k) {
        up[2 * k] = r.u[k].x ^ field_signs(6, 2 * k);
        up[2 * k + 1] = r.u[k].y ^ field_signs(6, 2 * k + 1);
    }
    up[6] = 0u;
    ktu_codes_fields<2>(up, r.s ^ field_signs(2, 0), 0u, i, w);
}
// Where element e of a row is among the operands, and back.
template <int U> __host__ __device__ __forceinline__ int ktu_place(int e) { return U == 4 ? (e & ~7) | (e & 1) << 2 | (e >> 1 & 3) : e; }
template <int U> __host__ __device__ __forceinline__ int ktu_element(int p) { return U == 4 ? (p & ~7) | (p >> 2 & 1) | (p & 3) << 1 : p; }

template <int U, int NR>
__global__ void __launch_bounds__(KTU_THREADS, 2)
kv_tree_umma_kernel(const KvTreeArgs a) {
    chain_wait();
    constexpr int NC = NR / 2;                                    // columns (query rows) of a thread in the softmax
    constexpr uint32_t OFFSET = 1024u + 128u + (1u << (U - 1));   // what the mantissa bytes stand above the codes
    extern __shared__ uint8_t ktu_smem_raw[];
    __shared__ __align__(8) uint64_t bar_s, bar_pv, bar_done;
    __shared__ uint32_t tmem_slot;
    __shared__ uint64_t mask_s[KT_MAX_T];
    __shared__ __align__(16) float2 ref[NR];                      // per row: score factor 2^x of the query row, 7 - m (+inf: nothing seen yet)
    __shared__ float m_s[NR], alpha_s[NR], cmax[4][NR];
    const uint32_t sbase = (smem_u32(ktu_smem_raw) + 1023u) & ~1023u;
    uint8_t* const smem = ktu_smem_raw + (sbase - smem_u32(ktu_smem_raw));

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, quad = warp & 3, half = warp >> 2;
    const bool issuer = __shfl_sync(0xffffffffu, warp, 0) == 0;    // the warp that issues the MMAs
    const int key = quad * 32 + lane;                             // this thread's key of a tile; its blocks are 2 half, 2 half + 1
    const int groups = gridDim.y / a.Hkv, hk = blockIdx.y / groups, grp = blockIdx.y % groups, b = blockIdx.z;
    const int G = a.Hq / a.Hkv, R = a.T * G, r0 = grp * NR, rows = min(NR, R - r0);
    const int len = kt_len(a, b);
    const int j0 = blockIdx.x * a.key_tile, j1 = min(j0 + a.key_tile, len + a.T);
    float* const out = a.partial + ((((int64_t)b * a.Hkv + hk) * R + r0) * a.S + blockIdx.x) * 130;
    if (j1 <= j0) {                                               // no keys of this sequence in this piece
        for (int r = tid; r < rows; r += KTU_THREADS) {
            out[(int64_t)r * a.S * 130 + 128] = -INFINITY;
            out[(int64_t)r * a.S * 130 + 129] = 0.0f;
        }
        return;
    }
    const int tiles = (j1 - j0 + KTU_KEYS - 1) / KTU_KEYS;
    const int64_t krow = (((int64_t)b * a.Hkv + hk) * 4) * a.Lcap;

    KtuRaw<U> kraw[2], vraw[2];
    int ke[4], ve[2];
    auto load_k = [&](int it) {
        const int j = j0 + it * KTU_KEYS + key;
        const bool ok = j < j1;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            if (ok) ktu_load(kraw[i], a.k, krow + (int64_t)(2 * half + i) * a.Lcap + j);
            else ktu_clear(kraw[i]);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) ke[i] = ok ? ldg_s8(a.k.s + krow + (int64_t)i * a.Lcap + j) : -127;
    };
    auto load_v = [&](int it) {
        const int j = j0 + it * KTU_KEYS + key;
        const bool ok = j < j1;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            if (ok) ktu_load(vraw[i], a.v, krow + (int64_t)(2 * half + i) * a.Lcap + j);
            else ktu_clear(vraw[i]);
            ve[i] = ok ? ldg_s8(a.v.s + krow + (int64_t)(2 * half + i) * a.Lcap + j) : 0;
        }
    };
    load_k(0);
    load_v(0);

    if (tid == 0) {
        mbar_init(smem_u32(&bar_s), 1);
        mbar_init(smem_u32(&bar_pv), 1);
        mbar_init(smem_u32(&bar_done), 1);
        mbar_init_fence();
    }
    if (warp == 0) {
        tmem_alloc(smem_u32(&tmem_slot), KTU_COLS);
        tmem_relinquish();
    }
    if (tid < a.T) mask_s[tid] = a.mask[b * a.mask_stride + tid];
    // ---- queries: rotated, scaled by a power of two per row, fp16, K-major with 128-byte swizzle ----
    for (int r = warp; r < NR; r += KTU_THREADS / 32) {
        float v[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        if (r < rows) {
            const int row = r0 + r;
            const __nv_bfloat16* qp = a.q + (((int64_t)b * a.T + row / G) * a.Hq + hk * G + row % G) * 128 + lane * 4;
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] = __bfloat162float(qp[i]);
        }
        if (a.qrot) {
            fwht_warp<4>(v, lane);
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] *= 0.08838834764831845f;     // 1 / sqrt(128)
        }
        uint32_t ax = 0u;
#pragma unroll
        for (int i = 0; i < 4; ++i) ax = max(ax, __float_as_uint(v[i]) & 0x7FFFFFFFu);
        ax = __reduce_max_sync(0xffffffffu, ax);
        const bool bad = ax >= 0x7F800000u;                       // an infinity or a NaN: the row is NaN, the others are not touched
        const int E = max((int)(ax >> 23) - 127, -100);
        const float up = __int_as_float((137 - E) << 23);          // largest element to [1024, 2048)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int p = ktu_place<U>(lane * 4 + i);
            const __half h = __float2half_rn(bad ? 0.0f : v[i] * up);
            *reinterpret_cast<__half*>(smem + KTU_Q + (p >> 6) * (NR * 128) + r * 128 + ((((p >> 3) & 7) ^ (r & 7)) << 4) + (p & 7) * 2) = h;
        }
        if (lane == 0) {
            ref[r] = make_float2(bad ? __int_as_float(0x7FC00000) : exp2_int(E - 10), INFINITY);
            m_s[r] = -INFINITY;
        }
    }
    fence_async_smem();
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tm = tmem_slot, tlane = tm + ((uint32_t)(quad * 32) << 16);
    const uint32_t idesc_qk = ktu_idesc(NR, 0, 0);
    const bool inject = a.skip_stage >= 0 && (blockIdx.x | blockIdx.y | blockIdx.z) == 0;

    float l[NC];
#pragma unroll
    for (int i = 0; i < NC; ++i) l[i] = 0.0f;
    bool ok = true;                                               // this thread's waits so far

#pragma unroll 1
    for (int it = 0; it < tiles; ++it) {
        // ---- keys to tensor memory ----
        const int emax = max(max(ke[0], ke[1]), max(ke[2], ke[3]));
        const float ck = a.sm_scale_log2 * exp2_int(emax);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const uint32_t sc = ktu_pow2_h2((half ? ke[2 + i] : ke[i]) - emax);
            const uint32_t off = hmul2(sc, 0xE400E400u + (OFFSET - 1024u) * 0x00010001u);      // -OFFSET (fp16 counts in ones from 1024 to 2048)
            uint32_t w[16];
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                uint32_t t[4];
                ktu_codes<U>(kraw[i], c, t);
#pragma unroll
                for (int x = 0; x < 4; ++x) w[4 * c + x] = hfma2(t[x], sc, off);
            }
            ktu_st16(tlane + KTU_COL_K + half * 32 + i * 16, w);
        }
        if (it + 1 < tiles) load_k(it + 1);
        // a value block outside the exponents that fp16 holds?
        bool far = false;
#pragma unroll
        for (int i = 0; i < 2; ++i) far = far || ((ve[i] < -24 - KTU_V_BITS || ve[i] > 5 - KTU_V_BITS) && !ktu_zero(vraw[i]));
        ktu_st_wait();
        tc_fence_before();
        const bool wide = __syncthreads_or(far);
        if (issuer && elect_lane()) {
            tc_fence_after();
            const uint32_t bhi = ktu_desc_hi(1024);
#pragma unroll
            for (int s = 0; s < 8; ++s)
                ktu_mma_ts(tm + KTU_COL_S, tm + KTU_COL_K + 8 * s, umma_desc_lo(sbase + KTU_Q + (s >> 2) * (NR * 128) + (s & 3) * 32, 16), bhi,
                           idesc_qk, s > 0);
            if (!(inject && it == a.skip_stage)) tc_commit(smem_u32(&bar_s));
        }
        // ---- values to shared memory, once the last tile's product has read them ----
        if (it > 0) ok = ok && mbar_wait_bounded(smem_u32(&bar_pv), (uint32_t)(it - 1) & 1u, a.max_polls);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const uint32_t row = sbase + KTU_V + half * 16384 + (key >> 3) * 1024 + (key & 7) * 128;
            if (!wide) {
                const uint32_t sc = ktu_pow2_h2(ktu_zero(vraw[i]) ? -100 : ve[i] + KTU_V_BITS);
                const uint32_t off = hmul2(sc, 0xE400E400u + (OFFSET - 1024u) * 0x00010001u);
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    uint32_t t[4];
                    ktu_codes<U>(vraw[i], c, t);
                    sts128(row + (((i * 4 + c) ^ (key & 7)) << 4), hfma2(t[0], sc, off), hfma2(t[1], sc, off), hfma2(t[2], sc, off),
                           hfma2(t[3], sc, off));
                }
            } else {
                const float sc = exp2_int(max(-126, min(116, ve[i] + KTU_V_BITS)));
#pragma unroll
                for (int c = 0; c < 4; ++c) {
                    uint32_t t[4];
                    ktu_codes<U>(vraw[i], c, t);
#pragma unroll
                    for (int x = 0; x < 4; ++x) {
                        const float f0 = (float)((int)(t[x] & 0xFFu) - (int)(OFFSET - 1024u)) * sc;
                        const float f1 = (float)((int)(t[x] >> 16 & 0xFFu) - (int)(OFFSET - 1024u)) * sc;
                        t[x] = prmt(__float_as_uint(f0), __float_as_uint(f1), 0x7632u);      // eight digits: exact
                    }
                    sts128(row + (((i * 4 + c) ^ (key & 7)) << 4), t[0], t[1], t[2], t[3]);
                }
            }
        }
        if (it + 1 < tiles) load_v(it + 1);
        // ---- scores ----
        ok = ok && mbar_wait_bounded(smem_u32(&bar_s), (uint32_t)it & 1u, a.max_polls);
        tc_fence_after();
        const int jb = j0 + it * KTU_KEYS;
        const bool tail = jb + KTU_KEYS > len;
        uint32_t vis = 0xFFFFFFFFu;                               // which of this thread's rows attend its key
        if (tail) {
            const int j = jb + key - len;                         // below 0: in front of the tree
            if (j >= 0) {
                vis = 0u;
                if (j < a.T)
                    for (int c = 0; c < NC; ++c) {
                        const int node = (r0 + half * NC + c) / G;
                        if (node < a.T && (mask_s[node] >> j & 1)) vis |= 1u << c;
                    }
            }
        }
        float x[NC];
#pragma unroll
        for (int c = 0; c < NC; c += 8) {
            ktu_ld8(tlane + KTU_COL_S + half * NC + c, &x[c]);
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                const float2 rf = ref[half * NC + c + k];
                x[c + k] = fmaf(x[c + k] * ck, rf.x, rf.y);
            }
        }
        if (tail)
#pragma unroll
            for (int c = 0; c < NC; ++c)
                if (!(vis >> c & 1)) x[c] = -INFINITY;
        float top = x[0];
#pragma unroll
        for (int c = 1; c < NC; ++c) top = fmaxf(top, x[c]);
        const bool move = it == 0 || top > KTU_MOVE;
        if (__syncthreads_or(move)) {
            // ---- references move: rows whose maximum of this tile is beyond theirs ----
#pragma unroll 1
            for (int c = 0; c < NC; c += 8) {
                float s[8];
                ktu_ld8(tlane + KTU_COL_S + half * NC + c, s);
#pragma unroll
                for (int k = 0; k < 8; ++k) {
                    float t = s[k] * ck * ref[half * NC + c + k].x;
                    if (!(vis >> (c + k) & 1) || t != t) t = -INFINITY;
                    const int o = __float_as_int(t);                      // in the order of whole numbers
                    const int mx = __reduce_max_sync(0xffffffffu, o ^ (o >> 31 & 0x7FFFFFFF));
                    if (lane == 0) cmax[quad][half * NC + c + k] = __int_as_float(mx ^ (mx >> 31 & 0x7FFFFFFF));
                }
            }
            if (it > 0) ok = ok && mbar_wait_bounded(smem_u32(&bar_pv), (uint32_t)(it - 1) & 1u, a.max_polls);
            __syncthreads();
            if (tid < NR) {
                const float mx = fmaxf(fmaxf(cmax[0][tid], cmax[1][tid]), fmaxf(cmax[2][tid], cmax[3][tid]));
                float al = 1.0f;
                const float m = m_s[tid];
                if (mx > -INFINITY && (m == -INFINITY || mx - m > KTU_MOVE - KTU_P_BITS)) {
                    al = m == -INFINITY ? 0.0f : ktu_exp2(m - mx);
                    m_s[tid] = mx;
                    ref[tid].y = KTU_P_BITS - mx;
                }
                alpha_s[tid] = al;
            }
            __syncthreads();
            tc_fence_after();
#pragma unroll
            for (int c = 0; c < NC; c += 8) {
                float o[8];
                if (it > 0) {
                    ktu_ld8(tlane + KTU_COL_O + half * NC + c, o);
#pragma unroll
                    for (int k = 0; k < 8; ++k) {
                        const float al = alpha_s[half * NC + c + k];
                        o[k] = al == 0.0f ? 0.0f : o[k] * al;
                    }
                    ktu_st8(tlane + KTU_COL_O + half * NC + c, o);
                }
                ktu_ld8(tlane + KTU_COL_S + half * NC + c, &x[c]);
#pragma unroll
                for (int k = 0; k < 8; ++k) {
                    const float al = alpha_s[half * NC + c + k];
                    l[c + k] = al == 0.0f ? 0.0f : l[c + k] * al;
                    const float2 rf = ref[half * NC + c + k];
                    x[c + k] = fmaf(x[c + k] * ck, rf.x, rf.y);
                    if (!(vis >> (c + k) & 1)) x[c + k] = -INFINITY;
                }
            }
            ktu_st_wait();
        }
        // ---- probabilities to shared memory ----
        auto store_p = [&](auto bf16) {
#pragma unroll
            for (int c = 0; c < NC; c += 8) {
                uint32_t w[4];
#pragma unroll
                for (int k = 0; k < 8; k += 2) {
                    const float p0 = ktu_exp2(x[c + k]), p1 = ktu_exp2(x[c + k + 1]);
                    l[c + k] += p0;
                    l[c + k + 1] += p1;
                    if constexpr (!decltype(bf16)::value) asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(w[k >> 1]) : "f"(p1), "f"(p0));
                    else asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(w[k >> 1]) : "f"(p1), "f"(p0));
                }
                sts128(sbase + KTU_P + (key >> 3) * 1024 + (key & 7) * 128 + (((half * (NC / 8) + c / 8) ^ (key & 7)) << 4), w[0], w[1], w[2], w[3]);
            }
        };
        if (wide) store_p(std::true_type{});
        else store_p(std::false_type{});
        fence_async_smem();
        tc_fence_before();
        const bool give_up = __syncthreads_or(!ok);
        if (give_up) {
            ok = false;
            break;
        }
        if (issuer && elect_lane()) {
            tc_fence_after();
            const uint32_t hi = ktu_desc_hi(1024), id = ktu_idesc(NR, wide ? 1u : 0u, 1u);
#pragma unroll
            for (int s = 0; s < 8; ++s)
                ktu_mma_ss(tm + KTU_COL_O, umma_desc_lo(sbase + KTU_V + s * 2048, 16384), hi, umma_desc_lo(sbase + KTU_P + s * 2048, 8192), hi, id,
                           it > 0 || s > 0);
            tc_commit(smem_u32(&bar_pv));
        }
    }

    // ---- the piece's result ----
    if (ok) ok = mbar_wait_bounded(smem_u32(&bar_pv), (uint32_t)(tiles - 1) & 1u, a.max_polls);
    const bool done = !__syncthreads_or(!ok);
    if (done) {
        tc_fence_after();
        float* const ls = reinterpret_cast<float*>(smem + KTU_V);         // [NR][132] sums of the 128 keys' threads
#pragma unroll
        for (int c = 0; c < NC; ++c) ls[(half * NC + c) * 132 + key] = l[c];
        const int ch = ktu_element<U>(key);                               // accumulator lane = operand place of the channel
#pragma unroll 1
        for (int c = 0; c < NC; c += 8) {
            float o[8];
            ktu_ld8(tlane + KTU_COL_O + half * NC + c, o);
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                const int r = half * NC + c + k;
                if (r < rows) out[(int64_t)r * a.S * 130 + ch] = o[k] * (1.0f / (1 << KTU_V_BITS));
            }
        }
        tc_fence_before();
        __syncthreads();
        for (int r = warp; r < rows; r += KTU_THREADS / 32) {
            float s = (ls[r * 132 + lane] + ls[r * 132 + 32 + lane]) + (ls[r * 132 + 64 + lane] + ls[r * 132 + 96 + lane]);
#pragma unroll
            for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
            if (lane == 0) {
                out[(int64_t)r * a.S * 130 + 128] = m_s[r];
                out[(int64_t)r * a.S * 130 + 129] = s;
            }
        }
    } else {
        for (int r = tid; r < rows; r += KTU_THREADS) out[(int64_t)r * a.S * 130 + 128] = __int_as_float(0x7FC00000);
        if (tid == 0) {
            report_wait_failure(a.sticky, WAIT_FAIL_KV_DECODE);
            tc_commit(smem_u32(&bar_done));                               // nothing may still write tensor memory when it is returned
            mbar_wait_bounded(smem_u32(&bar_done), 0);
        }
        tc_fence_before();
    }
    __syncthreads();
    if (warp == 0) {
        tc_fence_after();
        tmem_dealloc(tm, KTU_COLS);
    }
}

}  // namespace msaq
