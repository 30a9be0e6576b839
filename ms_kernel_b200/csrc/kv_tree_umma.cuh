// Tuned attention for a tree of drafted tokens over a packed cache: gs = 2, head_dim 128, any u, any Hq / Hkv, capacities
// that are multiples of 16 (the planes' rows begin on 16-byte boundaries then, as bulk copies need).
//
// A thread block (one per SM) takes up to 64 query rows (nodes x the heads of one kv head) against 128 keys at a time, with the KEYS on
// the tensor cores' wide side:
//     S^T[128 keys x rows] = K[128 x 128] . Q^T          P^T = 2^(S^T - m)          O^T[128 channels x rows] += V^T . P^T
// so that the tensor and exponential work follow the number of rows and every thread of the softmax owns one key (its scale is one
// register).  The roles meet on mbarriers:
//   * One warp brings the packed bytes of a tile (25 to 29 bytes per key and 32-block) into a ring in shared memory with TMA bulk
//     copies, three or four tiles ahead (with one tile ahead in registers the loads' latency alone held the kernel to 2.4 TB/s).
//   * Two teams of eight decode warps take alternate tiles, thread = (key, two 32-blocks).  Keys become fp16 operands q 2^(e - e_max) relative to the
//     largest exponent of THEIR row (exact down to 2^-24, 2^-31 of the row's largest value below) and go to tensor memory as
//     operand A; the factor 2^e_max is applied to the scores.  Values become fp16 operands q 2^(e - 1) in shared memory,
//     [key][channel] with the channel as the contiguous (M) dimension.
//   * One warp looks at the value exponents of a tile's attended keys first: a tile that holds one outside -23 .. 5 (2^-17 to 2^12 in magnitude) is done
//     in bf16 instead, values and probabilities: the range of fp32 (values exact, probabilities at sixteen digits), so that a row is
//     not touched by the range of a key it does not see.  From the first tile on whose values could take the sums beyond fp32 (2^110 / Lk)
//     the references of the item are 2^16 Lk lower: an average of finite values is finite.  A key with a block of exponent 122 or more
//     (127 is what infinities are written as) makes the rows that attend it NaN.  Exponents from -106 down, the
//     quantiser's for everything below 2^-99, zeros among them, count as zeros beside the others.
//   * Queries are staged once per item, rotated in fp32, scaled by a power of two and held as two fp16 numbers, the leading eleven digits and
//     what they leave: 22 digits.  So are probabilities (two bf16 numbers beside values in bf16), 2^7 above the reference's scale so that
//     they reach down to 2^-31.  With one number each the result before its rounding was off by 1.2e-4 (beside values in bf16 by 1.1e-3);
//     now by less than 2e-5 (over 32752 keys by 2.5e-5, 1.5e-6 of the average |v|), for 9 to 13 % more time with 64 rows, 5 % and less
//     with fewer.  The second numbers of the probabilities are further columns of the same products: the values are read once.  So are
//     those of up to 32 queries (4 sequences of 32752 keys, 16 rows 93 -> 83 us, 32 rows 102 -> 93: with few rows a product's time hardly
//     depends on them); with 64 the softmax pays as much for adding the two shares as the products gain (123 -> 124 us).
//   * Eight softmax warps, thread = (key, half of the rows) (four up to 16 rows: 16 sequences of 2000 keys 35.8 instead of 34.5 us, 8 nodes over
//     509 keys 13.4 instead of 12.5, but 4 sequences of 32752 83 instead of 85).  The maximum is lazy: a row's reference moves only when a score
//     exceeds it by more than 2^8 -- one vote per tile of the four warps that hold the row -- and then the accumulators of the
//     rows concerned are rescaled in tensor memory.  Sums and accumulators are fp32.
//   * One warp issues the MMAs: S(i + 1) before P.V(i), so that both run under the decoding and the softmax.
//   * The tiles of all (sequence, kv head, row group) items form one line, cut into equal runs, one per thread block: ragged
//     batches balance.  An item inside one run is finished there; one that is cut leaves partial results (acc, m, l), merged by a second
//     kernel in the order of the runs.
// What bounds it: the instructions of decoding and softmax, 7900 of a warp per tile of 128 keys and 64 rows (61 % of the issue
// slots), and the hand-overs between roles; the tensor cores are busy one cycle in four, HBM one in five.  16 sequences of 16 nodes,
// 32 / 8 heads, over up to 32752 keys (u = 4): 373 to 389 us by the draw, 640 MB at 1.7 TB/s; one of 61 nodes, 64 / 8 heads, over 16381 keys: 144 us, 229
// TFLOP/s; one of 8 nodes over 509 keys: 13.3 us, latency.
#pragma once

#include <cuda_fp16.h>

#include "tcgen05.cuh"
#include "kv_tree_generic.cuh"

namespace msaq {

constexpr int KTU_DEC_WARPS = 16, KTU_KEYS = 128, KTU_ROWS = 64;
constexpr int KTU_SOFT_WARPS = 8;                                                   // two halves of the rows by four quarters of the keys
constexpr int KTU_THREADS = (KTU_DEC_WARPS + KTU_SOFT_WARPS + 4) * 32;              // and four single ones
constexpr int KTU_COL_O = 0, KTU_COL_S = 128, KTU_COL_K = 256, KTU_COLS = 512;      // tensor memory columns: two O, two S, two K (384 used)
// Shared memory: two buffers of values, probabilities, queries, ring.  Probabilities and queries are stored as two numbers each, the
// leading digits and what they leave.  Probabilities of up to 32 rows: two buffers, the second numbers of a key right behind the
// first; 64 rows: one buffer, the second numbers in the half that follows (two buffers leave two tiles for the ring: 423 us against 408).
constexpr int KTU_V = 0, KTU_P = 2 * 32768, KTU_Q = KTU_P + 32768;
__host__ __device__ constexpr int ktu_p_buffers(int nr) { return nr > 32 ? 1 : 2; }
__host__ __device__ constexpr int ktu_p_second(int nr) { return nr > 32 ? 16384 : nr * 2; }
constexpr int KTU_PART = 132;                                                       // floats of a row's partial result: acc, m, l, padding
__host__ __device__ constexpr int ktu_ub(int u) { return 4 * (8 - u); }              // bytes of a block: upper codes, shared codes (and an exponent)
__host__ __device__ constexpr int ktu_sb(int u) { return 2 * u; }
// Queries, K-major in two halves of 64 channels: up to 32 rows a row's second numbers are further rows of the same product, 64 rows: of
// one that follows.  Distances between the halves and between the numbers:
__host__ __device__ constexpr bool ktu_q_joint(int nr) { return nr <= 32; }
__host__ __device__ constexpr int ktu_q_half(int nr) { return ktu_q_joint(nr) ? nr * 256 : nr * 128; }
__host__ __device__ constexpr int ktu_q_second(int nr) { return ktu_q_joint(nr) ? nr * 128 : nr * 256; }
__host__ __device__ constexpr int ktu_stages(int u, int nr) { return u == 4 && nr <= 32 ? 4 : 3; }
__host__ __device__ constexpr int ktu_stage_bytes(int u) { return 2 * 4 * KTU_KEYS * (ktu_ub(u) + ktu_sb(u) + 1); }
__host__ __device__ constexpr int ktu_smem_bytes(int u, int nr) { return KTU_Q + nr * 512 + ktu_stages(u, nr) * ktu_stage_bytes(u) + 1024; }
constexpr float KTU_P_BITS = 7.0f, KTU_MOVE = 15.0f;                                // 2^7 at the reference, which moves at 2^15
// What a tile's value exponents make of it: values and probabilities in fp16, in bf16, or in bf16 with the item's probabilities that much
// lower, from here to its end.  With lg = the bits of Lk: a value is below 2^(e + 8), a probability at most 2^15, so that the sum
// over Lk keys stays below 2^127 up to e = 103 - lg, and for any value with probabilities 2^(16 + lg) lower.
constexpr int KTU_NARROW = 0, KTU_WIDE = 1, KTU_HUGE = 2;
__device__ __forceinline__ int ktu_huge_from(int Lk) { return 104 - (32 - __clz(Lk)); }
__device__ __forceinline__ float ktu_huge_bits(int Lk) { return (float)(16 + 32 - __clz(Lk)); }
constexpr int KTU_TOP = 121;                                                        // the quantiser's largest exponent of finite values; half of them is finite whatever the codes

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
// Eight accumulator columns of this warp's lanes.
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
// N accumulator columns (8, 16 or 32) in one access.
template <int N> __device__ __forceinline__ void ktu_ld(uint32_t taddr, float (&v)[N]);
template <> __device__ __forceinline__ void ktu_ld<8>(uint32_t taddr, float (&v)[8]) { ktu_ld8(taddr, v); }
template <> __device__ __forceinline__ void ktu_ld<16>(uint32_t taddr, float (&v)[16]) { tmem_ld16(taddr, v); }
template <> __device__ __forceinline__ void ktu_ld<32>(uint32_t taddr, float (&v)[32]) {
    uint32_t r[32];
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,"
        "%26,%27,%28,%29,%30,%31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]),
          "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]),
          "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]),
          "=r"(r[31])
        : "r"(taddr)
        : "memory");
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
    for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(r[i]);
}
// Two fp32 operations in one instruction.
__device__ __forceinline__ uint64_t pack2(float a, float b) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ void unpack2(uint64_t r, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(r)); }
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
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
__device__ __forceinline__ float ktu_exp2(float x) {       // 2^x to about 2^-22 of it, x <= 15; -inf gives 0
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}

// 2^d, -24 <= d <= 15, in both halves; below 0.
__device__ __forceinline__ uint32_t ktu_pow2_h2(int d) {
    const uint32_t h = d >= -14 ? (uint32_t)(d + 15) << 10 : d >= -24 ? 1u << (d + 24) : 0u;
    return h * 0x00010001u;
}

// The packed bytes of one (key, 32-block).
template <int U> struct KtuRaw;
template <> struct KtuRaw<4> { uint4 u; uint2 s; };
template <> struct KtuRaw<3> { uint32_t u[5]; uint32_t s0, s1; };
template <> struct KtuRaw<2> { uint2 u[3]; uint32_t s; };

// The bytes of one block: up, sh are shared-memory addresses of this key's codes.
__device__ __forceinline__ void ktu_load(KtuRaw<4>& r, uint32_t up, uint32_t sh) {
    r.u = lds128(up);
    r.s = lds64<0>(sh);
}
__device__ __forceinline__ void ktu_load(KtuRaw<3>& r, uint32_t up, uint32_t sh) {
#pragma unroll
    for (int k = 0; k < 5; ++k) r.u[k] = lds32<0>(up + 4 * k);
    uint32_t x, y, z;
    asm volatile("ld.shared.u16 %0, [%1];" : "=r"(x) : "r"(sh));
    asm volatile("ld.shared.u16 %0, [%1+2];" : "=r"(y) : "r"(sh));
    asm volatile("ld.shared.u16 %0, [%1+4];" : "=r"(z) : "r"(sh));
    r.s0 = x | y << 16;
    r.s1 = z;
}
__device__ __forceinline__ void ktu_load(KtuRaw<2>& r, uint32_t up, uint32_t sh) {
#pragma unroll
    for (int k = 0; k < 3; ++k) r.u[k] = lds64<0>(up + 8 * k);
    r.s = lds32<0>(sh);
}

// ---- codes to fp16 -------------------------------------------------------------------------------
// The 32 values q s of a block (s a power of two up to 2^4 in both halves), eight to a chunk: emit(chunk, four words of two).
//
// q = 2^U (U' - 2^(7-U)) + (S' - 2^(U-1)) with both fields' sign bits flipped.  A field that lies in the mantissa of a fp16 number of
// exponent 2^k, its lowest bit worth 1, reads as 2^k + field: with U' + 64 (or 32) and S' + 1024 (or 16, 64)
//     A = (S' + 2^j) s - c s,    q s = (U' + 2^k) (2^U s) + A
// are two fused multiply-adds, the first shared by the two elements of a pair, with every intermediate exact (at most 2184 s).  The
// logic unit takes an instruction per two cycles and is what bounds the decoding: 8 (U = 4), 12 (U = 3) and 14 (U = 2) of its
// instructions go into eight elements here, where bytes assembled first and then permuted into mantissas took 11, 33 and 33.
__device__ __forceinline__ uint32_t hset2(float x) {
    const __half2 h = __float2half2_rn(x);
    return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t halves(uint32_t lo, uint32_t hi) {        // low half of lo, high half of hi
    uint32_t r;
    asm("lop3.b32 %0, %1, %2, 0xFFFF0000, 0xE4;" : "=r"(r) : "r"(hi), "r"(lo));
    return r;
}
// {s, 2^U s, -(2^j) s's of the two kinds of A} for s = 2^d.
template <int U> __device__ __forceinline__ uint4 ktu_scales(int d) {
    const uint32_t s = ktu_pow2_h2(d);
    if (U == 4) return make_uint4(s, hmul2(s, 0x4C004C00u), hmul2(s, hset2(-2184.0f)), hmul2(s, hset2(-1224.0f)));
    if (U == 3) return make_uint4(s, hmul2(s, 0x48004800u), hmul2(s, hset2(-1412.0f)), hmul2(s, hset2(-404.0f)));
    return make_uint4(s, hmul2(s, 0x44004400u), hmul2(s, hset2(-1410.0f)), hmul2(s, hset2(-450.0f)));
}
// Words of a chunk: elements (0 4) (1 5) (2 6) (3 7).
template <typename F> __device__ __forceinline__ void ktu_convert(const KtuRaw<4>& r, const uint4& s, F emit) {
#pragma unroll
    for (int c = 0; c < 4; ++c) {
        const uint32_t x = c == 0 ? r.u.x : c == 1 ? r.u.y : c == 2 ? r.u.z : r.u.w;
        const uint32_t y = prmt(c < 2 ? r.s.x : r.s.y, 0u, (c & 1) ? 0x4342u : 0x4140u);         // shared codes 1 0 | 3 2
        const uint32_t a0 = hfma2(and_xor(y, 0x000F000Fu, 0x64086408u), s.x, s.z), a1 = hfma2(and_xor(y, 0x00F000F0u, 0x54805480u), s.x, s.w);
        const uint32_t x8 = x >> 8;
        emit(c, hfma2(and_xor(x * 16u, 0x00F000F0u, 0x54805480u), s.y, a0), hfma2(and_xor(x, 0x00F000F0u, 0x54805480u), s.y, a0),
             hfma2(and_xor(x8 * 16u, 0x00F000F0u, 0x54805480u), s.y, a1), hfma2(and_xor(x8, 0x00F000F0u, 0x54805480u), s.y, a1));
    }
}
__device__ __forceinline__ uint32_t ktu_window(const uint32_t* w, int bit) {        // 32 bits of the run from `bit` on
    return (bit & 31) == 0 ? w[bit >> 5] : __funnelshift_r(w[bit >> 5], w[(bit >> 5) + 1], bit & 31);
}
// Words of a chunk: elements (0 2) (1 3) (4 6) (5 7).
template <typename F> __device__ __forceinline__ void ktu_convert(const KtuRaw<3>& r, const uint4& s, F emit) {
    const uint32_t w[6] = {r.u[0], r.u[1], r.u[2], r.u[3], r.u[4], 0u};
#pragma unroll
    for (int c = 0; c < 4; ++c) {
        const uint32_t t = c == 0 ? r.s0 : c == 1 ? r.s0 >> 12 : c == 2 ? __funnelshift_r(r.s0, r.s1, 24) : r.s1 >> 4;      // shared codes 4c ..
        const uint32_t ts = halves(t, t * 8192u);                                                  // 0 2 | 1 3 at bits 0, 6
        uint32_t o[4];
#pragma unroll
        for (int g = 0; g < 2; ++g) {
            const uint32_t x = ktu_window(w, 40 * c + 20 * g), y = halves(x, x * 64u);             // 1 0 | 3 2
            const uint32_t a = g == 0 ? hfma2(and_xor(ts, 0x00070007u, 0x64046404u), s.x, s.z) : hfma2(and_xor(ts, 0x01C001C0u, 0x4D004D00u), s.x, s.w);
            o[2 * g] = hfma2(and_xor(y * 32u, 0x03E003E0u, 0x52005200u), s.y, a);
            o[2 * g + 1] = hfma2(and_xor(y, 0x03E003E0u, 0x52005200u), s.y, a);
        }
        emit(c, o[0], o[1], o[2], o[3]);
    }
}
template <typename F> __device__ __forceinline__ void ktu_convert(const KtuRaw<2>& r, const uint4& s, F emit) {
    const uint32_t w[7] = {r.u[0].x, r.u[0].y, r.u[1].x, r.u[1].y, r.u[2].x, r.u[2].y, 0u};
#pragma unroll
    for (int c = 0; c < 4; ++c) {
        const uint32_t t = r.s >> (8 * c), ts = halves(t, t * 16384u);                             // 0 2 | 1 3 at bits 0, 4
        uint32_t o[4];
#pragma unroll
        for (int g = 0; g < 2; ++g) {
            const uint32_t x = ktu_window(w, 48 * c + 24 * g), y = halves(x, x * 16u);             // 1 0 | 3 2
            const uint32_t a = g == 0 ? hfma2(and_xor(ts, 0x00030003u, 0x64026402u), s.x, s.z) : hfma2(and_xor(ts, 0x00300030u, 0x54205420u), s.x, s.w);
            o[2 * g] = hfma2(and_xor(y * 16u, 0x03F003F0u, 0x56005600u), s.y, a);
            o[2 * g + 1] = hfma2(and_xor(y >> 2, 0x03F003F0u, 0x56005600u), s.y, a);
        }
        emit(c, o[0], o[1], o[2], o[3]);
    }
}
// Where element e of a row is among the operands, and back.
template <int U> __host__ __device__ __forceinline__ int ktu_place(int e) {
    return U == 4 ? (e & ~7) | (e & 3) << 1 | (e >> 2 & 1) : (e & ~3) | (e & 1) << 1 | (e >> 1 & 1);
}
template <int U> __host__ __device__ __forceinline__ int ktu_element(int p) {
    return U == 4 ? (p & ~7) | (p >> 1 & 3) | (p & 1) << 2 : (p & ~3) | (p & 1) << 1 | (p >> 1 & 1);
}

// ---- the line of tiles -------------------------------------------------------------------------
// Item (b, hk, group) has tiles_of(b) tiles; items in that order, sequences first.  Of the n tiles (below 2^31: kv_tree.cu) thread
// block c of C <= n takes [c n / C, (c + 1) n / C).
__device__ __forceinline__ uint32_t ktu_tiles(const KvTreeArgs& a, int len) { return (uint32_t)(len + a.T + KTU_KEYS - 1) / KTU_KEYS; }
struct KtuLine {
    uint32_t n, C, q, r;
    __device__ __forceinline__ KtuLine(uint32_t tiles, uint32_t blocks) : n(tiles), C(min(blocks, tiles)), q(tiles / C), r(tiles % C) {}
    __device__ __forceinline__ uint32_t run(uint32_t c) const { return q * c + r * c / C; }         // c n / C without overflow
    // The thread block whose run holds tile g.
    __device__ __forceinline__ uint32_t owner(uint32_t g) const {
        uint32_t c = min(C - 1u, (uint32_t)__fdividef((float)g * (float)C, (float)n));              // off by one at most
        while (c > 0u && run(c) > g) --c;
        while (c + 1u < C && run(c + 1u) <= g) ++c;
        return c;
    }
};

// A place on the line.
struct KtuCursor {
    int b, hk, grp, t;                                            // sequence, kv head, row group, tile
    int len, tiles;                                               // of the sequence
    __device__ __forceinline__ void sequence(const KvTreeArgs& a, int seq, int its_len) {
        b = seq;
        len = its_len;
        tiles = (int)ktu_tiles(a, len);
    }
    __device__ __forceinline__ void next(const KvTreeArgs& a, int groups, int B) {
        if (++t < tiles) return;
        t = 0;
        if (++grp < groups) return;
        grp = 0;
        if (++hk < a.Hkv) return;
        hk = 0;
        if (b + 1 < B) sequence(a, b + 1, kt_len(a, b + 1));
    }
};

// Barrier of `threads` threads under number `id`, with a vote.
__device__ __forceinline__ bool ktu_vote(int id, int threads, bool v) {
    uint32_t r;
    asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %1, 0;\n\tbarrier.cta.red.or.pred q, %2, %3, p;\n\tselp.u32 %0, 1, 0, q;\n\t}"
                 : "=r"(r) : "r"((uint32_t)v), "r"(id), "r"(threads) : "memory");
    return r != 0;
}
__device__ __forceinline__ void ktu_bar(int id, int threads) { asm volatile("barrier.cta.sync %0, %1;" ::"r"(id), "r"(threads) : "memory"); }

// Column sums over the 32 lanes: on return v[0] of lane c holds column c (N = 32), c % N below.
template <int N> __device__ __forceinline__ void ktu_column_sums(float (&v)[N], int lane) {
#pragma unroll
    for (int s = N / 2; s >= 1; s >>= 1)
#pragma unroll
        for (int i = 0; i < s; ++i) {
            const bool up = lane & s;
            const float give = up ? v[i] : v[i + s];
            v[i] = (up ? v[i + s] : v[i]) + __shfl_xor_sync(0xffffffffu, give, s);
        }
#pragma unroll
    for (int s = N; s < 32; s <<= 1) v[0] += __shfl_xor_sync(0xffffffffu, v[0], s);
}

struct __align__(16) KtuShared {
    uint64_t rfull[4], rempty[4], ready[4];                                   // ring: bytes landed, read, looked at
    uint64_t kfull[4], vfull[2], sfull[2], pfull[2], qfull[4];                // written: keys, values, scores, probabilities, queries
    uint64_t sempty[2], vempty[2], pempty[2], done;                           // read
    uint32_t tmem;
    int len;                                                      // of the first tile's sequence
    volatile int abort;
    int wide[8];                                                  // KTU_NARROW, KTU_WIDE, KTU_HUGE of the tile
    uint64_t mask[KT_MAX_T];
    float qf[4][KTU_ROWS], qscale[4];                             // score factors 2^x of the query rows; of all rows where they are the same
    int same[4], qtop[KTU_DEC_WARPS], qlow[KTU_DEC_WARPS];
    int64_t row[KTU_ROWS];                                        // where a row goes: in the output, among the partial results
    uint4 scales[32];                                             // of 2^d, d = 4 - i
    float ck[4][KTU_KEYS];                                        // score factors of the keys
    float4 ref4[KTU_ROWS / 4];                                    // per row 7 - m (+inf: nothing seen yet; NaN: not a number)
    float f[KTU_ROWS];                                            // per row the score factor, where they differ
    float m[KTU_ROWS], alpha[KTU_ROWS], part[4][KTU_ROWS];
};

template <int U, int NR>
__global__ void __launch_bounds__(KTU_THREADS, 1)
kv_tree_umma_kernel(const KvTreeArgs a, int B, int groups, __nv_bfloat16* __restrict__ out, float* __restrict__ out_f32) {
    chain_wait();
    constexpr int PB = ktu_p_buffers(NR);
    constexpr int SW = KTU_SOFT_WARPS, NC = NR / 2;               // columns (query rows) of a thread in the softmax
    constexpr int WARP_MMA = KTU_DEC_WARPS + SW, WARP_COPY = WARP_MMA + 1, WARP_SCOUT = WARP_MMA + 2, WARPS = WARP_MMA + 4;
    extern __shared__ uint8_t ktu_smem_raw[];
    __shared__ KtuShared sh;
    const uint32_t sbase = (smem_u32(ktu_smem_raw) + 1023u) & ~1023u;
    uint8_t* const smem = ktu_smem_raw + (sbase - smem_u32(ktu_smem_raw));

    const int tid = threadIdx.x, warp = __shfl_sync(0xffffffffu, tid >> 5, 0), lane = tid & 31;
    const int quad = warp & 3, half = warp >> 2 & 1;              // decode: which blocks; softmax: which rows
    const int key = quad * 32 + lane;                             // this thread's key of a tile
    const int G = a.Hq / a.Hkv, R = a.T * G, per_seq = a.Hkv * groups;

    // ---- this thread block's run of tiles, and where it begins: every warp for itself ----
    int len = lane < B ? kt_len(a, lane) : 0;
    uint32_t mine = lane < B ? ktu_tiles(a, len) : 0u, all = mine;
    for (int i = lane + 32; i < B; i += 32) all += ktu_tiles(a, kt_len(a, i));
    const KtuLine line(__reduce_add_sync(0xffffffffu, all) * (uint32_t)per_seq, gridDim.x);
    if (blockIdx.x >= line.C) return;                             // no run is empty
    const uint32_t g0 = line.run(blockIdx.x);
    const int n_run = (int)(line.run(blockIdx.x + 1) - g0);
    int seq = 0;
    uint32_t seq_tile = 0u;                                       // the sequence of tile g0, its first tile
    for (int i0 = 0; i0 < B; i0 += 32) {
        if (i0 > 0) {
            len = i0 + lane < B ? kt_len(a, i0 + lane) : 0;
            mine = i0 + lane < B ? ktu_tiles(a, len) : 0u;
        }
        const uint32_t n = mine * (uint32_t)per_seq;
        uint32_t upto = n;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const uint32_t t = __shfl_up_sync(0xffffffffu, upto, o);
            if (lane >= o) upto += t;
        }
        const uint32_t hit = __ballot_sync(0xffffffffu, seq_tile + upto > g0);
        if (hit) {
            const int src = __ffs(hit) - 1;
            seq = i0 + src;
            len = __shfl_sync(0xffffffffu, len, src);
            seq_tile += __shfl_sync(0xffffffffu, upto - n, src);
            break;
        }
        seq_tile += __shfl_sync(0xffffffffu, upto, 31);
    }
    if (tid == 0) sh.len = len;
    if (tid < 32) sh.scales[tid] = ktu_scales<U>(4 - tid);
    if (warp == WARP_MMA) {
        tmem_alloc(smem_u32(&sh.tmem), KTU_COLS);
        tmem_relinquish();
    }
    if (tid == 0) {
        for (int i = 0; i < 4; ++i) {
            mbar_init(smem_u32(&sh.rfull[i]), 1);
            mbar_init(smem_u32(&sh.rempty[i]), KTU_DEC_WARPS / 2);
            mbar_init(smem_u32(&sh.ready[i]), 1);
            mbar_init(smem_u32(&sh.kfull[i]), KTU_DEC_WARPS / 2);
            mbar_init(smem_u32(&sh.qfull[i]), KTU_DEC_WARPS);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(smem_u32(&sh.vfull[i]), KTU_DEC_WARPS / 2);
            mbar_init(smem_u32(&sh.sfull[i]), 1);
            mbar_init(smem_u32(&sh.pfull[i]), SW);
            mbar_init(smem_u32(&sh.sempty[i]), SW);
            mbar_init(smem_u32(&sh.vempty[i]), 1);
            mbar_init(smem_u32(&sh.pempty[i]), 1);
        }
        mbar_init(smem_u32(&sh.done), 1);
        mbar_init_fence();
        sh.abort = 0;
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tm = sh.tmem, tlane = tm + ((uint32_t)(quad * 32) << 16);
    KtuCursor cur;
    cur.sequence(a, seq, sh.len);
    {
        const uint32_t item = (g0 - seq_tile) / (uint32_t)cur.tiles;
        cur.t = (int)(g0 - seq_tile - item * (uint32_t)cur.tiles);
        cur.hk = (int)(item / (uint32_t)groups);
        cur.grp = (int)item - cur.hk * groups;
    }
    const KtuCursor start = cur;

    constexpr int UB = ktu_ub(U), SB = ktu_sb(U), NST = ktu_stages(U, NR);
    constexpr int K_SH = 4 * KTU_KEYS * UB, K_SC = K_SH + 4 * KTU_KEYS * SB, V_UP = K_SC + 4 * KTU_KEYS, V_SC = V_UP + K_SC;
    const uint32_t ring = sbase + KTU_Q + NR * 512;               // stages: upper, shared codes and exponents of the keys, of the values
    const uint32_t vrow = (sbase + KTU_V + (key >> 3) * 1024 + (key & 7) * 128) | (key & 7) << 4;      // with the swizzle of chunk 0

    // A bounded wait of the whole warp.  Where one runs out, it sets sh.abort: from then on no wait waits any more and all roles go on
    // through the motions to the end -- they meet at named barriers, so none may leave early --; the outputs are marked then.
    auto wait = [&](const uint64_t& bar, uint32_t phase) {
        uint32_t left = a.max_polls;                              // (a try sleeps for up to about two microseconds)
        while (!mbar_try_wait(smem_u32(&bar), phase & 1u))
            if (sh.abort || --left == 0) { sh.abort = 1; break; }
        __syncwarp();
    };
    auto arrive = [&](const uint64_t& bar) {
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&bar));
    };

    if (warp < KTU_DEC_WARPS) {
        // ================================ decode ================================
        asm volatile("setmaxnreg.dec.sync.aligned.u32 56;");
        const int team = warp >> 3;
        const uint32_t tab = smem_u32(sh.scales);
        int seg = -1;
        uint32_t n_slot = 0, r_phase = 0;                         // the tile's slot of the ring
#pragma unroll 1
        for (int j = 0; j < n_run; ++j) {
            if (j == 0 || cur.t == 0) {
                // ---- a new item: its queries, rotated, scaled by a power of two per row, fp16, K-major with 128-byte swizzle ----
                ++seg;
                if (j > 0) wait(sh.sfull[(j - 1) & 1], (uint32_t)(j - 1) >> 1);      // the last item's products have read theirs
                const int hk = cur.hk, r0 = cur.grp * NR, rows = min(NR, R - r0);
                constexpr int QR = NR / KTU_DEC_WARPS;            // rows of a warp
                float v[QR][4];
                int top = -128, low = 127;                        // exponents of the rows that are numbers and not zero
                uint32_t bad = 0u;                                // rows with an infinity or a NaN: NaN, the others are not touched
                int E[QR];
#pragma unroll
                for (int k = 0; k < QR; ++k) {
                    const int row = r0 + warp * QR + k;
                    if (warp * QR + k < rows) {
                        const uint2 raw = __ldcg(reinterpret_cast<const uint2*>(
                            a.q + (((int64_t)cur.b * a.T + row / G) * a.Hq + hk * G + row % G) * 128 + lane * 4));
                        v[k][0] = bf16_lo(raw.x); v[k][1] = bf16_hi(raw.x);
                        v[k][2] = bf16_lo(raw.y); v[k][3] = bf16_hi(raw.y);
                    } else {
                        v[k][0] = v[k][1] = v[k][2] = v[k][3] = 0.0f;
                    }
                }
#pragma unroll
                for (int k = 0; k < QR; ++k) {
                    if (a.qrot) {
                        fwht_warp<4>(v[k], lane);
#pragma unroll
                        for (int i = 0; i < 4; ++i) v[k][i] *= 0.08838834764831845f;     // 1 / sqrt(128)
                    }
                    uint32_t ax = 0u;
#pragma unroll
                    for (int i = 0; i < 4; ++i) ax = max(ax, __float_as_uint(v[k][i]) & 0x7FFFFFFFu);
                    ax = __reduce_max_sync(0xffffffffu, ax);
                    E[k] = max((int)(ax >> 23) - 127, -100);
                    if (ax >= 0x7F800000u) bad |= 1u << k;
                    else if (ax) { top = max(top, E[k]); low = min(low, E[k]); }
                }
                if (lane == 0) { sh.qtop[warp] = top; sh.qlow[warp] = low; }
                ktu_bar(1, KTU_DEC_WARPS * 32);
                top = __reduce_max_sync(0xffffffffu, sh.qtop[lane % KTU_DEC_WARPS]);
                low = __reduce_min_sync(0xffffffffu, sh.qlow[lane % KTU_DEC_WARPS]);
                // largest element to [1024, 2048): of all rows where the smallest row still has its eleven digits then, else of each row
                const bool same = low >= top - 12;
#pragma unroll
                for (int k = 0; k < QR; ++k) {
                    const int r = warp * QR + k, e = max(same ? top : E[k], -100);
                    const float up = __int_as_float((137 - e) << 23);
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int p = ktu_place<U>(lane * 4 + i);
                        const float x = bad >> k & 1 ? 0.0f : v[k][i] * up;
                        const __half h = __float2half_rn(x);
                        __half* const to = reinterpret_cast<__half*>(smem + KTU_Q + (p >> 6) * ktu_q_half(NR) + r * 128 + ((((p >> 3) & 7) ^ (r & 7)) << 4) + (p & 7) * 2);
                        to[0] = h;
                        to[ktu_q_second(NR) / 2] = __float2half_rn(x - __half2float(h));
                    }
                    if (lane == 0) sh.qf[seg & 3][r] = bad >> k & 1 ? __int_as_float(0x7FC00000) : exp2_int(e - 10);
                }
                if (tid == 0) { sh.same[seg & 3] = same; sh.qscale[seg & 3] = exp2_int(max(top, -100) - 10); }
                fence_async_smem();
                arrive(sh.qfull[seg & 3]);
            }
            const uint32_t slot = n_slot, phase = r_phase;
            if (++n_slot == NST) { n_slot = 0; r_phase ^= 1u; }
            cur.next(a, groups, B);
            if ((j & 1) != team) continue;                        // the other team's tile
            wait(sh.rfull[slot], phase);
            wait(sh.ready[slot], phase);                          // (before the keys: the softmax takes kfull for a sign that sh.wide is there)
            const uint32_t st = ring + slot * ktu_stage_bytes(U);
            // ---- keys to tensor memory, once the product before the last has read the buffer ----
            const uint32_t se = st + key;
            const int e0 = lds_s8<0>(se + K_SC + 2 * half * KTU_KEYS), e1 = lds_s8<KTU_KEYS>(se + K_SC + 2 * half * KTU_KEYS);
            const int emax = max(max(e0, e1), max((int)lds_s8<0>(se + K_SC + (2 - 2 * half) * KTU_KEYS), (int)lds_s8<KTU_KEYS>(se + K_SC + (2 - 2 * half) * KTU_KEYS)));
            const bool wide = sh.wide[j & 7] != KTU_NARROW;
            if (half == 0) {
                float f = a.sm_scale_log2 * exp2_int(emax);
                if (wide && max(max((int)lds_s8<0>(se + V_SC), (int)lds_s8<KTU_KEYS>(se + V_SC)), max((int)lds_s8<2 * KTU_KEYS>(se + V_SC), (int)lds_s8<3 * KTU_KEYS>(se + V_SC))) > KTU_TOP)
                    f = __int_as_float(0x7FC00000);               // no number: what attends this key is none either
                sh.ck[j & 3][key] = f;
            }
            if (j > 1) wait(sh.sfull[team], (uint32_t)(j - 2) >> 1);
            tc_fence_after();
            const uint32_t row = vrow + team * 32768 + half * 16384;
            // This thread's two blocks of the key, then of the value.  (One rolled loop for all: the roles share an instruction cache, and with
            // the blocks unrolled this kernel took a third longer.)
            uint32_t up = st + (2 * half * KTU_KEYS + key) * UB, shd = st + K_SH + (2 * half * KTU_KEYS + key) * SB;
#pragma unroll 1
            for (int i = 0; i < 4; ++i) {
                KtuRaw<U> raw;
                ktu_load(raw, up, shd);
                up += i == 1 ? V_UP - KTU_KEYS * UB : KTU_KEYS * UB;
                shd += i == 1 ? V_UP - KTU_KEYS * SB : KTU_KEYS * SB;
                int d = (i == 0 ? e0 : e1) - emax;
                if (i >= 2) {
                    if (i == 2) {
                        ktu_st_wait();
                        tc_fence_before();
                        arrive(sh.kfull[j & 3]);
                        // the product before the last has read the values' buffer
                        if (j > 1) wait(sh.vempty[team], (uint32_t)(j - 2) >> 1);
                    }
                    // (in bf16: the codes here, their exponent below; out of range otherwise: zeros, or a key that no row attends)
                    d = wide ? 0 : min(lds_s8<0>(se + V_SC + (2 * half + i - 2) * KTU_KEYS), 5) - 1;
                }
                const uint4 sc = lds128(tab + (4 - max(d, -27)) * 16);
                uint32_t w[16];
                ktu_convert(raw, sc, [&](int c, uint32_t w0, uint32_t w1, uint32_t w2, uint32_t w3) {
                    w[4 * c] = w0; w[4 * c + 1] = w1; w[4 * c + 2] = w2; w[4 * c + 3] = w3;
                });
                if (i < 2) {
                    ktu_st16(tlane + KTU_COL_K + team * 64 + half * 32 + i * 16, w);
                    continue;
                }
                if (wide) {
                    const float f = exp2_int(max(-126, min(KTU_TOP, lds_s8<0>(se + V_SC + (2 * half + i - 2) * KTU_KEYS)) - 1));
#pragma unroll
                    for (int c = 0; c < 16; ++c) {                            // eight digits: exact
                        const float2 q = __half22float2(*reinterpret_cast<const __half2*>(&w[c]));
                        w[c] = prmt(__float_as_uint(q.x * f), __float_as_uint(q.y * f), 0x7632u);
                    }
                }
                const uint32_t to = row ^ (i & 1) << 6;
#pragma unroll
                for (int c = 0; c < 4; ++c) sts128(to ^ c << 4, w[4 * c], w[4 * c + 1], w[4 * c + 2], w[4 * c + 3]);
            }
            arrive(sh.rempty[slot]);
            fence_async_smem();
            arrive(sh.vfull[team]);
        }
    } else if (warp < WARP_MMA) {
        // ================================ softmax ================================
        asm volatile("setmaxnreg.inc.sync.aligned.u32 120;");
        const uint32_t prow = (sbase + KTU_P + (key >> 3) * 1024 + (key & 7) * 128) | (key & 7) << 4;
        const int stid = tid - KTU_DEC_WARPS * 32, htid = stid & 127;             // thread of the role, of its half
        int seg = -1, n_seg = 0;
        bool same = true;                                         // the item's query rows have one score factor
        float qscale = 1.0f, lower = 0.0f;                        // lower: bits that the segment's probabilities are lower by
        uint64_t l[NC / 2];                                       // sums of pairs of rows over this thread's keys
#pragma unroll 1
        for (int j = 0; j < n_run; ++j) {
            const int r0 = cur.grp * NR;
            if (j == 0 || cur.t == 0) {
                ++seg;
                n_seg = 0;
                lower = 0.0f;
                wait(sh.qfull[seg & 3], (uint32_t)seg >> 2);
                ktu_bar(2, SW * 32);                       // the last item's masks and references are read
                if (stid < a.T) sh.mask[stid] = a.mask[cur.b * a.mask_stride + stid];
                if (stid < NR) {
                    const float f = sh.qf[seg & 3][stid];
                    sh.f[stid] = f;
                    reinterpret_cast<float*>(sh.ref4)[stid] = f != f ? f : INFINITY;
                    sh.m[stid] = -INFINITY;
                }
                same = sh.same[seg & 3] != 0;
                qscale = sh.qscale[seg & 3];
                ktu_bar(2, SW * 32);
#pragma unroll
                for (int c = 0; c < NC / 2; ++c) l[c] = 0ull;
            }
            const int jb = cur.t * KTU_KEYS;
            const bool tail = jb + KTU_KEYS > cur.len;            // the tile has nodes of the tree
            wait(sh.kfull[j & 3], (uint32_t)j >> 2);
            const float ck = same ? sh.ck[j & 3][key] * qscale : sh.ck[j & 3][key];
            const int range = sh.wide[j & 7];
            const bool wide = range != KTU_NARROW;
            uint32_t vis = 0xFFFFFFFFu;                           // which of this thread's rows attend its key
            if (tail) {
                const int k = jb + key - cur.len;                 // below 0: in front of the tree
                if (k >= 0) {
                    vis = 0u;
                    if (k < a.T)
                        for (int c = 0; c < NC; ++c) {
                            const int node = (r0 + half * NC + c) / G;
                            if (node < a.T && (sh.mask[node] >> k & 1)) vis |= 1u << c;
                        }
                }
            }
            wait(sh.sfull[j & 1], (uint32_t)j >> 1);
            tc_fence_after();
            const uint32_t scol = tlane + KTU_COL_S + (j & 1) * 64 + half * NC;
            float x[NC];
            auto scores = [&]() {                                 // exponents of this tile's probabilities on the present references
                ktu_ld<NC>(scol, x);
                if constexpr (ktu_q_joint(NR)) {                  // the second numbers' share
                    float x2[NC];
                    ktu_ld<NC>(scol + NR, x2);
#pragma unroll
                    for (int c = 0; c < NC; c += 2) unpack2(add2(pack2(x[c], x[c + 1]), pack2(x2[c], x2[c + 1])), x[c], x[c + 1]);
                }
                const uint64_t ck2 = pack2(ck, ck);
                if (!same)
#pragma unroll
                    for (int c = 0; c < NC; ++c) x[c] *= sh.f[half * NC + c];
#pragma unroll
                for (int c = 0; c < NC; c += 4) {
                    const float4 rf = sh.ref4[(half * NC + c) / 4];
                    unpack2(fma2(pack2(x[c], x[c + 1]), ck2, pack2(rf.x, rf.y)), x[c], x[c + 1]);
                    unpack2(fma2(pack2(x[c + 2], x[c + 3]), ck2, pack2(rf.z, rf.w)), x[c + 2], x[c + 3]);
                }
                if (tail)
#pragma unroll
                    for (int c = 0; c < NC; ++c)
                        if (!(vis >> c & 1)) x[c] = -INFINITY;
            };
            // the product that read this tile's buffer of the probabilities is done
            if (j >= PB) wait(sh.pempty[(j - PB) & 1], (uint32_t)(j - PB) >> 1);
            bool moved = false;
#pragma unroll 1
            for (;;) {
                scores();
                float top = x[0], top1 = x[1];
#pragma unroll
                for (int c = 2; c < NC; c += 2) {
                    top = fmaxf(top, x[c]);
                    top1 = fmaxf(top1, x[c + 1]);
                }
                const float drop = range == KTU_HUGE && lower == 0.0f ? ktu_huge_bits(a.Lk) : 0.0f;
                if (moved || !ktu_vote(3 + half, 128, n_seg == 0 || drop > 0.0f || fmaxf(top, top1) > KTU_MOVE - lower)) break;
                moved = true;
                lower += drop;
                // ---- references move: rows of this half whose maximum of this tile is beyond theirs; all, where they get lower ----
                if (n_seg > 0) wait(sh.pempty[(j - 1) & 1], (uint32_t)(j - 1) >> 1);  // the accumulators are at rest
#pragma unroll 1
                for (int c = 0; c < NC; c += 8) {
                    float s[8];
                    ktu_ld8(scol + c, s);
                    if constexpr (ktu_q_joint(NR)) {
                        float s2[8];
                        ktu_ld8(scol + NR + c, s2);
#pragma unroll
                        for (int k = 0; k < 8; ++k) s[k] += s2[k];
                    }
#pragma unroll
                    for (int k = 0; k < 8; ++k) {
                        const int r = half * NC + c + k;
                        float t = s[k] * ck * (same ? 1.0f : sh.f[r]);
                        if (!(vis >> (c + k) & 1) || t != t) t = -INFINITY;
                        float mx;
                        asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(mx) : "f"(t));
                        if (lane == 0) sh.part[quad][r] = mx;
                    }
                }
                ktu_bar(3 + half, 128);
                if (htid < NC) {
                    const int r = half * NC + htid;
                    const float mx = fmaxf(fmaxf(sh.part[0][r], sh.part[1][r]), fmaxf(sh.part[2][r], sh.part[3][r])), m = sh.m[r];
                    float al = -drop, to = m;
                    float* const rf = reinterpret_cast<float*>(sh.ref4) + r;
                    if (*rf == *rf && mx > -INFINITY && (m == -INFINITY || mx - m > KTU_MOVE - KTU_P_BITS)) {
                        al = m - mx - drop;                       // (-inf: nothing seen yet)
                        to = mx;
                    }
                    if (*rf == *rf && to > -INFINITY) {
                        sh.m[r] = to;
                        *rf = KTU_P_BITS - lower - to;
                    }
                    sh.alpha[r] = ktu_exp2(al);
                }
                ktu_bar(3 + half, 128);
                tc_fence_after();
                if (n_seg > 0) {
#pragma unroll 1
                    for (int c = 0; c < 2 * NC; c += 8) {         // both accumulators of a row
                        const int r = half * NC + c % NC, col = r + (c < NC ? 0 : NR);
                        float o[8];
                        ktu_ld8(tlane + KTU_COL_O + col, o);
#pragma unroll
                        for (int k = 0; k < 8; ++k) {
                            o[k] *= sh.alpha[r + k];
                        }
                        ktu_st8(tlane + KTU_COL_O + col, o);
                    }
#pragma unroll
                    for (int c = 0; c < NC; c += 2) {
                        const float al0 = sh.alpha[half * NC + c], al1 = sh.alpha[half * NC + c + 1];
                        float l0, l1;
                        unpack2(l[c / 2], l0, l1);
                        l[c / 2] = pack2(l0 * al0, l1 * al1);
                    }
                    ktu_st_wait();
                }
            }
            tc_fence_before();
            arrive(sh.sempty[j & 1]);
            // ---- probabilities to shared memory, in the type of the tile's values: the leading digits, then what they leave ----
            const uint32_t pr = prow + (PB == 2 ? (j & 1) * 16384 : 0), keep = wide ? 0xFFFF0000u : 0xFFFFE000u;
            const uint64_t minus = pack2(-1.0f, -1.0f);
#pragma unroll
            for (int c = 0; c < NC; c += 8) {
                uint32_t w[4], w2[4];
#pragma unroll
                for (int k = 0; k < 8; k += 2) {
                    x[c + k] = ktu_exp2(x[c + k]);
                    x[c + k + 1] = ktu_exp2(x[c + k + 1]);
                    l[(c + k) / 2] = add2(l[(c + k) / 2], pack2(x[c + k], x[c + k + 1]));
                    const float h0 = __uint_as_float(__float_as_uint(x[c + k]) & keep), h1 = __uint_as_float(__float_as_uint(x[c + k + 1]) & keep);
                    float r0, r1;
                    unpack2(fma2(pack2(h0, h1), minus, pack2(x[c + k], x[c + k + 1])), r0, r1);
                    if (wide) {
                        w[k >> 1] = prmt(__float_as_uint(h0), __float_as_uint(h1), 0x7632u);
                        asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(w2[k >> 1]) : "f"(r1), "f"(r0));
                    } else {
                        asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(w[k >> 1]) : "f"(h1), "f"(h0));
                        asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(w2[k >> 1]) : "f"(r1), "f"(r0));
                    }
                }
                const uint32_t to = pr ^ (half * (NC / 8) + c / 8) << 4;
                sts128(to, w[0], w[1], w[2], w[3]);
                sts128(NR > 32 ? to + ktu_p_second(NR) : to ^ ktu_p_second(NR), w2[0], w2[1], w2[2], w2[3]);
            }
            fence_async_smem();
            tc_fence_before();
            arrive(sh.pfull[j & 1]);
            ++n_seg;

            if (cur.t == cur.tiles - 1 || j == n_run - 1) {
                // ---- the segment's result ----
                if (j == n_run - 1) chain_release();              // the merge's blocks may come: they wait for this grid, and want no tensor memory
                const bool whole = n_seg == cur.tiles;            // finished here; else partial result 2 c (not the item's first) or 2 c + 1
                const int64_t part = ((int64_t)2 * blockIdx.x + (cur.t == n_seg - 1 ? 1 : 0)) * NR * KTU_PART;
                const int rows = min(NR, R - r0), hk = cur.hk;
                {
                    float v[NC];
#pragma unroll
                    for (int c = 0; c < NC; c += 2) unpack2(l[c / 2], v[c], v[c + 1]);
                    ktu_column_sums<NC>(v, lane);
                    if (lane < NC) sh.part[quad][half * NC + lane] = v[0];
                }
                ktu_bar(3 + half, 128);
                if (htid < NC) {
                    const int r = half * NC + htid;
                    const float s = (sh.part[0][r] + sh.part[1][r]) + (sh.part[2][r] + sh.part[3][r]);
                    sh.alpha[r] = s == 0.0f ? 0.0f : 2.0f / s;            // (values are held halved)
                    const int row = r0 + r;
                    sh.row[r] = whole ? (((int64_t)cur.b * a.T + row / G) * a.Hq + hk * G + row % G) * 128 : part + r * KTU_PART;
                    if (!whole) {
                        a.partial[part + r * KTU_PART + 128] = sh.m[r] + lower;
                        a.partial[part + r * KTU_PART + 129] = s;
                    }
                }
                ktu_bar(3 + half, 128);
                wait(sh.pempty[j & 1], (uint32_t)j >> 1);
                tc_fence_after();
                const int ch = ktu_element<U>(key);                           // accumulator lane = operand place of the channel
#pragma unroll 1
                for (int c = half * NC; c < min(half * NC + NC, rows); c += 8) {
                    float o[8], o2[8];
                    ktu_ld8(tlane + KTU_COL_O + c, o);
                    ktu_ld8(tlane + KTU_COL_O + NR + c, o2);
#pragma unroll
                    for (int k = 0; k < 8; ++k) {
                        o[k] += o2[k];
                        const int64_t at = sh.row[c + k] + ch;
                        if (!whole) {
                            a.partial[at] = o[k];
                        } else if (c + k < rows) {
                            const float f = sh.alpha[c + k], v = f == 0.0f ? 0.0f : o[k] * f;
                            out[at] = __float2bfloat16_rn(v);
                            if (out_f32) out_f32[at] = v;
                        }
                    }
                }
                tc_fence_before();
            }
            cur.next(a, groups, B);
        }
    } else {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 40;");
    }
    if (warp == WARP_MMA) {
        // ================================ MMAs ================================
        const uint32_t idesc_qk = ktu_idesc(ktu_q_joint(NR) ? 2 * NR : NR, 0, 0), hi = ktu_desc_hi(1024);
        const uint32_t q_lo = umma_desc_lo(sbase + KTU_Q, 16), v_lo = umma_desc_lo(sbase + KTU_V, 16384), p_lo = umma_desc_lo(sbase + KTU_P, 16384);
        int seg = -1;
        KtuCursor ahead = cur;                                    // of the scores' product, one tile in front
        auto issue_qk = [&](int j) {
            if (j == 0 || ahead.t == 0) {
                ++seg;
                wait(sh.qfull[seg & 3], (uint32_t)seg >> 2);
            }
            wait(sh.kfull[j & 3], (uint32_t)j >> 2);
            if (j > 1) wait(sh.sempty[j & 1], (uint32_t)(j - 2) >> 1);
            tc_fence_after();
            if (elect_lane()) {
#pragma unroll 1
                for (int s = 0; s < (ktu_q_joint(NR) ? 8 : 16); ++s)     // keys by the queries' first numbers and their second ones
                    ktu_mma_ts(tm + KTU_COL_S + (j & 1) * 64, tm + KTU_COL_K + (j & 1) * 64 + 8 * (s & 7),
                               q_lo + (s >> 2) * (ktu_q_half(NR) / 16) + (s & 3) * 2, hi, idesc_qk, s > 0);
                if (!(a.skip_stage == j && blockIdx.x == 0)) tc_commit(smem_u32(&sh.sfull[j & 1]));
            }
            __syncwarp();
            ahead.next(a, groups, B);
        };
        bool first = true;                                        // the next product begins a segment: it overwrites the accumulators
        issue_qk(0);
#pragma unroll 1
        for (int j = 0; j < n_run; ++j) {
            if (j + 1 < n_run) issue_qk(j + 1);
            wait(sh.vfull[j & 1], (uint32_t)j >> 1);
            wait(sh.pfull[j & 1], (uint32_t)j >> 1);
            tc_fence_after();
            const uint32_t id = ktu_idesc(2 * NR, sh.wide[j & 7] != KTU_NARROW, 1u);
            if (elect_lane()) {
#pragma unroll 1
                for (int s = 0; s < 8; ++s)                   // values by the probabilities' first and second numbers, side by side
                    ktu_mma_ss(tm + KTU_COL_O, v_lo + (j & 1) * 2048 + s * 128, hi, p_lo + (PB == 2 ? (j & 1) * 1024 : 0) + s * 128, hi, id, !first || s > 0);
                tc_commit(smem_u32(&sh.vempty[j & 1]));
                tc_commit(smem_u32(&sh.pempty[j & 1]));
            }
            __syncwarp();
            first = cur.t == cur.tiles - 1;
            cur.next(a, groups, B);
        }
        // nothing may still write tensor memory when it is returned
        if (elect_lane()) {
            tc_commit(smem_u32(&sh.done));
            mbar_wait_bounded(smem_u32(&sh.done), 0);
        }
        __syncwarp();
    } else if (warp == WARP_COPY) {
        // ================================ copies ================================
        // Lane 4 p + i brings plane p (keys: upper, shared, exponents; values: the same) of block i.
        const int p = lane >> 2, i = lane & 3, kind = p % 3, per_key = kind == 0 ? UB : kind == 1 ? SB : 1;
        const KvPlanes& pl = p < 3 ? a.k : a.v;
        const uint8_t* src = kind == 0 ? pl.u : kind == 1 ? pl.h : reinterpret_cast<const uint8_t*>(pl.s);
        const uint32_t dst = (p < 3 ? 0 : V_UP) + (kind == 0 ? 0 : kind == 1 ? K_SH : K_SC) + i * KTU_KEYS * per_key;
        uint32_t slot = 0, phase = 1;                             // passes at once on a fresh barrier
        int issued = 0;
        for (int j = 0; j < n_run; ++j) {
            wait(sh.rempty[slot], phase);
            // After a give-up the slot may still be on its way or being read: no more copies, and only what was issued is waited for below.  (The
            // other roles wait for nothing then, and this warp meets them at the block's last barrier only.)
            if (__any_sync(0xffffffffu, sh.abort)) break;
            const int n = min(KTU_KEYS, (cur.len + a.T - cur.t * KTU_KEYS + 15) & ~15);            // whole groups of 16 (so is the capacity)
            const int64_t row = (((int64_t)cur.b * a.Hkv + cur.hk) * 4 + i) * a.Lcap + cur.t * KTU_KEYS;
            const uint32_t bar = smem_u32(&sh.rfull[slot]);
            if (lane == 0) mbar_expect_tx(bar, (uint32_t)(n * 8 * (UB + SB + 1)));
            __syncwarp();
            if (lane < 24) bulk_g2s(ring + slot * ktu_stage_bytes(U) + dst, src + row * per_key, (uint32_t)(n * per_key), bar);
            ++issued;
            cur.next(a, groups, B);
            if (++slot == NST) { slot = 0; phase ^= 1u; }
        }
        // shared memory is not handed on with a copy in flight
        for (int j = max(0, issued - NST); j < issued; ++j) mbar_wait_bounded(smem_u32(&sh.rfull[j % NST]), (uint32_t)(j / NST) & 1u);
        __syncwarp();
    } else if (warp == WARP_SCOUT) {
        // ================================ value exponents ================================
        uint32_t slot = 0, phase = 0;
        bool huge = false;                                        // of a tile of this item so far
        uint64_t named = 0;                                       // nodes that some node of the sequence attends
        int whose = -1;                                           // that sequence
        for (int j = 0; j < n_run; ++j) {
            const int node = cur.t * KTU_KEYS + (lane & 7) * 16 - cur.len;         // of this lane's first key; below 0: in front of the tree
            if (whose != cur.b && (cur.t + 1) * KTU_KEYS > cur.len) {
                whose = cur.b;
                const uint64_t* const words = a.mask + cur.b * a.mask_stride;
                named = (lane < a.T ? words[lane] : 0ull) | (lane + 32 < a.T ? words[lane + 32] : 0ull);
                named = (uint64_t)__reduce_or_sync(0xffffffffu, (uint32_t)(named >> 32)) << 32 | __reduce_or_sync(0xffffffffu, (uint32_t)named);
                named &= ~0ull >> (64 - a.T);
            }
            // which of the lane's sixteen keys somebody attends
            const uint32_t keys = node <= -16 ? 0xFFFFu : node < 0 ? (uint32_t)(named << -node) | ((1u << -node) - 1u) : node < 64 ? (uint32_t)(named >> node) : 0u;
            wait(sh.rfull[slot], phase);
            const uint4 v = lds128<V_SC>(ring + slot * ktu_stage_bytes(U) + lane * 16);            // block lane / 8, keys 16 (lane % 8) ..
            int top = -128, low = 127;                            // of the exponents that are no zeros
            uint64_t lo = (uint64_t)v.y << 32 | v.x, hi = (uint64_t)v.w << 32 | v.z;
#pragma unroll 1
            for (int k = 0; k < 8; ++k, lo >>= 8, hi >>= 8) {
                const int e0 = (int8_t)lo, e1 = (int8_t)hi;
                if (keys >> k & 1 && e0 > -106) { top = max(top, e0); low = min(low, e0); }
                if (keys >> (k + 8) & 1 && e1 > -106) { top = max(top, e1); low = min(low, e1); }
            }
            top = __reduce_max_sync(0xffffffffu, top);
            low = __reduce_min_sync(0xffffffffu, low);
            huge = (huge && cur.t > 0) || top >= ktu_huge_from(a.Lk);
            if (lane == 0) sh.wide[j & 7] = huge ? KTU_HUGE : top > 5 || low < -23 ? KTU_WIDE : KTU_NARROW;
            arrive(sh.ready[slot]);
            cur.next(a, groups, B);
            if (++slot == NST) { slot = 0; phase ^= 1u; }
        }
    }

    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (warp == WARP_MMA) tmem_dealloc(tm, KTU_COLS);
    if (sh.abort) {
        // a wait gave up: everything of this run is marked
        if (tid == 0) report_wait_failure(a.sticky, WAIT_FAIL_KV_DECODE);
        cur = start;
        for (int j = 0, n_seg = 0; j < n_run; ++j) {
            ++n_seg;
            if (cur.t == cur.tiles - 1 || j == n_run - 1) {
                const int r0 = cur.grp * NR, rows = min(NR, R - r0), hk = cur.hk;
                float* const part = a.partial + ((int64_t)2 * blockIdx.x + (cur.t == n_seg - 1 ? 1 : 0)) * NR * KTU_PART;
                for (int i = tid; i < rows * 128; i += WARPS * 32) {
                    const int row = r0 + (i >> 7);
                    const int64_t o = (((int64_t)cur.b * a.T + row / G) * a.Hq + hk * G + row % G) * 128 + (i & 127);
                    if (n_seg == cur.tiles) {
                        out[o] = __float2bfloat16_rn(__int_as_float(0x7FC00000));
                        if (out_f32) out_f32[o] = __int_as_float(0x7FC00000);
                    } else if ((i & 127) == 0) {
                        part[(i >> 7) * KTU_PART + 128] = __int_as_float(0x7FC00000);
                    }
                }
                n_seg = 0;
            }
            cur.next(a, groups, B);
        }
    }
}

// Merge of the items that were cut: a warp per row, the runs' results in their order.  Run c left an item's first part in slot 2 c + 1 and
// any other in slot 2 c.  A NaN in m marks a run whose wait gave up.
template <int NR>
__global__ void __launch_bounds__(256)
kv_tree_merge_kernel(const KvTreeArgs a, int B, int groups, int blocks, __nv_bfloat16* __restrict__ out, float* __restrict__ out_f32) {
    chain_release();
    chain_wait();
    __shared__ uint32_t red[16];
    const int per_seq = a.Hkv * groups, G = a.Hq / a.Hkv, R = a.T * G;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int b = blockIdx.y, item = blockIdx.x / (NR / 8), r = blockIdx.x % (NR / 8) * 8 + warp;
    const int hk = item / groups, row = item % groups * NR + r;
    uint32_t before = 0u, all = 0u;                               // tiles of the sequences in front, of all
    for (int i = threadIdx.x; i < B; i += 256) {
        const uint32_t n = ktu_tiles(a, kt_len(a, i));
        all += n;
        if (i < b) before += n;
    }
    before = __reduce_add_sync(0xffffffffu, before);
    all = __reduce_add_sync(0xffffffffu, all);
    if (lane == 0) { red[warp] = before; red[8 + warp] = all; }
    __syncthreads();
    before = __reduce_add_sync(0xffffffffu, lane < 8 ? red[lane] : 0u);
    all = __reduce_add_sync(0xffffffffu, lane < 8 ? red[8 + lane] : 0u);
    const KtuLine line(all * (uint32_t)per_seq, (uint32_t)blocks);
    const uint32_t tiles = ktu_tiles(a, kt_len(a, b)), g = before * (uint32_t)per_seq + (uint32_t)item * tiles;
    const int first = (int)line.owner(g), last = (int)line.owner(g + tiles - 1u);
    if (first == last || row >= R) return;
    const int n = last - first + 1;
    auto slot = [&](int i) { return a.partial + (((int64_t)2 * (first + i) + (i == 0 ? 1 : 0)) * NR + r) * KTU_PART; };
    float mg = -INFINITY, acc[4] = {0.0f, 0.0f, 0.0f, 0.0f}, den = 0.0f;
    bool bad = false;
#pragma unroll 1
    for (int i0 = 0; i0 < n; i0 += 8) {                           // eight results on their way at a time, weights relative to the largest so far
        float4 v[8];
        float m[8], l[8], top = mg;
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            m[k] = -INFINITY;
            l[k] = 0.0f;
            if (i0 + k >= n) continue;
            const float* p = slot(i0 + k);
            v[k] = *reinterpret_cast<const float4*>(p + 4 * lane);
            m[k] = p[128];
            l[k] = p[129];
        }
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            bad = bad || m[k] != m[k];
            top = fmaxf(top, m[k]);
        }
        const float old = mg == top ? 1.0f : exp2f(mg - top);
        mg = top;
        den *= old;
#pragma unroll
        for (int k = 0; k < 4; ++k) acc[k] *= old;
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            if (m[k] == -INFINITY && l[k] == 0.0f) continue;       // a part of which the row attends nothing, or none
            const float w = exp2f(m[k] - mg);
            acc[0] = fmaf(v[k].x, w, acc[0]);
            acc[1] = fmaf(v[k].y, w, acc[1]);
            acc[2] = fmaf(v[k].z, w, acc[2]);
            acc[3] = fmaf(v[k].w, w, acc[3]);
            den = fmaf(l[k], w, den);
        }
    }
    const float f = den == 0.0f ? 0.0f : 2.0f / den;              // (values were held halved)
    const int64_t o = (((int64_t)b * a.T + row / G) * a.Hq + hk * G + row % G) * 128 + 4 * lane;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        float v = f == 0.0f ? 0.0f : acc[k] * f;
        if (bad) v = __int_as_float(0x7FC00000);
        out[o + k] = __float2bfloat16_rn(v);
        if (out_f32) out_f32[o + k] = v;
    }
}

}  // namespace msaq
