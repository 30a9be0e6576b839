// From the QKV projection's output to attention in one launch: norms of the query and key heads, rotary embedding, the query
// rows out in bf16, the key rows (Hadamard-rotated where the cache is) and the value rows quantised into the cache -- for one
// token, for the nodes of a drafted tree (whose positions differ from their slots) and for a prompt.  And the move that follows
// the verification of a drafted tree: the accepted nodes' rows become neighbours.
//
// A head row x with gain g becomes  y = bf16( rope( (x r) g ) ),  r = fl32( (mean(x^2) + eps)^(-1/2) ).  Mean and root are taken
// in 64 bits: r then depends on how the sum is split over lanes only where the 64-bit number lies within about 2^-52 of a border
// between two fp32 numbers, once in 2^28 rows, and so do the codes that the quantiser derives from y (in 32 bits one key row in about ten
// thousand would land on other codes).  The remaining steps are fp32 operations,
// each rounded by itself.
//
// A token moves 2 D (2 Hq + 2 Hkv) + 2 Hkv NB (UB + SB + 1) bytes and 4 D of tables: 185 MB for 8191 tokens of 32 + 2 x 8 heads (28 us).
// What bounds a prompt are the instructions (59 us: qkv_write8_kernel), one token the call (10 us, 2.6 of them on the device).
#include <algorithm>

#include "kv_quant_row.cuh"

namespace msaq {
namespace {

constexpr int QKV_WARPS = 4;
constexpr int KEEP_MAX_T = 64;

struct QkvArgs {
    const __nv_bfloat16* x;              // [B * T] tokens of Hq + 2 Hkv heads, ld elements from one token to the next
    __nv_bfloat16* q_out;                // [B * T][Hq][D]
    QuantJob k, v;
    int64_t ld, start, Lcap;
    const int32_t* start_per_seq;
    const int32_t* pos;                  // optional [B][T]: positions; null: the slots
    const int32_t* counts;               // optional [B]: tokens of a sequence, the rest is padding
    const void* q_gain;                  // optional [D]
    const void* k_gain;
    Rope rope;
    double eps;
    int* sticky;
    int B, T, Hq, Hkv, gain_f32;
    bool wide, rope_wide;                // x, ld and q_out, the tables allow 16-byte accesses
    int64_t q_blocks, k_blocks;          // lane per element: thread blocks of the query rows, of the key rows (as many of the value rows)
    int q_heads, kv_heads;               // eight values per lane: heads of a run
    int kv_chunks, chunks;               // runs of the key heads (as many of the value heads), of all heads of a token
};

// (mean + eps)^(-1/2) rounded to fp32: one Newton step of third order in 64 bits on the 32-bit estimate (what the series leaves out
// is below 2^-60, its roundings come to about 2^-52); a sum beyond the range of fp32 takes the slow root.
__device__ __forceinline__ float norm_factor(double ss, int D, double eps) {
    const double m = ss / (double)D + eps;
    if (!(m > 1e-36 && m < 1e36)) return (float)(1.0 / sqrt(m));
    float y32;
    asm("rsqrt.approx.ftz.f32 %0, %1;" : "=f"(y32) : "f"((float)m));
    const double y = (double)y32;
    const double e = fma(-m * y, y, 1.0);
    return (float)fma(y * e, fma(0.375, e, 0.5), y);
}

__device__ __forceinline__ float gain_at(const void* g, int f32, int i) {
    return f32 ? static_cast<const float*>(g)[i] : __bfloat162float(static_cast<const __nv_bfloat16*>(g)[i]);
}

// Where a token's rows go: its sequence, slot and position.  `live` on return: not padding (q), and its slot inside the cache (k, v).
struct QkvToken {
    int64_t token, key, at;
    int b;
    bool live;
};

__device__ __forceinline__ QkvToken qkv_token(const QkvArgs& a, int64_t token, bool into_cache, bool report) {
    QkvToken r;
    r.live = token < (int64_t)a.B * a.T;
    r.token = r.live ? token : 0;
    r.b = (int)((uint32_t)r.token / (uint32_t)a.T);            // B T fits 31 bits
    const int t = (int)(r.token - (int64_t)r.b * a.T);
    if (a.counts && t >= a.counts[r.b]) r.live = false;
    r.key = (a.start_per_seq ? (int64_t)a.start_per_seq[r.b] : a.start) + t;
    r.at = a.pos ? (int64_t)a.pos[r.token] : r.key;
    bool bad = into_cache && (r.key < 0 || r.key >= a.Lcap);
    if (a.rope.cos) {
        if (a.rope.rows == 1) r.at = 0;
        const int64_t p = min(max(r.at, (int64_t)0), a.rope.rows - 1);
        bad = bad || p != r.at;
        r.at = p;
    }
    if (bad && r.live) {                                       // a position from device memory: the row is skipped, the status word says so
        if (report && a.sticky) atomicOr(a.sticky, BAD_APPEND_POS);
        if (into_cache) r.live = false;
    }
    return r;
}

__device__ __forceinline__ void qkv_floats(const float* p, bool wide, float (&v)[4]) {
    if (wide) {
        const float4 t = *reinterpret_cast<const float4*>(p);
        v[0] = t.x; v[1] = t.y; v[2] = t.z; v[3] = t.w;
    } else
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = p[i];
}

// Eight bf16 as four words.
__device__ __forceinline__ uint4 qkv_load8(const __nv_bfloat16* p, bool wide) {
    if (wide) return *reinterpret_cast<const uint4*>(p);
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = (uint32_t)__bfloat16_as_ushort(p[2 * i]) | (uint32_t)__bfloat16_as_ushort(p[2 * i + 1]) << 16;
    return make_uint4(w[0], w[1], w[2], w[3]);
}

// The gs = 2 formats: eight values per lane, 4 EPL lanes to a token, 8 / EPL tokens to a warp, nothing through shared memory.  A
// lane keeps its token's sines and its gains in registers over a run of heads, and the next head's values are on their way while
// one is worked on; neighbouring tokens fill the sectors of the planes together.  What it spends its time on is instructions (a
// prompt of 8191 tokens, 32 + 2 x 8 heads: with one head per warp, its index arithmetic and narrow loads of gains and sines, 440
// per warp and row pair and 96 us; now 59 us, 185 MB at 3.1 TB/s, the schedulers busy four cycles in five).
template <int EPL, int U>
__global__ void __launch_bounds__(QKV_WARPS * 32)
qkv_write8_kernel(const QkvArgs a) {
    chain_release();
    chain_wait();
    constexpr int D = 32 * EPL, LANES = 4 * EPL, TOKENS = 8 / EPL * QKV_WARPS;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, l = lane % LANES;
    const uint32_t block = blockIdx.x / (uint32_t)a.chunks;
    int chunk = (int)(blockIdx.x - block * (uint32_t)a.chunks);
    const int kind = chunk < a.kv_chunks ? 1 : chunk < 2 * a.kv_chunks ? 2 : 0;
    chunk -= kind == 1 ? 0 : kind == 2 ? a.kv_chunks : 2 * a.kv_chunks;
    const int per = kind == 0 ? a.q_heads : a.kv_heads, heads = kind == 0 ? a.Hq : a.Hkv;
    const int h0 = chunk * per, h1 = min(h0 + per, heads);
    const int64_t token = (int64_t)block * TOKENS + warp * (8 / EPL) + lane / LANES;
    const QkvToken r = qkv_token(a, token, kind != 0, l == 0 && chunk == 0);
    const bool in_range = token < (int64_t)a.B * a.T;
    if (__ballot_sync(0xffffffffu, kind == 0 ? in_range : r.live) == 0u) return;

    const __nv_bfloat16* src = a.x + r.token * a.ld + (int64_t)((kind == 0 ? 0 : kind == 1 ? a.Hq : a.Hq + a.Hkv) + h0) * D + l * 8;
    uint4 next = r.live ? qkv_load8(src, a.wide) : make_uint4(0u, 0u, 0u, 0u);
    const void* gain = kind == 0 ? a.q_gain : kind == 1 ? a.k_gain : nullptr;
    const bool rope = kind != 2 && a.rope.cos;
    float g[8], cs[4], sn[4];
    if (gain)
#pragma unroll
        for (int i = 0; i < 8; ++i) g[i] = gain_at(gain, a.gain_f32, l * 8 + i);
    if (rope) {
        qkv_floats(a.rope.cos + r.at * (D / 2) + l * 4, a.rope_wide, cs);
        qkv_floats(a.rope.sin + r.at * (D / 2) + l * 4, a.rope_wide, sn);
    }
#pragma unroll 1
    for (int h = h0; h < h1; ++h) {
        uint32_t w[4] = {next.x, next.y, next.z, next.w};
        src += D;
        if (r.live && h + 1 < h1) next = qkv_load8(src, a.wide);
        float v[8];
#pragma unroll
        for (int i = 0; i < 4; ++i) { v[2 * i] = bf16_lo(w[i]); v[2 * i + 1] = bf16_hi(w[i]); }
        if (gain) {
            double ss = 0.0;
#pragma unroll
            for (int i = 0; i < 8; ++i) ss = fma((double)v[i], (double)v[i], ss);
#pragma unroll
            for (int m = 1; m < LANES; m <<= 1) ss += __shfl_xor_sync(0xffffffffu, ss, m);
            const float f = norm_factor(ss, D, a.eps);
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = __fmul_rn(__fmul_rn(v[i], f), g[i]);
        }
        if (gain || rope)
#pragma unroll
            for (int i = 0; i < 4; ++i) {                         // the pairs of rope_pair(), rounded two at a time
                float y0 = v[2 * i], y1 = v[2 * i + 1];
                if (rope) {
                    y0 = __fsub_rn(__fmul_rn(v[2 * i], cs[i]), __fmul_rn(v[2 * i + 1], sn[i]));
                    y1 = __fadd_rn(__fmul_rn(v[2 * i], sn[i]), __fmul_rn(v[2 * i + 1], cs[i]));
                }
                const __nv_bfloat162 y = __floats2bfloat162_rn(y0, y1);
                w[i] = *reinterpret_cast<const uint32_t*>(&y);
            }
        if (kind != 0) {
#pragma unroll
            for (int i = 0; i < 4; ++i) { v[2 * i] = bf16_lo(w[i]); v[2 * i + 1] = bf16_hi(w[i]); }
            quantize_values8_warp<EPL, U>(v, kind == 1 ? a.k : a.v, (int64_t)r.b * a.Hkv + h, r.key, a.Lcap, r.live, lane);
            continue;
        }
        if (!in_range) continue;
        if (!r.live) w[0] = w[1] = w[2] = w[3] = 0u;              // padding: zeros
        __nv_bfloat16* dst = a.q_out + (r.token * a.Hq + h) * D + l * 8;
        if (a.wide) *reinterpret_cast<uint4*>(dst) = make_uint4(w[0], w[1], w[2], w[3]);
        else
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                dst[2 * i] = __ushort_as_bfloat16((unsigned short)(w[i] & 0xFFFFu));
                dst[2 * i + 1] = __ushort_as_bfloat16((unsigned short)(w[i] >> 16));
            }
    }
}

// Every other group size: one warp per row, the lane-per-element quantiser.
template <int EPL>
__global__ void __launch_bounds__(QKV_WARPS * 32)
qkv_write_kernel(const QkvArgs a, Fmt f) {
    chain_release();
    chain_wait();
    constexpr int D = 32 * EPL, NB = EPL;
    __shared__ float rowbuf[QKV_WARPS][D];
    __shared__ uint32_t codes[QKV_WARPS][NB * QROW_CW];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    int64_t blk = blockIdx.x;
    const int kind = blk < a.q_blocks ? 0 : blk < a.q_blocks + a.k_blocks ? 1 : 2;
    blk -= kind == 0 ? 0 : kind == 1 ? a.q_blocks : a.q_blocks + a.k_blocks;
    const int heads = kind == 0 ? a.Hq : a.Hkv, head0 = kind == 0 ? 0 : kind == 1 ? a.Hq : a.Hq + a.Hkv;
    const int64_t row = blk * QKV_WARPS + warp;
    if (row >= (int64_t)a.B * a.T * heads) return;             // whole warps
    const int64_t token = row / heads;
    const int head = (int)(row - token * heads);
    const QkvToken r = qkv_token(a, token, kind != 0, lane == 0);
    if (!r.live) {
        if (kind == 0)
            for (int i = lane; i < D; i += 32) a.q_out[row * D + i] = __float2bfloat16_rn(0.0f);
        return;
    }
    float v[EPL];
    const __nv_bfloat16* src = a.x + r.token * a.ld + (int64_t)(head0 + head) * D + lane * EPL;
#pragma unroll
    for (int i = 0; i < EPL; ++i) v[i] = __bfloat162float(src[i]);
    if (kind != 2) {
        const void* gain = kind == 0 ? a.q_gain : a.k_gain;
        if (gain) {
            double ss = 0.0;
#pragma unroll
            for (int i = 0; i < EPL; ++i) ss = fma((double)v[i], (double)v[i], ss);
#pragma unroll
            for (int m = 1; m < 32; m <<= 1) ss += __shfl_xor_sync(0xffffffffu, ss, m);
            const float s = norm_factor(ss, D, a.eps);
#pragma unroll
            for (int i = 0; i < EPL; ++i) v[i] = __fmul_rn(__fmul_rn(v[i], s), gain_at(gain, a.gain_f32, lane * EPL + i));
        }
        if (a.rope.cos) rope_warp<EPL>(v, lane, a.rope, r.at);
        else if (gain)
#pragma unroll
            for (int i = 0; i < EPL; ++i) v[i] = __bfloat162float(__float2bfloat16_rn(v[i]));
    }
    if (kind == 0) {
#pragma unroll
        for (int i = 0; i < EPL; ++i) a.q_out[row * D + lane * EPL + i] = __float2bfloat16_rn(v[i]);
        return;
    }
    quantize_values_warp<EPL>(v, kind == 1 ? a.k : a.v, (int64_t)r.b * a.Hkv + head, r.key, a.Lcap, f, rowbuf[warp], codes[warp], lane);
}

template <int EPL>
int launch_qkv(QkvArgs& a, const Fmt& f, bool rows8, cudaStream_t st) {
    const int64_t tokens = (int64_t)a.B * a.T;
    int64_t blocks;
    if (rows8) {
        // Long runs of heads save instructions, many blocks keep the SMs busy: the longest run (of 8, 4, 2 query heads, half as many
        // key heads, or 1) that leaves six of seven resident blocks per SM.  Runs of 1 / 2 / 4 / 8 took, 32 + 2 x 8 heads: 128 tokens
        // 3.7 / 3.4 / 4.2 / 5.4 us, 512 tokens 8.3 / 6.9 / 6.0 / 6.9, 1024 tokens 14.2 / 11.9 / 10.1 / 9.7, 8191 tokens 105 / 86 / 67 /
        // 58 (16: 57, but 17.1 against 16.5 at 2048).
        const int64_t of_tokens = (tokens + QKV_WARPS * (8 / EPL) - 1) / (QKV_WARPS * (8 / EPL));
        for (a.q_heads = 8;; a.q_heads /= 2) {
            a.kv_heads = std::max(a.q_heads / 2, 1);
            a.kv_chunks = (a.Hkv + a.kv_heads - 1) / a.kv_heads;
            a.chunks = 2 * a.kv_chunks + (a.Hq + a.q_heads - 1) / a.q_heads;
            blocks = of_tokens * a.chunks;
            if (a.q_heads == 1 || blocks >= 6LL * sm_count()) break;
        }
    } else {
        a.q_blocks = (tokens * a.Hq + QKV_WARPS - 1) / QKV_WARPS;
        a.k_blocks = (tokens * a.Hkv + QKV_WARPS - 1) / QKV_WARPS;
        blocks = a.q_blocks + 2 * a.k_blocks;
    }
    if (blocks > INT32_MAX) return fail(MSAQ_ERR_ARG, "size exceeds the supported range");
    const dim3 grid((unsigned)blocks), block(QKV_WARPS * 32);
    if (!rows8) launch_chained(qkv_write_kernel<EPL>, grid, block, 0, st, a, f);
    else if (f.u == 4) launch_chained(qkv_write8_kernel<EPL, 4>, grid, block, 0, st, a);
    else if (f.u == 3) launch_chained(qkv_write8_kernel<EPL, 3>, grid, block, 0, st, a);
    else launch_chained(qkv_write8_kernel<EPL, 2>, grid, block, 0, st, a);
    count_launch();
    return check_launch("kv_write_qkv");
}

// ---- the accepted nodes' rows move together -------------------------------------------------------------
struct KeepArgs {
    int8_t* s[2];
    uint8_t* up[2];
    uint8_t* sh[2];
    const int32_t* path;                 // [B][T]
    const int32_t* count;                // [B]
    const int32_t* start_per_seq;
    int64_t start, Lcap;
    int* sticky;
    int T, Hkv, NB, UB, SB;
    int64_t planes;                      // B * Hkv * NB
};

// One warp per (sequence, head, block) of one cache reads every row that moves into registers before it writes one, so a row
// may go where another one comes from.  Two rows per lane cover the 64 nodes of the largest tree.  Latency: two round trips (path, rows)
// and the call; 6.5 us, 2.2 of them on the device for one small tree, 4.6 for 64 of 61 nodes.
__global__ void __launch_bounds__(128)
keep_kernel(const KeepArgs a) {
    chain_release();
    chain_wait();
    const int lane = threadIdx.x & 31, c = blockIdx.y;
    const int64_t plane = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
    if (plane >= a.planes) return;
    const int b = (int)(plane / (a.Hkv * a.NB));
    const int64_t start = a.start_per_seq ? (int64_t)a.start_per_seq[b] : a.start;
    const int n = min(max(a.count[b], 0), a.T);
    uint32_t up[2][6];
    uint64_t sh[2];
    int8_t e[2];
    bool move[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int k = lane + 32 * i;
        const int node = k < n ? a.path[(int64_t)b * a.T + k] : k;
        const bool ok = node >= 0 && node < a.T && start >= 0 && start + max(node, k) < a.Lcap;
        if (k < n && !ok && a.sticky) atomicOr(a.sticky, BAD_APPEND_POS);
        move[i] = k < n && ok && node != k;
        if (!move[i]) continue;
        const int64_t from = plane * a.Lcap + start + node;
        const uint32_t* u = reinterpret_cast<const uint32_t*>(a.up[c] + from * a.UB);
#pragma unroll
        for (int w = 0; w < 6; ++w) up[i][w] = w * 4 < a.UB ? u[w] : 0u;
        const uint8_t* h = a.sh[c] + from * a.SB;
        sh[i] = 0;
#pragma unroll
        for (int w = 0; w < 8; ++w) sh[i] |= w < a.SB ? (uint64_t)h[w] << (8 * w) : 0ull;
        e[i] = a.s[c][from];
    }
    __syncwarp();
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        if (!move[i]) continue;
        const int64_t to = plane * a.Lcap + start + lane + 32 * i;
        uint32_t* u = reinterpret_cast<uint32_t*>(a.up[c] + to * a.UB);
#pragma unroll
        for (int w = 0; w < 6; ++w)
            if (w * 4 < a.UB) u[w] = up[i][w];
        uint8_t* h = a.sh[c] + to * a.SB;
#pragma unroll
        for (int w = 0; w < 8; ++w)
            if (w < a.SB) h[w] = (uint8_t)(sh[i] >> (8 * w));
        a.s[c][to] = e[i];
    }
}

}  // namespace
}  // namespace msaq

using namespace msaq;

extern "C" int msaq_kv_write_qkv(const void* qkv, int64_t ld, void* q_out, int8_t* k_scale_exp, uint8_t* k_upper, uint8_t* k_shared,
                                 int8_t* v_scale_exp, uint8_t* v_upper, uint8_t* v_shared, int64_t B, int64_t T, int64_t H,
                                 int64_t Hkv, int64_t D, int64_t NB, int64_t start, const int32_t* start_per_seq, const int32_t* pos,
                                 const int32_t* counts, const void* q_gain, const void* k_gain, int gain_is_f32, double eps,
                                 const float* rope_cos, const float* rope_sin, int64_t rope_rows, int64_t Lcap, int u, int gs,
                                 int rotate_k, void* stream) {
    const DeviceScope device;
    Fmt f;
    if (!qkv || !q_out || !k_scale_exp || !k_upper || !k_shared || !v_scale_exp || !v_upper || !v_shared)
        return fail(MSAQ_ERR_ARG, "null pointer");
    if (!make_fmt(u, gs, &f)) return fail(MSAQ_ERR_UNSUPPORTED, "unsupported format u=%d gs=%d", u, gs);
    if (B <= 0 || T <= 0 || H <= 0 || Hkv <= 0 || Lcap <= 0) return fail(MSAQ_ERR_ARG, "B, T, H, Hkv and Lcap must be positive");
    if (B > INT32_MAX || T > INT32_MAX || H > 65535 || Hkv > 65535 || B * T > INT32_MAX)
        return fail(MSAQ_ERR_ARG, "size exceeds the supported range");
    if (D != 32 && D != 64 && D != 128 && D != 256)
        return fail(MSAQ_ERR_UNSUPPORTED, "head_dim %lld: must be 32, 64, 128 or 256", (long long)D);
    if (NB * BLOCK != D) return fail(MSAQ_ERR_ARG, "NB (%lld) must equal D/32 (D=%lld)", (long long)NB, (long long)D);
    if (ld < (H + 2 * Hkv) * D) return fail(MSAQ_ERR_ARG, "ld (%lld) is smaller than a token's heads", (long long)ld);
    if (!(eps >= 0.0)) return fail(MSAQ_ERR_ARG, "eps must not be negative");
    if (!start_per_seq && (start < 0 || start + T > Lcap))
        return fail(MSAQ_ERR_ARG, "slots [%lld, %lld) exceed the cache capacity %lld", (long long)start, (long long)(start + T), (long long)Lcap);
    if ((rope_cos == nullptr) != (rope_sin == nullptr)) return fail(MSAQ_ERR_ARG, "rope_cos and rope_sin come together");
    if (rope_cos) {
        // a row per position: every slot that a token can go to needs its table row (given positions are checked on the device)
        const int64_t need = pos ? 1 : start_per_seq ? Lcap : start + T;
        if (rope_rows < 1 || (rope_rows == 1 && T > 1) || (rope_rows > 1 && rope_rows < need))
            return fail(MSAQ_ERR_ARG, "the RoPE tables have %lld rows, %lld tokens with positions up to %lld are possible",
                        (long long)rope_rows, (long long)T, (long long)need - 1);
    }
    if ((reinterpret_cast<uintptr_t>(k_upper) | reinterpret_cast<uintptr_t>(v_upper)) & 3)
        return fail(MSAQ_ERR_ARG, "upper planes must be 4-byte aligned");
    if ((reinterpret_cast<uintptr_t>(q_gain) | reinterpret_cast<uintptr_t>(k_gain)) & (gain_is_f32 ? 3 : 1))
        return fail(MSAQ_ERR_ARG, "gains must be aligned to their type");
    if (int rc = require_sm100()) return rc;
    QkvArgs a{};
    a.x = static_cast<const __nv_bfloat16*>(qkv);
    a.q_out = static_cast<__nv_bfloat16*>(q_out);
    a.k = QuantJob{nullptr, k_scale_exp, k_upper, k_shared, rotate_k ? 1 : 0, 0, 0};
    a.v = QuantJob{nullptr, v_scale_exp, v_upper, v_shared, 0, 0, 0};
    a.ld = ld; a.start = start; a.Lcap = Lcap;
    a.start_per_seq = start_per_seq; a.pos = pos; a.counts = counts;
    a.q_gain = q_gain; a.k_gain = k_gain; a.gain_f32 = gain_is_f32 ? 1 : 0;
    a.rope = Rope{rope_cos, rope_sin, rope_rows};
    a.eps = eps;
    a.sticky = sticky_status();
    a.B = (int)B; a.T = (int)T; a.Hq = (int)H; a.Hkv = (int)Hkv;
    a.wide = !((reinterpret_cast<uintptr_t>(qkv) | reinterpret_cast<uintptr_t>(q_out)) & 15) && ld % 8 == 0;
    a.rope_wide = !((reinterpret_cast<uintptr_t>(rope_cos) | reinterpret_cast<uintptr_t>(rope_sin)) & 15);
    const bool rows8 = gs == 2 && !((reinterpret_cast<uintptr_t>(k_shared) | reinterpret_cast<uintptr_t>(v_shared)) & 1);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    switch (D) {
        case 32: return launch_qkv<1>(a, f, rows8, st);
        case 64: return launch_qkv<2>(a, f, rows8, st);
        case 128: return launch_qkv<4>(a, f, rows8, st);
        default: return launch_qkv<8>(a, f, rows8, st);
    }
}

extern "C" int msaq_kv_keep(int8_t* k_scale_exp, uint8_t* k_upper, uint8_t* k_shared, int8_t* v_scale_exp, uint8_t* v_upper,
                            uint8_t* v_shared, const int32_t* path, const int32_t* count, int64_t start,
                            const int32_t* start_per_seq, int64_t B, int64_t T, int64_t Hkv, int64_t NB, int64_t Lcap, int u,
                            int gs, void* stream) {
    const DeviceScope device;
    Fmt f;
    if (!k_scale_exp || !k_upper || !k_shared || !v_scale_exp || !v_upper || !v_shared || !path || !count)
        return fail(MSAQ_ERR_ARG, "null pointer");
    if (!make_fmt(u, gs, &f)) return fail(MSAQ_ERR_UNSUPPORTED, "unsupported format u=%d gs=%d", u, gs);
    if (B <= 0 || Hkv <= 0 || NB <= 0 || Lcap <= 0) return fail(MSAQ_ERR_ARG, "B, Hkv, NB and Lcap must be positive");
    if (T <= 0 || T > KEEP_MAX_T) return fail(MSAQ_ERR_ARG, "a tree has 1 to %d nodes", KEEP_MAX_T);
    if (Hkv > 65535 || NB > 65535 || B > INT32_MAX / (Hkv * NB)) return fail(MSAQ_ERR_ARG, "size exceeds the supported range");
    if (!start_per_seq && (start < 0 || start + T > Lcap))
        return fail(MSAQ_ERR_ARG, "slots [%lld, %lld) exceed the cache capacity %lld", (long long)start, (long long)(start + T), (long long)Lcap);
    if ((reinterpret_cast<uintptr_t>(k_upper) | reinterpret_cast<uintptr_t>(v_upper)) & 3)
        return fail(MSAQ_ERR_ARG, "upper planes must be 4-byte aligned");
    if (int rc = require_sm100()) return rc;
    const KeepArgs a{{k_scale_exp, v_scale_exp}, {k_upper, v_upper}, {k_shared, v_shared}, path, count, start_per_seq, start, Lcap,
                     sticky_status(), (int)T, (int)Hkv, (int)NB, f.UB, f.SB, B * Hkv * NB};
    launch_chained(keep_kernel, dim3((unsigned)((a.planes + 3) / 4), 2), dim3(128), 0, static_cast<cudaStream_t>(stream), a);
    count_launch();
    return check_launch("kv_keep");
}
