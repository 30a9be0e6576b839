// Host side of the attention for a tree of drafted tokens over a packed cache: argument checks, the split of the keys, kernel
// selection.
#include <algorithm>

#include "kv_tree_generic.cuh"
#include "kv_tree_umma.cuh"

namespace msaq {
namespace {

struct TreePlan {
    int S, key_tile, groups, rows;
};

// Rows per thread block by the rows there are: blocks of 16 / 32 / 64 took, us, over 4 sequences of 32752 keys and 8 kv heads: 16 rows 85 /
// 93 / 118, 32 rows 157 / 93 / 120, 64 rows 300 / 170 / 123; 16 sequences of 2000: 35 / 41 / 59, 57 / 43 / 64, 100 / 71 / 66; one of
// 16000: 16 rows 27 / 30 / 41, 32 rows 35 / 31 / 42.  Fewer where every block still has one tile at most: the keys are decoded more often, by
// SMs that had nothing to do (one sequence, 8 kv heads: 32 rows over 509 keys 14.1 -> 12.5, 64 rows over 100 keys 19.6 -> 11.1, over
// 509 20.5 -> 14.2; up to two tiles: 488 rows over 16 keys 14.8 -> 17.7, no) -- not under the hook that stops the first block's
// products, which then stops all rows of a small item.  As many runs of the line of tiles as there are SMs, or as there can be tiles.
TreePlan plan_tree_umma(int64_t B, int64_t T, int64_t H, int64_t Hkv, int64_t Lk) {
    TreePlan p;
    const int64_t R = T * (H / Hkv);
    p.rows = R <= 16 ? 16 : R <= 32 ? 32 : 64;
    const int64_t tiles = B * Hkv * ((Lk + KTU_KEYS - 1) / KTU_KEYS);
    while (p.rows > 16 && option_test_skip_stage() < 0 && tiles * ((2 * R + p.rows - 1) / p.rows) <= sm_count()) p.rows /= 2;
    p.groups = (int)((R + p.rows - 1) / p.rows);
    p.S = (int)std::min<int64_t>(sm_count(), tiles * p.groups);
    p.key_tile = KTU_KEYS;
    return p;
}

// The tuned kernel: head_dim 128, gs = 2, capacity a multiple of 16 (and planes on 16-byte boundaries: bulk copies), tiles counted in 31 bits.
// (The generic kernel takes 121 instead of 12.5 us at 8 nodes over 509 keys, 16.2 ms instead of 0.41 for 16 sequences of 16 nodes over up to
// 32752 keys.)
bool umma_eligible(int64_t D, int gs, int64_t Lcap, int64_t B, int64_t T, int64_t H, int64_t Hkv, int64_t Lk) {
    return D == 128 && gs == 2 && Lcap % 16 == 0 && B * Hkv * plan_tree_umma(B, T, H, Hkv, Lk).groups <= INT32_MAX / ((Lk + KTU_KEYS - 1) / KTU_KEYS);
}

template <int U, int NR>
int launch_tree_umma_rows(const KvTreeArgs& a, const TreePlan& p, int B, __nv_bfloat16* out, float* out_f32, cudaStream_t st) {
    static bool configured[64] = {};
    constexpr int smem = ktu_smem_bytes(U, NR);
    const int dev = current_device();
    if (dev >= 0 && dev < 64 && !configured[dev]) {
        if (cudaFuncSetAttribute(kv_tree_umma_kernel<U, NR>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) != cudaSuccess)
            return fail(MSAQ_ERR_CUDA, "cannot reserve %d bytes of shared memory", smem);
        configured[dev] = true;
    }
    launch_chained(kv_tree_umma_kernel<U, NR>, dim3((unsigned)p.S), dim3(KTU_THREADS), smem, st, a, B, p.groups, out, out_f32);
    count_launch();
    if (int rc = check_launch("kv_tree_umma")) return rc;
    launch_chained(kv_tree_merge_kernel<NR>, dim3((unsigned)(a.Hkv * p.groups * (NR / 8)), (unsigned)B), dim3(256), 0, st, a, B, p.groups, p.S, out,
                   out_f32);
    count_launch();
    return check_launch("kv_tree_merge");
}

template <int U>
int launch_tree_umma(const KvTreeArgs& a, const TreePlan& p, int B, __nv_bfloat16* out, float* out_f32, cudaStream_t st) {
    return p.rows == 16 ? launch_tree_umma_rows<U, 16>(a, p, B, out, out_f32, st)
         : p.rows == 32 ? launch_tree_umma_rows<U, 32>(a, p, B, out, out_f32, st) : launch_tree_umma_rows<U, 64>(a, p, B, out, out_f32, st);
}

// Row groups x kv heads x sequences thread blocks of one key piece each; pieces until about three blocks per SM are there.
TreePlan plan_tree_generic(int64_t B, int64_t T, int64_t H, int64_t Hkv, int64_t Lk) {
    TreePlan p;
    const int64_t R = T * (H / Hkv);
    p.rows = KTG_ROWS;
    p.groups = (int)((R + KTG_ROWS - 1) / KTG_ROWS);
    const int64_t blocks = B * Hkv * p.groups;
    int64_t want = (3LL * sm_count() + blocks - 1) / blocks;
    const int64_t most = (Lk + 127) / 128;
    if (want > most) want = most;
    if (want < 1) want = 1;
    const int64_t tile = ((Lk + want - 1) / want + KTG_KEYS - 1) / KTG_KEYS * KTG_KEYS;
    p.key_tile = (int)tile;
    p.S = (int)((Lk + tile - 1) / tile);
    return p;
}

template <int EPL>
int launch_tree_generic(const KvTreeArgs& a, const TreePlan& p, int B, cudaStream_t st) {
    static bool configured[64] = {};
    const int smem = (int)ktg_smem_bytes(32 * EPL), dev = current_device();
    if (dev >= 0 && dev < 64 && !configured[dev]) {
        if (cudaFuncSetAttribute(kv_tree_generic_kernel<EPL>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) != cudaSuccess)
            return fail(MSAQ_ERR_CUDA, "cannot reserve %d bytes of shared memory", smem);
        configured[dev] = true;
    }
    launch_chained(kv_tree_generic_kernel<EPL>, dim3((unsigned)p.S, (unsigned)(a.Hkv * p.groups), (unsigned)B), dim3(KTG_THREADS), smem, st, a);
    count_launch();
    return check_launch("kv_tree_generic");
}

// (Lk: key indexes, and the ends of tiles behind the last key, stay within 31 bits.)
bool tree_sizes_ok(int64_t B, int64_t T, int64_t H, int64_t Hkv, int64_t Lk, int64_t D) {
    return B > 0 && B <= 65535 && T > 0 && T <= KT_MAX_T && H > 0 && Hkv > 0 && H % Hkv == 0 && H <= 65535 && Lk >= T && Lk <= (1 << 30) &&
           (D == 32 || D == 64 || D == 128 || D == 256) && Hkv * ((T * (H / Hkv) + KTG_ROWS - 1) / KTG_ROWS) <= 65535;
}

}  // namespace
}  // namespace msaq

using namespace msaq;

extern "C" size_t msaq_kv_tree_workspace(int64_t B, int64_t T, int64_t H, int64_t Hkv, int64_t Lk, int64_t D) {
    const DeviceScope device;
    if (!tree_sizes_ok(B, T, H, Hkv, Lk, D)) return 0;
    size_t bytes = (size_t)B * T * H * plan_tree_generic(B, T, H, Hkv, Lk).S * (D + 2) * sizeof(float);
    if (D == 128) {                                               // the same size for every format
        const TreePlan p = plan_tree_umma(B, T, H, Hkv, Lk);
        bytes = std::max(bytes, (size_t)2 * p.S * p.rows * KTU_PART * sizeof(float));
    }
    return ((bytes + 255) & ~(size_t)255) + WS_CTL_BYTES;
}

extern "C" int msaq_kv_tree_attention(const void* q, const int8_t* ks, const uint8_t* ku, const uint8_t* kh, const int8_t* vs,
                                      const uint8_t* vu, const uint8_t* vh, void* out, float* out_f32, const int32_t* lens,
                                      const uint64_t* mask, int64_t mask_stride, int64_t B, int64_t T, int64_t H, int64_t Hkv,
                                      int64_t Lk, int64_t D, int64_t NB, int u, int gs, int64_t Lcap, int qrot, void* workspace,
                                      size_t workspace_bytes, void* stream) {
    const DeviceScope device;
    Fmt f;
    if (!q || !ks || !ku || !kh || !vs || !vu || !vh || !out || !mask) return fail(MSAQ_ERR_ARG, "null pointer");
    if (!make_fmt(u, gs, &f)) return fail(MSAQ_ERR_UNSUPPORTED, "unsupported format u=%d gs=%d", u, gs);
    if (B <= 0 || H <= 0 || Hkv <= 0) return fail(MSAQ_ERR_ARG, "B, H and Hkv must be positive");
    if (T <= 0 || T > KT_MAX_T) return fail(MSAQ_ERR_ARG, "a tree has 1 to %d nodes", KT_MAX_T);
    if (H % Hkv) return fail(MSAQ_ERR_ARG, "H (%lld) must be a multiple of Hkv (%lld)", (long long)H, (long long)Hkv);
    if (D != 32 && D != 64 && D != 128 && D != 256)
        return fail(MSAQ_ERR_UNSUPPORTED, "head_dim %lld: must be 32, 64, 128 or 256", (long long)D);
    if (NB * BLOCK != D) return fail(MSAQ_ERR_ARG, "NB (%lld) must equal D/32 (D=%lld)", (long long)NB, (long long)D);
    if (Lk < T) return fail(MSAQ_ERR_ARG, "Lk (%lld) does not hold the tree's %lld nodes", (long long)Lk, (long long)T);
    if (Lcap < Lk) return fail(MSAQ_ERR_ARG, "Lcap (%lld) is smaller than Lk (%lld)", (long long)Lcap, (long long)Lk);
    if (Lcap > INT32_MAX || !tree_sizes_ok(B, T, H, Hkv, Lk, D)) return fail(MSAQ_ERR_ARG, "size exceeds the supported range");
    if (mask_stride != 0 && mask_stride < T) return fail(MSAQ_ERR_ARG, "mask_stride must be 0 or at least T");
    if (reinterpret_cast<uintptr_t>(mask) & 7) return fail(MSAQ_ERR_ARG, "mask must be 8-byte aligned");
    if ((reinterpret_cast<uintptr_t>(ku) | reinterpret_cast<uintptr_t>(vu)) & 3)
        return fail(MSAQ_ERR_ARG, "upper planes must be 4-byte aligned");
    if (reinterpret_cast<uintptr_t>(workspace) & 15) return fail(MSAQ_ERR_ARG, "workspace must be 16-byte aligned");
    if (int rc = require_sm100()) return rc;
    const size_t need = msaq_kv_tree_workspace(B, T, H, Hkv, Lk, D);
    if (!workspace || workspace_bytes < need)
        return fail(MSAQ_ERR_WORKSPACE, "workspace of %zu bytes needed, %zu given", need, workspace ? workspace_bytes : (size_t)0);

    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const bool tuned = umma_eligible(D, gs, Lcap, B, T, H, Hkv, Lk) &&
                       !((reinterpret_cast<uintptr_t>(ks) | reinterpret_cast<uintptr_t>(vs) | reinterpret_cast<uintptr_t>(ku) | reinterpret_cast<uintptr_t>(kh) | reinterpret_cast<uintptr_t>(vu) |
                          reinterpret_cast<uintptr_t>(vh)) & 15) &&
                       !(reinterpret_cast<uintptr_t>(q) & 7);
    const TreePlan p = tuned ? plan_tree_umma(B, T, H, Hkv, Lk) : plan_tree_generic(B, T, H, Hkv, Lk);
    float* partial = reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) + WS_CTL_BYTES);
    const KvTreeArgs a{static_cast<const __nv_bfloat16*>(q), KvPlanes{ks, ku, kh}, KvPlanes{vs, vu, vh}, partial, lens, mask, mask_stride,
                       (int)T, (int)H, (int)Hkv, (int)Lk, (int)Lcap, (int)D, (int)NB, p.key_tile, p.S, qrot,
                       (float)(1.4426950408889634 / sqrt((double)D)), sticky_status(), option_wait_polls(), option_test_skip_stage(), f};
    if (tuned) {
        __nv_bfloat16* o = static_cast<__nv_bfloat16*>(out);
        return u == 4 ? launch_tree_umma<4>(a, p, (int)B, o, out_f32, st)
             : u == 3 ? launch_tree_umma<3>(a, p, (int)B, o, out_f32, st) : launch_tree_umma<2>(a, p, (int)B, o, out_f32, st);
    }
    int rc;
    switch (D) {
        case 32: rc = launch_tree_generic<1>(a, p, (int)B, st); break;
        case 64: rc = launch_tree_generic<2>(a, p, (int)B, st); break;
        case 128: rc = launch_tree_generic<4>(a, p, (int)B, st); break;
        default: rc = launch_tree_generic<8>(a, p, (int)B, st); break;
    }
    if (rc) return rc;
    launch_chained(kv_tree_combine_kernel, dim3((unsigned)(T * (H / Hkv)), (unsigned)Hkv, (unsigned)B), dim3(128), 0, st,
                   static_cast<const float*>(partial), static_cast<__nv_bfloat16*>(out), out_f32, (int)T, (int)H, (int)Hkv, (int)D, p.S);
    count_launch();
    return check_launch("kv_tree_combine");
}
