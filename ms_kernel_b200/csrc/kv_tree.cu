// Host side of the attention for a tree of drafted tokens over a packed cache: argument checks, the split of the keys, kernel
// selection.
#include "kv_tree_generic.cuh"

namespace msaq {
namespace {

struct TreePlan {
    int S, key_tile, groups;
};

// Row groups x kv heads x sequences thread blocks of one key piece each; pieces until about three blocks per SM are there.
TreePlan plan_tree_generic(int64_t B, int64_t T, int64_t H, int64_t Hkv, int64_t Lk) {
    TreePlan p;
    const int64_t R = T * (H / Hkv);
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

bool tree_sizes_ok(int64_t B, int64_t T, int64_t H, int64_t Hkv, int64_t Lk, int64_t D) {
    return B > 0 && B <= 65535 && T > 0 && T <= KT_MAX_T && H > 0 && Hkv > 0 && H % Hkv == 0 && H <= 65535 && Lk >= T && Lk <= INT32_MAX &&
           (D == 32 || D == 64 || D == 128 || D == 256) && Hkv * ((T * (H / Hkv) + KTG_ROWS - 1) / KTG_ROWS) <= 65535;
}

}  // namespace
}  // namespace msaq

using namespace msaq;

extern "C" size_t msaq_kv_tree_workspace(int64_t B, int64_t T, int64_t H, int64_t Hkv, int64_t Lk, int64_t D) {
    const DeviceScope device;
    if (!tree_sizes_ok(B, T, H, Hkv, Lk, D)) return 0;
    const TreePlan p = plan_tree_generic(B, T, H, Hkv, Lk);
    const size_t bytes = (size_t)B * T * H * p.S * (D + 2) * sizeof(float);
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
    if (int rc = require_sm100()) return rc;
    const size_t need = msaq_kv_tree_workspace(B, T, H, Hkv, Lk, D);
    if (!workspace || workspace_bytes < need)
        return fail(MSAQ_ERR_WORKSPACE, "workspace of %zu bytes needed, %zu given", need, workspace ? workspace_bytes : (size_t)0);

    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const TreePlan p = plan_tree_generic(B, T, H, Hkv, Lk);
    float* partial = reinterpret_cast<float*>(static_cast<uint8_t*>(workspace) + WS_CTL_BYTES);
    const KvTreeArgs a{static_cast<const __nv_bfloat16*>(q), KvPlanes{ks, ku, kh}, KvPlanes{vs, vu, vh}, partial, lens, mask, mask_stride,
                       (int)T, (int)H, (int)Hkv, (int)Lk, (int)Lcap, (int)D, (int)NB, p.key_tile, p.S, qrot,
                       (float)(1.4426950408889634 / sqrt((double)D)), sticky_status(), option_wait_polls(), option_test_skip_stage(), f};
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
