// attention_cached.hip — one query token a scene against a cache of keys and values.
//
// The kernel is gsv_cached.h's.
//
// Two caches of 200,003 rows, 4 heads of 128, bfloat16 (316 MB of live rows): 65 us, 4.9 TB/s, and 5 us
// for the join.  16 caches of 4,096, 2 heads of 64 (23 MB): 10.8 us and 3.9; there the time from
// launch to the first bytes and a wave's few steps one after the other bound it.
#include "gsv_cached.h"

// (a product and a difference stay two roundings where they are written as two)
#pragma clang fp contract(off)

namespace gsv {
namespace {

// One workgroup a scene and head.  Latency bounds it: 4 us at 16 splits a head, 5 at 32.
template <typename T>
__global__ __launch_bounds__(256) void k_cached_join(const float *__restrict__ part_o,
                                                     const float2 *__restrict__ part_ms, int splits,
                                                     int dim, T *__restrict__ out) {
    const int64_t row = blockIdx.x;
    join_row<T, 4>(part_o, part_ms, row * splits, 1, splits, dim, out + row * dim);
}

// Splits of a cache: one round of workgroups, as many as the CUs hold at once (their tiles fill the
// LDS), each with at least a step for all its waves.  Two caches of 200,003 rows, 4 heads of 128 (one
// workgroup a CU): 70 us in one round, 75 in two, 90 in four; 16 of 4,096 rows, 2 heads of 64
// (two a CU): 15 us in one round, 16 in half of one, 20 in two.
int cache_splits(const AttnArgs &a, int head_tiles, int dtype) {
    const int64_t size = dtype == GSV_BF16 ? 2 : 4, dp = a.dim <= 32 ? 32 : a.dim <= 64 ? 64 : 128;
    const int64_t waves = dp * size > 256 ? 2 : 4;
    const int64_t lds = waves * (4 * kKeys * dp * size + (a.slopes ? 6 * kKeys * (size == 2 ? 16 : 4) : 0)) + 2048;
    const int64_t round = 256 * imin64(163840 / lds, 4);
    const int64_t each = (int64_t)a.scenes * a.kv_heads * head_tiles;
    const int64_t most = (a.k_tokens + waves * kKeys - 1) / (waves * kKeys);
    return (int)imax64(1, imin64(round / each, most));
}

struct Cached {
    const AttnArgs &a;
    const CacheArgs &c;
    void *out;
    hipStream_t st;
    template <typename T, int DP, bool FAR, int CAP> void run() const {
        T *o = static_cast<T *>(out);
        hipLaunchKernelGGL((k_attention_cached<T, DP, FAR, CAP, kTogether>),
                           dim3((unsigned)(a.scenes * a.kv_heads * c.head_tiles * c.splits)),
                           dim3(64 * kWaves<T, DP, kTogether>), 0, st, a, c, o);
        if (c.splits > 1)
            hipLaunchKernelGGL(k_cached_join<T>, dim3((unsigned)(a.scenes * a.heads)), dim3(256), 0,
                               st, c.part_o, c.part_ms, c.splits, a.dim, o);
    }
};

int cached_plan(const gsv_attention *args, AttnArgs *a, int *head_tiles, int *splits) {
    if (!args || args->causal || args->prefix || args->q_starts || args->k_starts ||
        args->scenes < 0 || args->scenes != args->q_tokens)
        return GSV_ERR_INVALID_ARGUMENT;
    gsv_attention one = *args;
    one.scenes = 1;  // rows are addressed by scene here, not packed
    const int st = attention_args(&one, a);
    if (st != GSV_OK) return st;
    a->scenes = args->scenes;
    const int64_t tiles = (a->heads / a->kv_heads + kHeads - 1) / kHeads;
    if ((int64_t)a->scenes * a->kv_heads * tiles > (1 << 22) || (int64_t)a->scenes * a->heads > (1 << 24))
        return GSV_ERR_SIZE_OVERFLOW;
    *head_tiles = (int)tiles;
    *splits = a->scenes ? cache_splits(*a, (int)tiles, args->dtype) : 1;
    return GSV_OK;
}

size_t part_o_bytes(const AttnArgs &a, int splits) {
    return sizeof(float) * a.scenes * a.heads * splits * a.dim;  // a multiple of 32 bytes
}

}  // namespace
}  // namespace gsv

using namespace gsv;

extern "C" int gsv_attention_cached_workspace_bytes(const gsv_attention *args, size_t *bytes) {
    AttnArgs a;
    int tiles, splits;
    if (!bytes) return GSV_ERR_INVALID_ARGUMENT;
    const int st = cached_plan(args, &a, &tiles, &splits);
    if (st != GSV_OK) return st;
    *bytes = splits > 1 ? part_o_bytes(a, splits) + sizeof(float2) * a.scenes * a.heads * splits : 0;
    return GSV_OK;
}

extern "C" int gsv_attention_cached(const gsv_attention *args, const int32_t *lengths,
                                    int64_t k_scene, int64_t v_scene, int64_t k_pos_scene,
                                    int64_t keep_scene, void *out, void *workspace,
                                    size_t workspace_bytes, void *stream) {
    AttnArgs a;
    int tiles, splits;
    size_t need;
    int st = cached_plan(args, &a, &tiles, &splits);
    if (st != GSV_OK) return st;
    if (a.scenes == 0) return GSV_OK;
    if ((st = gsv_attention_cached_workspace_bytes(args, &need)) != GSV_OK) return st;
    if (need > workspace_bytes) return GSV_ERR_WORKSPACE_TOO_SMALL;
    const int64_t chunk = args->dtype == GSV_BF16 ? 8 : 4;
    k_scene = used_stride(k_scene, a.scenes);
    v_scene = used_stride(v_scene, a.scenes);
    if (!lengths || !out || (need && !workspace) || k_scene % chunk || v_scene % chunk ||
        reinterpret_cast<uintptr_t>(out) % 16 || reinterpret_cast<uintptr_t>(workspace) % 16)
        return GSV_ERR_INVALID_ARGUMENT;
    float *po = static_cast<float *>(workspace);
    CacheArgs c{lengths, k_scene, v_scene, k_pos_scene, keep_scene, splits, tiles, po,
                reinterpret_cast<float2 *>(static_cast<char *>(workspace) + part_o_bytes(a, splits))};
    Cached f{a, c, out, as_stream(stream)};
    attention_variant(a, args->dtype, f);
    return check_launch();
}
