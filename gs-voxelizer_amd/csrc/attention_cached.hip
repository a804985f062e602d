// attention_cached.hip — one query token a scene against a cache of keys and values.
//
// Same scores as attention_fwd.hip.  The bytes of the cache are the floor: each is read
// once, by coalesced 16-byte loads, and serves all query heads of its key head, which
// are the columns of a matrix product (32, those past the group idle: the matrix units
// have an order of magnitude to spare here).  A cache is split over workgroups, a split over
// four waves that never wait for each other; a second kernel joins the splits.
//
// Two caches of 200,003 rows, 4 heads of 128, bfloat16 (316 MB of live rows): 65 us, 4.9 TB/s, and 5 us
// for the join.  16 caches of 4,096, 2 heads of 64 (23 MB): 10.8 us and 3.9; there the time from
// launch to the first bytes and a wave's few steps one after the other bound it.
#include "gsv_attention.h"

// (a product and a difference stay two roundings where they are written as two)
#pragma clang fp contract(off)

namespace gsv {
namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr int kKeys = 32;   // keys of a wave's step
constexpr int kHeads = 32;  // query heads of a workgroup
constexpr float kSlack = 8.f;

struct CacheArgs {
    const int *lengths;
    int64_t k_scene, v_scene, k_pos_scene, keep_scene;
    int splits, head_tiles;
    float *part_o;   // (scenes, heads, splits, dim): sums of weights times values
    float2 *part_ms; // (scenes, heads, splits): maximum (log2) and sum of weights
};

// Waves of a workgroup: four, two where their tiles would pass the LDS of a CU.
template <typename T, int DP> constexpr int kWaves = DP * sizeof(T) > 256 ? 2 : 4;

// bfloat16 weights enter the product with the values in two parts: the results are as exact as their type
// (0.0017 in the 2-norm, in one part 0.0018 to 0.0020), for 0 to 4 % of the time beside the cache's bytes.
template <typename T> constexpr int kParts = sizeof(T) == 2 ? 2 : 1;

template <typename T, int DP, bool FAR, int CAP>
__global__ __launch_bounds__((64 * kWaves<T, DP>)) void k_attention_cached(const AttnArgs a, const CacheArgs c,
                                                          T *__restrict__ out) {
    typedef typename Elem<T>::frag frag;
    constexpr int W = kWaves<T, DP>;
    static_assert(4 * kKeys * DP * sizeof(T) >= kHeads * DP * sizeof(float), "sums reuse the tiles");
    __shared__ __align__(1024) T tiles[W][4 * kKeys * DP];  // a wave's keys and values, two buffers
    __shared__ __align__(16) typename Places<T>::Row spos[W][2][3 * kKeys];
    __shared__ float sm[W][kHeads], ss[W][kHeads];

    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int group = a.heads / a.kv_heads;
    int n = blockIdx.x;
    const int hk = n % a.kv_heads;
    n /= a.kv_heads;
    const int ht = n % c.head_tiles;
    n /= c.head_tiles;
    const int split = n % c.splits, s = n / c.splits;
    const int len = min(max(c.lengths[s], 0), a.k_tokens);
    const int per = ((len + c.splits - 1) / c.splits + kKeys - 1) / kKeys * kKeys;
    const int j_begin = min((int64_t)split * per, (int64_t)len), j_end = min(j_begin + per, len);
    const int col = ht * kHeads + (lane & 31);  // query head within the group
    const bool head = col < group;
    const int h = hk * group + (head ? col : 0);

    constexpr bool far = FAR, capped = CAP != kNoCap;
    const float slope = slope_of(a, h);
    const float unit = capped ? kLog2e : a.scale * kLog2e;
    const float far_unit = capped ? slope : slope / a.scale;
    const float in_cap = capped ? a.scale / a.cap : 0.f;
    frag q[DP / 16];
    load_column<T, DP>(q, static_cast<const T *>(a.q) + s * a.q_row + h * a.q_head, a.dim, head, lane);
    float x = 0.f, y = 0.f, z = 0.f;
    if (far) {
        const float *p = a.q_pos + s * a.q_pos_row;
        x = p[0], y = p[1], z = p[2];
    }
    Places<T> place;
        place.set(x, y, z, lane);
    const T *kbase = static_cast<const T *>(a.k) + s * c.k_scene + hk * a.k_head;
    const T *vbase = static_cast<const T *>(a.v) + s * c.v_scene + hk * a.v_head;
    T *const sk = tiles[wave], *const sv = sk + 2 * kKeys * DP;
    Tile<T, DP> at;
    at.plan(lane);
    Copy<T, DP, kKeys, 1> ck, cv;
    ck.plan(a.k_row, a.dim, 0, lane);
    cv.plan(a.v_row, a.dim, 0, lane);
    f32x16 o[DP / 32] = {};
    float m = -INFINITY, sum = 0.f;
    float gp[2] = {};
    int raw = 0;
    uint32_t live = ~0u, next_live = ~0u;
    const int step = W * kKeys;
    auto look = [&](int j0) {
        if (a.keep && j0 < j_end)
            raw = keep_raw(a, s * c.keep_scene + min(j0 + (lane & 31), j_end - 1));
    };
    auto fetch = [&](int b, int j0) {
        if (a.keep) next_live = (uint32_t)__ballot(raw != 0);
        look(j0 + step);
        const int left = j_end - j0;
        ck.start(sk + b * kKeys * DP, kbase + (int64_t)j0 * a.k_row, a.k_row, a.dim, left, a.keep,
                 next_live, 0, lane);
        cv.start(sv + b * kKeys * DP, vbase + (int64_t)j0 * a.v_row, a.v_row, a.dim, left, a.keep,
                 next_live, 0, lane);
        if (far)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const int r = min((i * 64 + lane) % kKeys, left - 1), ax = min((i * 64 + lane) / kKeys, 2);
                gp[i] = a.k_pos[s * c.k_pos_scene + (int64_t)(j0 + r) * a.k_pos_row + ax];
            }
    };
    // the tiles are this wave's own: its copies and LDS accesses need no barrier, only waits
    auto put = [&](int b) {
        if (far) {
            spos[wave][b][lane] = Places<T>::row(gp[0]);
            if (lane < kKeys) spos[wave][b][64 + lane] = Places<T>::row(gp[1]);
        }
        tile_wait();
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    };
    int b = 0;
    if (j_begin + wave * kKeys < j_end) {
        look(j_begin + wave * kKeys);
        fetch(0, j_begin + wave * kKeys);
        put(0);
    }
    for (int j0 = j_begin + wave * kKeys; j0 < j_end; j0 += step, b ^= 1) {
        const bool more = j0 + step < j_end;
        live = next_live;
        if (j_end - j0 < kKeys) live &= (1u << (j_end - j0)) - 1;
        if (more) fetch(b ^ 1, j0 + step);
        const T *kt = sk + b * kKeys * DP, *vt = sv + b * kKeys * DP;
        f32x16 d = {}, w = {};
        if (far) d = distances<T>(place, spos[wave][b], kKeys, 0, lane);
        if (far && !capped)
#pragma unroll
            for (int r = 0; r < 16; ++r) w[r] = -far_unit * d[r];
#pragma unroll
        for (int st = 0; st < DP / 16; ++st) w = mma(at.rows(kt, st), q[st], w);
        if (capped)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                w[r] = a.cap * tanh_of<T, CAP>(w[r] * in_cap);
                if (far) w[r] = fmaf(-far_unit, d[r], w[r]);
            }
        if (live != 0xffffffffu) {
            const uint32_t seen = live >> (4 * (lane >> 5));
#pragma unroll
            for (int r = 0; r < 16; ++r)
                if (!(seen & (1u << result_row(r)))) w[r] = -INFINITY;
        }
        // rounded here, so that the largest weight is a power of two exactly
#pragma unroll
        for (int r = 0; r < 16; ++r) w[r] *= unit;
        float top = -INFINITY;
#pragma unroll
        for (int r = 0; r < 16; ++r) top = fmaxf(top, w[r]);
        if (__any(top > m + kSlack)) {
            const float next = fmaxf(m, fmaxf(top, other_half(top)));
            const float by = next == -INFINITY ? 1.f : fast_exp2(m - next);
            m = next;
            sum *= by;
#pragma unroll
            for (int b = 0; b < DP / 32; ++b) o[b] *= by;
        }
        const float ref = m == -INFINITY ? 0.f : m;
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            w[r] = fast_exp2(w[r] - ref);
        }
#pragma unroll
        for (int part = 0; part < kParts<T>; ++part) {
            if (part) w = remainders<T>(w);
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                const frag p = to_frag<T>(w, half);
                sum = add_weights(p, sum);
#pragma unroll
                for (int e = 0; e < DP / 32; ++e)
                    o[e] = mma(at.columns(vt + half * 16 * DP, e, lane), p, o[e]);
            }
        }
        if (more) put(b ^ 1);
    }
    sum += other_half(sum);
    // the waves' sums, joined
    if (lane < 32) sm[wave][lane] = m, ss[wave][lane] = sum;
    float *so = reinterpret_cast<float *>(tiles[wave]);
#pragma unroll
    for (int b = 0; b < DP / 32; ++b)
#pragma unroll
        for (int g = 0; g < 4; ++g)
#pragma unroll
            for (int e = 0; e < 4; ++e)
                so[(lane & 31) * DP + b * 32 + 8 * g + 4 * (lane >> 5) + e] = o[b][4 * g + e];
    __syncthreads();
    const int heads = min(group - ht * kHeads, kHeads);
    for (int i = threadIdx.x; i < heads * DP; i += 64 * W) {
        const int r = i / DP, dd = i % DP;
        float top = -INFINITY, total = 0.f, val = 0.f;
#pragma unroll
        for (int w = 0; w < W; ++w) top = fmaxf(top, sm[w][r]);
#pragma unroll
        for (int w = 0; w < W; ++w) {
            // a wave without keys has the maximum -inf and the sum 0; NaN sums pass
            const float by = sm[w][r] == -INFINITY ? 1.f : fast_exp2(sm[w][r] - top);
            total = fmaf(by, ss[w][r], total);
            val = fmaf(by, reinterpret_cast<const float *>(tiles[w])[i], val);
        }
        if (dd >= a.dim) continue;
        const int hh = hk * group + ht * kHeads + r;
        if (c.splits == 1) {
            out[((int64_t)s * a.heads + hh) * a.dim + dd] = (T)(total == 0.f ? 0.f : val / total);
        } else {
            const int64_t at = ((int64_t)s * a.heads + hh) * c.splits + split;
            c.part_o[at * a.dim + dd] = val;
            if (dd == 0) c.part_ms[at] = make_float2(top, total);
        }
    }
}

// One workgroup a scene and head: four waves take the splits in turn, then their sums are joined,
// always in the same order.  Latency bounds it: 4 us at 16 splits a head, 5 at 32.
template <typename T>
__global__ __launch_bounds__(256) void k_cached_join(const float *__restrict__ part_o,
                                                     const float2 *__restrict__ part_ms, int splits,
                                                     int dim, T *__restrict__ out) {
    __shared__ float so[4][128], ss[4];
    const int64_t row = blockIdx.x;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const float2 *ms = part_ms + row * splits;
    float top = -INFINITY;
    for (int p = lane; p < splits; p += 64) top = fmaxf(top, ms[p].x);
#pragma unroll
    for (int k = 1; k < 64; k <<= 1) top = fmaxf(top, __shfl_xor(top, k));
    float total = 0.f, v0 = 0.f, v1 = 0.f;
    const int d0 = min(lane, dim - 1), d1 = min(lane + 64, dim - 1);
#pragma unroll 4
    for (int p = wave; p < splits; p += 4) {
        const float2 e = ms[p];
        const float by = e.x == -INFINITY ? 1.f : fast_exp2(e.x - top);
        total = fmaf(by, e.y, total);
        const float *o = part_o + (row * splits + p) * dim;
        v0 = fmaf(by, o[d0], v0);
        v1 = fmaf(by, o[d1], v1);
    }
    so[wave][lane] = v0, so[wave][64 + lane] = v1;
    if (lane == 0) ss[wave] = total;
    __syncthreads();
    if (threadIdx.x >= (unsigned)dim) return;
    const int d = threadIdx.x;
    total = ss[0] + ss[1] + ss[2] + ss[3];
    const float v = so[0][d] + so[1][d] + so[2][d] + so[3][d];
    out[row * dim + d] = (T)(total == 0.f ? 0.f : v / total);
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
        hipLaunchKernelGGL((k_attention_cached<T, DP, FAR, CAP>),
                           dim3((unsigned)(a.scenes * a.kv_heads * c.head_tiles * c.splits)),
                           dim3(64 * kWaves<T, DP>), 0, st, a, c, o);
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
    const CacheArgs c{lengths, k_scene, v_scene, k_pos_scene, keep_scene, splits, tiles, po,
                      reinterpret_cast<float2 *>(static_cast<char *>(workspace) + part_o_bytes(a, splits))};
    Cached f{a, c, out, as_stream(stream)};
    attention_variant(a, args->dtype, f);
    return check_launch();
}
