// gated_norm.hip — the norms around a block, fused with its gate and residual scale.
//
//   n = branch rstd(branch) branch_weight   (or branch)
//   y = x + gate scale n                    h = y rstd(y) weight
// with rstd(v) = 1 / sqrt(mean(v^2) + eps).  Bytes bound both directions: a row passes
// through registers once, in float32 throughout.  The backward forms y again from x and
// branch rather than reading it (the same bytes, and nothing rounded between), and
// sums two things over rows, from which every parameter's gradient follows:
//   A[c] = sum dy' branch_hat,  B[c] = sum dh y_hat    (dy': the whole gradient at y)
//   dgate = scale branch_weight A (a scene's), dscale = sum_s gate branch_weight A,
//   dbranch_weight = sum_s gate scale A, dweight = B
// first over each workgroup's rows of one scene, then over workgroups, in a fixed order.
//
// 20,000 rows of 1024, bfloat16 with a float32 residual (246 MB forward, 369 backward): 49 us (5.0 TB/s) and
// 75 (4.9 TB/s) + 13 for the sums.  200,000 rows of 500, bfloat16 (0.8 and 1.2 GB): 197 us (4.1 TB/s)
// and 339 (3.5 TB/s) + 21.
#include "gsv_device.h"

namespace gsv {
namespace {

typedef __bf16 bf16;

struct NormArgs {
    const void *x, *branch, *gate;
    const float *weight, *branch_weight, *scale;
    const int *starts;
    int64_t x_row, branch_row, gate_row;
    int tokens, channels, scenes, per_token, f32_gate;
    float eps;
    // forward
    void *y, *h;
    // backward
    const void *dy, *dh;
    int64_t dy_row, dh_row;
    void *dx, *dbranch, *dgate;
    float *part_a, *part_b;  // (places, channels)
    int places, rows;        // workgroups, and the rows of each
};

template <typename T, int N> struct __align__(sizeof(T) * N > 16 ? 16 : sizeof(T) * N) Pack {
    T v[N];
};

// One row's channels of a lane: item i covers VEC channels from (i * LANES + lane) * VEC.
template <int VEC, int E, int LANES> struct Lane {
    static constexpr int kItems = E / VEC;
    template <typename T>
    static __device__ __forceinline__ void load(float (&f)[E], const T *row, int lane, int channels,
                                                float other = 0.f) {
#pragma unroll
        for (int i = 0; i < kItems; ++i) {
            const int c = (i * LANES + lane) * VEC;
            Pack<T, VEC> p;
            if (c < channels) p = *reinterpret_cast<const Pack<T, VEC> *>(row + c);
#pragma unroll
            for (int e = 0; e < VEC; ++e) f[i * VEC + e] = c < channels ? (float)p.v[e] : other;
        }
    }
    template <typename T>
    static __device__ __forceinline__ void store(const float (&f)[E], T *row, int lane, int channels) {
#pragma unroll
        for (int i = 0; i < kItems; ++i) {
            const int c = (i * LANES + lane) * VEC;
            Pack<T, VEC> p;
#pragma unroll
            for (int e = 0; e < VEC; ++e) p.v[e] = (T)f[i * VEC + e];
            if (c < channels) *reinterpret_cast<Pack<T, VEC> *>(row + c) = p;
        }
    }
};

// The sum over a row's lanes: one wave, or several of them through LDS, in two places taken in turn:
// a wave writes to a place again only behind the next sum's barrier, which all have read before.
template <int WAVES> struct RowSum {
    float (*lds)[4];
    int turn = 0;
    __device__ __forceinline__ float operator()(float v) {
        v = wave_sum(v);
        if constexpr (WAVES > 1) {
            const int wave = threadIdx.x >> 6, first = wave / WAVES * WAVES;
            if ((threadIdx.x & 63) == 0) lds[turn][wave] = v;
            __syncthreads();
            v = 0.f;
#pragma unroll
            for (int w = 0; w < WAVES; ++w) v += lds[turn][first + w];
            turn ^= 1;
        }
        return v;
    }
};

__device__ __forceinline__ int start_of(const NormArgs &a, int s) {
    if (s <= 0) return 0;
    if (s >= a.scenes) return a.tokens;
    return min(max(a.starts[s], 0), a.tokens);
}

// The last scene with value(s) <= x, values that ascend from 0 to `end`: looked for among the 64 around
// where it is if they do so evenly, by one load, and past those by a search.  (200,000 rows of 512, bfloat16,
// forward: 190 scenes 126 us, 20,000 132, 200,000 152; by a look at all starts for each row 136, 1,624 and
// 15,230.)
template <typename F> __device__ __forceinline__ int scene_at(const NormArgs &a, int x, int end, const F &value) {
    if (a.scenes == 1) return 0;
    const int lane = threadIdx.x & 63, guess = (int)((float)x * ((float)a.scenes / (float)max(end, 1)));
    const int lo = __builtin_amdgcn_readfirstlane(max(min(guess - 32, a.scenes - 64), 0));
    const int n = __popcll(__ballot(lo + lane < a.scenes && value(lo + lane) <= x));
    if ((n == 0 && lo > 0) || (n == 64 && lo + 64 < a.scenes)) return last_at_most(a.scenes, x, value);
    return __builtin_amdgcn_readfirstlane(lo + max(n, 1) - 1);
}
__device__ __forceinline__ int scene_of(const NormArgs &a, int row) {
    return scene_at(a, row, a.tokens, [&](int s) { return start_of(a, s); });
}
// The backward's workgroups, scene after scene: scene s has those from start / rows + s on, at least one
// for each `rows` rows it begins, so that their number goes by the rows and scenes there are.
__device__ __forceinline__ int first_place(const NormArgs &a, int s) { return start_of(a, s) / a.rows + s; }

template <typename TF, typename L, int E>
__device__ __forceinline__ void load_gate(const NormArgs &a, float (&f)[E], int64_t row, int lane) {
    if (a.f32_gate)
        L::load(f, static_cast<const float *>(a.gate) + row * a.gate_row, lane, a.channels);
    else
        L::load(f, static_cast<const TF *>(a.gate) + row * a.gate_row, lane, a.channels);
}

template <typename TX, typename TF, int VEC, int E, int WAVES>
__global__ __launch_bounds__(256) void k_norm_fwd(const NormArgs a) {
    typedef Lane<VEC, E, 64 * WAVES> L;
    __shared__ float lds[2][4];
    RowSum<WAVES> row_sum{lds};
    const int lane = threadIdx.x % (64 * WAVES);
    constexpr int kPer = 4 / WAVES;  // rows of a workgroup at a time
    const float inv = 1.f / a.channels;
    float w[E];
    L::load(w, a.weight, lane, a.channels);
    const int stride = gridDim.x * kPer;
    for (int first = blockIdx.x * kPer; first < a.tokens; first += stride) {
        // waves past the last row form it again and store nothing: all meet at the sums' barriers
        const int mine = first + (threadIdx.x >> 6) / WAVES, row = min(mine, a.tokens - 1);
        float x[E], f[E];
        L::load(f, static_cast<const TF *>(a.branch) + row * a.branch_row, lane, a.channels);
        L::load(x, static_cast<const TX *>(a.x) + row * a.x_row, lane, a.channels);
        float by[E];
        if (a.gate) {
            load_gate<TF, L>(a, by, a.per_token ? row : a.scenes > 1 ? scene_of(a, row) : 0, lane);
        } else {
#pragma unroll
            for (int e = 0; e < E; ++e) by[e] = 1.f;
        }
        if (a.scale) {
            float t[E];
            L::load(t, a.scale, lane, a.channels);
#pragma unroll
            for (int e = 0; e < E; ++e) by[e] *= t[e];
        }
        if (a.branch_weight) {
            float t[E], sq = 0.f;
            L::load(t, a.branch_weight, lane, a.channels);
#pragma unroll
            for (int e = 0; e < E; ++e) sq = fmaf(f[e], f[e], sq);
            const float r = rsqrtf(row_sum(sq) * inv + a.eps);
#pragma unroll
            for (int e = 0; e < E; ++e) f[e] *= r * t[e];
        }
        float sq = 0.f;
#pragma unroll
        for (int e = 0; e < E; ++e) x[e] = fmaf(by[e], f[e], x[e]), sq = fmaf(x[e], x[e], sq);
        const float r = rsqrtf(row_sum(sq) * inv + a.eps);
        if (mine == row) L::store(x, static_cast<TX *>(a.y) + (int64_t)row * a.channels, lane, a.channels);
#pragma unroll
        for (int e = 0; e < E; ++e) x[e] *= r * w[e];
        if (mine == row) L::store(x, static_cast<TF *>(a.h) + (int64_t)row * a.channels, lane, a.channels);
    }
}

// TOKEN: a gate for each token.  What a lane keeps over its rows is weight, gate times scale times
// branch_weight (TOKEN: without the gate) and the two sums.
template <typename TX, typename TF, int VEC, int E, int WAVES, bool TOKEN>
__global__ __launch_bounds__(256) void k_norm_bwd(const NormArgs a) {
    typedef Lane<VEC, E, 64 * WAVES> L;
    __shared__ float lds[2][4];
    RowSum<WAVES> row_sum{lds};
    constexpr int kPer = 4 / WAVES;  // rows of a workgroup at a time
    __shared__ float sums[kPer > 1 ? (kPer - 1) * 64 * WAVES * E : 1];
    const int lane = threadIdx.x % (64 * WAVES), wave = threadIdx.x >> 6;
    const float inv = 1.f / a.channels;
    const int s = scene_at(a, blockIdx.x, a.places, [&](int s) { return first_place(a, s); });
    const int64_t r0 = start_of(a, s) + (int64_t)((int)blockIdx.x - first_place(a, s)) * a.rows;
    int64_t r1 = min(r0 + a.rows, (int64_t)start_of(a, s + 1));
    float wgt[E], by[E], sum_a[E], sum_b[E];
    L::load(wgt, a.weight, lane, a.channels);
#pragma unroll
    for (int e = 0; e < E; ++e) by[e] = 1.f, sum_a[e] = sum_b[e] = 0.f;
    if (a.branch_weight) L::load(by, a.branch_weight, lane, a.channels);
    if (a.scale) {
        float t[E];
        L::load(t, a.scale, lane, a.channels);
#pragma unroll
        for (int e = 0; e < E; ++e) by[e] *= t[e];
    }
    if (!TOKEN && a.gate) {
        float t[E];
        load_gate<TF, L>(a, t, s, lane);
#pragma unroll
        for (int e = 0; e < E; ++e) by[e] *= t[e];
    }
    if (r0 < start_of(a, s)) r1 = r0;  // (only where starts do not ascend)
    for (int64_t first = r0; first < r1; first += kPer) {
        // waves past the last row take it with zero gradients and store nothing
        const int64_t mine = first + wave / WAVES, row = min(mine, r1 - 1);
        const bool live = mine == row;
        float x[E], f[E], dy[E], dh[E], g[E];
        L::load(f, static_cast<const TF *>(a.branch) + row * a.branch_row, lane, a.channels);
        L::load(x, static_cast<const TX *>(a.x) + row * a.x_row, lane, a.channels);
        if (a.dh && live) {
            L::load(dh, static_cast<const TF *>(a.dh) + row * a.dh_row, lane, a.channels);
        } else {
#pragma unroll
            for (int e = 0; e < E; ++e) dh[e] = 0.f;
        }
        if (a.dy && live) {
            L::load(dy, static_cast<const TX *>(a.dy) + row * a.dy_row, lane, a.channels);
        } else {
#pragma unroll
            for (int e = 0; e < E; ++e) dy[e] = 0.f;
        }
        if constexpr (TOKEN) load_gate<TF, L>(a, g, row, lane);
        const auto weight = [&](int e) { return TOKEN ? by[e] * g[e] : by[e]; };
        float rb = 1.f;
        if (a.branch_weight) {
            float sq = 0.f;
#pragma unroll
            for (int e = 0; e < E; ++e) sq = fmaf(f[e], f[e], sq);
            rb = rsqrtf(row_sum(sq) * inv + a.eps);
        }
        float sq = 0.f;
#pragma unroll
        for (int e = 0; e < E; ++e) {
            f[e] *= rb;  // branch_hat
            x[e] = fmaf(weight(e), f[e], x[e]);
            sq = fmaf(x[e], x[e], sq);
        }
        const float ry = rsqrtf(row_sum(sq) * inv + a.eps);
        float m1 = 0.f;
#pragma unroll
        for (int e = 0; e < E; ++e) {
            x[e] *= ry;  // y_hat
            sum_b[e] = fmaf(dh[e], x[e], sum_b[e]);
            dh[e] *= wgt[e];
            m1 = fmaf(dh[e], x[e], m1);
        }
        m1 = row_sum(m1) * inv;
        float m2 = 0.f;
#pragma unroll
        for (int e = 0; e < E; ++e) {
            dy[e] = fmaf(ry, dh[e] - x[e] * m1, dy[e]);
            x[e] = dy[e] * weight(e);
            m2 = fmaf(x[e], f[e], m2);
            const float t = dy[e] * f[e];  // of A
            if constexpr (TOKEN) {
                sum_a[e] = fmaf(t, g[e], sum_a[e]);
                g[e] = t * by[e];
            } else {
                sum_a[e] += t;
            }
        }
        if (live) L::store(dy, static_cast<TX *>(a.dx) + row * a.channels, lane, a.channels);
        if (TOKEN && live) {
            if (a.f32_gate) L::store(g, static_cast<float *>(a.dgate) + row * a.channels, lane, a.channels);
            else L::store(g, static_cast<TF *>(a.dgate) + row * a.channels, lane, a.channels);
        }
        if (a.branch_weight) {
            m2 = row_sum(m2) * inv;
#pragma unroll
            for (int e = 0; e < E; ++e) x[e] = rb * (x[e] - f[e] * m2);
        }
        if (live) L::store(x, static_cast<TF *>(a.dbranch) + row * a.channels, lane, a.channels);
    }
    // the workgroup's sums: those of the first row's waves, then the other rows'
    if constexpr (kPer > 1) {
        constexpr int kLanes = 64 * WAVES;
        const int group = wave / WAVES;
#pragma unroll
        for (int turn = 0; turn < 2; ++turn) {
            float(&v)[E] = turn ? sum_b : sum_a;
            __syncthreads();
            if (group)
#pragma unroll
                for (int e = 0; e < E; ++e) sums[((group - 1) * E + e) * kLanes + lane] = v[e];
            __syncthreads();
            if (!group)
#pragma unroll
                for (int e = 0; e < E; ++e)
#pragma unroll
                    for (int o = 0; o < kPer - 1; ++o) v[e] += sums[(o * E + e) * kLanes + lane];
        }
        if (group) return;
    }
    L::store(sum_a, a.part_a + (int64_t)blockIdx.x * a.channels, lane, a.channels);
    L::store(sum_b, a.part_b + (int64_t)blockIdx.x * a.channels, lane, a.channels);
}

// Each scene's sums over its workgroups, into the first of them; a scene's gate gradient.  COLS columns
// and 256 / COLS row groups of a workgroup: 16 where scenes have many workgroups, 256 where there
// are so many scenes that most have one or two: 200,000 rows of 512 in 1,025 scenes train in 540 us with
// either, in 20,000 in 578 with 256 columns and 944 with 16, in 200,000 in 2,320 and 6,090.
template <int COLS>
__global__ __launch_bounds__(256) void k_norm_scene_sums(const NormArgs a, int first_scene) {
    constexpr int kCols = COLS, kGroups = 256 / COLS;
    __shared__ float la[kGroups][kCols], lb[kGroups][kCols];
    const int col = threadIdx.x % kCols, grp = threadIdx.x / kCols;
    const int c = blockIdx.x * kCols + col, s = first_scene + blockIdx.y;
    const int p0 = first_place(a, s), p1 = s + 1 < a.scenes ? first_place(a, s + 1) : a.places;
    float sa = 0.f, sb = 0.f;
    if (c < a.channels)
        for (int p = p0 + grp; p < p1; p += kGroups) {
            const int64_t at = (int64_t)p * a.channels + c;
            sa += a.part_a[at], sb += a.part_b[at];
        }
    la[grp][col] = sa, lb[grp][col] = sb;
    __syncthreads();
    if (grp || c >= a.channels) return;
#pragma unroll
    for (int g = 1; g < kGroups; ++g) sa += la[g][col], sb += lb[g][col];
    // no other workgroup reads these columns of this scene
    const int64_t at = (int64_t)p0 * a.channels + c;
    a.part_a[at] = sa, a.part_b[at] = sb;
    if (a.dgate && !a.per_token) {
        const float g = sa * (a.scale ? a.scale[c] : 1.f) * (a.branch_weight ? a.branch_weight[c] : 1.f);
        if (a.f32_gate) static_cast<float *>(a.dgate)[(int64_t)s * a.channels + c] = g;
        else static_cast<bf16 *>(a.dgate)[(int64_t)s * a.channels + c] = (bf16)g;
    }
}

// The parameters' gradients from the scenes' sums: kChunk scenes (every `step`-th, `count` in all) for a
// workgroup's columns.  With one chunk its sums are the whole; else they go where its first scene's were, and a
// further launch adds the chunks', which have the gate in them (step > 1).
constexpr int kCols = 16, kGroups = 16, kChunk = 1024;
__global__ __launch_bounds__(256) void k_norm_sums(const NormArgs a, int step, int count, float *dweight,
                                                   float *dbranch_weight, float *dscale) {
    __shared__ float la[kGroups][kCols], lb[kGroups][kCols];
    const int col = threadIdx.x % kCols, grp = threadIdx.x / kCols;
    const int c = blockIdx.x * kCols + col;
    const int i0 = blockIdx.y * kChunk, i1 = min(i0 + kChunk, count);
    float sa = 0.f, sb = 0.f;
    if (c < a.channels)
        for (int i = i0 + grp; i < i1; i += kGroups) {
            const int s = i * step;
            const int64_t at = (int64_t)first_place(a, s) * a.channels + c;
            float g = 1.f;
            if (a.gate && !a.per_token && step == 1)
                g = a.f32_gate ? static_cast<const float *>(a.gate)[s * a.gate_row + c]
                               : (float)static_cast<const bf16 *>(a.gate)[s * a.gate_row + c];
            sa = fmaf(a.part_a[at], g, sa), sb += a.part_b[at];
        }
    la[grp][col] = sa, lb[grp][col] = sb;
    __syncthreads();
    if (grp || c >= a.channels) return;
#pragma unroll
    for (int g = 1; g < kGroups; ++g) sa += la[g][col], sb += lb[g][col];
    if (gridDim.y > 1) {
        const int64_t at = (int64_t)first_place(a, i0 * step) * a.channels + c;
        a.part_a[at] = sa, a.part_b[at] = sb;
        return;
    }
    dweight[c] = sb;
    if (dscale) dscale[c] = sa * (a.branch_weight ? a.branch_weight[c] : 1.f);
    if (dbranch_weight) dbranch_weight[c] = sa * (a.scale ? a.scale[c] : 1.f);
}

template <typename TX, typename TF, int VEC, int E, int WAVES>
void launch_fwd(const NormArgs &a, hipStream_t s) {
    // a wave keeps the weights over its rows
    const int64_t want = ((int64_t)a.tokens * WAVES + 3) / 4;
    hipLaunchKernelGGL((k_norm_fwd<TX, TF, VEC, E, WAVES>), dim3((unsigned)imin64(want, 8192)),
                       dim3(256), 0, s, a);
}
template <typename TX, typename TF, int VEC, int E, int WAVES>
void launch_bwd(const NormArgs &a, hipStream_t s) {
    const dim3 grid((unsigned)a.places);
    if (a.per_token) hipLaunchKernelGGL((k_norm_bwd<TX, TF, VEC, E, WAVES, true>), grid, dim3(256), 0, s, a);
    else hipLaunchKernelGGL((k_norm_bwd<TX, TF, VEC, E, WAVES, false>), grid, dim3(256), 0, s, a);
}
// Channels of a lane and waves of a row.  The backward keeps eight vectors of them, so 8 channels a
// lane (105 registers, four waves a SIMD) and more waves a row: 20,000 rows of 1024 train in 127 us, with 16
// channels a lane and one wave (190 registers) in 143; of 768 in 97 and 111.
template <typename TX, typename TF, int VEC>
void launch_width(const NormArgs &a, bool backward, hipStream_t s) {
    if (!backward) {
        if (a.channels <= 512) launch_fwd<TX, TF, VEC, 8, 1>(a, s);
        else if (a.channels <= 1024) launch_fwd<TX, TF, VEC, 16, 1>(a, s);
        else if (a.channels <= 2048) launch_fwd<TX, TF, VEC, 32, 1>(a, s);
        else launch_fwd<TX, TF, VEC, 32, 4>(a, s);
    } else {
        if (a.channels <= 512) launch_bwd<TX, TF, VEC, 8, 1>(a, s);
        else if (a.channels <= 1024) launch_bwd<TX, TF, VEC, 8, 2>(a, s);
        else if (a.channels <= 2048) launch_bwd<TX, TF, VEC, 8, 4>(a, s);
        else launch_bwd<TX, TF, VEC, 32, 4>(a, s);
    }
}
template <typename TX, typename TF> void launch_types(const NormArgs &a, int vec, bool backward, hipStream_t s) {
    if (vec == 8) launch_width<TX, TF, 8>(a, backward, s);
    else if (vec == 4) launch_width<TX, TF, 4>(a, backward, s);
    else launch_width<TX, TF, 1>(a, backward, s);
}
void launch(const gsv_norm *n, const NormArgs &a, int vec, bool backward, hipStream_t s) {
    if (n->branch_dtype == GSV_F32) launch_types<float, float>(a, vec, backward, s);
    else if (n->dtype == GSV_F32) launch_types<float, bf16>(a, vec, backward, s);
    else launch_types<bf16, bf16>(a, vec, backward, s);
}

int norm_args(const gsv_norm *n, NormArgs *a) {
    if (!n) return GSV_ERR_INVALID_ARGUMENT;
    const auto type = [](int t) { return t == GSV_F32 || t == GSV_BF16; };
    if (!type(n->dtype) || !type(n->branch_dtype) || n->dtype > n->branch_dtype) return GSV_ERR_INVALID_ARGUMENT;
    if (n->tokens < 0 || n->channels < 1 || n->channels > 8192 || n->scenes < 1 || !(n->eps >= 0.f))
        return GSV_ERR_INVALID_ARGUMENT;
    if (n->tokens > GSV_MAX_TOKENS || n->scenes > GSV_MAX_TOKENS) return GSV_ERR_SIZE_OVERFLOW;
    if (n->scenes > 1 && !n->starts) return GSV_ERR_INVALID_ARGUMENT;
    if (n->gate && (!type(n->gate_dtype) || (n->gate_dtype == GSV_BF16 && n->branch_dtype == GSV_F32)))
        return GSV_ERR_INVALID_ARGUMENT;
    if (n->gate && n->gate_per_token && n->scenes != 1) return GSV_ERR_INVALID_ARGUMENT;
    if (n->tokens > 0 && (!n->x || !n->branch || !n->weight)) return GSV_ERR_INVALID_ARGUMENT;
    *a = NormArgs{};
    a->x = n->x, a->branch = n->branch, a->gate = n->gate, a->weight = n->weight;
    a->branch_weight = n->branch_weight, a->scale = n->scale, a->starts = n->starts;
    a->x_row = n->x_row, a->branch_row = n->branch_row, a->gate_row = n->gate_row;
    a->tokens = n->tokens, a->channels = n->channels, a->scenes = n->scenes;
    a->per_token = n->gate && n->gate_per_token, a->f32_gate = n->gate_dtype == GSV_F32;
    a->eps = n->eps;
    return GSV_OK;
}

// Channels of one access: 8, or 4, where every row and vector starts aligned for it (16 bytes,
// or what 4 or 8 channels take where that is less).
int norm_vec(const gsv_norm *n, const void *const *ptrs, const int *f32, const int64_t *rows, int count) {
    for (int vec : {8, 4}) {
        bool ok = n->channels % vec == 0;
        for (int i = 0; i < count && ok; ++i) {
            const int size = f32[i] ? 4 : 2, need = vec * size > 16 ? 16 : vec * size;
            ok = reinterpret_cast<uintptr_t>(ptrs[i]) % need == 0 && (rows[i] * size) % need == 0;
        }
        if (ok) return vec;
    }
    return 1;
}

// Rows and workgroups of the backward: about 1024 workgroups, at least 16 rows each, and one more a scene.
bool norm_places(const gsv_norm *n, NormArgs *a) {
    a->rows = (int)imax64(16, ((int64_t)n->tokens + 1023) / 1024);
    if (a->scenes > (1 << 22)) return false;
    a->places = n->tokens / a->rows + a->scenes;
    return true;
}

}  // namespace
}  // namespace gsv

using namespace gsv;

extern "C" int gsv_gated_norm_fwd(const gsv_norm *n, void *y, void *h, void *stream) {
    NormArgs a;
    const int st = norm_args(n, &a);
    if (st != GSV_OK) return st;
    if (a.tokens == 0) return GSV_OK;
    if (!y || !h) return GSV_ERR_INVALID_ARGUMENT;
    a.y = y, a.h = h;
    const int xf = n->dtype == GSV_F32, bf = n->branch_dtype == GSV_F32;
    const void *ptrs[] = {n->x, n->branch, n->gate, n->weight, n->branch_weight, n->scale, y, h};
    const int f32[] = {xf, bf, a.f32_gate, 1, 1, 1, xf, bf};
    const int64_t rows[] = {n->x_row, n->branch_row, n->gate ? n->gate_row : 0, 0, 0, 0, n->channels, n->channels};
    launch(n, a, norm_vec(n, ptrs, f32, rows, 8), false, as_stream(stream));
    return check_launch();
}

extern "C" int gsv_gated_norm_bwd_workspace_bytes(const gsv_norm *n, size_t *bytes) {
    NormArgs a;
    if (!bytes) return GSV_ERR_INVALID_ARGUMENT;
    const int st = norm_args(n, &a);
    if (st != GSV_OK) return st;
    if (!norm_places(n, &a)) return GSV_ERR_SIZE_OVERFLOW;
    const size_t one = ((size_t)a.places * a.channels * sizeof(float) + 255) / 256 * 256;
    *bytes = 2 * one;
    return GSV_OK;
}

extern "C" int gsv_gated_norm_bwd(const gsv_norm *n, const void *dy, int64_t dy_row, const void *dh,
                                  int64_t dh_row, void *dx, void *dbranch, float *dweight,
                                  float *dbranch_weight, float *dscale, void *dgate,
                                  void *workspace, size_t workspace_bytes, void *stream) {
    NormArgs a;
    int st = norm_args(n, &a);
    if (st != GSV_OK) return st;
    if (!norm_places(n, &a)) return GSV_ERR_SIZE_OVERFLOW;
    size_t need;
    if ((st = gsv_gated_norm_bwd_workspace_bytes(n, &need)) != GSV_OK) return st;
    if (need > workspace_bytes) return GSV_ERR_WORKSPACE_TOO_SMALL;
    if (!dweight || !workspace || (a.tokens > 0 && (!dx || !dbranch)) || (a.gate && !dgate) ||
        (a.branch_weight && !dbranch_weight) || (a.scale && !dscale) ||
        reinterpret_cast<uintptr_t>(workspace) % 256)
        return GSV_ERR_INVALID_ARGUMENT;
    a.dy = dy, a.dh = dh, a.dy_row = dy_row, a.dh_row = dh_row;
    a.dx = dx, a.dbranch = dbranch, a.dgate = a.gate ? dgate : nullptr;
    a.part_a = static_cast<float *>(workspace);
    a.part_b = reinterpret_cast<float *>(static_cast<char *>(workspace) + need / 2);
    const int xf = n->dtype == GSV_F32, bf = n->branch_dtype == GSV_F32;
    const int64_t C = n->channels;
    const void *ptrs[] = {n->x, n->branch, n->gate, n->weight, n->branch_weight, n->scale, dy, dh, dx, dbranch,
                          a.per_token ? dgate : nullptr};
    const int f32[] = {xf, bf, a.f32_gate, 1, 1, 1, xf, bf, xf, bf, a.f32_gate};
    const int64_t rows[] = {n->x_row, n->branch_row, n->gate ? n->gate_row : 0, 0, 0, 0, dy ? dy_row : 0,
                            dh ? dh_row : 0, C, C, C};
    hipStream_t s = as_stream(stream);
    launch(n, a, norm_vec(n, ptrs, f32, rows, 11), true, s);
    // scenes are the y axis of the grid, 65535 at most: the rest in further launches
    for (int s0 = 0; s0 < a.scenes; s0 += 65535) {
        const unsigned some = (unsigned)imin64(a.scenes - s0, 65535);
        if (a.scenes <= kChunk)
            hipLaunchKernelGGL(k_norm_scene_sums<16>, dim3((unsigned)((C + 15) / 16), some), dim3(256), 0, s, a, s0);
        else
            hipLaunchKernelGGL(k_norm_scene_sums<256>, dim3((unsigned)((C + 255) / 256), some), dim3(256), 0, s, a, s0);
    }
    for (int64_t count = a.scenes, step = 1, chunks; ; count = chunks, step *= kChunk) {
        chunks = (count + kChunk - 1) / kChunk;
        hipLaunchKernelGGL(k_norm_sums, dim3((unsigned)((C + kCols - 1) / kCols), (unsigned)chunks), dim3(256), 0, s,
                           a, (int)step, (int)count, dweight, dbranch_weight, dscale);
        if (chunks == 1) break;
    }
    return check_launch();
}
