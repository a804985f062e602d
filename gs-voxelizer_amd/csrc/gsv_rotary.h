// gsv_rotary.h — what the kernels that turn heads by their tokens' positions share.
#pragma once

#include "gsv_device.h"

namespace gsv {

typedef __bf16 bf16;

template <typename T, int N> struct __align__(sizeof(T) * N) Pack {
    T v[N];
};

// One pair turned; written as fused multiply-adds so that every access width gives the same bits.
__device__ __forceinline__ float2 turned(float x1, float x2, float2 w) {
    return make_float2(fmaf(x1, w.x, -(x2 * w.y)), fmaf(x1, w.y, x2 * w.x));
}

// cos and sin of a token's angle for one pair.  The angle in binary64, brought into -pi .. pi there: a
// binary32 product would lose 2^-24 of an angle of some hundred radians.
__device__ __forceinline__ float2 turn_of(const float *position, int64_t axis, const float *frequencies, int pairs,
                                          int axes) {
    double th = 0.0;
    for (int ax = 0; ax < axes; ++ax)
        th = fma((double)position[ax * axis], (double)frequencies[ax * pairs], th);
    const double turn = th * 0.15915494309189533577;
    const float r = (float)((turn - rint(turn)) * 6.283185307179586477);
    float sn, cs;
    sincosf(r, &sn, &cs);
    return make_float2(cs, sn);
}

// A row's items: its pairs, VEC at a time, then the channels past them, kPassed at a time.
template <int VEC, bool INTERLEAVED> constexpr int kPassed = INTERLEAVED && VEC > 1 ? 2 * VEC : VEC;

// One item of a head's row, loaded and then turned by `turns` (a token's cos and sin of each pair), or channels
// that pass through.  VEC pairs an item are two runs of VEC channels, or one of 2 VEC where pairs are interleaved.
template <typename T, int VEC, bool INTERLEAVED> struct TurnItem {
    static constexpr int kRun = INTERLEAVED ? 2 * VEC : VEC, W = kPassed<VEC, INTERLEAVED>;
    typedef Pack<T, kRun> Run;
    typedef Pack<T, W> Passed;
    Run x, z;
    // pairs: of the row; `turning` items of it are turned
    __device__ __forceinline__ void load(const T *in, int item, int turning, int pairs) {
        if (item >= turning) {
            const Passed p = *reinterpret_cast<const Passed *>(in + 2 * pairs + (item - turning) * W);
#pragma unroll
            for (int e = 0; e < W; ++e) x.v[e] = p.v[e];
        } else if constexpr (INTERLEAVED && VEC == 1) {  // (a pair may lie off its own alignment)
            x.v[0] = in[2 * item], x.v[1] = in[2 * item + 1];
        } else if constexpr (INTERLEAVED) {
            x = *reinterpret_cast<const Run *>(in + 2 * item * VEC);
        } else {
            x = *reinterpret_cast<const Run *>(in + item * VEC);
            z = *reinterpret_cast<const Run *>(in + pairs + item * VEC);
        }
    }
    __device__ __forceinline__ void store(T *out, int item, int turning, int pairs, const float2 *turns) {
        if (item >= turning) {
            Passed p;
#pragma unroll
            for (int e = 0; e < W; ++e) p.v[e] = x.v[e];
            *reinterpret_cast<Passed *>(out + 2 * pairs + (item - turning) * W) = p;
            return;
        }
        const float2 *tp = turns + item * VEC;
        if constexpr (INTERLEAVED) {
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                const float2 y = turned((float)x.v[2 * e], (float)x.v[2 * e + 1], tp[e]);
                x.v[2 * e] = (T)y.x, x.v[2 * e + 1] = (T)y.y;
            }
            if constexpr (VEC == 1) out[2 * item] = x.v[0], out[2 * item + 1] = x.v[1];
            else *reinterpret_cast<Run *>(out + 2 * item * VEC) = x;
        } else {
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                const float2 y = turned((float)x.v[e], (float)z.v[e], tp[e]);
                x.v[e] = (T)y.x, z.v[e] = (T)y.y;
            }
            *reinterpret_cast<Run *>(out + item * VEC) = x;
            *reinterpret_cast<Run *>(out + pairs + item * VEC) = z;
        }
    }
};

}  // namespace gsv
