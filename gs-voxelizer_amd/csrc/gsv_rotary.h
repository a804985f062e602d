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

// One item of a head's row: pairs turned by `turns` (a token's cos and sin of each pair), or channels that pass
// through.  VEC pairs an item are two runs of VEC channels, or one of 2 VEC where pairs are interleaved.
template <typename T, int VEC, bool INTERLEAVED>
__device__ __forceinline__ void turn_item(const T *in, T *out, int item, int turning, int pairs, const float2 *turns) {
    if (item >= turning) {
        constexpr int W = kPassed<VEC, INTERLEAVED>;
        typedef Pack<T, W> P;
        const int d = 2 * pairs + (item - turning) * W;
        *reinterpret_cast<P *>(out + d) = *reinterpret_cast<const P *>(in + d);
        return;
    }
    const int p = item * VEC;
    const float2 *tp = turns + p;
    if constexpr (INTERLEAVED && VEC == 1) {
        const float2 z = turned((float)in[2 * p], (float)in[2 * p + 1], *tp);
        out[2 * p] = (T)z.x, out[2 * p + 1] = (T)z.y;
    } else if constexpr (INTERLEAVED) {
        typedef Pack<T, 2 * VEC> P;
        P x = *reinterpret_cast<const P *>(in + 2 * p);
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
            const float2 z = turned((float)x.v[2 * e], (float)x.v[2 * e + 1], tp[e]);
            x.v[2 * e] = (T)z.x, x.v[2 * e + 1] = (T)z.y;
        }
        *reinterpret_cast<P *>(out + 2 * p) = x;
    } else {
        typedef Pack<T, VEC> P;
        P x = *reinterpret_cast<const P *>(in + p);
        P z = *reinterpret_cast<const P *>(in + pairs + p);
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
            const float2 y = turned((float)x.v[e], (float)z.v[e], tp[e]);
            x.v[e] = (T)y.x, z.v[e] = (T)y.y;
        }
        *reinterpret_cast<P *>(out + p) = x;
        *reinterpret_cast<P *>(out + pairs + p) = z;
    }
}

}  // namespace gsv
