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

}  // namespace gsv
