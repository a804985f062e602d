// rotary.hip — rotary positions with several axes.
//
//   theta[t, p] = sum_a positions[t, a] frequencies[a, p]
//   (y1, y2) = (x1 cos - x2 sin, x1 sin + x2 cos)  for each head's channel pair p
// The gradient is the rotation by -theta, so one kernel does both directions.  Bytes bound it:
// q and k are read and written once, in one launch; a token's angles are formed once, in LDS,
// and serve all its heads.
//
// 20,000 tokens, 8 + 8 heads of 64, bfloat16 (82 MB a direction): 15.7 us, 5.2 TB/s (the caches hold a
// part); 65,537 tokens, 12 + 4 heads of 40, float32, interleaved (336 MB): 84 us, 4.0 TB/s, 85 % of
// what a large copy reaches.
#include "gsv_rotary.h"

namespace gsv {
namespace {

struct RotaryArgs {
    const void *q, *k;
    void *q_out, *k_out;
    int64_t q_row, q_head, k_row, k_head;
    int tokens, heads, kv_heads, dim, pairs, axes;
    const float *positions, *frequencies;
    int64_t pos_row, pos_axis;
    float sign;
    int block_tokens;
    FastDiv by_pairs, by_items, by_heads;
};

// VEC pairs an item: two runs of VEC channels, or one of 2 VEC where pairs are interleaved.
template <typename T, int VEC, bool INTERLEAVED>
__global__ __launch_bounds__(256) void k_rotary(const RotaryArgs a) {
    extern __shared__ float2 turns[];  // cos, sin of block_tokens x pairs
    const int t0 = blockIdx.x * a.block_tokens, nt = min(a.block_tokens, a.tokens - t0);
    for (int i = threadIdx.x; i < nt * a.pairs; i += 256) {
        const int t = fastdiv(i, a.by_pairs), p = i - t * a.pairs;
        // the angle in binary64, brought into -pi .. pi there: a binary32 product would lose
        // 2^-24 of an angle of some hundred radians
        double th = 0.0;
        for (int ax = 0; ax < a.axes; ++ax)
            th = fma((double)a.positions[(t0 + t) * a.pos_row + ax * a.pos_axis],
                     (double)a.frequencies[ax * a.pairs + p], th);
        const double turn = th * 0.15915494309189533577;
        const float r = (float)((turn - rint(turn)) * 6.283185307179586477);
        float sn, cs;
        sincosf(r, &sn, &cs);
        turns[i] = make_float2(cs, a.sign * sn);
    }
    __syncthreads();
    // a row's items: its pairs, then the channels past them, which pass through
    constexpr int W = INTERLEAVED && VEC > 1 ? 2 * VEC : VEC;
    const int all = a.heads + a.kv_heads, turning = a.pairs / VEC;
    const int items = turning + (a.dim - 2 * a.pairs) / W;
    for (int i = threadIdx.x; i < nt * all * items; i += 256) {
        const int row = fastdiv(i, a.by_items), item = i - row * items, p = item * VEC;
        const int t = fastdiv(row, a.by_heads), h = row - t * all;
        const bool is_q = h < a.heads;
        const int64_t token = t0 + t;
        const T *in = is_q ? static_cast<const T *>(a.q) + token * a.q_row + h * a.q_head
                           : static_cast<const T *>(a.k) + token * a.k_row + (h - a.heads) * a.k_head;
        T *out = is_q ? static_cast<T *>(a.q_out) + (token * a.heads + h) * a.dim
                      : static_cast<T *>(a.k_out) + (token * a.kv_heads + h - a.heads) * a.dim;
        if (item >= turning) {
            typedef Pack<T, W> P;
            const int d = 2 * a.pairs + (item - turning) * W;
            *reinterpret_cast<P *>(out + d) = *reinterpret_cast<const P *>(in + d);
            continue;
        }
        const float2 *tp = turns + t * a.pairs + p;
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
            P z = *reinterpret_cast<const P *>(in + a.pairs + p);
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                const float2 y = turned((float)x.v[e], (float)z.v[e], tp[e]);
                x.v[e] = (T)y.x, z.v[e] = (T)y.y;
            }
            *reinterpret_cast<P *>(out + p) = x;
            *reinterpret_cast<P *>(out + a.pairs + p) = z;
        }
    }
}

template <typename T, bool INTERLEAVED> void launch_rotary(const RotaryArgs &a, int vec, hipStream_t s) {
    const dim3 grid((a.tokens + a.block_tokens - 1) / a.block_tokens), block(256);
    const size_t lds = sizeof(float2) * a.block_tokens * a.pairs;
    switch (vec) {
        case 8:
            if constexpr (!INTERLEAVED && sizeof(T) == 2) {
                hipLaunchKernelGGL((k_rotary<T, 8, INTERLEAVED>), grid, block, lds, s, a);
                break;
            }
            [[fallthrough]];
        case 4:
            if constexpr (!(INTERLEAVED && sizeof(T) == 4)) {
                hipLaunchKernelGGL((k_rotary<T, 4, INTERLEAVED>), grid, block, lds, s, a);
                break;
            }
            [[fallthrough]];
        case 2: hipLaunchKernelGGL((k_rotary<T, 2, INTERLEAVED>), grid, block, lds, s, a); break;
        default: hipLaunchKernelGGL((k_rotary<T, 1, INTERLEAVED>), grid, block, lds, s, a);
    }
}

}  // namespace
}  // namespace gsv

using namespace gsv;

extern "C" int gsv_rotary(const gsv_rotary_args *r, void *q_out, void *k_out, int32_t inverse,
                          void *stream) {
    if (!r || (r->dtype != GSV_F32 && r->dtype != GSV_BF16) || r->tokens < 0 || r->heads < 0 ||
        r->kv_heads < 0 || r->dim < 2 || r->dim > 1024 || r->pairs < 1 || 2 * r->pairs > r->dim ||
        r->axes < 1 || r->axes > 8)
        return GSV_ERR_INVALID_ARGUMENT;
    if (r->tokens > GSV_MAX_TOKENS) return GSV_ERR_SIZE_OVERFLOW;
    if (r->tokens == 0 || r->heads + r->kv_heads == 0) return GSV_OK;
    if ((int64_t)r->heads + r->kv_heads > 4096) return GSV_ERR_INVALID_ARGUMENT;
    if ((r->heads && (!r->q || !q_out)) || (r->kv_heads && (!r->k || !k_out)) || !r->positions ||
        !r->frequencies)
        return GSV_ERR_INVALID_ARGUMENT;
    // the widest access that every row, head and half starts aligned for, 16 bytes at most
    const int size = r->dtype == GSV_BF16 ? 2 : 4;
    uint64_t low = (uint64_t)r->dim * size | 16;
    if (r->heads)
        low |= (uint64_t)r->q_row * size | (uint64_t)r->q_head * size |
               reinterpret_cast<uintptr_t>(r->q) | reinterpret_cast<uintptr_t>(q_out);
    if (r->kv_heads)
        low |= (uint64_t)r->k_row * size | (uint64_t)r->k_head * size |
               reinterpret_cast<uintptr_t>(r->k) | reinterpret_cast<uintptr_t>(k_out);
    low |= (uint64_t)r->pairs * size * (r->interleaved ? 2 : 1);
    low |= (uint64_t)(r->dim - 2 * r->pairs) * size;
    const int bytes = (int)(low & (0 - low));
    if (bytes < size) return GSV_ERR_INVALID_ARGUMENT;
    const int vec = r->interleaved && bytes > size ? bytes / size / 2 : bytes / size;
    // Tokens of a workgroup: enough for four items a thread, fewer where the launch would
    // leave CUs idle, and angles within 16 KB of LDS.
    const int64_t per_token = (int64_t)(r->heads + r->kv_heads) * (r->pairs / vec);
    int64_t bt = imax64(1, 1024 / per_token);
    bt = imin64(bt, imax64(1, r->tokens / 1024));
    bt = imin64(bt, imax64(1, 2048 / r->pairs));
    const RotaryArgs a{r->q, r->k, q_out, k_out, r->q_row, r->q_head, r->k_row, r->k_head,
                       r->tokens, r->heads, r->kv_heads, r->dim, r->pairs, r->axes, r->positions,
                       r->frequencies, r->pos_row, r->pos_axis, inverse ? -1.f : 1.f, (int)bt,
                       make_fastdiv(r->pairs),
                       make_fastdiv(r->pairs / vec + (r->dim - 2 * r->pairs) /
                                                         (r->interleaved && vec > 1 ? 2 * vec : vec)),
                       make_fastdiv(r->heads + r->kv_heads)};
    hipStream_t s = as_stream(stream);
    if (r->dtype == GSV_BF16)
        r->interleaved ? launch_rotary<bf16, true>(a, vec, s) : launch_rotary<bf16, false>(a, vec, s);
    else
        r->interleaved ? launch_rotary<float, true>(a, vec, s) : launch_rotary<float, false>(a, vec, s);
    return check_launch();
}
