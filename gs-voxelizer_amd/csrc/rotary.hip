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
        const float2 w = turn_of(a.positions + (t0 + t) * a.pos_row, a.pos_axis, a.frequencies + p, a.pairs, a.axes);
        turns[i] = make_float2(w.x, a.sign * w.y);
    }
    __syncthreads();
    // a row's items: its pairs, then the channels past them, which pass through
    const int all = a.heads + a.kv_heads, turning = a.pairs / VEC;
    const int items = turning + (a.dim - 2 * a.pairs) / kPassed<VEC, INTERLEAVED>;
    for (int i = threadIdx.x; i < nt * all * items; i += 256) {
        const int row = fastdiv(i, a.by_items), item = i - row * items;
        const int t = fastdiv(row, a.by_heads), h = row - t * all;
        const bool is_q = h < a.heads;
        const int64_t token = t0 + t;
        const T *in = is_q ? static_cast<const T *>(a.q) + token * a.q_row + h * a.q_head
                           : static_cast<const T *>(a.k) + token * a.k_row + (h - a.heads) * a.k_head;
        T *out = is_q ? static_cast<T *>(a.q_out) + (token * a.heads + h) * a.dim
                      : static_cast<T *>(a.k_out) + (token * a.kv_heads + h - a.heads) * a.dim;
        TurnItem<T, VEC, INTERLEAVED> x;
        x.load(in, item, turning, a.pairs);
        x.store(out, item, turning, a.pairs, turns + t * a.pairs);
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
