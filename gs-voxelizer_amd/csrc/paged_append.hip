// paged_append.hip — new tokens' keys and values into a cache in pages, the keys turned on the way.
//
// Token i of scene s's n new ones becomes row r = lengths[s] - n + i of the scene, row r % page_rows of the page
// that its table names; keys (and the queries, which go to an output of their own) are turned as by rotary.hip.
// Bytes bound it: each head is read and written once, in one launch.  A workgroup takes a few tokens: one wave
// finds their rows, a lane each, while the others form the angles; both serve all heads from LDS.
#include "gsv_rotary.h"

namespace gsv {
namespace {

struct AppendArgs {
    const void *q, *k, *v;
    void *q_out, *k_pool, *v_pool;
    int64_t q_row, q_head, k_row, k_head, v_row, v_head;
    int64_t kp_page, kp_row, kp_head, vp_page, vp_row, vp_head;
    int tokens, heads, kv_heads, dim, pairs, axes;
    const float *positions, *frequencies;
    int64_t pos_row, pos_axis;
    float *pos_pool;
    int64_t pp_page, pp_row;
    const void *keep;
    void *keep_pool;
    int64_t keep_page;
    int keep_bytes, keep_pool_bytes;
    const int *lengths, *starts, *table;
    int64_t table_row;
    int scenes, pages, page_rows, capacity;
    int block_tokens;
    int token_items;  // of a token
    FastDiv by_rows, by_pairs, by_token, by_items, by_value;
};

// The row of a token's own in the pools: page, and row in it; page < 0: none.
struct Target {
    int page, row;
};

__device__ __forceinline__ int start_of(const AppendArgs &a, int s) {
    if (s <= 0) return 0;
    if (s >= a.scenes) return a.tokens;
    return min(max(a.starts[s], 0), a.tokens);
}

// Token t's scene is s0 or a later one: looked for in steps that double, then halve.
__device__ __forceinline__ Target target_of(const AppendArgs &a, int t, int s0) {
    int s = a.starts ? s0 : t, ahead = 1;
    if (a.starts) {
        int step = 1;
        while (s + step < a.scenes && start_of(a, s + step) <= t) s += step, step *= 2;
        for (; step > 1;) {
            step /= 2;
            if (s + step < a.scenes && start_of(a, s + step) <= t) s += step;
        }
        ahead = start_of(a, s + 1) - t;  // of the scene's tokens, this one and those behind it
    }
    const int64_t row = (int64_t)a.lengths[s] - ahead;
    if (ahead < 1 || row < 0 || row >= a.capacity) return {-1, 0};
    const int entry = fastdiv((uint32_t)row, a.by_rows);
    const int page = a.table[s * a.table_row + entry];
    if (page < 0 || page >= a.pages) return {-1, 0};
    return {page, (int)row - entry * a.page_rows};
}

// A thread's part of each token: some channels of one head.  It is found once, and then the same for all of the
// workgroup's tokens: found anew for each, its divisions took more time than the bytes.
template <typename T, int VEC, bool INTERLEAVED> struct Part {
    const T *in;   // of token 0 of the array
    T *out;        // of token 0 of q_out, or of page 0's first row
    int64_t in_row, out_page, out_row;
    int item, turning, pairs;
    bool q;
    __device__ __forceinline__ Part(const AppendArgs &a, int j) {
        constexpr int W = kPassed<VEC, INTERLEAVED>;
        const int items = a.pairs / VEC + (a.dim - 2 * a.pairs) / W, all = (a.heads + a.kv_heads) * items;
        q = false, turning = a.pairs / VEC, pairs = a.pairs;
        if (j >= all) {
            const int h = fastdiv(j - all, a.by_value);
            item = j - all - h * (a.dim / W), turning = pairs = 0;
            in = static_cast<const T *>(a.v) + h * a.v_head, in_row = a.v_row;
            out = static_cast<T *>(a.v_pool) + h * a.vp_head, out_page = a.vp_page, out_row = a.vp_row;
            return;
        }
        int h = fastdiv(j, a.by_items);
        item = j - h * items;
        if (h < a.heads) {
            q = true;
            in = static_cast<const T *>(a.q) + h * a.q_head, in_row = a.q_row;
            out = static_cast<T *>(a.q_out) + (int64_t)h * a.dim, out_page = 0, out_row = (int64_t)a.heads * a.dim;
        } else {
            h -= a.heads;
            in = static_cast<const T *>(a.k) + h * a.k_head, in_row = a.k_row;
            out = static_cast<T *>(a.k_pool) + h * a.kp_head, out_page = a.kp_page, out_row = a.kp_row;
        }
    }
};

// Tokens of a thread that are loaded at once (the first ones before their rows and angles are known), and all that it
// takes, over which the chains of loads at a workgroup's start spread.  20,000 tokens (below) take 28.9 us with 8 of
// them, 30.9 with 16 and 30.0 with 4 at once and no more; 65,537 104, 105 and 116.
constexpr int kDeep = 2, kTokens = 8;

template <typename T, int VEC, bool INTERLEAVED>
__global__ __launch_bounds__(256) void k_paged_append(const AppendArgs a) {
    extern __shared__ float2 turns[];  // cos, sin of block_tokens x pairs
    __shared__ Target target[64];
    const int t0 = blockIdx.x * a.block_tokens, nt = min(a.block_tokens, a.tokens - t0);
    // a thread's first part and token: as many tokens side by side as have room
    const int side = max(256 / a.token_items, 1);
    const int first_t = side > 1 ? fastdiv(threadIdx.x, a.by_token) : 0, first_j = threadIdx.x - first_t * a.token_items;
    const bool mine = first_t < side;
    bool begun = false;
    for (int j = first_j; j - first_j < a.token_items; j += 256) {
        const bool has = mine && j < a.token_items;
        const Part<T, VEC, INTERLEAVED> p(a, has ? j : 0);
        for (int tb = 0; tb < nt; tb += side * kDeep) {
            TurnItem<T, VEC, INTERLEAVED> x[kDeep];
#pragma unroll
            for (int k = 0; k < kDeep; ++k) {
                const int t = tb + k * side + first_t;
                if (has && t < nt) x[k].load(p.in + (t0 + t) * p.in_row, p.item, p.turning, p.pairs);
            }
            if (!begun) {
                begun = true;
                if (threadIdx.x >= 192) {  // the last wave: it has the fewest angles
                    const int lane = threadIdx.x & 63;
                    int s0 = 0;
                    if (a.starts) s0 = last_at_most(a.scenes, t0, [&](int s) { return start_of(a, s); });
                    if (lane < nt) target[lane] = target_of(a, t0 + lane, s0);
                }
                for (int i = threadIdx.x; i < nt * a.pairs; i += 256) {
                    const int t = fastdiv(i, a.by_pairs), r = i - t * a.pairs;
                    turns[i] = turn_of(a.positions + (t0 + t) * a.pos_row, a.pos_axis, a.frequencies + r, a.pairs,
                                       a.axes);
                }
                __syncthreads();
            }
#pragma unroll
            for (int k = 0; k < kDeep; ++k) {
                const int t = tb + k * side + first_t;
                if (!has || t >= nt) continue;
                Target to = target[t];
                if (p.q) to = {0, t0 + t};
                if (to.page < 0) continue;
                x[k].store(p.out + to.page * p.out_page + to.row * p.out_row, p.item, p.turning, p.pairs,
                           turns + t * a.pairs);
            }
        }
    }
    if (a.pos_pool && threadIdx.x < nt * 3) {
        const int t = threadIdx.x / 3, ax = threadIdx.x % 3;
        const Target to = target[t];
        if (to.page >= 0)
            a.pos_pool[to.page * a.pp_page + to.row * a.pp_row + ax] =
                a.positions[(t0 + t) * a.pos_row + ax * a.pos_axis];
    }
    if (a.keep_pool && threadIdx.x < nt) {
        const Target to = target[threadIdx.x];
        const int64_t t = t0 + threadIdx.x;
        const int on = a.keep_bytes == 1 ? static_cast<const uint8_t *>(a.keep)[t] != 0
                                         : static_cast<const int *>(a.keep)[t] != 0;
        if (to.page >= 0) {
            const int64_t at = to.page * a.keep_page + to.row;
            if (a.keep_pool_bytes == 1) static_cast<uint8_t *>(a.keep_pool)[at] = (uint8_t)on;
            else static_cast<int *>(a.keep_pool)[at] = on;
        }
    }
}

template <typename T, bool INTERLEAVED> void launch_append(const AppendArgs &a, int vec, hipStream_t s) {
    const dim3 grid((a.tokens + a.block_tokens - 1) / a.block_tokens), block(256);
    const size_t lds = sizeof(float2) * a.block_tokens * a.pairs;
    switch (vec) {
        case 8:
            if constexpr (!INTERLEAVED && sizeof(T) == 2) {
                hipLaunchKernelGGL((k_paged_append<T, 8, INTERLEAVED>), grid, block, lds, s, a);
                break;
            }
            [[fallthrough]];
        case 4:
            if constexpr (!(INTERLEAVED && sizeof(T) == 4)) {
                hipLaunchKernelGGL((k_paged_append<T, 4, INTERLEAVED>), grid, block, lds, s, a);
                break;
            }
            [[fallthrough]];
        case 2: hipLaunchKernelGGL((k_paged_append<T, 2, INTERLEAVED>), grid, block, lds, s, a); break;
        default: hipLaunchKernelGGL((k_paged_append<T, 1, INTERLEAVED>), grid, block, lds, s, a);
    }
}

// The stride of an axis of one entry is never used, whatever a caller's view holds there.
int64_t used(int64_t stride, int64_t entries) { return entries > 1 ? stride : 0; }

}  // namespace
}  // namespace gsv

using namespace gsv;

extern "C" int gsv_paged_append(const gsv_rotary_args *r, const void *v, int64_t v_row, int64_t v_head,
                                const gsv_pages *p, const int32_t *lengths, const int32_t *starts, int32_t scenes,
                                const void *keep, int32_t keep_bytes, void *q_out, void *stream) {
    if (!r || !p || (r->dtype != GSV_F32 && r->dtype != GSV_BF16) || r->tokens < 0 || r->heads < 0 ||
        r->kv_heads < 1 || r->dim < 8 || r->dim > 128 || r->dim % 8 || r->pairs < 0 || 2 * r->pairs > r->dim ||
        (r->pairs && (r->axes < 1 || r->axes > 8)) || (r->heads && !r->pairs) || scenes < 0 ||
        (!starts && scenes != r->tokens) || p->pages < 1 || p->page_rows < 16 || p->page_rows % 16 ||
        p->table_pages < 0 || p->table_row < 0)
        return GSV_ERR_INVALID_ARGUMENT;
    const int64_t rows = (int64_t)p->page_rows * p->table_pages;
    if (r->tokens > GSV_MAX_TOKENS || scenes > GSV_MAX_TOKENS || rows > GSV_MAX_TOKENS) return GSV_ERR_SIZE_OVERFLOW;
    if ((int64_t)r->heads + r->kv_heads > 4096 || (r->tokens && scenes < 1)) return GSV_ERR_INVALID_ARGUMENT;
    if (r->tokens == 0) return GSV_OK;
    if (!r->k || !v || (r->heads && (!r->q || !q_out)) || !p->k || !p->v || !lengths || (rows && !p->table) ||
        ((r->pairs || p->positions) && !r->positions) || (r->pairs && !r->frequencies) ||
        (p->positions && r->axes != 3) || (p->keep != nullptr) != (keep != nullptr) ||
        (keep && ((keep_bytes != 1 && keep_bytes != 4) || (p->keep_bytes != 1 && p->keep_bytes != 4))))
        return GSV_ERR_INVALID_ARGUMENT;
    const int64_t size = r->dtype == GSV_BF16 ? 2 : 4, K = r->kv_heads, T = r->tokens;
    uintptr_t all = reinterpret_cast<uintptr_t>(r->k) | reinterpret_cast<uintptr_t>(v) |
                    reinterpret_cast<uintptr_t>(p->k) | reinterpret_cast<uintptr_t>(p->v);
    if (r->heads)
        all |= reinterpret_cast<uintptr_t>(r->q) | reinterpret_cast<uintptr_t>(q_out) |
               (uintptr_t)(used(r->q_row, T) * size) | (uintptr_t)(used(r->q_head, r->heads) * size);
    for (int64_t x : {used(r->k_row, T), used(r->k_head, K), used(v_row, T), used(v_head, K),
                      used(p->k_page, p->pages), p->k_row, used(p->k_head, K), used(p->v_page, p->pages), p->v_row,
                      used(p->v_head, K)})
        all |= (uintptr_t)(x * size);
    if (all % 16) return GSV_ERR_INVALID_ARGUMENT;
    // the widest access that both halves of a row's pairs and what follows them are aligned for
    uint64_t low = 16 | (uint64_t)(r->dim * size) | (uint64_t)((r->dim - 2 * r->pairs) * size) |
                   (uint64_t)(r->pairs * size * (r->interleaved ? 2 : 1));
    const int bytes = (int)(low & (0 - low));
    const int vec = r->interleaved && bytes > size ? bytes / size / 2 : bytes / size;
    const int passed = r->interleaved && vec > 1 ? 2 * vec : vec;
    // Tokens of a workgroup: as many as its threads hold at once, fewer where the launch would leave CUs idle; their
    // angles within 16 KB of LDS, a lane for each.
    const int items = r->pairs / vec + (r->dim - 2 * r->pairs) / passed, values = r->dim / passed;
    const int64_t each = (r->heads + K) * items + K * values;
    int64_t bt = kTokens * imax64(1, 256 / each);
    bt = imin64(bt, imax64(1, T / 1024));
    bt = imin64(bt, r->pairs ? imax64(1, 2048 / r->pairs) : 64);
    bt = imin64(bt, 64);
    if ((T + bt - 1) / bt >= (1 << 24)) return GSV_ERR_SIZE_OVERFLOW;
    const AppendArgs a{r->q, r->k, v, q_out, p->k, p->v,
                       used(r->q_row, T), used(r->q_head, r->heads), used(r->k_row, T), used(r->k_head, K),
                       used(v_row, T), used(v_head, K),
                       used(p->k_page, p->pages), p->k_row, used(p->k_head, K),
                       used(p->v_page, p->pages), p->v_row, used(p->v_head, K),
                       r->tokens, r->heads, r->kv_heads, r->dim, r->pairs, r->axes, r->positions, r->frequencies,
                       r->pos_row, r->pos_axis, p->positions, p->pos_page, p->pos_row, keep, p->keep, p->keep_page,
                       keep_bytes, p->keep_bytes, lengths, starts, p->table, p->table_row, scenes, p->pages,
                       p->page_rows, (int)rows, (int)bt, (int)each, make_fastdiv(p->page_rows),
                       make_fastdiv(r->pairs ? r->pairs : 1), make_fastdiv(each), make_fastdiv(items),
                       make_fastdiv(values)};
    hipStream_t s = as_stream(stream);
    if (r->dtype == GSV_BF16)
        r->interleaved ? launch_append<bf16, true>(a, vec, s) : launch_append<bf16, false>(a, vec, s);
    else
        r->interleaved ? launch_append<float, true>(a, vec, s) : launch_append<float, false>(a, vec, s);
    return check_launch();
}
