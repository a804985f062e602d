// paged_append.hip — new tokens' keys and values into a cache in pages, the keys turned on the way.
//
// Token i of scene s's n new ones becomes row r = lengths[s] - n + i of the scene, row r % page_rows of the page
// that its table names; keys (and the queries, which go to an output of their own) are turned as by rotary.hip.
// Bytes bound it: each head is read and written once, in one launch.  A workgroup takes a few tokens: one wave
// finds their rows, a lane each, while the others form the angles; both serve all heads from LDS.
//
// 20,000 tokens in 7 scenes, 8 + 8 + 8 heads of 64, bfloat16 (123 MB): 29.6 us, 4.2 TB/s; 65,537 in 190, 12 + 4 + 4 heads
// of 40, 18 pairs, interleaved, float32 (421 MB): 87.0 us, 4.8 TB/s, what a large copy reaches.  One token for each
// of 16 scenes: 7.8 us a call, the host's; the kernel takes 5, its chain of loads (lengths, table, tokens).
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
    int token_items, head_items, value_items;  // parts of a token, of one of its turned heads, of one of its values
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
        uint32_t step = 1;  // (scenes may be near 2^31: s + step is formed where it is one)
        const auto takes = [&] { return step < (uint32_t)(a.scenes - s) && start_of(a, s + (int)step) <= t; };
        while (takes()) s += (int)step, step *= 2;
        for (; step > 1;) {
            step /= 2;
            if (takes()) s += (int)step;
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

// cos and sin of a token's angle for one pair, by the steps of rotary.hip: both give the same bits.  The angle
// in binary64, brought into -pi .. pi there: a binary32 product would lose 2^-24 of an angle of some hundred
// radians.
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

// A thread's part of each token: two runs of one head's channels, both turned or both passed through.  It is
// found once, and then the same for all of the workgroup's tokens: found anew for each, its divisions took more
// time than the bytes.  Two runs always (the second may be the first again, where a row's runs are odd in number),
// so that no load stands behind a branch: there the compiler waits for those before it.
//   not interleaved: RUN pairs, channels first .. and second = first + pairs ..; interleaved: RUN / 2 pairs each.
template <typename T, int RUN> struct Part {
    const T *in;  // of token 0 of the array
    T *out;       // of token 0 of q_out, or of page 0's first row
    int64_t in_row, out_page, out_row;
    int first, second;
    bool q, turns;
};
template <typename T, int RUN, bool INTERLEAVED> __device__ __forceinline__ Part<T, RUN> part_of(const AppendArgs &a, int j) {
    Part<T, RUN> p;
    const int all = (a.heads + a.kv_heads) * a.head_items;
    int runs = a.dim / RUN, from = 0, i, h;  // the runs that are taken two by two, from a channel on
    if (j >= all) {
        h = fastdiv(j - all, a.by_value), i = j - all - h * a.value_items;
        p.in = static_cast<const T *>(a.v) + h * a.v_head, p.in_row = a.v_row;
        p.out = static_cast<T *>(a.v_pool) + h * a.vp_head, p.out_page = a.vp_page, p.out_row = a.vp_row;
        p.q = p.turns = false;
    } else {
        h = fastdiv(j, a.by_items), i = j - h * a.head_items;
        p.q = h < a.heads;
        if (p.q) {
            p.in = static_cast<const T *>(a.q) + h * a.q_head, p.in_row = a.q_row;
            p.out = static_cast<T *>(a.q_out) + (int64_t)h * a.dim, p.out_page = 0, p.out_row = (int64_t)a.heads * a.dim;
        } else {
            h -= a.heads;
            p.in = static_cast<const T *>(a.k) + h * a.k_head, p.in_row = a.k_row;
            p.out = static_cast<T *>(a.k_pool) + h * a.kp_head, p.out_page = a.kp_page, p.out_row = a.kp_row;
        }
        const int turning = INTERLEAVED ? (2 * a.pairs / RUN + 1) / 2 : a.pairs / RUN;
        p.turns = i < turning;
        if (p.turns && !INTERLEAVED) {
            p.first = i * RUN, p.second = a.pairs + i * RUN;
            return p;
        }
        if (p.turns) runs = 2 * a.pairs / RUN;
        else i -= turning, from = 2 * a.pairs, runs -= from / RUN;
    }
    const int half = (runs + 1) / 2;
    p.first = from + i * RUN, p.second = i + half < runs ? p.first + half * RUN : p.first;
    return p;
}

// Tokens of a thread that are loaded at once (the first ones before their rows and angles are known), and all that it
// takes, over which the chains of loads at a workgroup's start spread.  The cases above: 29.6 and 87.0 us; with 8 tokens
// 29.7 and 92.0, with 4 at once 31.4 and 87.6, one at a time 32.0 and 90.7.
constexpr int kDeep = 2, kTokens = 4;

// A run as it lies in memory: words, which are loaded and stored in one piece (of a struct of bfloat16 the compiler
// makes loads of two and four bytes).
template <int BYTES> struct Words {
    typedef uint32_t type __attribute__((ext_vector_type(BYTES / 4)));
};
template <> struct Words<4> { typedef uint32_t type; };
template <> struct Words<2> { typedef uint16_t type; };

template <typename T, int RUN, bool INTERLEAVED>
__global__ __launch_bounds__(256) void k_paged_append(const AppendArgs a) {
    typedef typename Words<RUN * sizeof(T)>::type Run;
    typedef Pack<T, RUN> Values;
    extern __shared__ float2 turns[];  // cos, sin of block_tokens x pairs
    __shared__ Target target[64];
    const int t0 = blockIdx.x * a.block_tokens, nt = min(a.block_tokens, a.tokens - t0);
    // a thread's first part and token: as many tokens side by side as have room
    const int side = max(256 / a.token_items, 1);
    const int first_t = side > 1 ? fastdiv(threadIdx.x, a.by_token) : 0, first_j = threadIdx.x - first_t * a.token_items;
    bool begun = false;
    for (int j = first_j; j - first_j < a.token_items; j += 256) {
        const bool has = first_t < side && j < a.token_items;
        const Part<T, RUN> p = part_of<T, RUN, INTERLEAVED>(a, has ? j : 0);
        for (int tb = 0; tb < nt; tb += side * kDeep) {
            Run x[kDeep], z[kDeep];
#pragma unroll
            for (int k = 0; k < kDeep; ++k) {
                const T *in = p.in + (t0 + min(tb + k * side + first_t, nt - 1)) * p.in_row;
                x[k] = *reinterpret_cast<const Run *>(in + p.first);
                z[k] = *reinterpret_cast<const Run *>(in + p.second);
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
                if (p.turns) {
                    const float2 *w = turns + t * a.pairs;
                    Values u = __builtin_bit_cast(Values, x[k]), v = __builtin_bit_cast(Values, z[k]);
                    if constexpr (INTERLEAVED) {
#pragma unroll
                        for (int e = 0; e < RUN; e += 2) {
                            const float2 y = turned((float)u.v[e], (float)u.v[e + 1], w[(p.first + e) / 2]);
                            u.v[e] = (T)y.x, u.v[e + 1] = (T)y.y;
                            const float2 s = turned((float)v.v[e], (float)v.v[e + 1], w[(p.second + e) / 2]);
                            v.v[e] = (T)s.x, v.v[e + 1] = (T)s.y;
                        }
                    } else {
#pragma unroll
                        for (int e = 0; e < RUN; ++e) {
                            const float2 y = turned((float)u.v[e], (float)v.v[e], w[p.first + e]);
                            u.v[e] = (T)y.x, v.v[e] = (T)y.y;
                        }
                    }
                    x[k] = __builtin_bit_cast(Run, u), z[k] = __builtin_bit_cast(Run, v);
                }
                T *out = p.out + to.page * p.out_page + to.row * p.out_row;
                *reinterpret_cast<Run *>(out + p.first) = x[k];
                *reinterpret_cast<Run *>(out + p.second) = z[k];
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

template <typename T, bool INTERLEAVED> void launch_append(const AppendArgs &a, int run, hipStream_t s) {
    const dim3 grid((a.tokens + a.block_tokens - 1) / a.block_tokens), block(256);
    const size_t lds = sizeof(float2) * a.block_tokens * a.pairs;
    if constexpr (sizeof(T) == 2)
        if (run == 8) {
            hipLaunchKernelGGL((k_paged_append<T, 8, INTERLEAVED>), grid, block, lds, s, a);
            return;
        }
    if (run == 4) hipLaunchKernelGGL((k_paged_append<T, 4, INTERLEAVED>), grid, block, lds, s, a);
    else if (run == 2) hipLaunchKernelGGL((k_paged_append<T, 2, INTERLEAVED>), grid, block, lds, s, a);
    else if constexpr (!INTERLEAVED) hipLaunchKernelGGL((k_paged_append<T, 1, INTERLEAVED>), grid, block, lds, s, a);
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
    const int run = (int)((low & (0 - low)) / size);  // (2 at least where interleaved: rows and pairs are even)
    const auto twos = [&](int runs) { return (runs + 1) / 2; };
    const int items = (r->interleaved ? twos(2 * r->pairs / run) : r->pairs / run) + twos((r->dim - 2 * r->pairs) / run);
    const int values = twos(r->dim / run);
    // Tokens of a workgroup: as many as its threads take, fewer where the launch would leave CUs idle; their
    // angles within 16 KB of LDS, a lane for each.
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
                       p->page_rows, (int)rows, (int)bt, (int)each, items, values, make_fastdiv(p->page_rows),
                       make_fastdiv(r->pairs ? r->pairs : 1), make_fastdiv(each), make_fastdiv(items),
                       make_fastdiv(values)};
    hipStream_t s = as_stream(stream);
    if (r->dtype == GSV_BF16)
        r->interleaved ? launch_append<bf16, true>(a, run, s) : launch_append<bf16, false>(a, run, s);
    else
        r->interleaved ? launch_append<float, true>(a, run, s) : launch_append<float, false>(a, run, s);
    return check_launch();
}
