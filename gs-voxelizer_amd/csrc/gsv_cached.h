// gsv_cached.h — the kernel of one query token a scene against a cache of keys and values, whose rows
// lie together (attention_cached.hip) or in pages that a table names (attention_paged.hip).
//
// Same scores as attention_fwd.hip.  The bytes of the cache are the floor: each is read
// once, by coalesced 16-byte loads, and serves all query heads of its key head, which
// are the columns of a matrix product (32, those past the group idle: the matrix units
// have an order of magnitude to spare here).  A cache is split over workgroups, a split over
// four waves that never wait for each other; a second kernel joins the splits.
#pragma once

#include "gsv_attention.h"

// (a product and a difference stay two roundings where they are written as two)
#pragma clang fp contract(off)

namespace gsv {
namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr int kKeys = 32;   // keys of a wave's step
constexpr int kHeads = 32;  // query heads of a workgroup
constexpr float kSlack = 8.f;
constexpr int kPageUnit = 16;  // a page holds a multiple of so many rows: a copy never leaves one

struct CacheArgs {
    const int *lengths;
    // strides from scene to scene, or from page to page
    int64_t k_scene, v_scene, k_pos_scene, keep_scene;
    int splits, head_tiles;  // splits: of each scene; of paged scenes, 1 where none is split
    float *part_o;   // (scenes, heads, splits, dim) or (parts, heads, dim): sums of weights times values
    float2 *part_ms; // the same but the channels: maximum (log2) and sum of weights
    // paged: scene s's row j is row j % page_rows of page table[s table_row + j / page_rows]
    const int *table;
    int64_t table_row;
    int pages, page_rows;
    FastDiv by_rows;
    int2 *parts;  // of each scene: its first part, and how many it has
    int shares;   // workgroups of a key head
};

// How rows lie, and what a workgroup takes of them: a cache's rows together, an equal split of one; rows in
// pages, a piece of one scene, or an equal share of all scenes' steps.
enum Rows { kTogether, kPieces, kShares };

// What a workgroup takes of the paged scenes: `steps` from step `begin` of scene s on; s < 0: nothing.
struct Share {
    int s, begin, steps, most;  // most: of any workgroup
};
__device__ __forceinline__ int live_rows(const AttnArgs &a, const CacheArgs &c, int s) {
    return s < a.scenes ? min(max(c.lengths[s], 0), a.k_tokens) : 0;
}
// (an empty scene has a step, which writes its zeros)
__device__ __forceinline__ int steps_of(int len) { return len > 0 ? (len - 1) / kKeys + 1 : 1; }

// The scenes' lengths are known on the device alone, so each workgroup cuts the batch for itself.  A lane takes a
// run of scenes: up to 64 take one load and a scan over the lanes.
//   kPieces (few scenes): pieces of one scene each, of the least size with which all of them fit one round of
//     workgroups; `shares` of them do with steps / (shares - scenes) each.  Scene s's parts are its pieces.
//   kShares: one scene after the other, cut in equal shares, which go on from a scene into the next.  However
//     the lengths differ all workgroups end together, but one that has two scenes' keys starts twice.
//     The part of scene s that workgroup n has is number n + s: a scene's parts are neighbours, and
//     no two have one number.
// 16 caches of 4,096, 2 key heads of 64 (step of 16 scenes): 16.6 us in pieces, 20.7 in shares; 20 of 8,000, 4 of 128
// 53.5 and 57.4; 90 of 2,000 68.4 and 59.6; 100 of 3,000, 8 of 64 92.4 and 83.3.
template <int W, int ROWS> __device__ __forceinline__ Share share_of(const AttnArgs &a, const CacheArgs &c, int n) {
    if (c.splits == 1) {
        const int all = __builtin_amdgcn_readfirstlane(steps_of(live_rows(a, c, n)));
        return {n, 0, all, all};
    }
    const int lane = threadIdx.x & 63, each = (a.scenes + 63) / 64;
    const auto sum = [&](const auto &of) {  // of a lane's scenes
        int64_t x = 0;
        for (int i = 0; i < each; ++i)
            if (lane * each + i < a.scenes) x += of(steps_of(live_rows(a, c, lane * each + i)));
        return x;
    };
    const auto scan = [&](int64_t x) {  // over the lanes
#pragma unroll
        for (int k = 1; k < 64; k <<= 1) {
            const int64_t y = __shfl_up(x, k);
            if (lane >= k) x += y;
        }
        return x;
    };
    int64_t mine = sum([](int steps) { return steps; }), last = scan(mine);
    const int64_t all = __shfl(last, 63);
    // (a scene has less than 2^26 steps)
    int most = (int)imin64(imax64((all + c.shares - 1) / c.shares, W), INT32_MAX);
    int64_t from = (int64_t)n * most;
    if constexpr (ROWS == kPieces) {
        int high = (int)imin64(imax64(all / (c.shares - a.scenes) + 1, most), INT32_MAX);
        while (most < high) {
            const int mid = most + (high - most) / 2;
            const float count = wave_sum((float)sum([&](int steps) { return (steps - 1) / mid + 1; }));
            if (count <= (float)c.shares) high = mid;  // (less than 2^11: exact)
            else most = mid + 1;
        }
        most = __builtin_amdgcn_readfirstlane(most);
        mine = sum([&](int steps) { return (steps - 1) / most + 1; }), last = scan(mine);
        from = n;
    }
    const uint64_t past = __ballot(last > from);
    if (!past) return {-1, 0, 0, 0};
    const int holder = __builtin_amdgcn_readfirstlane((int)__builtin_ctzll(past));
    int steps = (int)imin64(most, all - from);
    from -= __shfl(last - mine, holder);
    int s = holder * each, own = 0;
    for (int i = 0; i < each; ++i, ++s) {  // among the holder's scenes
        own = steps_of(live_rows(a, c, s));
        const int has = ROWS == kPieces ? (own - 1) / most + 1 : own;
        if (from < has || i + 1 == each) break;
        from -= has;
    }
    if (ROWS == kPieces) from *= most, steps = min(most, own - (int)from);
    return {__builtin_amdgcn_readfirstlane(s), __builtin_amdgcn_readfirstlane((int)from),
            __builtin_amdgcn_readfirstlane(steps), __builtin_amdgcn_readfirstlane(most)};
}

// Waves of a workgroup: four, two where their tiles would pass the LDS of a CU.
template <typename T, int DP, int ROWS>
constexpr int kWaves = ROWS ? 512 / (DP * sizeof(T) < 128 ? 128 : DP * sizeof(T)) : DP * sizeof(T) > 256 ? 2 : 4;

// bfloat16 weights enter the product with the values in two parts: the results are as exact as their type
// (0.0017 in the 2-norm, in one part 0.0018 to 0.0020), for 0 to 4 % of the time beside the cache's bytes.
template <typename T> constexpr int kParts = sizeof(T) == 2 ? 2 : 1;

template <typename T, int DP, bool FAR, int CAP, int ROWS>
__global__ __launch_bounds__((64 * kWaves<T, DP, ROWS>)) void k_attention_cached(const AttnArgs a, const CacheArgs c,
                                                          T *__restrict__ out) {
    typedef typename Elem<T>::frag frag;
    constexpr int W = kWaves<T, DP, ROWS>;
    constexpr bool PAGED = ROWS != kTogether;
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
    int s, j_begin, j_end;
    bool whole;    // all of the scene's keys: the result goes to out
    int64_t part;  // else to this row, plus the head
    Share share;
    if constexpr (PAGED) {
        share = share_of<W, ROWS>(a, c, n);
        if (share.s < 0) return;
    }
    while (true) {
    if constexpr (PAGED) {
        s = share.s;
        const int len = __builtin_amdgcn_readfirstlane(live_rows(a, c, s));
        const int all = steps_of(len), take = min(all - share.begin, share.steps);
        j_begin = share.begin * kKeys, j_end = take < all - share.begin ? j_begin + take * kKeys : len;
        whole = share.begin == 0 && take == all;
        const int64_t number = (int64_t)n + (ROWS == kShares ? s : 0);
        part = number * a.heads;
        if (c.splits > 1 && share.begin == 0 && hk == 0 && ht == 0 && threadIdx.x == 0)
            c.parts[s] = make_int2((int)number, 1 + (all - take + share.most - 1) / share.most);
        share.steps -= take, share.begin = 0, ++share.s;
    } else {
        const int split = n % c.splits;
        s = n / c.splits;
        const int len = min(max(c.lengths[s], 0), a.k_tokens);
        const int per = ((len + c.splits - 1) / c.splits + kKeys - 1) / kKeys * kKeys;
        j_begin = min((int64_t)split * per, (int64_t)len), j_end = min(j_begin + per, len);
        whole = c.splits == 1;
        part = (int64_t)s * a.heads * c.splits + split;
    }
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
    const T *kbase = static_cast<const T *>(a.k) + (PAGED ? 0 : s * c.k_scene) + hk * a.k_head;
    const T *vbase = static_cast<const T *>(a.v) + (PAGED ? 0 : s * c.v_scene) + hk * a.v_head;
    T *const sk = tiles[wave], *const sv = sk + 2 * kKeys * DP;
    Tile<T, DP> at;
    at.plan(lane);
    // what one copy fills: a step's keys, or those of it in one page
    constexpr int kGroup = PAGED ? kPageUnit : kKeys, kGroups = kKeys / kGroup;
    Copy<T, DP, kGroup, 1> ck, cv;
    ck.plan(a.k_row, a.dim, 0, lane);
    cv.plan(a.v_row, a.dim, 0, lane);
    f32x16 o[DP / 32] = {};
    float m = -INFINITY, sum = 0.f;
    float gp[2] = {};
    int raw = 0;
    uint32_t live = ~0u, next_live = ~0u;
    const int step = W * kKeys;
    // paged: the pages of 32 of this wave's steps (two groups each), a lane each, and of the next 32;
    // of the step that is fetched next, each group's page (below 0: none) and its first row in it
    int ids = 0, next_ids = 0, page[kGroups], at_row[kGroups];
    auto entries = [&](int j0) {
        const int row = min(j0 + (lane >> 1) * step + (lane & 1) * kPageUnit, j_end - 1);
        return c.table[s * c.table_row + fastdiv(row, c.by_rows)];
    };
    auto look = [&](int j0) {
        if constexpr (PAGED) {
            const int first = j_begin + wave * kKeys, n = (j0 - first) / step;
            if ((n & 31) == 0 && n) ids = next_ids;
            if ((n & 31) == 16) next_ids = entries(j0 + 16 * step);
#pragma unroll
            for (int g = 0; g < kGroups; ++g) {
                const int row = j0 + g * kPageUnit;
                page[g] = __builtin_amdgcn_readlane(ids, (n & 31) * 2 + g);
                if (page[g] >= c.pages || row >= j_end) page[g] = -1;
                at_row[g] = row - fastdiv(min(row, j_end - 1), c.by_rows) * c.page_rows;
            }
        }
        if (a.keep && j0 < j_end) {
            if constexpr (PAGED) {
                const int r = min(lane & 31, j_end - 1 - j0), g = r / kPageUnit;
                const int p = g ? page[1 % kGroups] : page[0], first = g ? at_row[1 % kGroups] : at_row[0];
                raw = p < 0 ? 0 : keep_raw(a, p * c.keep_scene + first + r % kPageUnit);
            } else {
                raw = keep_raw(a, s * c.keep_scene + min(j0 + (lane & 31), j_end - 1));
            }
        }
    };
    auto fetch = [&](int b, int j0) {
        if (a.keep) next_live = (uint32_t)__ballot(raw != 0);
        if constexpr (PAGED) {
            const int left = j_end - j0;
            if (!a.keep) next_live = ~0u;
#pragma unroll
            for (int g = 0; g < kGroups; ++g) {
                // rows of a page that is none are not there
                const int rows = page[g] < 0 ? 0 : left - g * kPageUnit;
                if (page[g] < 0) next_live &= ~(0xffffu << (g * kPageUnit));
                const int64_t p = max(page[g], 0);
                ck.template start<true>(sk + (b * kKeys + g * kPageUnit) * DP, kbase + p * c.k_scene + at_row[g] * a.k_row, a.k_row,
                         a.dim, rows, a.keep, next_live >> (g * kPageUnit), 0, lane);
                cv.template start<true>(sv + (b * kKeys + g * kPageUnit) * DP, vbase + p * c.v_scene + at_row[g] * a.v_row, a.v_row,
                         a.dim, rows, a.keep, next_live >> (g * kPageUnit), 0, lane);
            }
            if (far)
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const int r = min((i * 64 + lane) % kKeys, left - 1), ax = min((i * 64 + lane) / kKeys, 2);
                    const int g = r / kPageUnit, p = g ? page[1 % kGroups] : page[0];
                    const int first = g ? at_row[1 % kGroups] : at_row[0];
                    gp[i] = p < 0 ? 0.f : a.k_pos[p * c.k_pos_scene + (first + r % kPageUnit) * a.k_pos_row + ax];
                }
            look(j0 + step);
        } else {
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
        if constexpr (PAGED) ids = entries(j_begin + wave * kKeys);
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
        if (whole) {
            out[((int64_t)s * a.heads + hh) * a.dim + dd] = (T)(total == 0.f ? 0.f : val / total);
        } else {
            const int64_t at = part + (int64_t)hh * (PAGED ? 1 : c.splits);
            c.part_o[at * a.dim + dd] = val;
            if (dd == 0) c.part_ms[at] = make_float2(top, total);
        }
    }
    if (ROWS != kShares || share.steps <= 0 || share.s >= a.scenes) return;
    __syncthreads();  // the next scene's copies go where the sums lay
    }
}

// The row of one scene and head from its `splits` parts, rows first, first + step .. of the workspace: the
// W waves take them in turn, then their sums are joined, always in the same order.
template <typename T, int W>
__device__ __forceinline__ void join_row(const float *__restrict__ part_o, const float2 *__restrict__ part_ms,
                                         int64_t first, int64_t step, int splits, int dim, T *__restrict__ out) {
    __shared__ float so[W][128], ss[W];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const float2 *ms = part_ms + first;
    float top = -INFINITY;
    for (int p = lane; p < splits; p += 64) top = fmaxf(top, ms[p * step].x);
#pragma unroll
    for (int k = 1; k < 64; k <<= 1) top = fmaxf(top, __shfl_xor(top, k));
    float total = 0.f, v0 = 0.f, v1 = 0.f;
    const int d0 = min(lane, dim - 1), d1 = min(lane + 64, dim - 1);
#pragma unroll 4
    for (int p = wave; p < splits; p += W) {
        const float2 e = ms[p * step];
        const float by = e.x == -INFINITY ? 1.f : fast_exp2(e.x - top);
        total = fmaf(by, e.y, total);
        const float *o = part_o + (first + p * step) * dim;
        v0 = fmaf(by, o[d0], v0);
        v1 = fmaf(by, o[d1], v1);
    }
    so[wave][lane] = v0, so[wave][64 + lane] = v1;
    if (lane == 0) ss[wave] = total;
    __syncthreads();
    if (threadIdx.x >= (unsigned)dim) return;
    const int d = threadIdx.x;
    total = ss[0];
    float v = so[0][d];
#pragma unroll
    for (int w = 1; w < W; ++w) total += ss[w], v += so[w][d];
    out[d] = (T)(total == 0.f ? 0.f : v / total);
}

}  // namespace
}  // namespace gsv
