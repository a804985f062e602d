// attention_paged.hip — one query token a scene against a cache whose rows lie in pages.
//
// Same scores as attention_fwd.hip.  The bytes of the cache are the floor: each is read once, by asynchronous
// 16-byte copies to LDS, and serves all query heads of its key head, which are the columns of a matrix product
// (16; a group of more takes several workgroups, neighbours on one XCD).  A wave takes steps of 32
// keys (float32 16), never waits for the others, and copies the next step while it works on one.
//   * A page holds a multiple of 16 rows, so 16 rows of a step have one page, and a buffer descriptor at its first
//     row.  The table's entries for 32 steps are one load, a lane each, made 16 steps ahead.
//   * Scenes differ in length, and their lengths are known on the device alone: every workgroup cuts the batch for
//     itself and takes its own part (share_of).  A second kernel joins the parts of a scene.
//
// Products run on v_mfma_f32_16x16x32_bf16, or v_mfma_f32_16x16x4_f32.  Lane l of a wave holds, of the left
// operand, row l % 16 and of the right one column l % 16, both with the contraction's indices of l / 16; of
// the result, column l % 16 and rows 4 (l / 16) + r, r = 0 .. 3.  A sum does not depend on which index is called
// which: scores come out with a lane's keys 4 (l / 16) + r (and 16 more), which are the right operand of the product
// with the values, in that order, straight from the registers.
//
// 2 caches of 200,003 rows, 16 heads on 4 of 128, bfloat16, capped, bias, pages of 256 (316 MB of live rows): 64.5 us,
// 4.9 TB/s, and 4.8 for the join; 128 of 2,000, 8 on 8 of 64 (350 MB) 74.4 us, 4.7 TB/s; 5 of 20,000, 12 on 4 of 40, float32 (66 MB)
// 20.6 us.  Bytes bound these: each is read once (counters), vector units are at work 15 to 20 % of the time, matrix units
// 1 to 20 %.  The last one's calls take 12 us (the start, the join) and their bytes at 5.3 TB/s, from 5 to 774 MB.  16 of 4,096, 8 on 2 of 64 (23 MB): 10.8 us and 3.6; there the chain from the launch to the first bytes
// (lengths, table, keys) and a wave's two steps bound it.
#include "gsv_attention.h"

// (a product and a difference stay two roundings where they are written as two)
#pragma clang fp contract(off)

namespace gsv {
namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kSlack = 8.f;
constexpr int kHeads = 16;     // query heads of a workgroup
constexpr int kPageUnit = 16;  // a page holds a multiple of so many rows: a copy never leaves one

// A wave's step, and the waves of a workgroup: two workgroups fit a CU (LDS), so that one starts while another works.
// 40 scenes of 4,000, 4 heads of 128: 46.8 us, with twice the waves 52.3 (2 of 200,003, long pieces only: 70.0 and 68.7).
template <typename T> constexpr int kKeys = sizeof(T) == 2 ? 32 : 16;
template <int DP> constexpr int kWaves = DP == 128 ? 2 : 4;

// bfloat16 weights enter the product with the values in two parts: the results are as exact as their type
// (0.0017 in the 2-norm, in one part 0.0018 to 0.0020).
template <typename T> constexpr int kParts = sizeof(T) == 2 ? 2 : 1;

struct PageArgs {
    const int *lengths, *table;
    int64_t table_row, k_page, v_page, pos_page, keep_page;
    int pages, page_rows;
    FastDiv by_rows;
    int head_tiles, split;  // split: whether scenes are cut
    int near;               // key heads that run side by side on one XCD
    int shares;             // workgroups of a key head and head tile
    float *part_o;          // (parts, heads, dim): sums of weights times values
    float2 *part_ms;        // (parts, heads): maximum (log2) and sum of weights
    int2 *parts;            // of each scene: its first part, and how many it has
};

__device__ __forceinline__ f32x4 mma16(bf16x8 a, bf16x8 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mma16(f32x4 a, f32x4 b, f32x4 c) {
#pragma unroll
    for (int e = 0; e < 4; ++e) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[e], b[e], c, 0, 0, 0);
    return c;
}
template <typename T> struct Operand;
template <> struct Operand<bf16> { typedef bf16x8 frag; };
template <> struct Operand<float> { typedef f32x4 frag; };

// A lane's parts of a tile (gsv_attention.h: rows of DP elements, chunk c of row r at place c ^ turn(r)).
template <typename T, int DP> struct Tile16 {
    typedef Tile<T, DP> Base;
    typedef typename Operand<T>::frag frag;
    static constexpr int kDepth = 4 * Elem<T>::kChunk;  // channels of one operand of the scores
    uint32_t row_at, col_at;
    __device__ __forceinline__ void plan(int lane) {
        const int r = lane & 15, g = lane >> 4;
        row_at = r * Base::kRowBytes + ((g ^ Base::turn(r)) << 4);
        const int r4 = 4 * g + (sizeof(T) == 2 ? r >> 2 : 0);
        col_at = sizeof(T) == 2 ? r4 * Base::kRowBytes + ((((r & 3) >> 1) ^ Base::turn(r4)) << 4) + (r & 1) * 8
                                : r4 * Base::kRowBytes + (((r >> 2) ^ Base::turn(r4)) << 4) + (r & 3) * 4;
    }
    // Channels kDepth st .. of 16 rows, from row 16 `tile` on.
    __device__ __forceinline__ frag rows(const T *t, int tile, int st) const {
        return Base::template read<frag>(((Base::base(t) + row_at) ^ (st << 6)) + tile * 16 * Base::kRowBytes);
    }
    // The transposed left operand of the values: channel 16 block + lane % 16 of rows 4 (lane / 16) .. + 3, and
    // for 16-bit elements of those 16 rows on.  There ds_read_b64_tr_b16 does it: of 16 lanes, lane i gives the
    // address of row i / 4, columns 4 (i % 4) .. + 3, and receives column i of the four rows.
    __device__ __forceinline__ frag columns(const T *t, int block) const {
        const uint32_t first = Base::base(t);
        if constexpr (sizeof(T) == 2) {
            typedef __attribute__((address_space(3))) s16x4 *lds_ptr;
            const uint32_t at = (first + col_at) ^ (block << 5);
            const s16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr)(uintptr_t)at);
            const s16x4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr)(uintptr_t)(at + 16 * Base::kRowBytes));
            const bf16x4 u = __builtin_bit_cast(bf16x4, a), v = __builtin_bit_cast(bf16x4, b);
            return bf16x8{u[0], u[1], u[2], u[3], v[0], v[1], v[2], v[3]};
        } else {
            // rows 4 g + e: turn differs by the row's low two bits
            f32x4 f;
#pragma unroll
            for (int e = 0; e < 4; ++e)
                f[e] = Base::template read<float>(
                    ((first + col_at) ^ ((4 * block) ^ (Base::turn(e) ^ Base::turn(0))) << 4) + e * Base::kRowBytes);
            return f;
        }
    }
};

// Inclusive sums over the lanes, by DPP: inside rows of 16, then their last lanes'.
__device__ __forceinline__ int wave_scan(int x) {
#define GSV_DPP_SCAN(ctrl, rows) x += __builtin_amdgcn_update_dpp(0, x, ctrl, rows, 0xf, true)
    GSV_DPP_SCAN(0x111, 0xf);  // row_shr 1, 2, 4, 8
    GSV_DPP_SCAN(0x112, 0xf);
    GSV_DPP_SCAN(0x114, 0xf);
    GSV_DPP_SCAN(0x118, 0xf);
    GSV_DPP_SCAN(0x142, 0xa);  // row_bcast 15: into rows 1 and 3
    GSV_DPP_SCAN(0x143, 0xc);  // row_bcast 31: into rows 2 and 3
#undef GSV_DPP_SCAN
    return x;
}
__device__ __forceinline__ int64_t wave_scan(int64_t x) {
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int k = 1; k < 64; k <<= 1) {
        const int64_t y = __shfl_up(x, k);
        if (lane >= k) x += y;
    }
    return x;
}

// What a workgroup takes of the scenes: `steps` from step `begin` of scene s on; s < 0: nothing.
struct Share {
    int s, begin, steps, most;  // most: of any workgroup
    int len;                    // rows of scene s
};
__device__ __forceinline__ int live_rows(const AttnArgs &a, const PageArgs &c, int s) {
    return s < a.scenes ? min(max(c.lengths[s], 0), a.k_tokens) : 0;
}
// (an empty scene has a step, which writes its zeros)
template <typename T> __device__ __forceinline__ int steps_of(int len) { return len > 0 ? (len - 1) / kKeys<T> + 1 : 1; }

// How a batch is cut.  Every workgroup does it for itself; a lane takes a run of scenes, so that up to 64 take one
// load and scans over the lanes.
//   kPieces (few scenes): pieces of one scene each, of the least size with which all of them fit one round of
//     workgroups (steps / (shares - scenes) do).  Scene s's parts are its pieces.
//   kShares: one scene after the other, cut in equal shares, which go on from a scene into the next.  However
//     the lengths differ all workgroups end together, but one that has two scenes' keys starts twice.
//     The part of scene s that workgroup n has is number n + s: a scene's parts are neighbours, and
//     no two have one number.
enum Cut { kPieces, kShares };
template <typename T, int W, Cut CUT> __device__ __forceinline__ Share share_of(const AttnArgs &a, const PageArgs &c, int n) {
    if (!c.split) {
        const int len = __builtin_amdgcn_readfirstlane(live_rows(a, c, n)), all = steps_of<T>(len);
        return {n, 0, all, all, len};
    }
    const int lane = threadIdx.x & 63, each = (a.scenes + 63) / 64;
    const int first = lane * each, behind = min(first + each, a.scenes);
    // the first (up to 64 scenes: the only) one's rows stay in a register: each further look at a length is a load
    const int len = live_rows(a, c, first);
    const auto sum = [&](auto x, const auto &of) {  // of a lane's scenes
        if (first < behind) x += of(steps_of<T>(len));
        for (int s = first + 1; s < behind; ++s) x += of(steps_of<T>(live_rows(a, c, s)));
        return x;
    };
    int holder, most, begin, steps;
    if constexpr (CUT == kPieces) {
        // (raised by more than what the sums of floats may have lost)
        const float all = wave_sum(sum(0.f, [](int steps) { return (float)steps; })) * 1.00002f;
        most = max((int)fminf(all / (float)c.shares, 1e9f), W);
        int high = max((int)fminf(all / (float)(c.shares - a.scenes), 1e9f) + 1, most);
        while (most < high) {
            const int mid = most + (high - most) / 2;
            const float count = wave_sum((float)sum(0, [&](int steps) { return (steps - 1) / mid + 1; }));
            if (count <= (float)c.shares) high = mid;  // (less than 2^12: exact)
            else most = mid + 1;
        }
        most = __builtin_amdgcn_readfirstlane(most);
        const int own = sum(0, [&](int steps) { return (steps - 1) / most + 1; }), last = wave_scan(own);
        const uint64_t past = __ballot(last > n);
        if (!past) return {-1, 0, 0, 0, 0};
        holder = __builtin_amdgcn_readfirstlane((int)__builtin_ctzll(past));
        begin = n - __builtin_amdgcn_readlane(last - own, holder);
        steps = most;
    } else {
        const int64_t own = sum((int64_t)0, [](int steps) { return steps; });
        const int64_t last = wave_scan(own), all = __shfl(last, 63);
        // (a scene has less than 2^27 steps)
        most = (int)imin64(imax64((all + c.shares - 1) / c.shares, W), INT32_MAX);
        const int64_t from = (int64_t)n * most;
        const uint64_t past = __ballot(last > from);
        if (!past) return {-1, 0, 0, 0, 0};
        holder = __builtin_amdgcn_readfirstlane((int)__builtin_ctzll(past));
        steps = (int)imin64(most, all - from);
        int64_t skip = from - __shfl(last - own, holder);
        // among the holder's scenes; what is left then lies in one scene
        int s = holder * each, rows = __builtin_amdgcn_readlane(len, holder);
        for (int i = 1; i < each && skip >= steps_of<T>(rows); ++i) {
            skip -= steps_of<T>(rows);
            rows = __builtin_amdgcn_readfirstlane(live_rows(a, c, ++s));
        }
        return {__builtin_amdgcn_readfirstlane(s), __builtin_amdgcn_readfirstlane((int)imin64(skip, INT32_MAX / kKeys<T>)),
                __builtin_amdgcn_readfirstlane(steps), __builtin_amdgcn_readfirstlane(most), __builtin_amdgcn_readfirstlane(rows)};
    }
    int s = holder * each, rows = __builtin_amdgcn_readlane(len, holder);
    for (int i = 1; i < each && begin >= (steps_of<T>(rows) - 1) / most + 1; ++i) {
        begin -= (steps_of<T>(rows) - 1) / most + 1;
        rows = __builtin_amdgcn_readfirstlane(live_rows(a, c, ++s));
    }
    return {__builtin_amdgcn_readfirstlane(s), __builtin_amdgcn_readfirstlane(begin * most), steps, most,
            __builtin_amdgcn_readfirstlane(rows)};
}

template <typename T, int DP, bool FAR, int CAP, Cut CUT>
__global__ __launch_bounds__((64 * kWaves<DP>)) void k_attention_paged(const AttnArgs a, const PageArgs c,
                                                                      T *__restrict__ out) {
    typedef Tile16<T, DP> Part;
    typedef typename Part::frag frag;
    constexpr int W = kWaves<DP>, KEYS = kKeys<T>, TILES = KEYS / 16, DEPTH = DP / Part::kDepth, BLOCKS = DP / 16;
    constexpr int kRow = DP + 4;  // of the sums in LDS: 16 rows lie in different banks
    static_assert(4 * KEYS * DP * sizeof(T) >= kHeads * kRow * sizeof(float), "sums reuse the tiles");
    __shared__ __align__(1024) T tiles[W][4 * KEYS * DP];  // a wave's keys and values, two buffers
    __shared__ __align__(16) float spos[W][2][3 * KEYS];
    __shared__ float sm[W][kHeads], ss[W][kHeads];

    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int g4 = 4 * (lane >> 4);  // a lane's keys of a tile, and channels of a block, are g4 .. g4 + 3
    const int group = a.heads / a.kv_heads;
    // those that read the same lines of memory (near): eight workgroups apart, on one XCD
    int n = blockIdx.x / kXcds;
    const int ht = n % c.head_tiles;
    n /= c.head_tiles;
    int hk = n % c.near;
    n = n / c.near * kXcds + blockIdx.x % kXcds;
    const int apart = a.kv_heads / c.near;
    hk += n % apart * c.near, n /= apart;
    if (n >= c.shares) return;
    Share share = share_of<T, W, CUT>(a, c, n);
    if (share.s < 0) return;

    constexpr bool capped = CAP != kNoCap;
    const int col = ht * kHeads + (lane & 15);  // query head within the group
    const bool head = col < group;
    const int h = hk * group + (head ? col : 0);
    const float slope = FAR ? slope_of(a, h) : 0.f;
    const float unit = capped ? kLog2e : a.scale * kLog2e;
    const float far_unit = capped ? slope : slope / a.scale;
    const float in_cap = capped ? a.scale / a.cap : 0.f;
    const T *kbase = static_cast<const T *>(a.k) + hk * a.k_head;
    const T *vbase = static_cast<const T *>(a.v) + hk * a.v_head;
    T *const sk = tiles[wave], *const sv = sk + 2 * KEYS * DP;
    Part at;
    at.plan(lane);
    Copy<T, DP, kPageUnit, 1> ck, cv;
    ck.plan(a.k_row, a.dim, 0, lane);
    cv.plan(a.v_row, a.dim, 0, lane);
    constexpr int step = W * KEYS;

    while (true) {
        const int s = share.s, len = share.len;
        const int all = steps_of<T>(len), take = min(all - share.begin, share.steps);
        const int j_begin = share.begin * KEYS, j_end = take < all - share.begin ? j_begin + take * KEYS : len;
        const bool whole = share.begin == 0 && take == all;
        const int64_t number = (int64_t)n + (CUT == kShares ? s : 0);
        if (c.split && share.begin == 0 && hk == 0 && ht == 0 && threadIdx.x == 0)
            c.parts[s] = make_int2((int)number, 1 + (all - take + share.most - 1) / share.most);
        share.steps -= take, share.begin = 0, ++share.s;
        if (CUT == kShares) share.len = __builtin_amdgcn_readfirstlane(live_rows(a, c, share.s));

        // the pages of 32 of this wave's steps, a lane each, and of the next 32; of the step that is
        // fetched next, each tile's page (below 0: none) and its first row in it
        int ids = 0, next_ids = 0, page[TILES], at_row[TILES];
        const int first = j_begin + wave * KEYS;
        const auto entries = [&](int j0) {
            const int row = TILES == 2 ? j0 + (lane >> 1) * step + (lane & 1) * 16 : j0 + (lane & 31) * step;
            return c.table[s * c.table_row + fastdiv(min(row, j_end - 1), c.by_rows)];
        };
        if (first < j_end) ids = entries(first);
        frag q[DEPTH];
#pragma unroll
        for (int st = 0; st < DEPTH; ++st) {
            const int d = st * Part::kDepth + (lane >> 4) * Elem<T>::kChunk;
            q[st] = {};
            if (head && d < a.dim)
                q[st] = *reinterpret_cast<const frag *>(static_cast<const T *>(a.q) + s * a.q_row + h * a.q_head + d);
        }
        float qx = 0.f, qy = 0.f, qz = 0.f;
        if (FAR) {
            const float *p = a.q_pos + s * a.q_pos_row;
            qx = p[0], qy = p[1], qz = p[2];
        }
        f32x4 o[BLOCKS] = {};
        float m = -INFINITY, sum = 0.f, gp[2] = {};
        int raw = 0;
        uint32_t live = ~0u, next_live = ~0u;
        const auto look = [&](int j0) {
            const int k = (j0 - first) / step;
            if ((k & 31) == 0 && k) ids = next_ids;
            if ((k & 31) == 16) next_ids = entries(j0 + 16 * step);
#pragma unroll
            for (int t = 0; t < TILES; ++t) {
                const int row = j0 + t * 16;
                page[t] = __builtin_amdgcn_readlane(ids, (k & 31) * TILES + t);
                if (page[t] >= c.pages || row >= j_end) page[t] = -1;
                at_row[t] = row - fastdiv(min(row, j_end - 1), c.by_rows) * c.page_rows;
            }
            if (a.keep && j0 < j_end) {
                const int r = min(lane & (KEYS - 1), j_end - 1 - j0), t = r / 16;
                const int p = t ? page[TILES - 1] : page[0], from = t ? at_row[TILES - 1] : at_row[0];
                raw = p < 0 ? 0 : keep_raw(a, p * c.keep_page + from + r % 16);
            }
        };
        const auto fetch = [&](int b, int j0) {
            const int left = j_end - j0;
            next_live = a.keep ? (uint32_t)__ballot(raw != 0) : ~0u;
#pragma unroll
            for (int t = 0; t < TILES; ++t) {
                // rows of a page that is none are not there
                const int rows = page[t] < 0 ? 0 : left - t * 16;
                if (page[t] < 0) next_live &= ~(0xffffu << (t * 16));
                const int64_t p = max(page[t], 0);
                const uint32_t those = next_live >> (t * 16);
                ck.template start<true>(sk + (b * KEYS + t * 16) * DP, kbase + p * c.k_page + at_row[t] * a.k_row,
                                        a.k_row, a.dim, rows, a.keep, those, 0, lane);
                cv.template start<true>(sv + (b * KEYS + t * 16) * DP, vbase + p * c.v_page + at_row[t] * a.v_row,
                                        a.v_row, a.dim, rows, a.keep, those, 0, lane);
            }
            if (FAR)
#pragma unroll
                for (int i = 0; i < (3 * KEYS + 63) / 64; ++i) {
                    const int r = min((i * 64 + lane) % KEYS, left - 1), ax = min((i * 64 + lane) / KEYS, 2);
                    const int t = r / 16, p = t ? page[TILES - 1] : page[0], from = t ? at_row[TILES - 1] : at_row[0];
                    gp[i] = p < 0 ? 0.f : a.k_pos[p * c.pos_page + (from + r % 16) * a.k_pos_row + ax];
                }
            look(j0 + step);
        };
        // the tiles are this wave's own: its copies and LDS accesses need no barrier, only waits
        const auto put = [&](int b) {
            if (FAR) {
                if (lane < 3 * KEYS) spos[wave][b][lane] = gp[0];
                if (3 * KEYS > 64 && lane < 3 * KEYS - 64) spos[wave][b][64 + lane] = gp[1];
            }
            tile_wait();
            __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
            __builtin_amdgcn_wave_barrier();
            __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
        };
        int b = 0;
        if (first < j_end) {
            look(first);
            fetch(0, first);
            put(0);
        }
        for (int j0 = first; j0 < j_end; j0 += step, b ^= 1) {
            const bool more = j0 + step < j_end;
            live = next_live;
            if (j_end - j0 < KEYS) live &= (1u << (j_end - j0)) - 1;
            if (more) fetch(b ^ 1, j0 + step);
            const T *kt = sk + b * KEYS * DP, *vt = sv + b * KEYS * DP;
            f32x4 d[TILES] = {}, w[TILES] = {};
            if (FAR)
#pragma unroll
                for (int t = 0; t < TILES; ++t) {
                    const float *p = spos[wave][b] + t * 16 + g4;
                    const f32x4 x = *reinterpret_cast<const f32x4 *>(p), y = *reinterpret_cast<const f32x4 *>(p + KEYS),
                                z = *reinterpret_cast<const f32x4 *>(p + 2 * KEYS);
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        const float dx = x[r] - qx, dy = y[r] - qy, dz = z[r] - qz;
                        d[t][r] = __builtin_amdgcn_sqrtf(fmaf(dz, dz, fmaf(dy, dy, dx * dx)));
                    }
                }
#pragma unroll
            for (int st = 0; st < DEPTH; ++st)
#pragma unroll
                for (int t = 0; t < TILES; ++t) w[t] = mma16(at.rows(kt, t, st), q[st], w[t]);
            // the distances' part last: begun with it, each of the products' sums would round at its size
#pragma unroll
            for (int t = 0; t < TILES; ++t)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    if (capped) w[t][r] = a.cap * tanh_of<T, CAP>(w[t][r] * in_cap);
                    if (FAR) w[t][r] = fmaf(-far_unit, d[t][r], w[t][r]);
                }
            constexpr uint32_t kAll = KEYS == 32 ? ~0u : (1u << (KEYS & 31)) - 1;
            if ((live & kAll) != kAll) {
                const uint32_t seen = live >> g4;
#pragma unroll
                for (int t = 0; t < TILES; ++t)
#pragma unroll
                    for (int r = 0; r < 4; ++r)
                        if (!(seen & (1u << (16 * t + r)))) w[t][r] = -INFINITY;
            }
            // rounded here, so that the largest weight is a power of two exactly
            float top = -INFINITY;
#pragma unroll
            for (int t = 0; t < TILES; ++t)
#pragma unroll
                for (int r = 0; r < 4; ++r) w[t][r] *= unit, top = fmaxf(top, w[t][r]);
            if (__any(top > m + kSlack)) {
                top = fmaxf(top, __shfl_xor(top, 16));
                const float next = fmaxf(m, fmaxf(top, __shfl_xor(top, 32)));
                const float by = next == -INFINITY ? 1.f : fast_exp2(m - next);
                m = next;
                sum *= by;
#pragma unroll
                for (int e = 0; e < BLOCKS; ++e) o[e] *= by;
            }
            const float ref = m == -INFINITY ? 0.f : m;
#pragma unroll
            for (int t = 0; t < TILES; ++t)
#pragma unroll
                for (int r = 0; r < 4; ++r) w[t][r] = fast_exp2(w[t][r] - ref);
#pragma unroll
            for (int part = 0; part < kParts<T>; ++part) {
                frag p;
                if constexpr (sizeof(T) == 2) {
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        p[e] = (T)w[e / 4][e % 4];
                        w[e / 4][e % 4] -= (float)p[e];
                    }
                    sum = add_weights(p, sum);
                } else {
                    p = w[0];
#pragma unroll
                    for (int e = 0; e < 4; ++e) sum += p[e];
                }
#pragma unroll
                for (int e = 0; e < BLOCKS; ++e) o[e] = mma16(at.columns(vt, e), p, o[e]);
            }
            if (more) put(b ^ 1);
        }
        sum += __shfl_xor(sum, 16);
        sum += __shfl_xor(sum, 32);
        // the waves' sums, joined
        if (lane < kHeads) sm[wave][lane] = m, ss[wave][lane] = sum;
        float *so = reinterpret_cast<float *>(tiles[wave]);
        if (head)
#pragma unroll
            for (int e = 0; e < BLOCKS; ++e) *reinterpret_cast<f32x4 *>(so + (lane & 15) * kRow + e * 16 + g4) = o[e];
        __syncthreads();
        const int heads = min(group - ht * kHeads, kHeads);
        for (int i = threadIdx.x; i < heads * (DP / 4); i += 64 * W) {
            const int r = i / (DP / 4), dd = i % (DP / 4) * 4;
            if (dd >= a.dim) continue;
            float top = -INFINITY, total = 0.f;
            f32x4 val = {};
#pragma unroll
            for (int w = 0; w < W; ++w) top = fmaxf(top, sm[w][r]);
#pragma unroll
            for (int w = 0; w < W; ++w) {
                // a wave without keys has the maximum -inf and the sum 0; NaN sums pass
                const float by = sm[w][r] == -INFINITY ? 1.f : fast_exp2(sm[w][r] - top);
                total = fmaf(by, ss[w][r], total);
                const f32x4 x = *reinterpret_cast<const f32x4 *>(reinterpret_cast<const float *>(tiles[w]) + r * kRow + dd);
#pragma unroll
                for (int e = 0; e < 4; ++e) val[e] = fmaf(by, x[e], val[e]);
            }
            const int hh = hk * group + ht * kHeads + r;
            if (whole) {
                typedef T t4 __attribute__((ext_vector_type(4)));
                t4 y;
#pragma unroll
                for (int e = 0; e < 4; ++e) y[e] = (T)(total == 0.f ? 0.f : val[e] / total);
                *reinterpret_cast<t4 *>(out + ((int64_t)s * a.heads + hh) * a.dim + dd) = y;
            } else {
                const int64_t to = number * a.heads + hh;
                *reinterpret_cast<f32x4 *>(c.part_o + to * a.dim + dd) = val;
                if (dd == 0) c.part_ms[to] = make_float2(top, total);
            }
        }
        if (CUT == kPieces || share.steps <= 0 || share.s >= a.scenes) return;
        __syncthreads();  // the next scene's copies go where the sums lay
    }
}

// One workgroup a scene and head; scenes of one part have their row already.  The waves take the parts in turn,
// then their sums are joined, always in the same order.  Latency bounds it: 3.6 us at 16 parts, 4.8 at 64.
constexpr int kJoinWaves = 8;
template <typename T>
__global__ __launch_bounds__((64 * kJoinWaves)) void k_paged_join(const float *__restrict__ part_o,
                                                                  const float2 *__restrict__ part_ms,
                                                                  const int2 *__restrict__ parts, FastDiv by_heads,
                                                                  int rows, int heads, int dim, T *__restrict__ out) {
    constexpr int kOnce = 4;  // parts of a wave whose maxima, sums and rows are loaded together
    __shared__ float so[kJoinWaves][128], sm[kJoinWaves], ss[kJoinWaves];
    const int row = blockIdx.y * gridDim.x + blockIdx.x;
    if (row >= rows) return;
    const int s = fastdiv(row, by_heads), h = row - s * heads;
    const int2 own = parts[s];
    if (own.y == 1) return;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int64_t first = (int64_t)own.x * heads + h;
    const int d0 = min(lane, dim - 1), d1 = min(lane + 64, dim - 1);
    float m = -INFINITY, total = 0.f, v0 = 0.f, v1 = 0.f;
    for (int p = wave; p < own.y; p += kJoinWaves * kOnce) {
        float2 e[kOnce];
        float x0[kOnce], x1[kOnce], top = m;
#pragma unroll
        for (int i = 0; i < kOnce; ++i) {
            const int64_t at = first + (int64_t)min(p + i * kJoinWaves, own.y - 1) * heads;
            e[i] = part_ms[at], x0[i] = part_o[at * dim + d0], x1[i] = part_o[at * dim + d1];
        }
#pragma unroll
        for (int i = 0; i < kOnce; ++i)
            if (p + i * kJoinWaves < own.y) top = fmaxf(top, e[i].x);
        const float keep = m == -INFINITY ? 1.f : fast_exp2(m - top);
        m = top, total *= keep, v0 *= keep, v1 *= keep;
#pragma unroll
        for (int i = 0; i < kOnce; ++i) {
            if (p + i * kJoinWaves >= own.y) continue;
            // parts without keys have the maximum -inf and the sum 0; NaN sums pass
            const float by = e[i].x == -INFINITY ? 1.f : fast_exp2(e[i].x - m);
            total = fmaf(by, e[i].y, total), v0 = fmaf(by, x0[i], v0), v1 = fmaf(by, x1[i], v1);
        }
    }
    so[wave][lane] = v0, so[wave][64 + lane] = v1;
    if (lane == 0) sm[wave] = m, ss[wave] = total;
    __syncthreads();
    const int d = threadIdx.x;
    if (d >= dim) return;
    float top = -INFINITY, v = 0.f;
    total = 0.f;
#pragma unroll
    for (int w = 0; w < kJoinWaves; ++w) top = fmaxf(top, sm[w]);
#pragma unroll
    for (int w = 0; w < kJoinWaves; ++w) {
        const float by = sm[w] == -INFINITY ? 1.f : fast_exp2(sm[w] - top);
        total = fmaf(by, ss[w], total), v = fmaf(by, so[w][d], v);
    }
    out[(int64_t)row * dim + d] = (T)(total == 0.f ? 0.f : v / total);
}

// Sets the workgroups of a key head and head tile: one round of them in all, as many as the CUs have room for at
// once.  Scenes of few steps for each wave stay whole.
void paged_shares(const AttnArgs &a, int dtype, PageArgs *c) {
    const int64_t size = dtype == GSV_BF16 ? 2 : 4, dp = a.dim <= 32 ? 32 : a.dim <= 64 ? 64 : 128;
    const int64_t waves = dp == 128 ? 2 : 4, keys = size == 2 ? 32 : 16;
    c->split = 0, c->shares = a.scenes;
    if (!a.scenes || a.k_tokens <= imax64(waves * keys, 64)) return;
    const int64_t lds = waves * (4 * keys * dp * size + 6 * keys * 4) + 2048;
    const int64_t round = 256 * imin64(163840 / lds, 4);
    const int64_t most = ((int64_t)a.k_tokens + waves * keys - 1) / (waves * keys) * a.scenes;
    c->split = 1;
    c->shares = (int)imax64(1, imin64(round / ((int64_t)a.kv_heads * c->head_tiles), most + a.scenes));
}

struct Paged {
    const AttnArgs &a;
    const PageArgs &c;
    void *out;
    hipStream_t st;
    template <typename T, int DP, bool FAR, int CAP> void run() const {
        T *o = static_cast<T *>(out);
        const int64_t apart = ((int64_t)c.shares * (a.kv_heads / c.near) + kXcds - 1) / kXcds * kXcds;
        const dim3 grid((unsigned)(apart * c.near * c.head_tiles)), block(64 * kWaves<DP>);
        // Pieces and shares, us: 16 caches of 4,096, 2 key heads of 64 (256 workgroups each) 13.0 and 15.9; 20 of 100,003
        // and less, 4 of 128 (128) 61.3 and 68.0; 40 of 4,000 46.8 and 51.5; 90 of 2,000 56.7 and 56.5, 120 of 1,500 57.3
        // and 56.4; 50 of 3,000, 8 of 64 (64) 53.0 and 46.4.
        if (a.scenes * 2 < c.shares || !c.split)
            hipLaunchKernelGGL((k_attention_paged<T, DP, FAR, CAP, kPieces>), grid, block, 0, st, a, c, o);
        else
            hipLaunchKernelGGL((k_attention_paged<T, DP, FAR, CAP, kShares>), grid, block, 0, st, a, c, o);
        if (c.split) {
            // (an axis of a grid holds less than 2^32 threads: 2^23 of these workgroups; rows are less than 2^24)
            const int rows = a.scenes * a.heads, x = rows < (1 << 22) ? rows : 1 << 22;
            hipLaunchKernelGGL(k_paged_join<T>, dim3((unsigned)x, (unsigned)((rows + x - 1) / x)), dim3(64 * kJoinWaves),
                               0, st, c.part_o, c.part_ms, c.parts, make_fastdiv(a.heads), rows, a.heads, a.dim, o);
        }
    }
};

int paged_plan(const gsv_attention *args, const gsv_pages *p, AttnArgs *a, PageArgs *c) {
    if (!args || !p || args->causal || args->prefix || args->q_starts || args->k_starts ||
        args->scenes < 0 || args->scenes != args->q_tokens || p->pages < 1 || p->page_rows < kPageUnit ||
        p->page_rows % kPageUnit || p->table_pages < 0 || p->table_row < 0)
        return GSV_ERR_INVALID_ARGUMENT;
    const int64_t rows = (int64_t)p->page_rows * p->table_pages;
    if (rows > GSV_MAX_TOKENS) return GSV_ERR_SIZE_OVERFLOW;
    gsv_attention one = *args;
    one.scenes = 1;  // rows are addressed by scene and page here, not packed
    one.k = p->k, one.v = p->v, one.k_positions = p->positions, one.k_pos_row = p->pos_row;
    one.k_row = p->k_row, one.v_row = p->v_row, one.k_head = p->k_head, one.v_head = p->v_head;
    one.keep = p->keep, one.keep_bytes = p->keep_bytes;
    one.k_tokens = (int)rows;
    const int st = attention_args(&one, a);
    if (st != GSV_OK) return st;
    a->scenes = args->scenes;
    const int64_t tiles = (a->heads / a->kv_heads + kHeads - 1) / kHeads;
    if ((int64_t)a->scenes * a->kv_heads * tiles > (1 << 22) || (int64_t)a->scenes * a->heads >= (1 << 24))
        return GSV_ERR_SIZE_OVERFLOW;
    *c = PageArgs{};
    c->head_tiles = (int)tiles;
    // All key heads where they share lines of 128 bytes, which one L2 so fetches once: 128 scenes, 8 key heads of 32
    // bfloat16, 356 MB 92 us, on 8 XCDs 125.  Heads of whole lines are 2 % faster apart.
    c->near = a->dim * (args->dtype == GSV_BF16 ? 2 : 4) % 128 ? a->kv_heads : 1;
    paged_shares(*a, args->dtype, c);
    return GSV_OK;
}

// The workspace: parts of the sums, their maxima and sums of weights, and which are a scene's.
struct Workspace {
    size_t rows, ms, parts, bytes;
};
Workspace paged_workspace(const AttnArgs &a, const PageArgs &c) {
    if (!c.split) return {};
    Workspace w;
    w.rows = ((size_t)c.shares + a.scenes) * a.heads;
    w.ms = w.rows * a.dim * sizeof(float);  // a multiple of 32 bytes
    w.parts = w.ms + w.rows * sizeof(float2);
    w.bytes = w.parts + a.scenes * sizeof(int2);
    return w;
}

}  // namespace
}  // namespace gsv

using namespace gsv;

extern "C" int gsv_attention_paged_workspace_bytes(const gsv_attention *args, const gsv_pages *pages,
                                                   size_t *bytes) {
    AttnArgs a;
    PageArgs c;
    if (!bytes) return GSV_ERR_INVALID_ARGUMENT;
    const int st = paged_plan(args, pages, &a, &c);
    if (st != GSV_OK) return st;
    *bytes = paged_workspace(a, c).bytes;
    return GSV_OK;
}

extern "C" int gsv_attention_paged(const gsv_attention *args, const gsv_pages *pages, const int32_t *lengths,
                                   void *out, void *workspace, size_t workspace_bytes, void *stream) {
    AttnArgs a;
    PageArgs c;
    int st = paged_plan(args, pages, &a, &c);
    if (st != GSV_OK) return st;
    if (a.scenes == 0) return GSV_OK;
    const Workspace ws = paged_workspace(a, c);
    if (ws.bytes > workspace_bytes) return GSV_ERR_WORKSPACE_TOO_SMALL;
    const int64_t chunk = args->dtype == GSV_BF16 ? 8 : 4;
    c.k_page = used_stride(pages->k_page, pages->pages);
    c.v_page = used_stride(pages->v_page, pages->pages);
    if (!lengths || (pages->table_pages && !pages->table) || !out || (ws.bytes && !workspace) ||
        c.k_page % chunk || c.v_page % chunk || reinterpret_cast<uintptr_t>(out) % 16 ||
        reinterpret_cast<uintptr_t>(workspace) % 16)
        return GSV_ERR_INVALID_ARGUMENT;
    c.lengths = lengths;
    c.pos_page = pages->pos_page, c.keep_page = pages->keep_page;
    c.part_o = static_cast<float *>(workspace);
    c.part_ms = reinterpret_cast<float2 *>(static_cast<char *>(workspace) + ws.ms);
    c.parts = reinterpret_cast<int2 *>(static_cast<char *>(workspace) + ws.parts);
    c.table = pages->table, c.table_row = pages->table_row;
    c.pages = pages->pages, c.page_rows = pages->page_rows;
    c.by_rows = make_fastdiv(pages->page_rows);
    Paged f{a, c, out, as_stream(stream)};
    attention_variant(a, args->dtype, f);
    return check_launch();
}
