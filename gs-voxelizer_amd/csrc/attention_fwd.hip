// attention_fwd.hip — attention inside packed scenes, forward.
//
//   t_ij = cap tanh(scale q_i.k_j / cap) - slope_h |p_i - p_j|   (cap, slope optional)
//   o_i = sum_j softmax_j(t_ij) v_j     over the keys j that row i sees; 0 if it sees none
//
// A workgroup of four waves takes 128 query rows of one head; a wave 32 of them, one in
// each lane pair (l, l + 32).  Keys pass through LDS in tiles, the scores are formed
// transposed (K Q^T), so a row's running maximum and sum stay with its lanes, and the weights are in
// place as the right operand of the product with the values (V^T P^T).
//
// The two products are 4 dim operations an element; beside them an element costs an exponential, a
// square root and about eight further vector instructions (differences of positions come from the
// matrix units too), which at 64 channels take more cycles than the products.  One scene of 16,000 tokens, 8
// heads of 64, bias, bfloat16: 1.00 ms, 526 TFLOP/s in the products; vector instructions issue in 64 % of the
// cycles, the matrix units work in 27 %, and what is left is their overlap.  Shorter scenes wait: 8,001 tokens in
// 8 scenes take 89 us (39 and 11 %, 4.3 waves a CU: a workgroup's chain of about 20 tiles and its start);
// 10,007 in 4 causal scenes, 16 heads of 128 on 4, capped, with a bias 323 us (55 and 19 %).
#include "gsv_attention.h"

// (a product and a difference stay two roundings where they are written as two)
#pragma clang fp contract(off)

namespace gsv {
namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr int WAVES = 4, kRows = 32 * WAVES;  // a workgroup's waves and query rows
// The maximum follows the scores only when one exceeds it by 2^8: weights then stay
// below 2^8, and a rescale of the sums (one multiply a register) is rare.
constexpr float kSlack = 8.f;

// HEADS query heads of a wave share its distances (a third of the vector work of one head: 2
// multiply-adds, a multiply and a root an element, at the matrix units' differences).  With one
// key head for both (SHARED) they share the tiles too.
// TRAIN: the log sums and out_low are wanted.
template <typename T, int DP, bool FAR, int CAP, int HEADS, bool SHARED, bool TRAIN>
__global__ __launch_bounds__(256, sizeof(T) == 2 || DP <= 64 ? 2 : 1) void k_attention_fwd(
    const AttnArgs a, T *__restrict__ out, T *__restrict__ out_low, float *__restrict__ lse) {
    constexpr int KB = sizeof(T) == 2 ? 64 : 32;  // keys of a tile
    constexpr int KV = SHARED ? 1 : HEADS;        // key heads of the workgroup
    constexpr bool far = FAR, capped = CAP != kNoCap;
    // float32: scores are rounded to powers of two before their maximum is taken off, so that the
    // largest has the weight 1 exactly, as the rounding to bfloat16 gives it there
    constexpr bool kExact = sizeof(T) == 4;
    typedef typename Elem<T>::frag frag;
    __shared__ __align__(1024) T sk[2][KV][KB * DP];
    __shared__ __align__(1024) T sv[2][KV][KB * DP];
    __shared__ __align__(16) typename Places<T>::Row spos[2][3 * KB];

    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int sets = a.heads / HEADS;
    const int h0 = blockIdx.x % sets * HEADS, place_n = grid_place(sets);
    if (place_n >= a.places) return;
    const Place where = tile_place<kRows>(a.q_starts, a.scenes, a.q_tokens, place_n, a.slots);
    const Scene c = scene_of(a, where.scene, true);
    const int nq = c.q1 - c.q0;
    const int tiles = (nq + kRows - 1) / kRows;
    const int group = a.heads / a.kv_heads;
    const bool fine = in_two_parts<T>(c.k1 - c.k0);
    const T *kbase[KV], *vbase[KV];
#pragma unroll
    for (int n = 0; n < KV; ++n) {
        const int hk = (h0 + n) / group;
        kbase[n] = static_cast<const T *>(a.k) + (int64_t)c.k0 * a.k_row + hk * a.k_head;
        vbase[n] = static_cast<const T *>(a.v) + (int64_t)c.k0 * a.v_row + hk * a.v_head;
    }
    // scores leave the matrix product in units of 1 / scale (or 1 where they are capped);
    // unit turns them into powers of two
    const float unit = capped ? kLog2e : a.scale * kLog2e;
    const float left_unit = fine ? 1.f : unit;  // two parts: as for float32 (kExact)
    const float in_cap = capped ? a.scale / a.cap : 0.f;
    float far_unit[HEADS];
#pragma unroll
    for (int n = 0; n < HEADS; ++n) far_unit[n] = slope_of(a, h0 + n) / (capped ? 1.f : a.scale);
    Tile<T, DP> at;
    at.plan(lane);
    Copy<T, DP, KB, WAVES> ck, cv;
    ck.plan(a.k_row, a.dim, wave, lane);
    cv.plan(a.v_row, a.dim, wave, lane);

    for (int tile = where.tile; tile < tiles; tile += where.step) {
        // the last rows of a causal scene see the most keys: they start first
        const int first = (tiles - 1 - tile) * kRows;
        const int i = first + wave * 32 + (lane & 31);
        const bool row = i < nq;
        const int64_t qi = c.q0 + i;
        frag q[HEADS][DP / 16];
#pragma unroll
        for (int n = 0; n < HEADS; ++n)
            load_column<T, DP>(q[n], static_cast<const T *>(a.q) + qi * a.q_row + (h0 + n) * a.q_head,
                               a.dim, row, lane);
        Places<T> place;
        if (far) {
            float x = 0.f, y = 0.f, z = 0.f;
            if (row) {
                const float *p = a.q_pos + qi * a.q_pos_row;
                x = p[0], y = p[1], z = p[2];
            }
            place.set(x, y, z, lane);
        }
        const int limit = row ? key_limit(a, c, i) : 0;
        const int all = first + wave * 32 + 31 < nq ? key_limit(a, c, first + wave * 32) : 0;
        const int most = key_limit(a, c, min(first + kRows, nq) - 1);  // of the workgroup
        const int mine = first + wave * 32 < nq
                             ? key_limit(a, c, min(first + wave * 32 + 32, nq) - 1) : 0;
        f32x16 o[HEADS][DP / 32] = {};
        // the weights' sums as the product takes them and, for the log sums, unrounded
        float m[HEADS], sum[HEADS], exact[HEADS];
#pragma unroll
        for (int n = 0; n < HEADS; ++n) m[n] = -INFINITY, sum[n] = exact[n] = 0.f;

        float gp = 0.f;
        int raw = 0;
        uint64_t live = ~0ull, next_live = ~0ull;
        auto look = [&](int j0) {  // the mask of a tile
            if (a.keep && j0 < most) raw = keep_raw(a, c.k0 + min(j0 + lane, most - 1));
        };
        auto fetch = [&](int b, int j0) {
            const int left = most - j0;
            if (a.keep) next_live = __ballot(raw != 0);
            look(j0 + KB);
#pragma unroll
            for (int n = 0; n < KV; ++n) {
                ck.start(sk[b][n], kbase[n] + j0 * a.k_row, a.k_row, a.dim, left, a.keep, next_live,
                         wave, lane);
                cv.start(sv[b][n], vbase[n] + j0 * a.v_row, a.v_row, a.dim, left, a.keep, next_live,
                         wave, lane);
            }
            if (far && threadIdx.x < 3 * KB)
                gp = a.k_pos[(c.k0 + j0 + min((int)threadIdx.x % KB, left - 1)) * a.k_pos_row +
                             threadIdx.x / KB];
        };
        auto put = [&](int b) {
            if (far && threadIdx.x < 3 * KB) spos[b][threadIdx.x] = Places<T>::row(gp);
            tile_wait();
        };
        __syncthreads();  // the previous tile's last reads
        if (most > 0) {
            look(0);
            fetch(0, 0);
            put(0);
        }
        __syncthreads();
        int b = 0;
        for (int j0 = 0; j0 < most; j0 += KB, b ^= 1) {
            const bool more = j0 + KB < most;
            live = next_live;
            if (more) fetch(b ^ 1, j0 + KB);
            if (j0 < mine) {
                // (a branch of its own for the scores of two parts costs long scenes 2 %)
                const bool masked = fine || j0 + KB > all || (KB == 64 ? ~live : (uint32_t)~live) != 0;
#pragma unroll 1
                for (int kb = 0; kb < KB / 32; ++kb) {
                    f32x16 d = {}, w[HEADS] = {};
#pragma unroll
                    for (int st = 0; st < DP / 16; ++st)
#pragma unroll
                        for (int n = 0; n < HEADS; ++n)
                            w[n] = mma(at.rows(sk[b][SHARED ? 0 : n] + kb * 32 * DP, st), q[n][st], w[n]);
                    // the distances' vector work runs while the products above do
                    if (far) d = distances<T>(place, spos[b], KB, kb * 32, lane);
#pragma unroll
                    for (int n = 0; n < HEADS; ++n)
#pragma unroll
                        for (int r = 0; r < 16; ++r) {
                            if (capped) w[n][r] = a.cap * tanh_of<T, CAP>(w[n][r] * in_cap);
                            if (far) w[n][r] = fmaf(-far_unit[n], d[r], w[n][r]);
                        }
                    if (masked) {
                        const uint32_t seen = seen_rows(live, kb, limit - j0 - kb * 32, lane);
#pragma unroll
                        for (int n = 0; n < HEADS; ++n)
#pragma unroll
                            for (int r = 0; r < 16; ++r)
                                if (!(seen & (1u << result_row(r)))) w[n][r] = -INFINITY;
                        if (fine)
#pragma unroll
                            for (int n = 0; n < HEADS; ++n)
#pragma unroll
                                for (int r = 0; r < 16; ++r) w[n][r] *= unit;
                    }
                    if constexpr (kExact)
#pragma unroll
                        for (int n = 0; n < HEADS; ++n)
#pragma unroll
                            for (int r = 0; r < 16; ++r) w[n][r] *= unit;
                    float top[HEADS];
                    bool grown = false;
#pragma unroll
                    for (int n = 0; n < HEADS; ++n) {
                        top[n] = -INFINITY;
#pragma unroll
                        for (int r = 0; r < 16; ++r) top[n] = fmaxf(top[n], w[n][r]);
                        if (!kExact) top[n] *= left_unit;
                        grown |= top[n] > m[n] + kSlack;
                    }
                    if (__any(grown)) {
#pragma unroll
                        for (int n = 0; n < HEADS; ++n) {
                            const float next = fmaxf(m[n], fmaxf(top[n], other_half(top[n])));
                            const float by = next == -INFINITY ? 1.f : fast_exp2(m[n] - next);
                            m[n] = next;
                            sum[n] *= by, exact[n] *= by;
#pragma unroll
                            for (int e = 0; e < DP / 32; ++e) o[n][e] *= by;
                        }
                    }
#pragma unroll
                    for (int n = 0; n < HEADS; ++n) {
                        const float ref = m[n] == -INFINITY ? 0.f : m[n];
#pragma unroll
                        for (int r = 0; r < 16; ++r) {
                            w[n][r] = fast_exp2(kExact ? w[n][r] - ref : fmaf(w[n][r], left_unit, -ref));
                            if (TRAIN) exact[n] += w[n][r];
                        }
                        for (int part = 0; part <= (fine ? 1 : 0); ++part) {
                            if (part) w[n] = remainders<T>(w[n]);
                            Tile<T, DP> cols = at;
                            cols.forget();
#pragma unroll
                            for (int half = 0; half < 2; ++half) {
                                const frag p = to_frag<T>(w[n], half);
                                sum[n] = add_weights(p, sum[n]);
                                const T *vt = sv[b][SHARED ? 0 : n] + (kb * 32 + half * 16) * DP;
#pragma unroll
                                for (int e = 0; e < DP / 32; ++e)
                                    o[n][e] = mma(cols.columns(vt, e, lane), p, o[n][e]);
                            }
                        }
                    }
                }
            }
            if (more) put(b ^ 1);
            __syncthreads();
        }
#pragma unroll
        for (int n = 0; n < HEADS; ++n) {
            sum[n] += other_half(sum[n]);
            exact[n] += other_half(exact[n]);
            if (!row) continue;
            const int64_t at_out = (qi * a.heads + h0 + n) * a.dim;
            store_column<T, DP>(out + at_out, o[n], sum[n] == 0.f ? 0.f : 1.f / sum[n], a.dim, lane,
                                TRAIN && out_low ? out_low + at_out : nullptr);
            // log2 of the row's sum of exponentials; +inf for an empty row, whose weights
            // in the backward are exp2(-inf)
            if (TRAIN && lane < 32)
                lse[(int64_t)(h0 + n) * a.q_tokens + qi] =
                    exact[n] == 0.f ? INFINITY : m[n] + log2f(exact[n]);
        }
    }
}

// The same for few rows, where a wave's chain of tiles, one after the other, bounds it (601 float32
// tokens in 6 scenes, 4 heads of 32: 10 us): a workgroup takes 32 rows of one head, its waves every
// W-th tile of 32 keys each.  The tiles are a wave's own (its copies need no barrier, only waits);
// the waves' sums are joined through LDS at the end.  Four times as many workgroups, each a quarter as
// long.  Scores are rounded to powers of two before their
// maximum is taken off, so that the largest weight is exactly a power of two.
template <typename T, int DP, bool FAR, int CAP, bool TRAIN>
__global__ __launch_bounds__((64 * kFewWaves<T, DP>)) void k_attention_fwd_few(
    const AttnArgs a, T *__restrict__ out, T *__restrict__ out_low, float *__restrict__ lse) {
    constexpr int W = kFewWaves<T, DP>, KB = 32;
    constexpr bool far = FAR, capped = CAP != kNoCap;
    typedef typename Elem<T>::frag frag;
    static_assert(4 * KB * DP * sizeof(T) >= 32 * DP * sizeof(float), "sums reuse the tiles");
    __shared__ __align__(1024) T tiles[W][4 * KB * DP];  // a wave's keys and values, two buffers
    __shared__ __align__(16) typename Places<T>::Row spos[W][2][3 * KB];
    __shared__ float sm[W][32], ss[W][32], se[W][32];

    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int h = blockIdx.x % a.heads, place_n = grid_place(a.heads);
    if (place_n >= a.places) return;
    const Place where = tile_place<32>(a.q_starts, a.scenes, a.q_tokens, place_n, a.slots);
    const Scene c = scene_of(a, where.scene, true);
    const int nq = c.q1 - c.q0, row_tiles = (nq + 31) / 32;
    const bool fine = in_two_parts<T>(c.k1 - c.k0);
    const int hk = h / (a.heads / a.kv_heads);
    const T *kbase = static_cast<const T *>(a.k) + (int64_t)c.k0 * a.k_row + hk * a.k_head;
    const T *vbase = static_cast<const T *>(a.v) + (int64_t)c.k0 * a.v_row + hk * a.v_head;
    const float unit = capped ? kLog2e : a.scale * kLog2e;
    const float in_cap = capped ? a.scale / a.cap : 0.f;
    const float far_unit = slope_of(a, h) / (capped ? 1.f : a.scale);
    T *const sk = tiles[wave], *const sv = sk + 2 * KB * DP;
    Tile<T, DP> at;
    at.plan(lane);
    Copy<T, DP, KB, 1> ck, cv;
    ck.plan(a.k_row, a.dim, 0, lane);
    cv.plan(a.v_row, a.dim, 0, lane);

    for (int tile = where.tile; tile < row_tiles; tile += where.step) {
        const int first = (row_tiles - 1 - tile) * 32, i = first + (lane & 31);
        const bool row = i < nq;
        const int64_t qi = c.q0 + i;
        frag q[DP / 16];
        load_column<T, DP>(q, static_cast<const T *>(a.q) + qi * a.q_row + h * a.q_head, a.dim, row, lane);
        Places<T> place;
        if (far) {
            float x = 0.f, y = 0.f, z = 0.f;
            if (row) {
                const float *p = a.q_pos + qi * a.q_pos_row;
                x = p[0], y = p[1], z = p[2];
            }
            place.set(x, y, z, lane);
        }
        const int limit = row ? key_limit(a, c, i) : 0;
        const int all = first + 31 < nq ? key_limit(a, c, first) : 0;
        const int most = key_limit(a, c, min(first + 32, nq) - 1);
        f32x16 o[DP / 32] = {};
        float m = -INFINITY, sum = 0.f, exact = 0.f;

        float gp[2] = {};
        int raw = 0;
        uint64_t live = ~0ull, next_live = ~0ull;
        auto look = [&](int j0) {
            if (a.keep && j0 < most) raw = keep_raw(a, c.k0 + min(j0 + (lane & 31), most - 1));
        };
        auto fetch = [&](int b, int j0) {
            if (a.keep) next_live = __ballot(raw != 0);
            look(j0 + W * KB);
            const int left = most - j0;
            ck.start(sk + b * KB * DP, kbase + j0 * a.k_row, a.k_row, a.dim, left, a.keep, next_live, 0, lane);
            cv.start(sv + b * KB * DP, vbase + j0 * a.v_row, a.v_row, a.dim, left, a.keep, next_live, 0, lane);
            if (far)
#pragma unroll
                for (int n = 0; n < 2; ++n) {
                    const int r = min(lane & 31, left - 1), ax = min(2 * n + (lane >> 5), 2);
                    gp[n] = a.k_pos[(c.k0 + j0 + r) * a.k_pos_row + ax];
                }
        };
        auto put = [&](int b) {
            if (far) {
                spos[wave][b][lane] = Places<T>::row(gp[0]);
                if (lane < KB) spos[wave][b][64 + lane] = Places<T>::row(gp[1]);
            }
            tile_wait();
            __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
            __builtin_amdgcn_wave_barrier();
            __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
        };
        __syncthreads();  // the previous rows' sums in the tiles have been read
        int b = 0;
        if (wave * KB < most) {
            look(wave * KB);
            fetch(0, wave * KB);
            put(0);
        }
        for (int j0 = wave * KB; j0 < most; j0 += W * KB, b ^= 1) {
            const bool more = j0 + W * KB < most;
            live = next_live;
            if (more) fetch(b ^ 1, j0 + W * KB);
            const T *kt = sk + b * KB * DP, *vt = sv + b * KB * DP;
            f32x16 d = {}, w = {};
#pragma unroll
            for (int st = 0; st < DP / 16; ++st) w = mma(at.rows(kt, st), q[st], w);
            if (far) d = distances<T>(place, spos[wave][b], KB, 0, lane);
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                if (capped) w[r] = a.cap * tanh_of<T, CAP>(w[r] * in_cap);
                if (far) w[r] = fmaf(-far_unit, d[r], w[r]);
            }
            if (j0 + KB > all || (uint32_t)~live) {
                const uint32_t seen = seen_rows(live, 0, limit - j0, lane);
#pragma unroll
                for (int r = 0; r < 16; ++r)
                    if (!(seen & (1u << result_row(r)))) w[r] = -INFINITY;
            }
#pragma unroll
            for (int r = 0; r < 16; ++r) w[r] *= unit;
            float top = -INFINITY;
#pragma unroll
            for (int r = 0; r < 16; ++r) top = fmaxf(top, w[r]);
            if (__any(top > m + kSlack)) {
                const float next = fmaxf(m, fmaxf(top, other_half(top)));
                const float by = next == -INFINITY ? 1.f : fast_exp2(m - next);
                m = next;
                sum *= by, exact *= by;
#pragma unroll
                for (int e = 0; e < DP / 32; ++e) o[e] *= by;
            }
            const float ref = m == -INFINITY ? 0.f : m;
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                w[r] = fast_exp2(w[r] - ref);
                if (TRAIN) exact += w[r];
            }
            for (int part = 0; part <= (fine ? 1 : 0); ++part) {
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
        exact += other_half(exact);
        if (lane < 32) sm[wave][lane] = m, ss[wave][lane] = sum, se[wave][lane] = exact;
        // the waves' sums: row r's channel d at d * 32 + r, so that lanes read and write in a line
        float *so = reinterpret_cast<float *>(tiles[wave]);
#pragma unroll
        for (int e = 0; e < DP / 32; ++e)
#pragma unroll
            for (int r = 0; r < 16; ++r)
                so[(e * 32 + result_row(r) + 4 * (lane >> 5)) * 32 + (lane & 31)] = o[e][r];
        __syncthreads();
        float by[W], top = -INFINITY, total = 0.f, log_total = 0.f;
        const int r = threadIdx.x & 31;
#pragma unroll
        for (int w = 0; w < W; ++w) top = fmaxf(top, sm[w][r]);
#pragma unroll
        for (int w = 0; w < W; ++w) {
            by[w] = sm[w][r] == -INFINITY ? 1.f : fast_exp2(sm[w][r] - top);  // else its sum is 0
            total = fmaf(by[w], ss[w][r], total);
            log_total = fmaf(by[w], se[w][r], log_total);
        }
        const float inv = total == 0.f ? 0.f : 1.f / total;
        if (first + r < nq) {
            const int64_t at_out = ((int64_t)(c.q0 + first + r) * a.heads + h) * a.dim;
            // eight channels of a row at a time
            for (int d0 = (threadIdx.x >> 5) * 8; d0 < a.dim; d0 += 2 * W * 8) {
                typedef T t8 __attribute__((ext_vector_type(8)));
                t8 v, low;
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    float x = 0.f;
#pragma unroll
                    for (int w = 0; w < W; ++w)
                        x = fmaf(by[w], reinterpret_cast<const float *>(tiles[w])[(d0 + e) * 32 + r], x);
                    x *= inv;
                    v[e] = (T)x;
                    low[e] = (T)(x - (float)v[e]);
                }
                *reinterpret_cast<t8 *>(out + at_out + d0) = v;
                if (TRAIN && out_low) *reinterpret_cast<t8 *>(out_low + at_out + d0) = low;
            }
            if (TRAIN && threadIdx.x < 32)
                lse[(int64_t)h * a.q_tokens + c.q0 + first + r] =
                    log_total == 0.f ? INFINITY : top + log2f(log_total);
        }
    }
}

struct Forward {
    AttnArgs a;
    int longest;
    void *out, *out_low;
    float *lse;
    hipStream_t st;
    int status;
    bool plan(int rows, int heads, dim3 *grid) {
        const int64_t slots = attention_slots(a, a.q_tokens, longest, rows);
        const int64_t places = attention_places(a, a.q_tokens, rows, slots);
        a.slots = (int)slots, a.places = (int)places;
        status = attention_grid(places, heads, grid) ? GSV_OK : GSV_ERR_SIZE_OVERFLOW;
        return status == GSV_OK;
    }
    template <typename T, int DP, bool FAR, int CAP, int HEADS, bool SHARED> void start() {
        dim3 grid;
        if (!plan(kRows, a.heads / HEADS, &grid)) return;
        T *o = static_cast<T *>(out), *low = static_cast<T *>(out_low);
        if (lse)
            hipLaunchKernelGGL((k_attention_fwd<T, DP, FAR, CAP, HEADS, SHARED, true>), grid,
                               dim3(256), 0, st, a, o, low, lse);
        else
            hipLaunchKernelGGL((k_attention_fwd<T, DP, FAR, CAP, HEADS, SHARED, false>), grid,
                               dim3(256), 0, st, a, o, low, lse);
        status = check_launch();
    }
    template <typename T, int DP, bool FAR, int CAP> void few() {
        dim3 grid, block(64 * kFewWaves<T, DP>);
        if (!plan(32, a.heads, &grid)) return;
        T *o = static_cast<T *>(out), *low = static_cast<T *>(out_low);
        if (lse)
            hipLaunchKernelGGL((k_attention_fwd_few<T, DP, FAR, CAP, true>), grid, block, 0, st, a, o, low, lse);
        else
            hipLaunchKernelGGL((k_attention_fwd_few<T, DP, FAR, CAP, false>), grid, block, 0, st, a, o, low, lse);
        status = check_launch();
    }
    template <typename T, int DP, bool FAR, int CAP> void run() {
        if (attention_few(a)) return few<T, DP, FAR, CAP>();
        if constexpr (FAR && sizeof(T) == 2 && DP <= 64 && CAP != kAnyCap) {
            if (attention_pairs(a)) {
                if (a.heads / a.kv_heads % 2 == 0) start<T, DP, FAR, CAP, 2, true>();
                else start<T, DP, FAR, CAP, 2, false>();
                return;
            }
        }
        start<T, DP, FAR, CAP, 1, true>();
    }
};

}  // namespace

int attention_args(const gsv_attention *in, AttnArgs *a) {
    if (!in) return GSV_ERR_INVALID_ARGUMENT;
    const gsv_attention &g = *in;
    if (g.dtype != GSV_F32 && g.dtype != GSV_BF16) return GSV_ERR_INVALID_ARGUMENT;
    if (g.q_tokens < 0 || g.k_tokens < 0 || g.heads < 1 || g.kv_heads < 1 ||
        g.heads % g.kv_heads || g.dim < 8 || g.dim > 128 || g.dim % 8 || g.scenes < 1)
        return GSV_ERR_INVALID_ARGUMENT;
    if (g.q_tokens > GSV_MAX_TOKENS || g.k_tokens > GSV_MAX_TOKENS || g.scenes > (1 << 29))
        return GSV_ERR_SIZE_OVERFLOW;
    const int64_t chunk = g.dtype == GSV_BF16 ? 8 : 4;
    const int64_t q_row = used_stride(g.q_row, g.q_tokens), q_head = used_stride(g.q_head, g.heads);
    const int64_t k_row = used_stride(g.k_row, g.k_tokens), k_head = used_stride(g.k_head, g.kv_heads);
    const int64_t v_row = used_stride(g.v_row, g.k_tokens), v_head = used_stride(g.v_head, g.kv_heads);
    for (int64_t x : {q_row, q_head, k_row, k_head, v_row, v_head})
        if (x % chunk) return GSV_ERR_INVALID_ARGUMENT;
    for (int64_t x : {q_row, k_row, v_row})
        if (x < 0 || x * (16 / chunk) > kMaxRowBytes) return GSV_ERR_INVALID_ARGUMENT;
    const void *ptrs[] = {g.q, g.k, g.v};
    for (const void *p : ptrs)
        if (reinterpret_cast<uintptr_t>(p) % 16) return GSV_ERR_INVALID_ARGUMENT;
    if ((g.q_tokens > 0 && !g.q) || (g.k_tokens > 0 && (!g.k || !g.v)))
        return GSV_ERR_INVALID_ARGUMENT;
    if (g.scenes > 1 && (!g.q_starts || !g.k_starts)) return GSV_ERR_INVALID_ARGUMENT;
    if (!(g.scale > 0.f) || !(g.cap >= 0.f)) return GSV_ERR_INVALID_ARGUMENT;
    if (g.slopes && ((!g.q_positions && g.q_tokens > 0) || (!g.k_positions && g.k_tokens > 0) ||
                     (g.slopes_dtype != GSV_F32 && g.slopes_dtype != GSV_BF16)))
        return GSV_ERR_INVALID_ARGUMENT;
    if (g.keep && g.keep_bytes != 1 && g.keep_bytes != 4) return GSV_ERR_INVALID_ARGUMENT;
    *a = AttnArgs{g.q, g.k, g.v, q_row, q_head, k_row, k_head, v_row, v_head,
                  g.q_tokens, g.k_tokens, g.heads, g.kv_heads, g.dim, g.scenes, g.q_starts,
                  g.k_starts, g.prefix, g.causal, g.scale, g.cap, g.q_positions, g.k_positions,
                  g.q_pos_row, g.k_pos_row, g.slopes, g.slopes_dtype == GSV_F32, g.keep,
                  g.keep_bytes, 0, 0};
    return GSV_OK;
}

}  // namespace gsv

using namespace gsv;

extern "C" int gsv_attention_fwd(const gsv_attention *args, void *out, void *out_low, float *lse,
                                 void *stream) {
    AttnArgs a;
    const int st = attention_args(args, &a);
    if (st != GSV_OK) return st;
    if (a.q_tokens == 0) return GSV_OK;
    if (!out || reinterpret_cast<uintptr_t>(out) % 16 || reinterpret_cast<uintptr_t>(out_low) % 16) return GSV_ERR_INVALID_ARGUMENT;
    Forward f{a, args->longest_q, out, out_low, lse, as_stream(stream), GSV_OK};
    attention_variant(a, args->dtype, f);
    return f.status;
}
