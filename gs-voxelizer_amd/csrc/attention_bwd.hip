// attention_bwd.hip — attention inside packed scenes, backward.
//
// With p_ij the weights, recomputed from the saved log sums, and D_i = do_i.o_i:
//   dv_j = sum_i p_ij do_i            dt_ij = p_ij (do_i.v_j - D_i)
//   dslope = - sum_ij dt_ij |p_i - p_j|
//   ds_ij = dt_ij (1 - tanh^2)        dq_i = scale sum_j ds_ij k_j
//                                     dk_j = scale sum_i ds_ij q_i
// D_i is formed from o_i in two parts (out, and out_low, what its rounding took): where one key has
// nearly all of a row's weight, do_i.v_j - D_i is a small difference, and 8 bits of o_i would leave
// little of it.  Two kernels form the scores twice, one with the rows' sums (dq, D, dslope) and one with
// the keys' (dk, dv): each sum stays in the registers of one wave, in a fixed order, with no atomics
// (and partial gradients in memory only where few key tiles have many rows: bwd_parts).
//
// The rows' kernel does 6 dim operations an element in its products, the keys' 8 dim; both pay
// the forward's vector instructions for an element's weight again and some for its gradient, and
// two waves a SIMD (one at 128 channels, where dk and dv alone take 128 registers) overlap the two only
// in part.  16,000 tokens, 8 heads of 64, bias, bfloat16: rows 1.44 ms (545 TFLOP/s; vector instructions issue in
// 71 % of the cycles, the matrix units work in 30 %), keys 1.64 ms (639 TFLOP/s; 56 and 33 %).  8,001 tokens in
// 8 scenes: 110 us each (43 and 13 %, 32 and 16 %, at 4.4 waves a CU).  10,007 tokens in 4 causal scenes, 16
// heads of 128 on 4, capped: 414 us (54 and 23 %) and 673 us (35 and 17 %, one wave a SIMD: it waits).
#include "gsv_attention.h"

namespace gsv {
namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr int kRows = 128;  // rows (dq) or keys (dk, dv) of a workgroup, 32 a wave

// Rows of the other side in a tile.
template <typename T> constexpr int kOther = sizeof(T) == 2 ? 64 : 32;

struct BwdArgs {
    const void *out, *out_low, *dout;
    int64_t dout_row, dout_head;
    const float *lse;
    float *delta;   // (heads, q_tokens)
    double *dslope;  // (heads, n_slopes) partial sums
    void *dslopes;
    int n_slopes;    // the rows' places
    void *dq, *dk, *dv;
    int parts;             // workgroups that share a key tile's rows
    float *part_k, *part_v;  // (parts, k_tokens, kv_heads, dim) partial sums, with parts > 1
};

// A block's scores from the matrix product: capped (u: the tanh), with their bias.
template <typename T, bool FAR, int CAP>
__device__ __forceinline__ void finish_scores(f32x16 &w, f32x16 &u, const f32x16 &d, float in_cap,
                                              float cap, float far_unit) {
#pragma unroll
    for (int r = 0; r < 16; ++r) {
        if (CAP != kNoCap) {
            u[r] = tanh_of<T, CAP>(w[r] * in_cap);
            w[r] = cap * u[r];
        }
        if (FAR) w[r] = fmaf(-far_unit, d[r], w[r]);
    }
}

// dq, D and dslope.  A wave's lanes are query rows, as in the forward.
template <typename T, int DP, bool FAR, int CAP>
__global__ __launch_bounds__(256, sizeof(T) == 2 || DP <= 32 ? 2 : 1) void k_attention_dq(
    const AttnArgs a, const BwdArgs g) {
    constexpr int KB = kOther<T>, WAVES = 4;
    constexpr bool far = FAR, capped = CAP != kNoCap;
    typedef typename Elem<T>::frag frag;
    __shared__ __align__(1024) T sk[2][KB * DP];
    __shared__ __align__(1024) T sv[2][KB * DP];
    __shared__ __align__(16) typename Places<T>::Row spos[2][3 * KB];
    __shared__ double sums[4];

    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int h = blockIdx.x % a.heads, place_n = grid_place(a.heads);
    if (place_n >= a.places) return;
    const Place where = tile_place<kRows>(a.q_starts, a.scenes, a.q_tokens, place_n, a.slots);
    const Scene c = scene_of(a, where.scene, true);
    const int nq = c.q1 - c.q0;
    const int tiles = (nq + kRows - 1) / kRows;
    const bool fine = in_two_parts<T>(c.k1 - c.k0);
    const int hk = h / (a.heads / a.kv_heads);
    const T *kbase = static_cast<const T *>(a.k) + (int64_t)c.k0 * a.k_row + hk * a.k_head;
    const T *vbase = static_cast<const T *>(a.v) + (int64_t)c.k0 * a.v_row + hk * a.v_head;
    const float unit = capped ? kLog2e : a.scale * kLog2e;
    const float in_cap = capped ? a.scale / a.cap : 0.f;
    const float far_unit = slope_of(a, h) / (capped ? 1.f : a.scale);
    double dslope = 0.0;
    Tile<T, DP> at;
    at.plan(lane);
    Copy<T, DP, KB, WAVES> ck, cv;
    ck.plan(a.k_row, a.dim, wave, lane);
    cv.plan(a.v_row, a.dim, wave, lane);

    for (int tile = where.tile; tile < tiles; tile += where.step) {
        const int first = (tiles - 1 - tile) * kRows;
        const int i = first + wave * 32 + (lane & 31);
        const bool row = i < nq;
        const int64_t qi = c.q0 + i;
        frag q[DP / 16], dO[DP / 16];
        load_column<T, DP>(q, static_cast<const T *>(a.q) + qi * a.q_row + h * a.q_head, a.dim, row,
                           lane);
        load_column<T, DP>(dO, static_cast<const T *>(g.dout) + qi * g.dout_row + h * g.dout_head,
                           a.dim, row, lane);
        // D_i: where the row sees one key, out is that key's value and D_i its do_i.v_j bit for bit, so
        // that the row's gradients are exactly 0
        frag o[DP / 16];
        load_column<T, DP>(o, static_cast<const T *>(g.out) + (qi * a.heads + h) * a.dim, a.dim, row, lane);
        float delta = own_product<T>(o, dO, lane);
        if (g.out_low) {
            load_column<T, DP>(o, static_cast<const T *>(g.out_low) + (qi * a.heads + h) * a.dim, a.dim,
                               row, lane);
            delta += own_product<T>(o, dO, lane);
        }
        if (row && lane < 32) g.delta[(int64_t)h * a.q_tokens + qi] = delta;
        const float lse = row ? g.lse[(int64_t)h * a.q_tokens + qi] : INFINITY;
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
        const int most = key_limit(a, c, min(first + kRows, nq) - 1);
        const int mine = first + wave * 32 < nq
                             ? key_limit(a, c, min(first + wave * 32 + 32, nq) - 1) : 0;
        f32x16 dq[DP / 32] = {};
        float mean = 0.f, rest = 0.f;

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
            ck.start(sk[b], kbase + j0 * a.k_row, a.k_row, a.dim, left, a.keep, next_live, wave, lane);
            cv.start(sv[b], vbase + j0 * a.v_row, a.v_row, a.dim, left, a.keep, next_live, wave, lane);
            if (far && threadIdx.x < 3 * KB)
                gp = a.k_pos[(c.k0 + j0 + min((int)threadIdx.x % KB, left - 1)) * a.k_pos_row +
                             threadIdx.x / KB];
        };
        auto put = [&](int b) {
            if (far && threadIdx.x < 3 * KB) spos[b][threadIdx.x] = Places<T>::row(gp);
            tile_wait();
        };
        __syncthreads();
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
                const bool masked = j0 + KB > all || (KB == 64 ? ~live : (uint32_t)~live) != 0;
                float here = 0.f;
#pragma unroll 1
                for (int kb = 0; kb < KB / 32; ++kb) {
                    f32x16 d = {};
                    uint32_t seen = 0;
                    if (far) d = distances<T>(place, spos[b], KB, kb * 32, lane);
                    if (masked) {
                        seen = seen_rows(live, kb, limit - j0 - kb * 32, lane);
                        if (far)  // a masked key's position may be anything
#pragma unroll
                            for (int r = 0; r < 16; ++r)
                                if (!(seen & (1u << result_row(r)))) d[r] = 0.f;
                    }
                    f32x16 w = {}, u = {}, dp = {};
                    const T *kt = sk[b] + kb * 32 * DP, *vt = sv[b] + kb * 32 * DP;
#pragma unroll
                    for (int st = 0; st < DP / 16; ++st) {
                        w = mma(at.rows(kt, st), q[st], w);
                        dp = mma(at.rows(vt, st), dO[st], dp);
                    }
                    finish_scores<T, FAR, CAP>(w, u, d, in_cap, a.cap, far_unit);
                    if (masked)
#pragma unroll
                        for (int r = 0; r < 16; ++r)
                            if (!(seen & (1u << result_row(r)))) w[r] = -INFINITY;
#pragma unroll
                    for (int r = 0; r < 16; ++r) w[r] = fast_exp2(fmaf(w[r], unit, -lse));
#pragma unroll
                    for (int r = 0; r < 16; ++r) {
                        dp[r] = (dp[r] - delta) * w[r];
                        if (far) {
                            here = fmaf(dp[r], d[r], here);
                            if (sizeof(T) == 2) mean = fmaf(w[r], d[r], mean), rest += dp[r];
                        }
                        if (capped) dp[r] *= fmaf(-u[r], u[r], 1.f);
                    }
                    for (int part = 0; part <= (fine ? 1 : 0); ++part) {
                        if (part) dp = remainders<T>(dp);
                        Tile<T, DP> cols = at;
                        cols.forget();
#pragma unroll
                        for (int half = 0; half < 2; ++half) {
                            const frag ds = to_frag<T>(dp, half);
#pragma unroll
                            for (int e = 0; e < DP / 32; ++e)
                                dq[e] = mma(cols.columns(kt + half * 16 * DP, e, lane), ds, dq[e]);
                        }
                    }
                }
                dslope -= here;
            }
            if (more) put(b ^ 1);
            __syncthreads();
        }
        // D_i comes from an output whose weights were rounded to T.  dslope sums over all rows, and in
        // it a row's rest, sum_j p_ij (do_i.v_j - D_i), which ought to be 0, would meet its mean
        // distance: taken out, dslope is as good as float32 weights make it.
        if (far && sizeof(T) == 2) {
            rest += other_half(rest);
            dslope += rest * mean;
        }
        if (row)
            store_column<T, DP>(static_cast<T *>(g.dq) + (qi * a.heads + h) * a.dim, dq, a.scale, a.dim,
                                lane);
    }
    if (!far) return;
#pragma unroll
    for (int k = 1; k < 64; k <<= 1) dslope += __shfl_xor(dslope, k);
    if (lane == 0) sums[wave] = dslope;
    __syncthreads();
    if (threadIdx.x == 0)
        g.dslope[(int64_t)h * a.places + place_n] = sums[0] + sums[1] + sums[2] + sums[3];
}

// The same for few rows: 32 of them for a workgroup, whose waves take every W-th tile of 32 keys, as
// k_attention_fwd_few does.
template <typename T, int DP, bool FAR, int CAP>
__global__ __launch_bounds__((64 * kFewWaves<T, DP>)) void k_attention_dq_few(const AttnArgs a,
                                                                              const BwdArgs g) {
    constexpr int W = kFewWaves<T, DP>, KB = 32;
    constexpr bool far = FAR, capped = CAP != kNoCap;
    typedef typename Elem<T>::frag frag;
    static_assert(4 * KB * DP * sizeof(T) >= 32 * DP * sizeof(float), "sums reuse the tiles");
    __shared__ __align__(1024) T tiles[W][4 * KB * DP];  // a wave's keys and values, two buffers
    __shared__ __align__(16) typename Places<T>::Row spos[W][2][3 * KB];
    __shared__ float srest[W][32], smean[W][32];
    __shared__ double sums[W];

    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int h = blockIdx.x % a.heads, place_n = grid_place(a.heads);
    if (place_n >= a.places) return;
    const Place where = tile_place<32>(a.q_starts, a.scenes, a.q_tokens, place_n, a.slots);
    const Scene c = scene_of(a, where.scene, true);
    const int nq = c.q1 - c.q0, row_tiles = (nq + 31) / 32;
    const bool fine = in_two_parts<T>(c.k1 - c.k0);  // ds, as the forward's weights
    const int hk = h / (a.heads / a.kv_heads);
    const T *kbase = static_cast<const T *>(a.k) + (int64_t)c.k0 * a.k_row + hk * a.k_head;
    const T *vbase = static_cast<const T *>(a.v) + (int64_t)c.k0 * a.v_row + hk * a.v_head;
    const float unit = capped ? kLog2e : a.scale * kLog2e;
    const float in_cap = capped ? a.scale / a.cap : 0.f;
    const float far_unit = slope_of(a, h) / (capped ? 1.f : a.scale);
    double dslope = 0.0;
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
        frag q[DP / 16], dO[DP / 16];
        load_column<T, DP>(q, static_cast<const T *>(a.q) + qi * a.q_row + h * a.q_head, a.dim, row,
                           lane);
        load_column<T, DP>(dO, static_cast<const T *>(g.dout) + qi * g.dout_row + h * g.dout_head,
                           a.dim, row, lane);
        // D_i: where the row sees one key, out is that key's value and D_i its do_i.v_j bit for bit, so
        // that the row's gradients are exactly 0
        frag o[DP / 16];
        load_column<T, DP>(o, static_cast<const T *>(g.out) + (qi * a.heads + h) * a.dim, a.dim, row, lane);
        float delta = own_product<T>(o, dO, lane);
        if (g.out_low) {
            load_column<T, DP>(o, static_cast<const T *>(g.out_low) + (qi * a.heads + h) * a.dim, a.dim,
                               row, lane);
            delta += own_product<T>(o, dO, lane);
        }
        if (row && threadIdx.x < 32) g.delta[(int64_t)h * a.q_tokens + qi] = delta;
        const float lse = row ? g.lse[(int64_t)h * a.q_tokens + qi] : INFINITY;
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
        f32x16 dq[DP / 32] = {};
        float mean = 0.f, rest = 0.f;

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
            const bool masked = j0 + KB > all || (uint32_t)~live;
            const T *kt = sk + b * KB * DP, *vt = sv + b * KB * DP;
            f32x16 d = {}, w = {}, u = {}, dp = {};
            uint32_t seen = 0;
            float here = 0.f;
            if (far) d = distances<T>(place, spos[wave][b], KB, 0, lane);
            if (masked) {
                seen = seen_rows(live, 0, limit - j0, lane);
                if (far)  // a masked key's position may be anything
#pragma unroll
                    for (int r = 0; r < 16; ++r)
                        if (!(seen & (1u << result_row(r)))) d[r] = 0.f;
            }
#pragma unroll
            for (int st = 0; st < DP / 16; ++st) {
                w = mma(at.rows(kt, st), q[st], w);
                dp = mma(at.rows(vt, st), dO[st], dp);
            }
            finish_scores<T, FAR, CAP>(w, u, d, in_cap, a.cap, far_unit);
            if (masked)
#pragma unroll
                for (int r = 0; r < 16; ++r)
                    if (!(seen & (1u << result_row(r)))) w[r] = -INFINITY;
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const float p = fast_exp2(fmaf(w[r], unit, -lse));
                dp[r] = (dp[r] - delta) * p;
                if (far) {
                    here = fmaf(dp[r], d[r], here);
                    if (sizeof(T) == 2) mean = fmaf(p, d[r], mean), rest += dp[r];
                }
                if (capped) dp[r] *= fmaf(-u[r], u[r], 1.f);
            }
            for (int part = 0; part <= (fine ? 1 : 0); ++part) {
                if (part) dp = remainders<T>(dp);
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    const frag ds = to_frag<T>(dp, half);
#pragma unroll
                    for (int e = 0; e < DP / 32; ++e)
                        dq[e] = mma(at.columns(kt + half * 16 * DP, e, lane), ds, dq[e]);
                }
            }
            dslope -= here;
            if (more) put(b ^ 1);
        }
        if (far && sizeof(T) == 2) {  // a row's, over all waves (see k_attention_dq)
            rest += other_half(rest);
            mean += other_half(mean);
            if (lane < 32) srest[wave][lane] = rest, smean[wave][lane] = mean;
        }
        // row r's channel d at d * 32 + r
        float *so = reinterpret_cast<float *>(tiles[wave]);
#pragma unroll
        for (int e = 0; e < DP / 32; ++e)
#pragma unroll
            for (int r = 0; r < 16; ++r)
                so[(e * 32 + result_row(r) + 4 * (lane >> 5)) * 32 + (lane & 31)] = dq[e][r];
        __syncthreads();
        const int r = threadIdx.x & 31;
        if (far && sizeof(T) == 2 && threadIdx.x < 32) {
            float row_rest = 0.f, row_mean = 0.f;
#pragma unroll
            for (int w = 0; w < W; ++w) row_rest += srest[w][r], row_mean += smean[w][r];
            dslope += row_rest * row_mean;
        }
        if (first + r < nq) {
            T *to = static_cast<T *>(g.dq) + ((int64_t)(c.q0 + first + r) * a.heads + h) * a.dim;
            for (int d0 = (threadIdx.x >> 5) * 8; d0 < a.dim; d0 += 2 * W * 8) {
                typedef T t8 __attribute__((ext_vector_type(8)));
                t8 v;
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    float x = 0.f;
#pragma unroll
                    for (int w = 0; w < W; ++w)
                        x += reinterpret_cast<const float *>(tiles[w])[(d0 + e) * 32 + r];
                    v[e] = (T)(x * a.scale);
                }
                *reinterpret_cast<t8 *>(to + d0) = v;
            }
        }
    }
    if (!far) return;
#pragma unroll
    for (int k = 1; k < 64; k <<= 1) dslope += __shfl_xor(dslope, k);
    if (lane == 0) sums[wave] = dslope;
    __syncthreads();
    if (threadIdx.x == 0) {
        double sum = 0.0;
#pragma unroll
        for (int w = 0; w < W; ++w) sum += sums[w];
        g.dslope[(int64_t)h * a.places + place_n] = sum;
    }
}

// dk and dv.  A wave's lanes are keys; the rows of all query heads of the key head pass by, so a shared
// key head's gradient is summed in its wave's registers.
template <typename T, int DP, bool FAR, int CAP>
__global__ __launch_bounds__(256, DP <= 64 ? 2 : 1) void k_attention_dkv(const AttnArgs a, const BwdArgs g) {
    constexpr int QB = kOther<T>, WAVES = 4;
    typedef typename Elem<T>::frag frag;
    __shared__ __align__(1024) T sq[2][QB * DP];
    __shared__ __align__(1024) T sdo[2][QB * DP];
    __shared__ __align__(16) typename Places<T>::Row spos[2][3 * QB];
    __shared__ __align__(16) float srow[2][2 * QB];  // log sums, D

    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int hk = blockIdx.x % a.kv_heads, part = blockIdx.x / a.kv_heads % g.parts;
    const int place_n = grid_place(a.kv_heads * g.parts);
    if (place_n >= a.places) return;
    const Place where = tile_place<kRows>(a.k_starts, a.scenes, a.k_tokens, place_n, a.slots);
    const Scene c = scene_of(a, where.scene, false);
    const int nq = c.q1 - c.q0, nk = c.k1 - c.k0, off = nk - nq;
    const int group = a.heads / a.kv_heads;
    const int tiles = (nk + kRows - 1) / kRows;
    const bool fine = in_two_parts<T>(nk);  // weights and ds
    constexpr bool far = FAR, capped = CAP != kNoCap;
    const float unit = capped ? kLog2e : a.scale * kLog2e;
    const float in_cap = capped ? a.scale / a.cap : 0.f;

    Tile<T, DP> tl;
    tl.plan(lane);
    Copy<T, DP, QB, WAVES> cq, cd;
    cq.plan(a.q_row, a.dim, wave, lane);
    cd.plan(g.dout_row, a.dim, wave, lane);

    // the rows' kernel has ended: a head's partial sums of dslope, in order
    if (far && place_n == 0 && part == 0)
        for (int h = hk * group + wave; h < (hk + 1) * group; h += WAVES) {
            double sum = 0.0;
#pragma unroll 8
            for (int n = lane; n < g.n_slopes; n += 64) sum += g.dslope[(int64_t)h * g.n_slopes + n];
#pragma unroll
            for (int n = 1; n < 64; n <<= 1) sum += __shfl_xor(sum, n);
            if (lane == 0) {
                if (a.slopes_f32) static_cast<float *>(g.dslopes)[h] = (float)sum;
                else static_cast<bf16 *>(g.dslopes)[h] = (bf16)(float)sum;
            }
        }

    for (int tile = where.tile; tile < tiles; tile += where.step) {
        const int first = tile * kRows;
        const int j = first + wave * 32 + (lane & 31);
        const int64_t kj = c.k0 + j;
        const bool live = j < nk && kept(a, kj);
        frag k[DP / 16], v[DP / 16];
        load_column<T, DP>(k, static_cast<const T *>(a.k) + kj * a.k_row + hk * a.k_head, a.dim,
                           live, lane);
        load_column<T, DP>(v, static_cast<const T *>(a.v) + kj * a.v_row + hk * a.v_head, a.dim,
                           live, lane);
        float x = 0.f, y = 0.f, z = 0.f;
        if (far && live) {
            const float *p = a.k_pos + kj * a.k_pos_row;
            x = p[0], y = p[1], z = p[2];
        }
        Places<T> place;
        place.set(x, y, z, lane);
        // the first query row that sees this key; one that no row sees
        const int from = !live ? INT32_MAX : a.causal && j >= c.prefix ? j - off : 0;
        const bool dead_here = __any(!live);
        const int wave_from = a.causal && first + wave * 32 >= c.prefix ? first + wave * 32 - off : 0;
        const int wave_all = dead_here ? INT32_MAX
                             : a.causal && first + wave * 32 + 31 >= c.prefix
                                 ? first + wave * 32 + 31 - off : 0;
        const int q_from =
            a.causal && first >= c.prefix ? max(first - off, 0) / QB * QB : 0;
        const int per_head = q_from < nq ? (nq - q_from + QB - 1) / QB : 0;
        const int first_step = (int64_t)per_head * group * part / g.parts;
        const int steps = (int64_t)per_head * group * (part + 1) / g.parts;
        f32x16 dk[DP / 32] = {}, dv[DP / 32] = {};

        float gr[2] = {};
        auto fetch = [&](int b, int step) {
            const int h = hk * group + step % group, i0 = q_from + step / group * QB;
            const int64_t q0 = c.q0 + i0;
            const int left = nq - i0;
            cq.start(sq[b], static_cast<const T *>(a.q) + q0 * a.q_row + h * a.q_head, a.q_row, a.dim,
                     left, false, 0, wave, lane);
            cd.start(sdo[b], static_cast<const T *>(g.dout) + q0 * g.dout_row + h * g.dout_head,
                     g.dout_row, a.dim, left, false, 0, wave, lane);
            // log sums, D and positions of the rows, five arrays in turn
#pragma unroll
            for (int n = 0; n < 2; ++n) {
                const int at = n * 256 + threadIdx.x, r = at % QB, what = at / QB;
                if (what >= 5) continue;
                const int64_t row = q0 + min(r, left - 1);
                if (what < 2)
                    gr[n] = (what ? g.delta : g.lse)[(int64_t)h * a.q_tokens + row];
                else if (far)
                    gr[n] = a.q_pos[row * a.q_pos_row + what - 2];
                if (what == 0 && r >= left) gr[n] = INFINITY;  // no weights past the last row
            }
        };
        auto put = [&](int b) {
#pragma unroll
            for (int n = 0; n < 2; ++n)
                if (const int at = n * 256 + threadIdx.x; at >= 2 * QB && at < 5 * QB) {
                    if (far) spos[b][at - 2 * QB] = Places<T>::row(gr[n]);
                } else if (at < 2 * QB) {
                    srow[b][at] = gr[n];
                }
            tile_wait();
        };
        __syncthreads();
        if (first_step < steps) {
            fetch(0, first_step);
            put(0);
        }
        __syncthreads();
        int b = 0;
        for (int step = first_step; step < steps; ++step, b ^= 1) {
            const bool more = step + 1 < steps;
            if (more) fetch(b ^ 1, step + 1);
            const int i0 = q_from + step / group * QB;
            if (i0 + QB > wave_from && first + wave * 32 < nk) {
                const float slope = slope_of(a, hk * group + step % group);
                const float far_unit = capped ? slope : slope / a.scale;
                const bool masked = i0 < wave_all;
#pragma unroll 1
                for (int qb = 0; qb < QB / 32; ++qb) {
                    f32x16 d = {}, w = {}, u = {}, dp = {}, lse, delta;
                    if (far) d = distances<T>(place, spos[b], QB, qb * 32, lane);
#pragma unroll
                    for (int n = 0; n < 4; ++n) {
                        const float *p = srow[b] + qb * 32 + 8 * n + 4 * (lane >> 5);
                        const f32x4 ls = *reinterpret_cast<const f32x4 *>(p);
                        const f32x4 de = *reinterpret_cast<const f32x4 *>(p + QB);
#pragma unroll
                        for (int e = 0; e < 4; ++e) lse[4 * n + e] = ls[e], delta[4 * n + e] = de[e];
                    }
#pragma unroll
                    for (int st = 0; st < DP / 16; ++st) {
                        w = mma(tl.rows(sq[b] + qb * 32 * DP, st), k[st], w);
                        dp = mma(tl.rows(sdo[b] + qb * 32 * DP, st), v[st], dp);
                    }
                    finish_scores<T, FAR, CAP>(w, u, d, in_cap, a.cap, far_unit);
                    if (masked) {
                        const int lo = from == INT32_MAX ? from : from - i0 - qb * 32 - 4 * (lane >> 5);
#pragma unroll
                        for (int r = 0; r < 16; ++r)
                            if (result_row(r) < lo) w[r] = -INFINITY;
                    }
#pragma unroll
                    for (int r = 0; r < 16; ++r) {
                        w[r] = fast_exp2(fmaf(w[r], unit, -lse[r]));
                        dp[r] = (dp[r] - delta[r]) * w[r];
                        if (capped) dp[r] *= fmaf(-u[r], u[r], 1.f);
                    }
                    for (int part = 0; part <= (fine ? 1 : 0); ++part) {
                        if (part) w = remainders<T>(w), dp = remainders<T>(dp);
                        Tile<T, DP> cols = tl;
                        cols.forget();
#pragma unroll
                        for (int half = 0; half < 2; ++half) {
                            const frag p = to_frag<T>(w, half), ds = to_frag<T>(dp, half);
                            const int at = (qb * 32 + half * 16) * DP;
#pragma unroll
                            for (int n = 0; n < DP / 32; ++n) {
                                dv[n] = mma(cols.columns(sdo[b] + at, n, lane), p, dv[n]);
                                dk[n] = mma(cols.columns(sq[b] + at, n, lane), ds, dk[n]);
                            }
                        }
                    }
                }
            }
            if (more) put(b ^ 1);
            __syncthreads();
        }
        if (j < nk) {
            const int64_t at = (kj * a.kv_heads + hk) * a.dim;
            if (g.parts == 1) {
                store_column<T, DP>(static_cast<T *>(g.dk) + at, dk, a.scale, a.dim, lane);
                store_column<T, DP>(static_cast<T *>(g.dv) + at, dv, 1.f, a.dim, lane);
            } else {
                const int64_t all = (int64_t)a.k_tokens * a.kv_heads * a.dim * part;
                store_column<float, DP>(g.part_k + all + at, dk, a.scale, a.dim, lane);
                store_column<float, DP>(g.part_v + all + at, dv, 1.f, a.dim, lane);
            }
        }
    }
}

// The parts' sums of dk and dv, in order: four values a thread, 16 bytes of each part.  Bytes bound
// it: four parts of 10,007 tokens, 4 heads of 128 (164 MB read, from the last-level cache in part) take 27 us.
template <typename T>
__global__ __launch_bounds__(256) void k_parts_sum(const float *__restrict__ pk,
                                                   const float *__restrict__ pv, int parts,
                                                   int64_t fours, T *__restrict__ dk,
                                                   T *__restrict__ dv) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= 2 * fours) return;
    const bool second = i >= fours;
    const int64_t at = second ? i - fours : i;
    const f32x4 *p = reinterpret_cast<const f32x4 *>(second ? pv : pk) + at;
    f32x4 sum = p[0];
    for (int n = 1; n < parts; ++n) sum += p[n * fours];
    typedef T t4 __attribute__((ext_vector_type(4)));
    t4 r;
#pragma unroll
    for (int e = 0; e < 4; ++e) r[e] = (T)sum[e];
    reinterpret_cast<t4 *>(second ? dv : dk)[at] = r;
}

size_t delta_bytes(const AttnArgs &a) {
    return ((size_t)a.heads * a.q_tokens * sizeof(float) + 255) / 256 * 256;
}

// Parts of a key tile's rows: more workgroups where the tiles alone leave CUs idle or, as under a
// causal mask, a few of them have most of the work.  About four rounds of workgroups at one a CU
// (128 channels), one at two a CU; eight parts at most, each with four tiles of a mean scene's
// rows at least (sizes alone decide: the longest scene's length is a hint that changes no sum of these).
// Partial sums then pass through memory.  Training, against one part: 10,007 tokens of 4 causal scenes, 16
// heads on 4, 128 channels 1,318 and 1,673 us, 3 scenes of 3,000, 8 heads of 64 on 1 602 and 1,359; 8 heads of 64
// on 8, 8 scenes of 1,000, gain nothing (189 and 190).
int bwd_parts(const AttnArgs &a, int elem) {
    const int64_t tiles = ((int64_t)a.k_tokens / kRows + a.scenes) * a.kv_heads;
    const int64_t want = (a.dim > 64 ? 1024 : 512) / tiles + (a.dim > 64);
    const int64_t rows = elem == GSV_BF16 ? kOther<bf16> : kOther<float>;
    const int64_t most = (int64_t)a.q_tokens / a.scenes * (a.heads / a.kv_heads) / (4 * rows);
    return (int)imax64(1, imin64(imin64(want, most), 8));
}

size_t parts_bytes(const AttnArgs &a, int parts) {
    return parts == 1 ? 0 : sizeof(float) * parts * a.k_tokens * a.kv_heads * a.dim;  // of 32 bytes each
}

// The two launches: of the rows' places (a->places, a->slots) and of the keys' in their parts.
struct BwdPlan {
    dim3 rows, keys;
    int key_places, key_slots, parts;
};
int bwd_plan(const gsv_attention *args, AttnArgs *a, BwdPlan *p) {
    const int st = attention_args(args, a);
    if (st != GSV_OK) return st;
    p->parts = bwd_parts(*a, args->dtype);
    const int rows = attention_few(*a) ? 32 : kRows;
    const int64_t slots = attention_slots(*a, a->q_tokens, args->longest_q, rows);
    const int64_t key_slots = attention_slots(*a, a->k_tokens, args->longest_k, kRows);
    const int64_t places = attention_places(*a, a->q_tokens, rows, slots);
    const int64_t key_places = attention_places(*a, a->k_tokens, kRows, key_slots);
    a->slots = (int)slots, a->places = (int)places;
    p->key_slots = (int)key_slots, p->key_places = (int)key_places;
    return attention_grid(places, a->heads, &p->rows) &&
                   attention_grid(key_places, (int64_t)a->kv_heads * p->parts, &p->keys)
               ? GSV_OK : GSV_ERR_SIZE_OVERFLOW;
}

struct Backward {
    const AttnArgs &a;
    const BwdArgs &g;
    const BwdPlan &plan;
    hipStream_t st;
    template <typename T, int DP, bool FAR, int CAP> void run() const {
        if (a.q_tokens > 0 && attention_few(a))
            hipLaunchKernelGGL((k_attention_dq_few<T, DP, FAR, CAP>), plan.rows,
                               dim3(64 * kFewWaves<T, DP>), 0, st, a, g);
        else if (a.q_tokens > 0)
            hipLaunchKernelGGL((k_attention_dq<T, DP, FAR, CAP>), plan.rows, dim3(256), 0, st, a, g);
        AttnArgs k = a;
        k.slots = plan.key_slots, k.places = plan.key_places;
        hipLaunchKernelGGL((k_attention_dkv<T, DP, FAR, CAP>), plan.keys, dim3(256), 0, st, k, g);
        if (g.parts == 1 || a.k_tokens == 0) return;
        const int64_t fours = (int64_t)a.k_tokens * a.kv_heads * a.dim / 4;
        hipLaunchKernelGGL(k_parts_sum<T>, dim3((unsigned)((2 * fours + 255) / 256)), dim3(256), 0, st,
                           g.part_k, g.part_v, g.parts, fours, static_cast<T *>(g.dk),
                           static_cast<T *>(g.dv));
    }
};

}  // namespace
}  // namespace gsv

using namespace gsv;

extern "C" int gsv_attention_bwd_workspace_bytes(const gsv_attention *args, size_t *bytes) {
    AttnArgs a;
    BwdPlan plan;
    if (!bytes) return GSV_ERR_INVALID_ARGUMENT;
    const int st = bwd_plan(args, &a, &plan);
    if (st != GSV_OK) return st;
    *bytes = delta_bytes(a) + 2 * parts_bytes(a, plan.parts) +
             (a.slopes ? sizeof(double) * a.places * a.heads : 0);
    return GSV_OK;
}

extern "C" int gsv_attention_bwd(const gsv_attention *args, const void *out, const void *out_low,
                                 const float *lse, const void *dout, int64_t dout_row, int64_t dout_head, void *dq,
                                 void *dk, void *dv, void *dslopes, void *workspace,
                                 size_t workspace_bytes, void *stream) {
    AttnArgs a;
    BwdPlan plan;
    size_t need;
    int st = bwd_plan(args, &a, &plan);
    if (st != GSV_OK) return st;
    if ((st = gsv_attention_bwd_workspace_bytes(args, &need)) != GSV_OK) return st;
    if (need > workspace_bytes) return GSV_ERR_WORKSPACE_TOO_SMALL;
    const int64_t chunk = args->dtype == GSV_BF16 ? 8 : 4;
    dout_row = used_stride(dout_row, a.q_tokens);
    dout_head = used_stride(dout_head, a.heads);
    if (dout_row % chunk || dout_head % chunk || dout_row < 0 ||
        dout_row * (16 / chunk) > kMaxRowBytes)
        return GSV_ERR_INVALID_ARGUMENT;
    if (a.q_tokens > 0 && (!out || !lse || !dout || !dq || !workspace)) return GSV_ERR_INVALID_ARGUMENT;
    if ((a.k_tokens > 0 && (!dk || !dv)) || (a.slopes && !dslopes)) return GSV_ERR_INVALID_ARGUMENT;
    const void *ptrs[] = {out, out_low, dout, dq, dk, dv, workspace};
    for (const void *p : ptrs)
        if (reinterpret_cast<uintptr_t>(p) % 16) return GSV_ERR_INVALID_ARGUMENT;
    float *delta = static_cast<float *>(workspace);
    char *next = static_cast<char *>(workspace) + delta_bytes(a);
    float *part_k = reinterpret_cast<float *>(next);
    float *part_v = reinterpret_cast<float *>(next + parts_bytes(a, plan.parts));
    double *slopes = reinterpret_cast<double *>(next + 2 * parts_bytes(a, plan.parts));
    const BwdArgs g{out, out_low, dout, dout_row, dout_head, lse, delta, slopes, dslopes,
                    a.q_tokens > 0 ? a.places : 0, dq, dk, dv, plan.parts, part_k, part_v};
    Backward f{a, g, plan, as_stream(stream)};
    attention_variant(a, args->dtype, f);
    return check_launch();
}
