// gsv_attention.h — what the attention kernels share: the two element types, the
// fragments of their matrix instructions, tiles in LDS, and the rows' masks.
//
// Products run on v_mfma_f32_32x32x16_bf16, or on eight v_mfma_f32_32x32x2_f32 for
// float32.  Lane l of a wave holds, of the left operand, row l % 32 and the eight
// contraction indices 8 (l / 32) + e; of the right operand, column l % 32 and the same
// indices; of the result, column l % 32 and the rows 8 (r / 4) + 4 (l / 32) + r % 4,
// r = 0 .. 15.  (A sum does not depend on which index is called e: the float32 form
// feeds element e of both fragments to step e.)  So a 32 x 32 result is, eight registers
// at a time, the right operand of a further product whose contraction runs over the
// result's rows, in the order {4 g .. 4 g + 3, 8 + 4 g .. 8 + 4 g + 3}, g = l / 32: the
// weights go from the softmax into their product with V in registers, and only
// the left operand (V transposed) has to be read in that order (tr_frag).
#pragma once

#include "gsv_device.h"

// m0 is named as written by the copies below; the compiler warns that it is a reserved register
#pragma clang diagnostic ignored "-Winline-asm"

namespace gsv {

typedef __bf16 bf16;
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));

template <typename T> struct Elem;
template <> struct Elem<bf16> {
    typedef bf16x8 frag;
    static constexpr int kChunk = 8;  // elements of a 16-byte chunk
};
template <> struct Elem<float> {
    typedef f32x8 frag;
    static constexpr int kChunk = 4;
};

__device__ __forceinline__ f32x16 mma(bf16x8 a, bf16x8 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x16 mma(f32x8 a, f32x8 b, f32x16 c) {
#pragma unroll
    for (int e = 0; e < 8; ++e) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a[e], b[e], c, 0, 0, 0);
    return c;
}

// Eight results as a right operand, rounded to T.  bfloat16 keeps 8 bits of a weight:
// an error of 2^-9 of each term, as large as the rounding of the result itself.
template <typename T> __device__ __forceinline__ typename Elem<T>::frag to_frag(f32x16 s, int half) {
    typename Elem<T>::frag f;
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] = (T)s[half * 8 + e];
    return f;
}

// The eight contraction indices of one lane: 16 bytes (bf16) or 32 (float32) of a row.
__device__ __forceinline__ bf16x8 row_frag(const bf16 *p) {
    return *reinterpret_cast<const bf16x8 *>(p);
}
__device__ __forceinline__ f32x8 row_frag(const float *p) {
    const f32x4 a = *reinterpret_cast<const f32x4 *>(p), b = *reinterpret_cast<const f32x4 *>(p + 4);
    return f32x8{a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
}

// A tile of one head in LDS: rows of DP elements, no padding (the copies below fill 1024
// bytes in lane order), chunk c of row r at place c ^ turn(r).  turn spreads what one access reads over
// all 64 banks: chunk c of eight rows in sequence, and four chunks of four rows in sequence.  It
// depends on the row's low four bits.
template <typename T, int DP> struct Tile {
    static constexpr int kPerRow = DP / Elem<T>::kChunk, kRowBytes = kPerRow * 16;
    static __device__ __forceinline__ int turn(int r) {
        if constexpr (kPerRow == 4) return (r >> 2) & 3;
        if constexpr (kPerRow == 8) return (r & 2) << 1 | (r & 4) >> 1 | (r & 8) >> 3;
        return (r & 3) << 2 | ((r >> 2) & 3);
    }
    uint32_t row_at, col_at;  // byte offsets of the lane's parts below
    __device__ __forceinline__ void plan(int lane) {
        const int r = lane & 31, g = lane >> 5;
        row_at = r * kRowBytes + (((sizeof(T) == 2 ? g : 2 * g) ^ turn(r)) << 4);
        const int i = lane & 15, r4 = 4 * g + (i >> 2);
        col_at = r4 * kRowBytes + ((((lane >> 3) & 2) + ((i & 3) >> 1)) ^ turn(r4)) * 16 + (i & 1) * 8;
    }
    // At 128 channels, lets the compiler know nothing of the columns' offset in a loop over the parts of the
    // weights: it would form all their addresses before the loop, and keep them in registers there are
    // not.  (Below they fit; formed again for each block, they cost the forward 4 %.)
    __device__ __forceinline__ void forget() {
        if constexpr (DP == 128) asm volatile("" : "+v"(col_at));
    }
    // An address in LDS, as a number.  A tile starts at a multiple of 1024 bytes, so a lane's part
    // `bits` from its first is (base + at) ^ bits or base + (at ^ bits).  The first form keeps one
    // register, the second one for each part and saves an instruction a read (5 % of the training time
    // of 16,000 tokens, 64 channels, when it was chosen); at 128 channels its registers do not fit (the
    // rows' kernel of the backward took 590 instead of 440 us for 10,007 tokens).
    static __device__ __forceinline__ uint32_t part(uint32_t base, uint32_t at, uint32_t bits) {
        return DP == 128 ? (base + at) ^ bits : base + (at ^ bits);
    }
    template <typename V> static __device__ __forceinline__ V read(uint32_t at) {
        return *(const __attribute__((address_space(3))) V *)(uintptr_t)at;
    }
    static __device__ __forceinline__ uint32_t base(const T *tile) {
        return (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) T *)tile;
    }
    // Columns 16 st + 8 (lane / 32) .. + 7 of row lane % 32; the tile from a multiple of 16 rows on.
    __device__ __forceinline__ typename Elem<T>::frag rows(const T *tile, int st) const {
        const uint32_t first = base(tile);
        if constexpr (sizeof(T) == 2) {
            return read<bf16x8>(part(first, row_at, st << 5));
        } else {
            const f32x4 a = read<f32x4>(part(first, row_at, st << 6));
            const f32x4 b = read<f32x4>(part(first, row_at, st << 6 | 16));
            return f32x8{a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
        }
    }
    // The transposed left operand: column 32 block + lane % 32, rows 4 g .. 4 g + 3 and 8 + 4 g ..
    // 8 + 4 g + 3.  For 16-bit elements ds_read_b64_tr_b16 does it: of 16 lanes, lane i gives the
    // address of row i / 4, columns 4 (i % 4) .. + 3, and receives column i of the four rows.
    __device__ __forceinline__ typename Elem<T>::frag columns(const T *tile, int block, int lane) const {
        if constexpr (sizeof(T) == 2) {
            typedef __attribute__((address_space(3))) s16x4 *lds_ptr;
            const uint32_t first = base(tile);
            const s16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                (lds_ptr)(uintptr_t)part(first, col_at, block << 6));
            const s16x4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                (lds_ptr)(uintptr_t)(part(first, col_at, block << 6 | turn(8) << 4) + 8 * kRowBytes));
            const bf16x4 u = __builtin_bit_cast(bf16x4, a), v = __builtin_bit_cast(bf16x4, b);
            return bf16x8{u[0], u[1], u[2], u[3], v[0], v[1], v[2], v[3]};
        } else {
            f32x8 f;
            const int chunk = 8 * block + ((lane & 31) >> 2);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const int r = 4 * (lane >> 5) + (e & 3) + 8 * (e >> 2);
                f[e] = read<float>(base(tile) + r * kRowBytes + ((chunk ^ turn(r)) << 4) + (lane & 3) * 4);
            }
            return f;
        }
    }
};

// The sum of a fragment's weights as the product with V takes them, rounded: a row divided by this
// sum is a mean of values, so that where one key has all the weight its value comes out exactly.
__device__ __forceinline__ float add_weights(bf16x8 p, float sum) {
    typedef bf16 bf16x2 __attribute__((ext_vector_type(2)));
    const bf16x2 one = {(bf16)1.f, (bf16)1.f};
#pragma unroll
    for (int e = 0; e < 8; e += 2) sum = __builtin_amdgcn_fdot2_f32_bf16(bf16x2{p[e], p[e + 1]}, one, sum, false);
    return sum;
}
__device__ __forceinline__ float add_weights(f32x8 p, float sum) {
#pragma unroll
    for (int e = 0; e < 8; ++e) sum += p[e];
    return sum;
}

__device__ __forceinline__ float fast_exp2(float x) { return __builtin_amdgcn_exp2f(x); }

// tanh.  For bfloat16 scores 1 - 2 / (exp(2 x) + 1): absolute error 2^-22.7, far
// below the 2^-9 of the operands; ends at +-1 where exp overflows or vanishes.  Times a cap of
// thousands that error is one of the scores (all near 0 then): past kWideCap, where it is 2^-12.7, tanhf.
constexpr float kWideCap = 1024.f;
enum Cap { kNoCap, kCap, kAnyCap };
template <typename T, int CAP> __device__ __forceinline__ float tanh_of(float x) {
    if constexpr (sizeof(T) == 4 || CAP == kAnyCap) return tanhf(x);
    const float e = fast_exp2(2.885390082f * x);  // 2 log2(e)
    return 1.f - 2.f * __builtin_amdgcn_rcpf(e + 1.f);
}

__device__ __forceinline__ float other_half(float x) { return __shfl_xor(x, 32); }

// Everything a launch of the packed attention needs; strides in elements.
struct AttnArgs {
    const void *q, *k, *v;
    int64_t q_row, q_head, k_row, k_head, v_row, v_head;
    int q_tokens, k_tokens, heads, kv_heads, dim, scenes;
    const int *q_starts, *k_starts, *prefix;
    int causal;
    float scale, cap;
    const float *q_pos, *k_pos;  // rows of x, y, z
    int64_t q_pos_row, k_pos_row;
    const void *slopes;
    int slopes_f32;
    const void *keep;
    int keep_bytes;
    int places;  // workgroups for each head
    int slots;   // places a scene where they go by scene, 0 where they are tiles (tile_place)
};

// The stride of an axis of one entry is never used, whatever a caller's view holds there.
inline int64_t used_stride(int64_t stride, int64_t entries) { return entries > 1 ? stride : 0; }

// Checks the C arguments and lays them out for a launch.
int attention_args(const gsv_attention *in, AttnArgs *a);

// The kernel variant of a call: element type, channels (up to 32, 64 or 128; the columns past
// dim are zeros), distance bias, score cap (with another tanh past kWideCap for bfloat16).
template <typename T, int DP, typename F> void attention_options(const AttnArgs &a, F &f) {
    const bool far = a.slopes, capped = a.cap > 0.f;
    if constexpr (sizeof(T) == 2)
        if (a.cap > kWideCap)
            return far ? f.template run<T, DP, true, kAnyCap>() : f.template run<T, DP, false, kAnyCap>();
    if (far && capped) f.template run<T, DP, true, kCap>();
    else if (far) f.template run<T, DP, true, kNoCap>();
    else if (capped) f.template run<T, DP, false, kCap>();
    else f.template run<T, DP, false, kNoCap>();
}
template <typename T, typename F> void attention_channels(const AttnArgs &a, F &f) {
    if (a.dim <= 32) attention_options<T, 32>(a, f);
    else if (a.dim <= 64) attention_options<T, 64>(a, f);
    else attention_options<T, 128>(a, f);
}
template <typename F> void attention_variant(const AttnArgs &a, int dtype, F &f) {
    if (dtype == GSV_BF16) attention_channels<bf16>(a, f);
    else attention_channels<float>(a, f);
}

// Workgroups of 128 rows of one head, all scenes'.
inline int64_t attention_tiles(const AttnArgs &a) {
    return ((int64_t)a.q_tokens / 128 + a.scenes) * a.heads;
}
// Whether a wave takes two heads (for their distances): where the workgroups of one head pass a round of
// three a CU, so that half as many, each 1.7 times as long, end sooner.  Not under a causal mask, whose
// workgroups differ in length and fill the rounds' ends better the smaller they are, nor for short scenes, whose
// last tiles are part empty.  8 heads of 64, forward: one scene of 12,000 tokens (752 workgroups) takes 687 us in
// pairs and 585 without, 14,000 (880) 830 and 920, 16,000 913 and 1,059, and causal 703 and 521; 8 scenes of
// 2,000 (1,064) 133 and 148; 32 scenes of 1,000, 16 heads 273 and 293; 200 scenes of 200 81 and 76.
inline bool attention_pairs(const AttnArgs &a) {
    return a.heads % 2 == 0 && !a.causal && attention_tiles(a) > 3 * 256 && a.q_tokens / a.scenes >= 512;
}
// Whether rows are so few that the waves of a workgroup share them and split the keys: below three
// workgroups of 128 rows for four CUs.  8 heads of 64, one scene: 500 tokens forward 10 us so and 21
// otherwise, 2,000 35 and 68, 2,900 68 and 94, 4,000 111 and 112, where training takes 455 and 381.
inline bool attention_few(const AttnArgs &a) { return attention_tiles(a) < 192; }
// Whether a scene's bfloat16 weights and ds enter the products in two parts (16 bits): where its rows see
// too few keys to average their roundings.  The gradients of scenes of two tokens are 0.0017 off (2-norm:
// the rounding of the results) so and 0.0025 in one part, of 64 tokens 0.0017 and 0.0024.  Its own keys alone
// decide, so that no other scene of the batch changes how exact it is.  500 scenes of 120 tokens, 8 heads
// of 64: 78 us (forward) and 461 (training), in one part 67 and 445.  Long scenes stay with one part, 0.0024
// off: 16,000 tokens train in 3.76 ms so and 5.00 in two.
template <typename T> __device__ __forceinline__ bool in_two_parts(int keys) {
    return sizeof(T) == 2 && keys < 128;
}
// The waves of such a workgroup: as many as the LDS holds their tiles.
template <typename T, int DP> constexpr int kFewWaves = DP * sizeof(T) > 256 ? 2 : 4;

// Places a scene of one side where fewer workgroups come of it than of its tiles (tile_place), else 0.
// longest: rows of the longest scene, if known; places go by it, and no result.
inline int64_t attention_slots(const AttnArgs &a, int tokens, int longest, int rows) {
    if (longest < 1 || longest > tokens) return 0;
    const int64_t slots = (longest + rows - 1) / rows;
    return slots * a.scenes < (int64_t)tokens / rows + a.scenes ? slots : 0;
}
inline int64_t attention_places(const AttnArgs &a, int tokens, int rows, int64_t slots) {
    return slots ? slots * a.scenes : (int64_t)tokens / rows + a.scenes;
}
// A launch of a workgroup for each place and `each` heads (or parts of them), which vary fastest: with
// eight (or a multiple) of them each XCD's L2 holds the keys of its own heads.  The places past
// four million workgroups are the grid's y axis.  False where that would pass its limit.
inline bool attention_grid(int64_t places, int64_t each, dim3 *grid) {
    if (each > (1 << 22)) return false;
    const int64_t x = imin64(places, (1 << 22) / each), y = (places + x - 1) / x;
    *grid = dim3((unsigned)(x * each), (unsigned)y);
    return y <= 65535;
}
__device__ __forceinline__ int grid_place(int each) {
    return blockIdx.y * (gridDim.x / each) + blockIdx.x / each;
}

// One scene's rows.  Starts are clamped to the arrays, the first scene begins at row 0
// and the last ends with the arrays: whatever the starts hold, each access stays inside.
struct Scene {
    int q0, q1, k0, k1, prefix;
};
__device__ __forceinline__ int scene_start(const int *starts, int s, int scenes, int tokens) {
    if (s <= 0) return 0;
    if (s >= scenes) return tokens;
    return min(max(starts[s], 0), tokens);
}
// Scene s and its rows first .. last - 1 of one side.
struct Span {
    int s, first, last;
};
__device__ __forceinline__ Span span(const int *starts, int s, int scenes, int tokens) {
    const int first = __builtin_amdgcn_readfirstlane(scene_start(starts, s, scenes, tokens));
    return {s, first, max(__builtin_amdgcn_readfirstlane(scene_start(starts, s + 1, scenes, tokens)), first)};
}
// What a workgroup does on one side: of a scene's tiles of ROWS rows, `tile` and every `step` further.
struct Place {
    Span scene;
    int tile, step;
};
// By tiles (slots 0), scene after scene: scene s has those from first / ROWS + s on.  That leaves it one
// for each ROWS rows it begins, and often one without rows; a launch then needs to know nothing of the
// scenes but their number, however their lengths differ, and a scene's longest rows start first.  The scene of
// a place is looked for among the 64 around where it is if all have one length, by one load, and past
// those by a search.  By slots, a scene has as many as its launch gives each.
// Training, 8 heads of 64: 500 scenes of 128 tokens take 453 us in one slot each and 756 by tiles, of
// which half are without rows (and 5,674 in slots for as many rows as there are); one scene of
// 16,000 beside 999 of 10 takes 4.1 ms by tiles, and 20 in 125 slots each; 16 of 1,500 and 2,300 in turn,
// 16 heads of 128 on 4, 4.2 ms by 253 tiles and 5.3 in 288 slots.
template <int ROWS>
__device__ __forceinline__ Place tile_place(const int *starts, int scenes, int tokens, int n, int slots) {
    if (slots) return {span(starts, n % scenes, scenes, tokens), n / scenes, slots};
    constexpr int kOnce = 1 << 30;
    if (scenes == 1) return {{0, 0, tokens}, n, kOnce};
    const int lane = threadIdx.x & 63;
    const int guess = (int)((float)n * ((float)scenes / (float)(tokens / ROWS + scenes)));
    const int lo = __builtin_amdgcn_readfirstlane(max(min(guess - 32, scenes - 64), 0));
    const int start = scene_start(starts, lo + lane, scenes, tokens);
    int at = __popcll(__ballot(lo + lane < scenes && start / ROWS + lo + lane <= n));
    Span s;
    if ((at == 0 && lo > 0) || (at == 64 && lo + 64 < scenes)) {
        const auto before = [&](int s) { return scene_start(starts, s, scenes, tokens) / ROWS + s; };
        s = span(starts, last_at_most(scenes, n, before), scenes, tokens);
    } else {
        at = __builtin_amdgcn_readfirstlane(max(at, 1));
        const int first = __builtin_amdgcn_readlane(start, at - 1);
        const int last = at < 64 ? __builtin_amdgcn_readlane(start, at) : tokens;
        s = {lo + at - 1, first, max(last, first)};
    }
    const int tile = n - (s.first / ROWS + s.s);
    return {s, tile >= 0 ? tile : kOnce, kOnce};  // (below 0 only where starts do not ascend)
}
// The scene whose rows of one side are known; the other side's are the same where both have the same starts.
__device__ __forceinline__ Scene scene_of(const AttnArgs &a, const Span &p, bool queries) {
    const bool same = a.q_starts == a.k_starts && a.q_tokens == a.k_tokens;
    const Span q = queries || same ? p : span(a.q_starts, p.s, a.scenes, a.q_tokens);
    const Span k = !queries || same ? p : span(a.k_starts, p.s, a.scenes, a.k_tokens);
    Scene c{q.first, q.last, k.first, k.last, 0};
    if (a.prefix) c.prefix = min(max(__builtin_amdgcn_readfirstlane(a.prefix[p.s]), 0), c.k1 - c.k0);
    return c;
}
// Keys of the scene that its query row i sees (those below the limit): with the causal mask
// a prefix or what precedes the query, whose rows end where the keys end.
__device__ __forceinline__ int key_limit(const AttnArgs &a, const Scene &c, int i) {
    const int n = c.k1 - c.k0;
    if (!a.causal) return n;
    return min(max(c.prefix, n - (c.q1 - c.q0 - i) + 1), n);
}
__device__ __forceinline__ bool kept(const AttnArgs &a, int64_t row) {
    if (!a.keep) return true;
    return a.keep_bytes == 1 ? static_cast<const uint8_t *>(a.keep)[row] != 0
                             : static_cast<const int *>(a.keep)[row] != 0;
}
__device__ __forceinline__ float slope_of(const AttnArgs &a, int h) {
    if (!a.slopes) return 0.f;
    return a.slopes_f32 ? static_cast<const float *>(a.slopes)[h]
                        : (float)static_cast<const bf16 *>(a.slopes)[h];
}

// The widest row stride: 64 rows have to lie within a buffer descriptor's 2^31 bytes.
constexpr int64_t kMaxRowBytes = 1 << 24;

// Copies ROWS rows of one head from global memory into a tile, asynchronously and past the
// registers (buffer_load_dwordx4 ... lds: a wave's 64 chunks of 16 bytes, to LDS in lane order).
// The buffer descriptor ends with the last live row: rows past it, columns from dim up to DP and
// rows that a mask drops are given offsets past its end, where the hardware reads zeros, so that no
// value of theirs, NaN among them, meets a weight of 0.  tile_wait() before the barrier behind
// which the tile is read.
template <typename T, int DP, int ROWS, int WAVES> struct Copy {
    static constexpr int kPerRow = DP / Elem<T>::kChunk, kAll = ROWS * kPerRow / 64;
    static constexpr int kN = (kAll + WAVES - 1) / WAVES;
    // Past every descriptor's end, also with a tile's rows added (offsets are unsigned).
    static constexpr uint32_t kNowhere = INT32_MAX - 15;
    // Rows between a wave's copies.  Where that is a multiple of 16 its chunks lie alike in them
    // (turn), and one offset a lane serves all.
    static constexpr int kStep = WAVES * 64 / kPerRow;
    static constexpr bool kAlike = kStep % 16 == 0;
    uint32_t at[kAlike ? 1 : kN];
    static __device__ __forceinline__ int row_of(int i, int wave, int lane) {
        return ((i * WAVES + wave) * 64 + lane) / kPerRow;
    }
    __device__ __forceinline__ void plan(int64_t stride, int dim, int wave, int lane) {
#pragma unroll
        for (int i = 0; i < (kAlike ? 1 : kN); ++i) {
            const int row = row_of(i, wave, lane);
            const int col = ((lane % kPerRow) ^ Tile<T, DP>::turn(row)) * Elem<T>::kChunk;
            at[i] = col < dim ? (uint32_t)(row * (int)stride + col) * (uint32_t)sizeof(T) : kNowhere;
        }
    }
    // rows: live rows from base on, 1 at least; with `some`, those whose bit is set in `live`
    __device__ __forceinline__ void start(T *tile, const T *base, int64_t stride, int dim, int rows,
                                          bool some, uint64_t live, int wave, int lane) const {
        // (the same in all lanes, but loaded in a loop: said so, it lies in scalar registers)
        const int bytes = __builtin_amdgcn_readfirstlane(((min(rows, ROWS) - 1) * (int)stride + dim) * (int)sizeof(T));
        const uint64_t p = reinterpret_cast<uintptr_t>(base);
        const uint64_t first_byte = (uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(p >> 32)) << 32 |
                                    (uint32_t)__builtin_amdgcn_readfirstlane((int)p);
        const auto rsrc = __builtin_amdgcn_make_buffer_rsrc(reinterpret_cast<void *>(first_byte), 0, bytes, 0x00020000);
        typedef __attribute__((address_space(3))) const void *lds_ptr;
        // the later rows' offsets and bits come from the first's here, not from registers kept all
        // along (at 128 channels those would not fit)
        uint32_t first = at[0];
        asm volatile("" : "+v"(first));
        const uint64_t from = some ? live >> row_of(0, wave, lane) : ~0ull;
#pragma unroll
        for (int i = 0; i < kN; ++i) {
            if (kAll % WAVES && i * WAVES + wave >= kAll) break;
            uint32_t x = kAlike ? first + (uint32_t)(i * kStep * (int)stride * (int)sizeof(T)) : at[i];
            if (!((from >> (i * kStep)) & 1)) x = kNowhere;
            // As assembly, without register outputs: for the builtin the compiler waits before
            // every read of LDS, also of the other buffer.  The only readers of this tile
            // stand behind tile_wait() and a barrier.
            asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds"
                         :
                         : "s"((uint32_t)(uintptr_t)(lds_ptr)(tile + (i * WAVES + wave) * 64 *
                                                                        Elem<T>::kChunk)),
                           "v"(x), "s"(rsrc)
                         : "m0", "memory");
        }
    }
};
// Waits for this wave's copies (vmcnt 0, the other counters as they are).
__device__ __forceinline__ void tile_wait() { __builtin_amdgcn_s_waitcnt(0x0f70); }

// A key's mask value as it lies in memory; compared only where it is used, so that nothing
// waits for it where it is loaded.
__device__ __forceinline__ int keep_raw(const AttnArgs &a, int64_t row) {
    return a.keep_bytes == 1 ? static_cast<const uint8_t *>(a.keep)[row]
                             : static_cast<const int *>(a.keep)[row];
}

// A row of global memory as the right operand's column of one lane.
template <typename T, int DP>
__device__ __forceinline__ void load_column(typename Elem<T>::frag (&f)[DP / 16], const T *row,
                                            int dim, bool live, int lane) {
#pragma unroll
    for (int s = 0; s < DP / 16; ++s) {
        const int d = s * 16 + 8 * (lane >> 5);
        f[s] = {};
        if (live && d < dim) f[s] = row_frag(row + d);
    }
}

// A 32 x DP result (columns of DP values) to one row of global memory, scaled; with `low`, what the
// rounding to T took away goes there.
template <typename T, int DP>
__device__ __forceinline__ void store_column(T *row, const f32x16 (&o)[DP / 32], float scale,
                                             int dim, int lane, T *low = nullptr) {
#pragma unroll
    for (int b = 0; b < DP / 32; ++b)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            const int d = b * 32 + 8 * g + 4 * (lane >> 5);
            if (d >= dim) continue;
            typedef T t4 __attribute__((ext_vector_type(4)));
            t4 v, w;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const float x = o[b][4 * g + e] * scale;
                v[e] = (T)x;
                w[e] = (T)(x - (float)v[e]);
            }
            *reinterpret_cast<t4 *>(row + d) = v;
            if (low) *reinterpret_cast<t4 *>(low + d) = w;
        }
}

// The row of a block that result register r of a lane's half holds, less 4 (lane / 32).
__device__ __forceinline__ constexpr int result_row(int r) { return 8 * (r >> 2) + (r & 3); }

// What the rounding to T takes from each value.
template <typename T> __device__ __forceinline__ f32x16 remainders(const f32x16 &w) {
    f32x16 low;
#pragma unroll
    for (int r = 0; r < 16; ++r) low[r] = w[r] - (float)(T)w[r];
    return low;
}

// The product of each lane's own row with its column, the diagonal of a 32 x 32 product: formed by
// the instructions and in the order of any other element, so that equal rows give equal bits.
template <typename T, int N>
__device__ __forceinline__ float own_product(const typename Elem<T>::frag (&row)[N],
                                             const typename Elem<T>::frag (&column)[N], int lane) {
    f32x16 w = {};
#pragma unroll
    for (int st = 0; st < N; ++st) w = mma(row[st], column[st], w);
    float x = 0.f;
#pragma unroll
    for (int r = 0; r < 16; ++r)
        if (result_row(r) + 4 * (lane >> 5) == (lane & 31)) x = w[r];
    return x + other_half(x);  // the other half's is 0
}

// Positions for distances: differences of two sides' coordinates formed by the matrix units.
// float32: x_row * 1 + 1 * -x_column, one v_mfma_f32_32x32x2_f32 an axis, the rounding of a
// subtraction.  bfloat16: each coordinate as the exact sum of three bfloat16 (24 bits), so a
// difference is six exact products with one, in one v_mfma_f32_32x32x16_bf16 an axis; the
// products' sum is rounded like a binary32 sum of six terms.  That form runs beside the vector
// instructions, where 48 subtractions a block would queue with them (the float32 matrix
// instructions do not: they share the vector units, measured).
template <typename T> struct Places;

template <> struct Places<float> {
    typedef float Row;
    float own[3];
    static __device__ __forceinline__ Row row(float x) { return x; }
    __device__ __forceinline__ void set(float x, float y, float z, int lane) {
        own[0] = lane < 32 ? 1.f : -x, own[1] = lane < 32 ? 1.f : -y, own[2] = lane < 32 ? 1.f : -z;
    }
    __device__ __forceinline__ f32x16 minus(Row r, int ax, int lane) const {
        return __builtin_amdgcn_mfma_f32_32x32x2f32(lane < 32 ? r : 1.f, own[ax], f32x16{}, 0, 0, 0);
    }
};

template <> struct Places<bf16> {
    typedef bf16x8 Row;
    bf16x8 own[3];
    static __device__ __forceinline__ Row row(float x) {
        const bf16 a = (bf16)x;
        x -= (float)a;
        const bf16 b = (bf16)x, c = (bf16)(x - (float)b), one = (bf16)1.f, no = (bf16)0.f;
        return bf16x8{a, b, c, one, one, one, no, no};
    }
    // the upper lanes' contraction indices meet zeros
    __device__ __forceinline__ void set(float x, float y, float z, int lane) {
        const float c[3] = {x, y, z};
#pragma unroll
        for (int ax = 0; ax < 3; ++ax) {
            const bf16x8 r = row(-c[ax]);
            own[ax] = lane < 32 ? bf16x8{r[3], r[4], r[5], r[0], r[1], r[2], r[6], r[7]} : bf16x8{};
        }
    }
    __device__ __forceinline__ f32x16 minus(Row r, int ax, int) const {
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(r, own[ax], f32x16{}, 0, 0, 0);
    }
};

// Distances of the lanes' columns to the 32 rows of a block, in the result's layout; xyz: three
// arrays of `n` rows in LDS, `first` the block's first row in them.
template <typename T>
__device__ __forceinline__ f32x16 distances(const Places<T> &to, const typename Places<T>::Row *xyz,
                                            int n, int first, int lane) {
    const typename Places<T>::Row *p = xyz + first + (lane & 31);
    f32x16 d;
#pragma unroll
    for (int ax = 0; ax < 3; ++ax) {
        const f32x16 e = to.minus(p[ax * n], ax, lane);
#pragma unroll
        for (int r = 0; r < 16; ++r) d[r] = ax ? fmaf(e[r], e[r], d[r]) : e[r] * e[r];
    }
#pragma unroll
    for (int r = 0; r < 16; ++r) d[r] = __builtin_amdgcn_sqrtf(d[r]);
    return d;
}

// The rows of a block that a lane sees, a bit each at result_row(r): those kept (bits of the tile)
// below the lane's limit, counted from the block's first row.
__device__ __forceinline__ uint32_t seen_rows(uint64_t live, int block, int limit, int lane) {
    const uint32_t below = limit >= 32 ? ~0u : limit > 0 ? (1u << limit) - 1 : 0u;
    return ((uint32_t)(live >> (32 * block)) & below) >> (4 * (lane >> 5));
}

}  // namespace gsv
