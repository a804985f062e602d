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
    static constexpr int kPad = 8;    // LDS row padding, elements
    static constexpr int kChunk = 8;  // elements of a 16-byte chunk
};
template <> struct Elem<float> {
    typedef f32x8 frag;
    static constexpr int kPad = 4;
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

// The transposed left operand: column l % 32 of 32 columns, rows 4 g .. 4 g + 3 and
// 8 + 4 g .. 8 + 4 g + 3 of 16 rows.  `tile` points at the first row and column.  For 16-bit
// elements ds_read_b64_tr_b16 does it: of 16 lanes, lane i gives the address of
// row i / 4, columns 4 (i % 4) .. + 3, and receives column i of the four rows.
template <int LD> __device__ __forceinline__ bf16x8 tr_frag(const bf16 *tile, int lane) {
    const int i = lane & 15, g = lane >> 5;
    const bf16 *p = tile + (4 * g + (i >> 2)) * LD + (lane & 16) + 4 * (i & 3);
    typedef __attribute__((address_space(3))) s16x4 *lds_ptr;
    const s16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr)(p));
    const s16x4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_ptr)(p + 8 * LD));
    const bf16x4 x = __builtin_bit_cast(bf16x4, a), y = __builtin_bit_cast(bf16x4, b);
    return bf16x8{x[0], x[1], x[2], x[3], y[0], y[1], y[2], y[3]};
}
template <int LD> __device__ __forceinline__ f32x8 tr_frag(const float *tile, int lane) {
    const float *p = tile + 4 * (lane >> 5) * LD + (lane & 31);
    f32x8 f;
#pragma unroll
    for (int e = 0; e < 4; ++e) f[e] = p[e * LD], f[4 + e] = p[(8 + e) * LD];
    return f;
}

__device__ __forceinline__ float fast_exp2(float x) { return __builtin_amdgcn_exp2f(x); }

// tanh.  For bfloat16 scores 1 - 2 / (exp(2 x) + 1): absolute error near 2^-23, far
// below the 2^-9 of the operands; ends at +-1 where exp overflows or vanishes.
template <typename T> __device__ __forceinline__ float tanh_of(float x) {
    if constexpr (sizeof(T) == 4) return tanhf(x);
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
    int slots;  // workgroups a scene and head: they take its tiles in turn
};

// Checks the C arguments and lays them out for a launch; longest_*: rows of the longest scene.
int attention_args(const gsv_attention *in, AttnArgs *a, int *longest_q, int *longest_k);

// The kernel variant of a call: element type, channels (up to 32, 64 or 128; the columns past
// dim are zeros), distance bias, score cap.
template <typename T, int DP, typename F> void attention_options(const AttnArgs &a, const F &f) {
    const bool far = a.slopes, capped = a.cap > 0.f;
    if (far && capped) f.template run<T, DP, true, true>();
    else if (far) f.template run<T, DP, true, false>();
    else if (capped) f.template run<T, DP, false, true>();
    else f.template run<T, DP, false, false>();
}
template <typename T, typename F> void attention_channels(const AttnArgs &a, const F &f) {
    if (a.dim <= 32) attention_options<T, 32>(a, f);
    else if (a.dim <= 64) attention_options<T, 64>(a, f);
    else attention_options<T, 128>(a, f);
}
template <typename F> void attention_variant(const AttnArgs &a, int dtype, const F &f) {
    if (dtype == GSV_BF16) attention_channels<bf16>(a, f);
    else attention_channels<float>(a, f);
}

// Whether a wave takes two heads (for their distances): an even number of them.
inline bool attention_pairs(const AttnArgs &a) { return a.heads % 2 == 0; }

// Workgroups for each scene and head: one for each tile of the longest scene, fewer where the
// launch would pass a million (they take the tiles in turn, so any number is right).
inline bool attention_slots(AttnArgs *a, int longest, int rows, int heads) {
    const int64_t each = (int64_t)a->scenes * heads;
    if (each > (1 << 24) - 1) return false;
    a->slots = (int)imin64((longest + rows - 1) / rows, imax64((1 << 20) / each, 1));
    return true;
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
__device__ __forceinline__ Scene scene_rows(const AttnArgs &a, int s) {
    Scene c;
    c.q0 = scene_start(a.q_starts, s, a.scenes, a.q_tokens);
    c.q1 = max(scene_start(a.q_starts, s + 1, a.scenes, a.q_tokens), c.q0);
    c.k0 = scene_start(a.k_starts, s, a.scenes, a.k_tokens);
    c.k1 = max(scene_start(a.k_starts, s + 1, a.scenes, a.k_tokens), c.k0);
    c.prefix = a.prefix ? min(max(a.prefix[s], 0), c.k1 - c.k0) : 0;
    return c;
}
// Keys of the scene that its query row i sees (those below the limit): with the causal mask
// a prefix or what precedes the query, whose rows end where the keys end.
__device__ __forceinline__ int key_limit(const AttnArgs &a, const Scene &c, int i) {
    const int n = c.k1 - c.k0;
    if (!a.causal) return n;
    return min(max(c.prefix, i + n - (c.q1 - c.q0) + 1), n);
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

// A tile of ROWS rows of one head on its way from global memory to LDS: 256 threads, 16-byte
// chunks through a buffer descriptor that ends with the last live row, so that rows past it and
// columns from dim up to DP arrive as zeros without a branch.  Rows of a mask are zeroed
// as they are stored: no value of theirs, NaN among them, meets a weight of 0.
template <typename T, int DP, int ROWS> struct Staged {
    static constexpr int kCh = Elem<T>::kChunk, kPerRow = DP / kCh, LD = DP + Elem<T>::kPad;
    static constexpr int kN = ROWS * kPerRow / 256;
    static_assert(ROWS * kPerRow % 256 == 0, "whole chunks for each thread");
    typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
    u32x4 r[kN];
    int at[kN];  // byte offsets in the tile
    __device__ __forceinline__ void plan(int64_t stride, int dim) {
#pragma unroll
        for (int i = 0; i < kN; ++i) {
            const int c = i * 256 + threadIdx.x, row = c / kPerRow, col = (c % kPerRow) * kCh;
            at[i] = col < dim ? (row * (int)stride + col) * (int)sizeof(T) : INT32_MAX - 15;
        }
    }
    // rows: live rows from base on, 1 at least
    __device__ __forceinline__ void load(const T *base, int64_t stride, int dim, int rows) {
        const int bytes = ((min(rows, ROWS) - 1) * (int)stride + dim) * (int)sizeof(T);
        const auto rsrc = __builtin_amdgcn_make_buffer_rsrc(const_cast<T *>(base), 0, bytes, 0x00020000);
#pragma unroll
        for (int i = 0; i < kN; ++i) r[i] = __builtin_amdgcn_raw_buffer_load_b128(rsrc, at[i], 0, 0);
    }
    __device__ __forceinline__ void store(T *tile) const {
#pragma unroll
        for (int i = 0; i < kN; ++i) {
            const int c = i * 256 + threadIdx.x, row = c / kPerRow, col = (c % kPerRow) * kCh;
            *reinterpret_cast<u32x4 *>(tile + row * LD + col) = r[i];
        }
    }
    __device__ __forceinline__ void keep(uint64_t live) {
#pragma unroll
        for (int i = 0; i < kN; ++i)
            if (!((live >> ((i * 256 + threadIdx.x) / kPerRow)) & 1)) r[i] = u32x4{};
    }
};

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

// A 32 x DP result (columns of DP values) to one row of global memory, scaled.
template <typename T, int DP>
__device__ __forceinline__ void store_column(T *row, const f32x16 (&o)[DP / 32], float scale,
                                             int dim, int lane) {
#pragma unroll
    for (int b = 0; b < DP / 32; ++b)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            const int d = b * 32 + 8 * g + 4 * (lane >> 5);
            if (d >= dim) continue;
            typedef T t4 __attribute__((ext_vector_type(4)));
            t4 v;
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = (T)(o[b][4 * g + e] * scale);
            *reinterpret_cast<t4 *>(row + d) = v;
        }
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

__device__ __forceinline__ int result_row(int r, int lane) {
    return 8 * (r >> 2) + 4 * (lane >> 5) + (r & 3);
}

}  // namespace gsv
