// adamw.hip — one AdamW step over many tensors.
//
//   g' = g min(1, max_norm / (|all g| + 1e-6))
//   m = b1 m + (1 - b1) g',  v = b2 v + (1 - b2) g'^2
//   w = w (1 - lr decay) - lr / (1 - b1^t) m / (sqrt(v) / sqrt(1 - b2^t) + eps)
//
// Bytes bound it: 28 an element in float32, or in bfloat16 with 32-bit masters.  The tensors' addresses and sizes
// are a table in the kernel's own arguments, so a launch takes as many as fit there (kTensors) and copies
// nothing to the device first; a workgroup finds its tensor from its number.  The norm needs all gradients before
// the first update: a pass of its own, whose sums one workgroup adds up, and which the
// update then reads again, from the caches where they hold it.
//
// 83 million bfloat16 weights with masters, clipped (2.3 GB): 479 us, 4.8 TB/s, what a large copy reaches; 200,000 Gaussians'
// 2.2 million values (62 MB, which the caches hold): 11.2 us; four tensors of 1,500 values: 6.0 us, the host's; the
// kernel takes 3.7.
#include "gsv_device.h"

#include <algorithm>
#include <cmath>
#include <functional>
#include <new>
#include <type_traits>

namespace gsv {
namespace {

typedef __bf16 bf16;

struct Entry {
    void *p;
    const void *g;
    float *m, *v, *w;  // w: the 32-bit master, or unused
    const float *lr_device;
    int64_t n;
    double lr;  // lr decay is formed in binary64: 1 less it is near 1
    float decay, by_m, by_v;  // by_m = 1 / (1 - b1^t), by_v = 1 / sqrt(1 - b2^t)
    int own;                  // below 0: these; else the place of those of the tensor's own counter
};
// Tensors of a launch: as many as its arguments hold, which end at 4 KB; where there are few, a table of few, since the
// host copies all of it (four tensors: 6.03 us a call, in the large table 6.32).
constexpr int kTensors = 44, kFew = 8;
template <int N> struct Table {
    static constexpr int kMost = N;
    int count;
    int first[N];  // the tensors' first workgroups
    Entry t[N];
    void put(int i, const gsv_adamw_tensor &x, float by_m, float by_v, int own) {
        t[i] = Entry{x.param, x.grad, x.exp_avg, x.exp_avg_sq, x.master, x.lr_device, x.numel, x.lr,
                     (float)x.weight_decay, by_m, by_v, own};
    }
};
// For the norm: the gradients alone (148 tensors of 83 million values, one launch in place of four: 478 us, in the tables
// above 490; 28 tensors 16.2 both ways).  4 KB would hold 200; what is not used is copied all the same: 28 tensors in a
// table of 32 14.2 or 16.1 us (the host runs at one of two speeds, from process to process), in one of 160 14.3 or 16.4.
constexpr int kGradients = 160, kFewGradients = 32;
template <int N> struct Gradients {
    static constexpr int kMost = N;
    int count;
    int first[N];
    const void *g[N];
    int64_t n[N];
    void put(int i, const gsv_adamw_tensor &x, float, float, int) { g[i] = x.grad, n[i] = x.numel; }
};
struct Rates {
    float b1, c1, b2, c2, eps;  // c = 1 - b
    const float *shared;        // by_m, by_v, the gradients' factor; NULL: the entries', and 1
    int counted;                // by_m and by_v are those of `shared`
    // few sums of squares: each workgroup forms what k_adamw_shared does, and no launch is needed for it
    const double *sums;
    int count;
    double max_norm, beta1, beta2;
    const int *counter;  // advanced already
    float *norm;         // for the first workgroup of a launch, or NULL
    const float2 *own;   // by_m, by_v of the tensors' own counters
};

// Elements of a thread's step: 16 bytes of the 32-bit arrays.
constexpr int kVec = 4;
template <typename T> struct __align__(sizeof(T) * kVec) Four {
    T v[kVec];
};

// The tensor of a workgroup: loads over the lanes (a search one step after the other cost 2 us).
template <typename Tensors> __device__ __forceinline__ int tensor_of(const Tensors &t, int block) {
    const int lane = threadIdx.x & 63;
    int begun = 0;
#pragma unroll
    for (int i = 0; i < Tensors::kMost; i += 64) {
        const int first = t.first[min(i + lane, Tensors::kMost - 1)];
        begun += __popcll(__ballot(i + lane < t.count && first <= block));
    }
    return __builtin_amdgcn_readfirstlane(begun - 1);
}

struct Step {
    float b1, c1, b2, c2, eps, factor, keep, rate, by_v;
};

__device__ __forceinline__ void update(float g, float &m, float &v, float &w, const Step &s) {
    g *= s.factor;
    m = fmaf(s.b1, m, s.c1 * g);
    v = fmaf(s.b2, v, s.c2 * (g * g));
    w = fmaf(-s.rate, m / fmaf(sqrtf(v), s.by_v, s.eps), w * s.keep);
}

// The sum over a workgroup of 256.
__device__ __forceinline__ double block_sum(double x) {
    __shared__ double part[4];
#pragma unroll
    for (int k = 1; k < 64; k <<= 1) x += __shfl_xor(x, k);
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = x;
    __syncthreads();
    return (part[0] + part[1]) + (part[2] + part[3]);
}

// The norm, and the factor that brings it to max_norm at most.
__device__ __forceinline__ float norm_of(const double *sums, int count, double max_norm, float *factor) {
    double sum = 0.0;
#pragma unroll 8
    for (int i = threadIdx.x; i < count; i += 256) sum += sums[i];
    const double all = sqrt(block_sum(sum)), by = max_norm / (all + 1e-6);
    *factor = by < 1.0 || by != by ? (float)by : 1.f;
    return (float)all;
}
// 1 / (1 - beta1^t) and 1 / sqrt(1 - beta2^t)
__device__ __forceinline__ float2 corrections(double beta1, double beta2, int t) {
    return make_float2((float)(1.0 / (1.0 - pow(beta1, (double)t))), (float)(1.0 / sqrt(1.0 - pow(beta2, (double)t))));
}

// STEPS: steps of a thread.  P, G: types of the param and its gradient; MASTER: a bfloat16 param's 32-bit copy.
template <typename P, typename G, bool MASTER, int STEPS, int N>
__global__ __launch_bounds__(256) void k_adamw(const Table<N> table, const Rates r) {
    const int at = tensor_of(table, blockIdx.x);
    const Entry &e = table.t[at];
    const double lr = e.lr_device ? (double)*e.lr_device : e.lr;
    Step s{r.b1, r.c1, r.b2, r.c2, r.eps, 1.f, (float)(1.0 - lr * (double)e.decay), 0.f, e.by_v};
    float by_m = e.by_m;
    if (r.shared) {
        s.factor = r.shared[2];
        if (r.counted) by_m = r.shared[0], s.by_v = r.shared[1];
    } else if (r.sums) {
        const float all = norm_of(r.sums, r.count, r.max_norm, &s.factor);
        if (r.norm && blockIdx.x == 0 && threadIdx.x == 0) *r.norm = all;
        if (r.counter) {
            const float2 by = corrections(r.beta1, r.beta2, *r.counter);
            by_m = by.x, s.by_v = by.y;
        }
    }
    if (e.own >= 0) {
        const float2 by = r.own[e.own];
        by_m = by.x, s.by_v = by.y;
    }
    s.rate = (float)(lr * (double)by_m);
    P *const p = static_cast<P *>(e.p);
    const G *const g = static_cast<const G *>(e.g);
    float *const m = e.m, *const v = e.v, *const w = e.w;
    const int64_t n = e.n, base = (int64_t)(blockIdx.x - table.first[at]) * (256 * kVec * STEPS);
    // An array off alignment, or the tensor's last elements: by single elements, 256 apart for a thread.
    const bool wide = (reinterpret_cast<uintptr_t>(m) | reinterpret_cast<uintptr_t>(v) |
                       (MASTER ? reinterpret_cast<uintptr_t>(w) : 0)) % 16 == 0 &&
                      reinterpret_cast<uintptr_t>(p) % sizeof(Four<P>) == 0 &&
                      reinterpret_cast<uintptr_t>(g) % sizeof(Four<G>) == 0 && base + 256 * kVec * STEPS <= n;
    Four<float> mm[STEPS], vv[STEPS], ww[STEPS];
    Four<G> gg[STEPS];
    Four<P> pp[STEPS];
    if (wide) {
#pragma unroll
        for (int k = 0; k < STEPS; ++k) {
            const int64_t i = base + (k * 256 + threadIdx.x) * kVec;
            gg[k] = *reinterpret_cast<const Four<G> *>(g + i);
            mm[k] = *reinterpret_cast<const Four<float> *>(m + i);
            vv[k] = *reinterpret_cast<const Four<float> *>(v + i);
            if constexpr (MASTER) ww[k] = *reinterpret_cast<const Four<float> *>(w + i);
            else pp[k] = *reinterpret_cast<const Four<P> *>(p + i);
        }
    } else {
#pragma unroll
        for (int k = 0; k < STEPS; ++k)
#pragma unroll
            for (int j = 0; j < kVec; ++j) {
                const int64_t i = base + (k * kVec + j) * 256 + threadIdx.x;
                if (i >= n) continue;
                gg[k].v[j] = g[i], mm[k].v[j] = m[i], vv[k].v[j] = v[i];
                if constexpr (MASTER) ww[k].v[j] = w[i];
                else pp[k].v[j] = p[i];
            }
    }
#pragma unroll
    for (int k = 0; k < STEPS; ++k) {
#pragma unroll
        for (int j = 0; j < kVec; ++j) {
            float wi = MASTER ? ww[k].v[j] : (float)pp[k].v[j];
            update((float)gg[k].v[j], mm[k].v[j], vv[k].v[j], wi, s);
            ww[k].v[j] = wi, pp[k].v[j] = (P)wi;
        }
        if (wide) {
            const int64_t i = base + (k * 256 + threadIdx.x) * kVec;
            *reinterpret_cast<Four<float> *>(m + i) = mm[k];
            *reinterpret_cast<Four<float> *>(v + i) = vv[k];
            *reinterpret_cast<Four<P> *>(p + i) = pp[k];
            if constexpr (MASTER) *reinterpret_cast<Four<float> *>(w + i) = ww[k];
        } else {
#pragma unroll
            for (int j = 0; j < kVec; ++j) {
                const int64_t i = base + (k * kVec + j) * 256 + threadIdx.x;
                if (i >= n) continue;
                m[i] = mm[k].v[j], v[i] = vv[k].v[j], p[i] = pp[k].v[j];
                if constexpr (MASTER) w[i] = ww[k].v[j];
            }
        }
    }
}

// Sums of squares in binary64: no overflow, and no length at which the small terms are lost.
constexpr int kNormSteps = 8;
template <typename G, int N>
__global__ __launch_bounds__(256) void k_adamw_squares(const Gradients<N> table, double *sums, int *counter) {
    if (counter && blockIdx.x == 0 && threadIdx.x == 0) *counter += 1;
    const int at = tensor_of(table, blockIdx.x);
    const G *const g = static_cast<const G *>(table.g[at]);
    constexpr int64_t kAll = 256 * kVec * kNormSteps;
    const int64_t n = table.n[at], base = (int64_t)(blockIdx.x - table.first[at]) * kAll;
    Four<G> x[kNormSteps];
    if (reinterpret_cast<uintptr_t>(g) % sizeof(Four<G>) == 0 && base + kAll <= n) {
#pragma unroll
        for (int k = 0; k < kNormSteps; ++k)
            x[k] = *reinterpret_cast<const Four<G> *>(g + base + (k * 256 + threadIdx.x) * kVec);
    } else {
#pragma unroll
        for (int k = 0; k < kNormSteps; ++k)
#pragma unroll
            for (int j = 0; j < kVec; ++j) {
                const int64_t i = base + (k * kVec + j) * 256 + threadIdx.x;
                x[k].v[j] = i < n ? g[i] : (G)0.f;
            }
    }
    double sum = 0.0;
#pragma unroll
    for (int k = 0; k < kNormSteps; ++k)
#pragma unroll
        for (int j = 0; j < kVec; ++j) sum = fma((double)(float)x[k].v[j], (double)(float)x[k].v[j], sum);
    sum = block_sum(sum);
    if (threadIdx.x == 0) sums[blockIdx.x] = sum;
}

// What all tensors share, by one workgroup: the norm from the squares' sums, and the step that `counter` counts.
__global__ __launch_bounds__(256) void k_adamw_shared(const double *sums, int count, double max_norm, double b1,
                                                      double b2, int *counter, float *norm, float *shared) {
    float factor = 1.f, all = 0.f;
    if (max_norm > 0.0) all = norm_of(sums, count, max_norm, &factor);
    if (threadIdx.x) return;
    if (max_norm > 0.0 && norm) *norm = all;
    shared[2] = factor;
    if (counter) {
        const int t = *counter + 1;
        *counter = t;
        const float2 by = corrections(b1, b2, t);
        shared[0] = by.x, shared[1] = by.y;
    }
}

// Counters of their own that tensors have: each counts its step, a thread each, and the corrections of that step
// go to the workspace for the update.  A launch before the update: one workgroup of a tensor could not
// advance what the others still read.  2.6 us, of 4 tensors or 148; calls of 28 tensors, not clipped, take 14.9 us so and
// 13.6 with one counter, which k_adamw_shared counts (or the norm's pass, without a launch).
constexpr int kCounters = 256;
struct CounterTable {
    int count;
    int *of[kCounters];
};
__global__ __launch_bounds__(kCounters) void k_adamw_counters(const CounterTable table, double b1, double b2, float2 *own) {
    const int i = threadIdx.x;
    if (i >= table.count) return;
    int *const counter = table.of[i];
    const int t = *counter + 1;
    *counter = t;
    own[i] = corrections(b1, b2, t);
}

struct Sizes {
    int64_t elements, squares;  // workgroups of the norm's pass
    int64_t counters;           // tensors with a counter of their own
};

// All workgroups of a launch then fit its grid: at most 2^22 of 4,096 elements (where there are fewer than 8.4 million,
// 2^13 of 1,024), or 2^21 of the norm's 8,192, and one more for each tensor of a table.
constexpr int64_t kMostElements = (int64_t)1 << 34;

int adamw_check(const gsv_adamw_args *a, Sizes *out) {
    if (!a || a->count < 0 || (a->count && !a->tensors) || !(a->beta1 >= 0 && a->beta1 < 1) ||
        !(a->beta2 >= 0 && a->beta2 < 1) || !(a->eps >= 0) || !(a->max_norm >= 0))
        return GSV_ERR_INVALID_ARGUMENT;
    *out = Sizes{};
    for (int64_t i = 0; i < a->count; ++i) {
        const gsv_adamw_tensor &t = a->tensors[i];
        if (t.numel < 0 || (a->counter ? t.counter != nullptr : !t.counter && t.step < 1) ||
            reinterpret_cast<uintptr_t>(t.counter) % 4 || (t.dtype != GSV_F32 && t.dtype != GSV_BF16) ||
            (t.grad_dtype != GSV_F32 && t.grad_dtype != GSV_BF16) || (t.master && t.dtype != GSV_BF16))
            return GSV_ERR_INVALID_ARGUMENT;
        out->counters += t.counter != nullptr;
        if (t.numel > kMostElements || out->elements > kMostElements) return GSV_ERR_SIZE_OVERFLOW;
        if (t.numel == 0) continue;
        const uintptr_t words = reinterpret_cast<uintptr_t>(t.exp_avg) | reinterpret_cast<uintptr_t>(t.exp_avg_sq) |
                                reinterpret_cast<uintptr_t>(t.master) | reinterpret_cast<uintptr_t>(t.lr_device);
        if (!t.param || !t.grad || !t.exp_avg || !t.exp_avg_sq || words % 4 ||
            reinterpret_cast<uintptr_t>(t.param) % (t.dtype == GSV_BF16 ? 2 : 4) ||
            reinterpret_cast<uintptr_t>(t.grad) % (t.grad_dtype == GSV_BF16 ? 2 : 4))
            return GSV_ERR_INVALID_ARGUMENT;
        out->elements += t.numel;
    }
    if (out->elements > kMostElements) return GSV_ERR_SIZE_OVERFLOW;
    const int64_t each = 256 * kVec * kNormSteps;
    for (int64_t i = 0; i < a->count; ++i) out->squares += (a->tensors[i].numel + each - 1) / each;
    return GSV_OK;
}

// The tensors' own counters, each once, and which of them a tensor has (-1: none).
struct Counters {
    int32_t **each = nullptr;
    int *of = nullptr;  // NULL: no tensor has one
    int count = 0;
    bool fits = true;
    Counters(const gsv_adamw_args *a, const Sizes &s) {
        if (!s.counters) return;
        each = new (std::nothrow) int32_t *[s.counters];
        of = new (std::nothrow) int[a->count];
        if (!each || !of) {
            fits = false;
            return;
        }
        for (int64_t i = 0; i < a->count; ++i)
            if (a->tensors[i].counter) each[count++] = a->tensors[i].counter;
        std::sort(each, each + count, std::less<int32_t *>());
        count = (int)(std::unique(each, each + count) - each);
        for (int64_t i = 0; i < a->count; ++i) {
            int32_t *const c = a->tensors[i].counter;
            of[i] = c ? (int)(std::lower_bound(each, each + count, c, std::less<int32_t *>()) - each) : -1;
        }
    }
    ~Counters() { delete[] each, delete[] of; }
    Counters(const Counters &) = delete;
};

// Tables of the tensors that `takes`, each handed to `launch` with its workgroups when it is full.
template <typename Tensors, typename Takes, typename Launch>
void tables(const gsv_adamw_args *a, int64_t per_block, const int *counter_of, const Takes &takes, const Launch &launch) {
    Tensors t;
    t.count = 0;
    int64_t blocks = 0;
    for (int64_t i = 0; i < a->count; ++i) {
        const gsv_adamw_tensor &x = a->tensors[i];
        if (!x.numel || !takes(x)) continue;
        const int64_t own = (x.numel + per_block - 1) / per_block;
        if (t.count == Tensors::kMost) {
            launch(t, blocks);
            t.count = 0, blocks = 0;
        }
        float by_m = 1.f, by_v = 1.f;
        if (!a->counter && !x.counter) {
            by_m = (float)(1.0 / (1.0 - std::pow(a->beta1, (double)x.step)));
            by_v = (float)(1.0 / std::sqrt(1.0 - std::pow(a->beta2, (double)x.step)));
        }
        t.first[t.count] = (int)blocks;
        t.put(t.count++, x, by_m, by_v, counter_of ? counter_of[i] : -1);
        blocks += own;
    }
    if (t.count) launch(t, blocks);
}
template <typename Takes> bool at_most(const gsv_adamw_args *a, int most, const Takes &takes) {
    for (int64_t i = 0; i < a->count; ++i)
        if (a->tensors[i].numel && takes(a->tensors[i]) && --most < 0) return false;
    return true;
}

template <typename P, typename G, bool MASTER>
void update_all(const gsv_adamw_args *a, const Rates &r, const int *own, int steps, hipStream_t st) {
    constexpr int p = sizeof(P) == 2 ? GSV_BF16 : GSV_F32, g = sizeof(G) == 2 ? GSV_BF16 : GSV_F32;
    const auto takes = [](const gsv_adamw_tensor &t) {
        return t.dtype == p && t.grad_dtype == g && (t.master != nullptr) == MASTER;
    };
    if (steps == 4)
        tables<Table<kTensors>>(a, 256 * kVec * 4, own, takes, [&](const Table<kTensors> &t, int64_t blocks) {
            hipLaunchKernelGGL((k_adamw<P, G, MASTER, 4, kTensors>), dim3((unsigned)blocks), dim3(256), 0, st, t, r);
        });
    else if (at_most(a, kFew, takes))
        tables<Table<kFew>>(a, 256 * kVec, own, takes, [&](const Table<kFew> &t, int64_t blocks) {
            hipLaunchKernelGGL((k_adamw<P, G, MASTER, 1, kFew>), dim3((unsigned)blocks), dim3(256), 0, st, t, r);
        });
    else
        tables<Table<kTensors>>(a, 256 * kVec, own, takes, [&](const Table<kTensors> &t, int64_t blocks) {
            hipLaunchKernelGGL((k_adamw<P, G, MASTER, 1, kTensors>), dim3((unsigned)blocks), dim3(256), 0, st, t, r);
        });
}

template <typename G> void squares_all(const gsv_adamw_args *a, double *sums, int *counter, int64_t *at, hipStream_t st) {
    constexpr int g = sizeof(G) == 2 ? GSV_BF16 : GSV_F32;
    const auto takes = [](const gsv_adamw_tensor &t) { return t.grad_dtype == g; };
    const auto launch = [&](const auto &t, int64_t blocks) {
        constexpr int N = std::decay_t<decltype(t)>::kMost;
        hipLaunchKernelGGL((k_adamw_squares<G, N>), dim3((unsigned)blocks), dim3(256), 0, st, t, sums + *at,
                           *at ? nullptr : counter);
        *at += blocks;
    };
    if (at_most(a, kFewGradients, takes)) tables<Gradients<kFewGradients>>(a, 256 * kVec * kNormSteps, nullptr, takes, launch);
    else tables<Gradients<kGradients>>(a, 256 * kVec * kNormSteps, nullptr, takes, launch);
}

// Whether a tensor that the step writes shares memory with another that it writes, or with a gradient.
bool share_memory(const gsv_adamw_args *a) {
    struct Span {
        uintptr_t first, end;
    };
    Span *spans = new (std::nothrow) Span[4 * a->count];
    if (!spans) return true;
    int64_t n = 0;
    for (int64_t i = 0; i < a->count; ++i) {
        const gsv_adamw_tensor &t = a->tensors[i];
        if (!t.numel) continue;
        const auto add = [&](const void *p, int64_t size) {
            const uintptr_t at = reinterpret_cast<uintptr_t>(p);
            spans[n++] = Span{at, at + (uintptr_t)(t.numel * size)};
        };
        add(t.param, t.dtype == GSV_BF16 ? 2 : 4);
        add(t.exp_avg, 4);
        add(t.exp_avg_sq, 4);
        if (t.master) add(t.master, 4);
    }
    std::sort(spans, spans + n, [](const Span &x, const Span &y) { return x.first < y.first; });
    bool twice = false;
    for (int64_t i = 1; i < n; ++i) twice |= spans[i].first < spans[i - 1].end;
    for (int64_t i = 0; i < a->count && !twice; ++i) {
        const gsv_adamw_tensor &t = a->tensors[i];
        if (!t.numel) continue;
        const uintptr_t first = reinterpret_cast<uintptr_t>(t.grad);
        const uintptr_t end = first + (uintptr_t)(t.numel * (t.grad_dtype == GSV_BF16 ? 2 : 4));
        // the first written span that ends behind the gradient's start (they do not overlap: their ends ascend too)
        const Span *s = std::upper_bound(spans, spans + n, first, [](uintptr_t x, const Span &y) { return x < y.end; });
        twice = s < spans + n && s->first < end;
    }
    delete[] spans;
    return twice;
}

// The workspace: sums of squares, the tensors' own corrections, what all share.
struct Workspace {
    size_t own, shared, bytes;
};
Workspace adamw_workspace(const gsv_adamw_args *a, const Sizes &s) {
    Workspace w;
    w.own = a->max_norm > 0 ? sizeof(double) * (size_t)s.squares : 0;
    w.shared = w.own + sizeof(float2) * (size_t)s.counters;
    w.bytes = w.shared + (a->max_norm > 0 || a->counter ? 4 * sizeof(float) : 0);
    return w;
}

}  // namespace
}  // namespace gsv

using namespace gsv;

extern "C" int gsv_adamw_workspace_bytes(const gsv_adamw_args *args, size_t *bytes) {
    Sizes s;
    if (!bytes) return GSV_ERR_INVALID_ARGUMENT;
    const int st = adamw_check(args, &s);
    if (st != GSV_OK) return st;
    *bytes = adamw_workspace(args, s).bytes;
    return GSV_OK;
}

extern "C" int gsv_adamw(const gsv_adamw_args *args, void *workspace, size_t workspace_bytes, void *stream) {
    Sizes s;
    const int st = adamw_check(args, &s);
    if (st != GSV_OK) return st;
    const Workspace ws = adamw_workspace(args, s);
    if (ws.bytes > workspace_bytes) return GSV_ERR_WORKSPACE_TOO_SMALL;
    if ((ws.bytes && !workspace) || reinterpret_cast<uintptr_t>(workspace) % 16 || share_memory(args))
        return GSV_ERR_INVALID_ARGUMENT;
    const Counters counters(args, s);
    if (!counters.fits) return GSV_ERR_INVALID_ARGUMENT;
    hipStream_t stm = as_stream(stream);
    Rates r{(float)args->beta1, (float)(1.0 - args->beta1), (float)args->beta2, (float)(1.0 - args->beta2),
            (float)args->eps, nullptr, args->counter != nullptr, nullptr, 0, args->max_norm, args->beta1, args->beta2,
            args->counter, args->norm, reinterpret_cast<const float2 *>(static_cast<char *>(workspace) + ws.own)};
    for (int first = 0; first < counters.count; first += kCounters) {
        CounterTable t;
        t.count = std::min(counters.count - first, kCounters);
        std::copy_n(counters.each + first, t.count, t.of);
        hipLaunchKernelGGL(k_adamw_counters, dim3(1), dim3(kCounters), 0, stm, t, args->beta1, args->beta2,
                           reinterpret_cast<float2 *>(static_cast<char *>(workspace) + ws.own) + first);
    }
    if (args->max_norm > 0 || args->counter) {
        double *sums = static_cast<double *>(workspace);
        // Few sums are added up by every workgroup of the update, many by a launch of one.  28 tensors of 235,000
        // elements: 15.6 us, with the launch 20.6 (before the tables of few gradients).
        const bool few = args->max_norm > 0 && s.squares > 0 && s.squares <= 256;
        int64_t count = 0;
        if (args->max_norm > 0) {
            squares_all<float>(args, sums, few ? args->counter : nullptr, &count, stm);
            squares_all<bf16>(args, sums, few ? args->counter : nullptr, &count, stm);
        }
        if (few) {
            r.sums = sums, r.count = (int)count;
        } else {
            float *shared = reinterpret_cast<float *>(static_cast<char *>(workspace) + ws.shared);
            hipLaunchKernelGGL(k_adamw_shared, dim3(1), dim3(256), 0, stm, sums, (int)count, args->max_norm,
                               args->beta1, args->beta2, args->counter, args->norm, shared);
            r.shared = shared;
        }
    }
    // Elements of a workgroup: 1,024, and 4,096 (more loads at once) where that leaves workgroups enough.
    const int steps = s.elements >= (int64_t)4096 * 2048 ? 4 : 1;
    update_all<float, float, false>(args, r, counters.of, steps, stm);
    update_all<float, bf16, false>(args, r, counters.of, steps, stm);
    update_all<bf16, float, false>(args, r, counters.of, steps, stm);
    update_all<bf16, bf16, false>(args, r, counters.of, steps, stm);
    update_all<bf16, float, true>(args, r, counters.of, steps, stm);
    update_all<bf16, bf16, true>(args, r, counters.of, steps, stm);
    return check_launch();
}
