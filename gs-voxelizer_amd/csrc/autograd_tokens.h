// autograd_tokens.h — the native autograd nodes of the operators on packed tokens, a part of
// autograd.cpp (it uses that file's helpers).
//
// As there: only plain calls come here, with tensors that the kernels take as they are; the
// functions return nothing for any other, and the Python modules (rotary.py, gated_norm.py,
// attention.py) do those, and raise every error.
#pragma once

#include <torch/csrc/autograd/functions/basic_ops.h>

namespace {

// A tensor argument that may be absent.
using Maybe = c10::optional<Tensor>;

Tensor given(const Maybe &t) { return t.has_value() ? *t : Tensor(); }
// As a node's input: an undefined tensor must not be one.
Maybe maybe(const Tensor &t) { return t.defined() ? Maybe(t) : Maybe(); }

bool token_type(const Tensor &t) {
    return t.scalar_type() == at::kFloat || t.scalar_type() == at::kBFloat16;
}
int type_code(const Tensor &t) { return t.scalar_type() == at::kBFloat16 ? GSV_BF16 : GSV_F32; }

bool wants_grad(const Tensor &t) {
    return t.defined() && at::GradMode::is_enabled() && t.requires_grad();
}

// Activations: float32 or bfloat16, `dims` axes, the last one contiguous, on this device.
bool is_tokens(const Tensor &t, int64_t dims, const at::Device &dev) {
    return t.defined() && t.layout() == at::kStrided && token_type(t) && t.device() == dev &&
           t.dim() == dims && t.stride(-1) == 1;
}
// Rows that start 16-byte aligned and lie within the attention kernels' reach; the stride of an axis
// of one entry says nothing.
bool is_aligned(const Tensor &t) {
    const int64_t size = t.element_size();
    if (reinterpret_cast<uintptr_t>(t.data_ptr()) % 16) return false;
    if (t.size(-3) > 1 && t.stride(-3) * size > (1 << 24)) return false;
    for (int64_t i = 0; i + 1 < t.dim(); ++i)
        if (t.size(i) > 1 && t.stride(i) * size % 16) return false;
    return true;
}
// Float32 rows of x, y, z.
bool is_positions(const Tensor &t, at::IntArrayRef shape, const at::Device &dev) {
    return t.defined() && t.layout() == at::kStrided && t.scalar_type() == at::kFloat &&
           t.device() == dev && t.sizes() == shape && t.stride(-1) == 1 && !wants_grad(t);
}
bool is_mask(const Tensor &t, at::IntArrayRef shape, const at::Device &dev) {
    const auto type = t.scalar_type();
    return t.layout() == at::kStrided && (type == at::kInt || type == at::kBool || type == at::kByte) &&
           t.device() == dev && t.sizes() == shape && t.stride(-1) == 1;
}
bool is_parameter(const Tensor &t, int64_t n, const at::Device &dev) {
    return !t.defined() || is_vector(t, at::kFloat, dev, n);
}

// The gradients of a backward whose kernels have no gradients themselves: differentiating
// them again raises, as it does after the Python classes.
variable_list once(variable_list grads) {
    if (!at::GradMode::is_enabled()) return grads;
    variable_list out;
    for (Tensor &g : grads) {
        if (!g.defined()) {
            out.push_back(g);
            continue;
        }
        auto node = std::make_shared<torch::autograd::DelayedError>(
            "gs_voxelizer: this operator's gradients can be differentiated once only", 1);
        out.push_back((*node)({g.detach().requires_grad_()})[0]);
    }
    return out;
}

// ------------------------------------------------------------------ rotary --

Tensor rotary_out(const Tensor &t) {
    return t.defined() ? at::empty(t.sizes(), t.options().memory_format(at::MemoryFormat::Contiguous)) : t;
}

// q or k may be undefined.
variable_list turn(const Tensor &q, const Tensor &k, const Tensor &positions,
                   const Tensor &frequencies, bool interleaved, bool inverse) {
    const Tensor &one = q.defined() ? q : k;
    gsv_rotary_args a{};
    a.positions = ptr<float>(positions);
    a.frequencies = ptr<float>(frequencies);
    a.pos_row = positions.stride(0), a.pos_axis = positions.stride(1);
    a.dtype = type_code(one), a.tokens = (int)one.size(0), a.dim = (int)one.size(2);
    a.pairs = (int)frequencies.size(1), a.axes = (int)frequencies.size(0), a.interleaved = interleaved;
    if (q.defined())
        a.q = ptr<void>(q), a.q_row = q.stride(0), a.q_head = q.stride(1), a.heads = (int)q.size(1);
    if (k.defined())
        a.k = ptr<void>(k), a.k_row = k.stride(0), a.k_head = k.stride(1), a.kv_heads = (int)k.size(1);
    const Tensor q_out = rotary_out(q), k_out = rotary_out(k);
    check(lib.gsv_rotary(&a, ptr<void>(q_out), ptr<void>(k_out), inverse, stream_of(one)), "rotary");
    return {q_out, k_out};
}

struct Rotate : public torch::autograd::Function<Rotate> {
    static variable_list forward(AutogradContext *ctx, const Tensor &q, const Tensor &k,
                                 const Tensor &positions, const Tensor &frequencies, bool interleaved) {
        ctx->saved_data["interleaved"] = interleaved;
        ctx->saved_data["shape"] = std::vector<int64_t>{q.size(0), q.get_device()};
        ctx->save_for_backward({positions, frequencies});
        ctx->set_materialize_grads(false);
        return turn(q, k, positions, frequencies, interleaved, false);
    }
    static variable_list backward(AutogradContext *ctx, const variable_list &grads) {
        const auto saved = ctx->get_saved_variables();
        const auto shape = ctx->saved_data["shape"].toIntVector();
        const at::Device dev = gpu(shape[1]);
        const Tensor &pos = saved[0], &freq = saved[1];
        TORCH_CHECK(pos.device() == dev && pos.scalar_type() == at::kFloat && pos.dim() == 2 &&
                        pos.size(0) == shape[0] && freq.device() == dev &&
                        freq.scalar_type() == at::kFloat && freq.is_contiguous() &&
                        freq.dim() == 2 && freq.size(0) == pos.size(1),
                    "positions and frequencies: expected the forward's");
        Tensor g[2];
        for (int i = 0; i < 2; ++i) {
            if (!ctx->needs_input_grad(i) || !grads[i].defined()) continue;
            TORCH_CHECK(grads[i].device() == dev && grads[i].dim() == 3 && token_type(grads[i]),
                        "the gradients of q and k must have their type and shape");
            g[i] = grads[i].stride(-1) == 1 ? grads[i] : grads[i].contiguous();
        }
        if (!g[0].defined() && !g[1].defined()) return variable_list(5);
        const c10::DeviceGuard guard(dev);
        variable_list d = turn(g[0], g[1], pos, freq, ctx->saved_data["interleaved"].toBool(), true);
        return once({d[0], d[1], Tensor(), Tensor(), Tensor()});
    }
};

std::vector<Tensor> rotate(const Tensor &q, const Tensor &k, const Tensor &positions,
                           const Tensor &frequencies, bool interleaved) {
    if (!q.defined() || !q.is_cuda()) return {};
    const at::Device dev = q.device();
    if (!is_tokens(q, 3, dev) || !is_tokens(k, 3, dev) || k.scalar_type() != q.scalar_type()) return {};
    const int64_t T = q.size(0), D = q.size(2);
    if (k.size(0) != T || k.size(2) != D || T < 1 || T > GSV_MAX_TOKENS || D > 1024 ||
        q.size(1) + k.size(1) > 4096 || positions.dim() != 2 || frequencies.dim() != 2 ||
        positions.scalar_type() != at::kFloat || frequencies.scalar_type() != at::kFloat ||
        positions.device() != dev || frequencies.device() != dev || !frequencies.is_contiguous() ||
        wants_grad(positions) || wants_grad(frequencies))
        return {};
    const int64_t A = frequencies.size(0), P = frequencies.size(1);
    if (positions.size(0) != T || positions.size(1) != A || A < 1 || A > 8 || P < 1 || 2 * P > D) return {};
    const c10::DeviceGuard guard(dev);
    if (!wants_grad(q) && !wants_grad(k)) return turn(q, k, positions, frequencies, interleaved, false);
    return Rotate::apply(q, k, positions, frequencies, interleaved);
}

// -------------------------------------------------------------- gated norm --

struct NormCall {
    Tensor x, branch, weight, branch_weight, scale, gate, starts;
    int64_t scenes;
    bool per_token;
    double eps;

    gsv_norm args() const {
        gsv_norm n{};
        n.x = ptr<void>(x), n.branch = ptr<void>(branch), n.gate = ptr<void>(gate);
        n.weight = ptr<float>(weight), n.branch_weight = ptr<float>(branch_weight);
        n.scale = ptr<float>(scale), n.starts = ptr<int32_t>(starts);
        n.x_row = x.stride(0), n.branch_row = branch.stride(0);
        n.gate_row = gate.defined() ? gate.stride(0) : 0;
        n.dtype = type_code(x), n.branch_dtype = type_code(branch);
        n.gate_dtype = gate.defined() ? type_code(gate) : 0;
        n.gate_per_token = per_token;
        n.tokens = (int)x.size(0), n.channels = (int)x.size(1), n.scenes = (int)scenes;
        n.eps = (float)eps;
        return n;
    }
    variable_list forward() const {
        const gsv_norm n = args();
        Tensor y = empty(x.sizes(), x, x.scalar_type()), h = empty(x.sizes(), x, branch.scalar_type());
        check(lib.gsv_gated_norm_fwd(&n, ptr<void>(y), ptr<void>(h), stream_of(x)), "gated_norm_fwd");
        return {y, h};
    }
};

struct GatedNorm : public torch::autograd::Function<GatedNorm> {
    static variable_list forward(AutogradContext *ctx, const Tensor &x, const Tensor &branch,
                                 const Tensor &weight, const Maybe &, const Maybe &, const Maybe &,
                                 const NormCall *c) {
        const Tensor &branch_weight = c->branch_weight, &scale = c->scale, &gate = c->gate;
        ctx->saved_data["kept"] = std::vector<int64_t>{
            x.size(0), x.size(1), x.get_device(), c->scenes, c->per_token,
            gate.defined() ? gate.size(0) : 0, type_code(x), type_code(branch),
            gate.defined() ? type_code(gate) : 0};
        ctx->saved_data["eps"] = c->eps;
        ctx->save_for_backward({x, branch, weight, branch_weight, scale, gate, c->starts});
        ctx->set_materialize_grads(false);
        return c->forward();
    }
    static variable_list backward(AutogradContext *ctx, const variable_list &grads) {
        const auto saved = ctx->get_saved_variables();
        const auto k = ctx->saved_data["kept"].toIntVector();
        const int64_t T = k[0], C = k[1];
        const at::Device dev = gpu(k[2]);
        if (!grads[0].defined() && !grads[1].defined()) return variable_list(7);
        const auto type = [](int64_t code) { return code == GSV_BF16 ? at::kBFloat16 : at::kFloat; };
        const auto rows = [&](const Tensor &t, int64_t code, int64_t n, const char *what) {
            TORCH_CHECK(t.defined() && t.device() == dev && t.scalar_type() == type(code) &&
                            t.dim() == 2 && t.size(0) == n && t.size(1) == C,
                        what, ": expected ", n, " rows of ", C, " values on ", dev);
            return t.stride(1) == 1 ? t : t.contiguous();
        };
        const auto vec = [&](const Tensor &t, const char *what) {
            return t.defined() ? unpacked(t, at::kFloat, dev, C, what) : t;
        };
        NormCall c{rows(saved[0], k[6], T, "x"), rows(saved[1], k[7], T, "branch"),
                   vec(saved[2], "weight"), vec(saved[3], "branch_weight"), vec(saved[4], "scale"),
                   saved[5].defined() ? rows(saved[5], k[8], k[5], "gate") : saved[5], saved[6],
                   k[3], k[4] != 0, ctx->saved_data["eps"].toDouble()};
        if (c.starts.defined())
            c.starts = unpacked(c.starts, at::kInt, dev, c.scenes + 1, "scene_starts");
        const c10::DeviceGuard guard(dev);
        const Tensor dy = grads[0].defined() ? rows(grads[0], k[6], T, "the gradient of y") : Tensor();
        const Tensor dh = grads[1].defined() ? rows(grads[1], k[7], T, "the gradient of h") : Tensor();
        const gsv_norm n = c.args();
        const auto like = [&](const Tensor &t) {
            return t.defined() ? empty(t.sizes(), t, t.scalar_type()) : Tensor();
        };
        Tensor dx = like(c.x), db = like(c.branch), dw = like(c.weight), dbw = like(c.branch_weight);
        Tensor ds = like(c.scale), dg = like(c.gate);
        size_t bytes = 0;
        check(lib.gsv_gated_norm_bwd_workspace_bytes(&n, &bytes), "gated_norm_bwd_workspace_bytes");
        const Tensor ws = workspace(bytes, c.x);
        check(lib.gsv_gated_norm_bwd(&n, ptr<void>(dy), dy.defined() ? dy.stride(0) : 0, ptr<void>(dh),
                                     dh.defined() ? dh.stride(0) : 0, ptr<void>(dx), ptr<void>(db),
                                     ptr<float>(dw), ptr<float>(dbw), ptr<float>(ds), ptr<void>(dg),
                                     ptr<void>(ws), bytes, stream_of(c.x)),
              "gated_norm_bwd");
        return once({dx, db, dw, dbw, ds, dg, Tensor()});
    }
};

std::vector<Tensor> gated_norm(const Tensor &x, const Tensor &branch, const Tensor &weight,
                               const Maybe &branch_weight, const Maybe &scale, const Maybe &gate,
                               const Maybe &scene_starts, double eps) {
    if (!x.defined() || !x.is_cuda()) return {};
    const at::Device dev = x.device();
    if (!is_tokens(x, 2, dev) || !is_tokens(branch, 2, dev) || branch.sizes() != x.sizes() ||
        !(branch.scalar_type() == x.scalar_type() || x.scalar_type() == at::kFloat))
        return {};
    const int64_t T = x.size(0), C = x.size(1);
    NormCall c{x, branch, weight, given(branch_weight), given(scale), given(gate), given(scene_starts),
               1, false, eps};
    if (T < 1 || T > GSV_MAX_TOKENS || C < 1 || C > 8192 || !(eps >= 0) ||
        !weight.defined() || !is_parameter(weight, C, dev) || !is_parameter(c.branch_weight, C, dev) ||
        !is_parameter(c.scale, C, dev))
        return {};
    if (c.starts.defined()) {
        c.scenes = c.starts.numel() - 1;
        if (c.scenes < 1 || !is_vector(c.starts, at::kInt, dev, c.scenes + 1)) return {};
    }
    if (c.gate.defined()) {
        if (!is_tokens(c.gate, 2, dev) || c.gate.size(1) != C ||
            !(c.gate.scalar_type() == at::kFloat || c.gate.scalar_type() == branch.scalar_type()))
            return {};
        c.per_token = !c.starts.defined() && c.gate.size(0) == T && T != 1;
        if (!c.per_token && c.gate.size(0) != c.scenes) return {};
    }
    if (!c.gate.defined() || c.per_token) c.starts = Tensor(), c.scenes = 1;
    const c10::DeviceGuard guard(dev);
    bool grad = false;
    for (const Tensor *t : {&c.x, &c.branch, &c.weight, &c.branch_weight, &c.scale, &c.gate})
        grad |= wants_grad(*t);
    if (!grad) return c.forward();
    return GatedNorm::apply(c.x, c.branch, c.weight, maybe(c.branch_weight), maybe(c.scale),
                            maybe(c.gate), (const NormCall *)&c);
}

// --------------------------------------------------------------- attention --

struct AttentionCall {
    Tensor q, k, v, slopes, q_starts, k_starts, prefix, q_pos, k_pos, keep;
    int64_t scenes, longest;
    bool causal;
    double scale, cap;

    gsv_attention args() const {
        gsv_attention a{};
        a.q = ptr<void>(q), a.q_row = q.stride(0), a.q_head = q.stride(1);
        a.k = ptr<void>(k), a.k_row = k.stride(-3), a.k_head = k.stride(-2);
        a.v = ptr<void>(v), a.v_row = v.stride(-3), a.v_head = v.stride(-2);
        a.q_starts = ptr<int32_t>(q_starts), a.k_starts = ptr<int32_t>(k_starts);
        a.prefix = ptr<int32_t>(prefix);
        if (slopes.defined()) {
            a.slopes = ptr<void>(slopes), a.slopes_dtype = type_code(slopes);
            a.q_positions = ptr<float>(q_pos), a.q_pos_row = q_pos.stride(0);
            a.k_positions = ptr<float>(k_pos), a.k_pos_row = k_pos.stride(-2);
        }
        if (keep.defined()) a.keep = ptr<void>(keep), a.keep_bytes = (int)keep.element_size();
        a.dtype = type_code(q), a.causal = causal;
        a.q_tokens = (int)q.size(0), a.k_tokens = (int)k.size(-3);
        a.heads = (int)q.size(1), a.kv_heads = (int)k.size(-2), a.dim = (int)q.size(2);
        a.scenes = (int)scenes, a.longest_q = a.longest_k = (int)longest;
        a.scale = (float)scale, a.cap = (float)cap;
        return a;
    }
    // The checks of both entry points; dims: the key tensors' axes.
    bool plain(int64_t dims, double scale_or_0) {
        if (!q.defined() || !q.is_cuda()) return false;
        const at::Device dev = q.device();
        if (!is_tokens(q, 3, dev) || !is_tokens(k, dims, dev) || !is_tokens(v, dims, dev) ||
            k.scalar_type() != q.scalar_type() || v.scalar_type() != q.scalar_type() ||
            k.sizes() != v.sizes())
            return false;
        const int64_t H = q.size(1), K = k.size(-2), D = q.size(2);
        if (k.size(-1) != D || D < 8 || D > 128 || D % 8 || H < 1 || K < 1 || H % K ||
            q.size(0) < 1 || q.size(0) > GSV_MAX_TOKENS || k.size(-3) < 1 || k.size(-3) > GSV_MAX_TOKENS ||
            longest < 0 || longest > INT32_MAX)
            return false;
        if (!is_aligned(q) || !is_aligned(k) || !is_aligned(v)) return false;
        scale = scale_or_0 == 0 ? 1.0 / std::sqrt((double)D) : scale_or_0;
        if (!((float)scale > 0) || !(cap >= 0) || !std::isfinite((float)scale) || !std::isfinite((float)cap)) return false;
        return !slopes.defined() ||
               (token_type(slopes) && is_vector(slopes, slopes.scalar_type(), dev, H));
    }
};

struct SceneAttention : public torch::autograd::Function<SceneAttention> {
    static Tensor forward(AutogradContext *ctx, const Tensor &q, const Tensor &k, const Tensor &v,
                          const Maybe &, const AttentionCall *c) {
        const Tensor &slopes = c->slopes;
        const gsv_attention a = c->args();
        Tensor out = empty(q.sizes(), q, q.scalar_type());
        Tensor lse = empty({q.size(1), q.size(0)}, q, at::kFloat);
        // what rounding took from the output: the backward needs it whole
        Tensor low = q.scalar_type() == at::kBFloat16 ? empty(q.sizes(), q, q.scalar_type()) : Tensor();
        check(lib.gsv_attention_fwd(&a, ptr<void>(out), ptr<void>(low), ptr<float>(lse), stream_of(q)),
              "attention_fwd");
        ctx->saved_data["kept"] = std::vector<int64_t>{
            q.get_device(), q.size(0), q.size(1), q.size(2), k.size(0), k.size(1), c->scenes,
            c->longest, c->causal, type_code(q), slopes.defined() ? type_code(slopes) : -1};
        ctx->saved_data["scale"] = c->scale;
        ctx->saved_data["cap"] = c->cap;
        ctx->save_for_backward({q, k, v, slopes, out, low, lse, c->q_starts, c->k_starts, c->prefix,
                                c->q_pos, c->k_pos, c->keep});
        ctx->set_materialize_grads(false);
        return out;
    }
    static variable_list backward(AutogradContext *ctx, const variable_list &grads) {
        if (!grads[0].defined()) return variable_list(5);
        const auto s = ctx->get_saved_variables();
        const auto m = ctx->saved_data["kept"].toIntVector();
        const at::Device dev = gpu(m[0]);
        const int64_t T = m[1], H = m[2], D = m[3], N = m[4], K = m[5], scenes = m[6];
        const auto type = m[9] == GSV_BF16 ? at::kBFloat16 : at::kFloat;
        const auto heads = [&](const Tensor &t, int64_t n, int64_t h, const char *what) {
            TORCH_CHECK(t.defined() && t.device() == dev && t.scalar_type() == type && t.dim() == 3 &&
                            t.size(0) == n && t.size(1) == h && t.size(2) == D,
                        what, ": expected shape (", n, ", ", h, ", ", D, ") on ", dev);
            return t.stride(2) == 1 && is_aligned(t) ? t : t.clone(at::MemoryFormat::Contiguous);
        };
        const auto ints = [&](const Tensor &t, int64_t n, const char *what) {
            return t.defined() ? unpacked(t, at::kInt, dev, n, what) : t;
        };
        const auto places = [&](const Tensor &t, int64_t n, const char *what) {
            if (!t.defined()) return t;
            TORCH_CHECK(t.device() == dev && t.scalar_type() == at::kFloat && t.dim() == 2 &&
                            t.size(0) == n && t.size(1) == 3,
                        what, ": expected ", n, " rows of 3 float32 values on ", dev);
            return t.stride(1) == 1 ? t : t.contiguous();
        };
        AttentionCall c{heads(s[0], T, H, "q"), heads(s[1], N, K, "k"), heads(s[2], N, K, "v"),
                        s[3], ints(s[7], scenes + 1, "scene_starts"), ints(s[8], scenes + 1, "key_starts"),
                        ints(s[9], scenes, "prefix"), places(s[10], T, "positions"),
                        places(s[11], N, "key_positions"), s[12], scenes, m[7], m[8] != 0,
                        ctx->saved_data["scale"].toDouble(), ctx->saved_data["cap"].toDouble()};
        if (c.slopes.defined())
            c.slopes = unpacked(c.slopes, m[10] == GSV_BF16 ? at::kBFloat16 : at::kFloat, dev, H, "slopes");
        TORCH_CHECK(!c.keep.defined() || is_mask(c.keep, {N}, dev), "keep: expected ", N, " values on ", dev);
        const Tensor out = heads(s[4], T, H, "out").contiguous();
        const Tensor low = s[5].defined() ? heads(s[5], T, H, "out_low").contiguous() : s[5];
        const Tensor lse = unpacked(s[6], at::kFloat, dev, H * T, "the log sums");
        const Tensor dout = heads(grads[0], T, H, "the gradient");
        const c10::DeviceGuard guard(dev);
        const gsv_attention a = c.args();
        Tensor dq = empty({T, H, D}, out, type), dk = empty({N, K, D}, out, type);
        Tensor dv = empty({N, K, D}, out, type);
        Tensor ds = c.slopes.defined() ? empty({H}, out, c.slopes.scalar_type()) : Tensor();
        size_t bytes = 0;
        check(lib.gsv_attention_bwd_workspace_bytes(&a, &bytes), "attention_bwd_workspace_bytes");
        const Tensor ws = workspace(bytes, out);
        check(lib.gsv_attention_bwd(&a, ptr<void>(out), ptr<void>(low), ptr<float>(lse), ptr<void>(dout),
                                    dout.stride(0), dout.stride(1), ptr<void>(dq), ptr<void>(dk), ptr<void>(dv),
                                    ptr<void>(ds), ptr<void>(ws), bytes, stream_of(out)),
              "attention_bwd");
        return once({dq, dk, dv, ds, Tensor()});
    }
};

std::vector<Tensor> scene_attention(const Tensor &q, const Tensor &k, const Tensor &v,
                                    const Maybe &scene_starts, const Maybe &key_starts, int64_t longest,
                                    bool causal, const Maybe &prefix, double scale, double cap,
                                    const Maybe &positions, const Maybe &key_positions,
                                    const Maybe &slopes, const Maybe &keep) {
    AttentionCall c{q, k, v, given(slopes), given(scene_starts), given(key_starts), given(prefix),
                    given(positions), given(key_positions), given(keep), 1, longest, causal, 0.0, cap};
    if (!c.plain(3, scale)) return {};
    const at::Device dev = q.device();
    const int64_t T = q.size(0), N = k.size(0);
    if (c.q_starts.defined()) {
        c.scenes = c.q_starts.numel() - 1;
        if (c.scenes < 1 || !is_vector(c.q_starts, at::kInt, dev, c.scenes + 1)) return {};
    }
    if (c.k_starts.defined()) {
        if (!is_vector(c.k_starts, at::kInt, dev, c.scenes + 1)) return {};
    } else {
        if (c.scenes != 1 && N != T) return {};
        c.k_starts = c.q_starts;
    }
    if (c.prefix.defined() && (!causal || !is_vector(c.prefix, at::kInt, dev, c.scenes))) return {};
    if (c.slopes.defined()) {
        if (!c.k_pos.defined()) c.k_pos = c.q_pos;
        if (!is_positions(c.q_pos, {T, 3}, dev) || !is_positions(c.k_pos, {N, 3}, dev)) return {};
    } else if (c.q_pos.defined() || c.k_pos.defined()) {
        return {};
    }
    if (c.keep.defined() && !is_mask(c.keep, {N}, dev)) return {};
    const c10::DeviceGuard guard(dev);
    if (wants_grad(q) || wants_grad(k) || wants_grad(v) || wants_grad(c.slopes))
        return {SceneAttention::apply(q, k, v, maybe(c.slopes), (const AttentionCall *)&c)};
    const gsv_attention a = c.args();
    Tensor out = empty(q.sizes(), q, q.scalar_type());
    check(lib.gsv_attention_fwd(&a, ptr<void>(out), nullptr, nullptr, stream_of(q)), "attention_fwd");
    return {out};
}

std::vector<Tensor> cached_attention(const Tensor &q, const Tensor &k, const Tensor &v,
                                     const Tensor &lengths, double scale, double cap,
                                     const Maybe &positions, const Maybe &key_positions,
                                     const Maybe &slopes, const Maybe &keep) {
    AttentionCall c{q, k, v, given(slopes), Tensor(), Tensor(), Tensor(), given(positions),
                    given(key_positions), given(keep), q.defined() && q.dim() == 3 ? q.size(0) : 0, 0,
                    false, 0.0, cap};
    if (!c.plain(4, scale)) return {};
    const at::Device dev = q.device();
    const int64_t S = q.size(0), N = k.size(1);
    if (k.size(0) != S || !is_vector(lengths, at::kInt, dev, S) || wants_grad(q) || wants_grad(k) ||
        wants_grad(v) || wants_grad(c.slopes))
        return {};
    if (c.slopes.defined()) {
        if (!is_positions(c.q_pos, {S, 3}, dev) || !is_positions(c.k_pos, {S, N, 3}, dev)) return {};
    } else if (c.q_pos.defined() || c.k_pos.defined()) {
        return {};
    }
    if (c.keep.defined() && !is_mask(c.keep, {S, N}, dev)) return {};
    const c10::DeviceGuard guard(dev);
    const gsv_attention a = c.args();
    Tensor out = empty(q.sizes(), q, q.scalar_type());
    size_t bytes = 0;
    check(lib.gsv_attention_cached_workspace_bytes(&a, &bytes), "attention_cached_workspace_bytes");
    const Tensor ws = bytes ? workspace(bytes, q) : Tensor();
    check(lib.gsv_attention_cached(&a, ptr<int32_t>(lengths), k.stride(0), v.stride(0),
                                   c.slopes.defined() ? c.k_pos.stride(0) : 0,
                                   c.keep.defined() ? c.keep.stride(0) : 0, ptr<void>(out),
                                   ptr<void>(ws), bytes, stream_of(q)),
          "attention_cached");
    return {out};
}

}  // namespace
