// autograd_paged.h — the plain calls of the operators on a cache in pages, a part of autograd.cpp (after
// autograd_tokens.h, whose helpers it uses).  No gradients: a call that asks for one goes to paged.py, and raises.
#pragma once

namespace {

// A tensor that the kernels write into: autograd sees that it changed.
void written(const Tensor &t) {
    if (t.defined() && !t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

// No two elements in one place, of a tensor or of `copies` of it `between` elements apart.
bool is_apart(const Tensor &t, int64_t copies = 1, int64_t between = 0) {
    std::vector<std::pair<int64_t, int64_t>> axes;
    for (int64_t i = 0; i < t.dim(); ++i)
        if (t.size(i) > 1) axes.emplace_back(t.stride(i), t.size(i));
    if (copies > 1) axes.emplace_back(between, copies);
    std::sort(axes.begin(), axes.end());
    int64_t reach = 0;
    for (const auto &a : axes) {
        if (a.first <= reach) return false;
        reach += a.first * (a.second - 1);
    }
    return true;
}
int64_t reach_of(const Tensor &t) {
    int64_t reach = 1;
    for (int64_t i = 0; i < t.dim(); ++i) reach += t.stride(i) * (t.size(i) - 1);
    return reach;
}
// Two pools of one shape that share no element: one behind the other, or the halves of one pool.
bool are_apart(const Tensor &a, const Tensor &b) {
    const auto first = [](const Tensor &t) { return static_cast<int64_t>(reinterpret_cast<uintptr_t>(t.data_ptr())); };
    const int64_t size = a.element_size(), by = first(a) < first(b) ? first(b) - first(a) : first(a) - first(b);
    return by >= reach_of(first(a) < first(b) ? a : b) * size ||
           (a.strides() == b.strides() && by % size == 0 && is_apart(a, 2, by / size));
}

// Whether the memory from one's first element to its last one meets the other's.
bool meet(const Tensor &a, const Tensor &b) {
    const uintptr_t x = reinterpret_cast<uintptr_t>(a.data_ptr()), y = reinterpret_cast<uintptr_t>(b.data_ptr());
    return x < y + reach_of(b) * b.element_size() && y < x + reach_of(a) * a.element_size();
}

struct PagedCache {
    Tensor k, v, table, positions, keep;

    // Whether the kernels take the pools and the table as they are.
    bool plain(const at::Device &dev, at::ScalarType type, int64_t scenes) const {
        if (!is_tokens(k, 4, dev) || !is_tokens(v, 4, dev) || k.scalar_type() != type || v.scalar_type() != type ||
            k.sizes() != v.sizes())
            return false;
        const int64_t P = k.size(0), R = k.size(1), D = k.size(3);
        if (P < 1 || P > INT32_MAX || R < 16 || R % 16 || R > GSV_MAX_TOKENS || D < 8 || D > 128 || D % 8 ||
            !is_aligned(k) || !is_aligned(v))
            return false;
        if (table.layout() != at::kStrided || table.scalar_type() != at::kInt || table.device() != dev ||
            table.dim() != 2 || table.size(0) != scenes || (table.size(1) > 1 && table.stride(1) != 1) ||
            table.size(1) > GSV_MAX_TOKENS / R)
            return false;
        if (positions.defined() && !is_positions(positions, {P, R, 3}, dev)) return false;
        return !keep.defined() || is_mask(keep, {P, R}, dev);
    }
    gsv_pages args() const {
        gsv_pages p{};
        p.k = ptr<void>(k), p.v = ptr<void>(v);
        p.k_page = k.stride(0), p.k_row = k.stride(1), p.k_head = k.stride(2);
        p.v_page = v.stride(0), p.v_row = v.stride(1), p.v_head = v.stride(2);
        if (positions.defined())
            p.positions = ptr<float>(positions), p.pos_page = positions.stride(0), p.pos_row = positions.stride(1);
        if (keep.defined())
            p.keep = ptr<void>(keep), p.keep_page = keep.stride(0), p.keep_bytes = (int)keep.element_size();
        p.table = ptr<int32_t>(table), p.table_row = table.stride(0);
        p.pages = (int)k.size(0), p.page_rows = (int)k.size(1), p.table_pages = (int)table.size(1);
        return p;
    }
};

// {the turned queries, or nothing in their place}; empty for a call that paged.py takes.
std::vector<Maybe> append_tokens(const Tensor &k, const Tensor &v, const Tensor &k_pages, const Tensor &v_pages,
                                 const Tensor &table, const Tensor &lengths, const Maybe &queries,
                                 const Maybe &scene_starts, const Maybe &where, const Maybe &turns, bool interleaved,
                                 const Maybe &position_pages, const Maybe &keep, const Maybe &keep_pages) {
    if (!k.defined() || !k.is_cuda()) return {};
    const at::Device dev = k.device();
    const Tensor q = given(queries), starts = given(scene_starts), positions = given(where), freq = given(turns);
    const Tensor kept = given(keep);
    const PagedCache c{k_pages, v_pages, table, given(position_pages), given(keep_pages)};
    if (!is_tokens(k, 3, dev) || !is_tokens(v, 3, dev) || v.scalar_type() != k.scalar_type() ||
        v.sizes() != k.sizes() || table.dim() != 2)
        return {};
    const int64_t T = k.size(0), K = k.size(1), D = k.size(2), S = table.size(0);
    if (T < 1 || T > GSV_MAX_TOKENS || S > GSV_MAX_TOKENS || K < 1 || K > 4096 || !c.plain(dev, k.scalar_type(), S) ||
        c.k.size(2) != K || c.k.size(3) != D || !is_aligned(k) || !is_aligned(v) || !is_apart(c.k) || !is_apart(c.v) ||
        !are_apart(c.k, c.v) ||
        !is_vector(lengths, at::kInt, dev, S))
        return {};
    if (starts.defined() ? !is_vector(starts, at::kInt, dev, S + 1) : S != T) return {};
    if (positions.defined() &&
        (positions.layout() != at::kStrided || positions.scalar_type() != at::kFloat || positions.device() != dev ||
         positions.dim() != 2 || positions.size(0) != T))
        return {};
    if (freq.defined() &&
        (freq.scalar_type() != at::kFloat || freq.device() != dev || freq.dim() != 2 || !freq.is_contiguous() ||
         !positions.defined() || freq.size(0) != positions.size(1) || freq.size(0) < 1 || freq.size(0) > 8 ||
         freq.size(1) < 1 || 2 * freq.size(1) > D))
        return {};
    if (c.positions.defined() && (!positions.defined() || positions.size(1) != 3 || !is_apart(c.positions))) return {};
    if (positions.defined() && !freq.defined() && !c.positions.defined()) return {};
    if (kept.defined() != c.keep.defined() || (kept.defined() && (!is_mask(kept, {T}, dev) || !is_apart(c.keep))))
        return {};
    if (q.defined() && (!freq.defined() || !is_tokens(q, 3, dev) || q.scalar_type() != k.scalar_type() ||
                        q.size(0) != T || q.size(2) != D || q.size(1) < 1 || q.size(1) + K > 4096 || !is_aligned(q)))
        return {};
    for (const Tensor *t : {&k, &v, &q, &positions, &freq, &c.k, &c.v, &c.positions})
        if (wants_grad(*t)) return {};
    for (const Tensor *t : {&k, &v, &q})
        if (t->defined() && (meet(*t, c.k) || meet(*t, c.v))) return {};
    if ((c.positions.defined() && meet(positions, c.positions)) || (kept.defined() && meet(kept, c.keep))) return {};
    const c10::DeviceGuard guard(dev);
    gsv_rotary_args a{};
    a.k = ptr<void>(k), a.k_row = k.stride(0), a.k_head = k.stride(1), a.kv_heads = (int)K;
    Tensor out;
    if (q.defined()) {
        a.q = ptr<void>(q), a.q_row = q.stride(0), a.q_head = q.stride(1), a.heads = (int)q.size(1);
        out = empty(q.sizes(), q, q.scalar_type());
    }
    if (positions.defined()) {
        a.positions = ptr<float>(positions), a.axes = (int)positions.size(1);
        a.pos_row = positions.stride(0), a.pos_axis = positions.stride(1);
    }
    if (freq.defined()) a.frequencies = ptr<float>(freq), a.pairs = (int)freq.size(1);
    a.dtype = type_code(k), a.tokens = (int)T, a.dim = (int)D, a.interleaved = interleaved;
    const gsv_pages p = c.args();
    check(lib.gsv_paged_append(&a, ptr<void>(v), v.stride(0), v.stride(1), &p, ptr<int32_t>(lengths),
                               ptr<int32_t>(starts), (int)S, ptr<void>(kept),
                               kept.defined() ? (int)kept.element_size() : 0, ptr<void>(out), stream_of(k)),
          "paged_append");
    for (const Tensor *t : {&c.k, &c.v, &c.positions, &c.keep}) written(*t);
    return {maybe(out)};
}

std::vector<Tensor> paged_attention(const Tensor &q, const Tensor &k_pages, const Tensor &v_pages, const Tensor &table,
                                    const Tensor &lengths, double scale, double cap, const Maybe &positions,
                                    const Maybe &position_pages, const Maybe &slopes, const Maybe &keep_pages) {
    if (!q.defined() || !q.is_cuda()) return {};
    const at::Device dev = q.device();
    const PagedCache c{k_pages, v_pages, table, given(position_pages), given(keep_pages)};
    if (!is_tokens(q, 3, dev)) return {};
    const int64_t S = q.size(0);
    if (table.dim() != 2 || table.size(1) < 1 || !c.plain(dev, q.scalar_type(), S)) return {};
    AttentionCall a{q, c.k, c.v, given(slopes), Tensor(), Tensor(), Tensor(), given(positions), Tensor(), Tensor(), S,
                    0, false, 0.0, cap};
    if (!a.plain(4, scale) || !is_vector(lengths, at::kInt, dev, S) || wants_grad(q) || wants_grad(c.k) ||
        wants_grad(c.v) || wants_grad(a.slopes))
        return {};
    if (a.slopes.defined() ? !is_positions(a.q_pos, {S, 3}, dev) || !c.positions.defined()
                           : a.q_pos.defined() || c.positions.defined())
        return {};
    const c10::DeviceGuard guard(dev);
    a.k_pos = c.positions;  // (read by the pages' own members)
    const gsv_attention args = a.args();
    const gsv_pages p = c.args();
    Tensor out = empty(q.sizes(), q, q.scalar_type());
    size_t bytes = 0;
    check(lib.gsv_attention_paged_workspace_bytes(&args, &p, &bytes), "attention_paged_workspace_bytes");
    const Tensor ws = bytes ? workspace(bytes, q) : Tensor();
    check(lib.gsv_attention_paged(&args, &p, ptr<int32_t>(lengths), ptr<void>(out), ptr<void>(ws), bytes,
                                  stream_of(q)),
          "attention_paged");
    return {out};
}

}  // namespace
