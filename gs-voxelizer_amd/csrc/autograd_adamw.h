// autograd_adamw.h — the plain calls of the optimiser's step, a part of autograd.cpp (after autograd_paged.h).
#pragma once

#include <c10/hip/HIPGraphsC10Utils.h>

namespace {

// A tensor with memory of its own in one run, no subclass's that answers calls itself.
bool is_dense(const Tensor &t, const at::Device &dev) {
    return t.defined() && t.layout() == at::kStrided && t.device() == dev &&
           !t.key_set().has(c10::DispatchKey::Python) && t.unsafeGetTensorImpl()->has_storage() &&
           t.is_non_overlapping_and_dense();
}
// The same shape, laid out alike.
bool is_like(const Tensor &t, const Tensor &p, const at::Device &dev) {
    return is_dense(t, dev) && t.sizes() == p.sizes() && t.strides() == p.strides();
}

// {whether it was done; the norm, where it is asked for}: adamw.py does the other calls.
std::pair<bool, Maybe> adamw_step(const std::vector<Tensor> &params, const std::vector<Tensor> &grads,
                                  const std::vector<Tensor> &exp_avgs, const std::vector<Tensor> &exp_avg_sqs,
                                  const std::vector<Maybe> &masters, const std::vector<int64_t> &steps,
                                  const Maybe &counted, const std::vector<double> &rates,
                                  const std::vector<double> &decays, double beta1, double beta2, double eps,
                                  double max_norm) {
    const std::pair<bool, Maybe> other{false, Maybe()};
    const size_t n = params.size();
    const Tensor counter = given(counted);
    if (!n || grads.size() != n || exp_avgs.size() != n || exp_avg_sqs.size() != n ||
        (!masters.empty() && masters.size() != n) || (!counter.defined() && steps.size() != n) || rates.size() != n ||
        decays.size() != n || !(beta1 >= 0 && beta1 < 1) || !(beta2 >= 0 && beta2 < 1) || !(eps >= 0) ||
        !(max_norm >= 0) || !params[0].defined() || !params[0].is_cuda())
        return other;
    const at::Device dev = params[0].device();
    if (counter.defined() ? !is_vector(counter, at::kInt, dev, 1)
                          : c10::hip::currentStreamCaptureStatusMayInitCtx() != c10::hip::CaptureStatus::None)
        return other;
    std::vector<gsv_adamw_tensor> all(n);
    for (size_t i = 0; i < n; ++i) {
        const Tensor &p = params[i], &g = grads[i], &m = exp_avgs[i], &v = exp_avg_sqs[i];
        const Tensor w = masters.empty() ? Tensor() : given(masters[i]);
        if (!is_dense(p, dev) || !token_type(p) || !is_like(g, p, dev) || !token_type(g) || !is_like(m, p, dev) ||
            m.scalar_type() != at::kFloat || !is_like(v, p, dev) || v.scalar_type() != at::kFloat ||
            (w.defined() && (!is_like(w, p, dev) || w.scalar_type() != at::kFloat || p.scalar_type() == at::kFloat)) ||
            (!counter.defined() && steps[i] < 1) || !(rates[i] >= 0) || !(decays[i] >= 0))
            return other;
        gsv_adamw_tensor &t = all[i];
        t = gsv_adamw_tensor{};
        t.param = ptr<void>(p), t.grad = ptr<void>(g), t.exp_avg = ptr<float>(m), t.exp_avg_sq = ptr<float>(v);
        t.master = ptr<float>(w), t.numel = p.numel(), t.step = counter.defined() ? 0 : steps[i];
        t.lr = rates[i], t.weight_decay = decays[i], t.dtype = type_code(p), t.grad_dtype = type_code(g);
    }
    const c10::DeviceGuard guard(dev);
    gsv_adamw_args a{};
    a.tensors = all.data(), a.count = (int64_t)n;
    a.beta1 = beta1, a.beta2 = beta2, a.eps = eps, a.max_norm = max_norm, a.counter = ptr<int32_t>(counter);
    Tensor norm;
    if (max_norm > 0) {
        norm = empty({}, exp_avgs[0], at::kFloat);
        a.norm = ptr<float>(norm);
    }
    size_t bytes = 0;
    check(lib.gsv_adamw_workspace_bytes(&a, &bytes), "adamw_workspace_bytes");
    const Tensor ws = bytes ? workspace(bytes, params[0]) : Tensor();
    const int status = lib.gsv_adamw(&a, ptr<void>(ws), bytes, stream_of(params[0]));
    if (status == GSV_ERR_INVALID_ARGUMENT) return other;  // tensors share memory; nothing was launched
    check(status, "adamw");
    for (size_t i = 0; i < n; ++i) {
        written(params[i]), written(exp_avgs[i]), written(exp_avg_sqs[i]);
        if (!masters.empty()) written(given(masters[i]));
    }
    written(counter);
    return {true, maybe(norm)};
}

}  // namespace
