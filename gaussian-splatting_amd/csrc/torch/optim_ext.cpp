// Host layer of the gradient norm, clipping, the Adam step under a ceiling and the eviction to a row budget
// (grad_clip.hip, evict.hip): lists of tensors are checked and turned into the C ABI's tables here, because a list of
// several hundred tensors costs Python more than the kernels take.  Host code only.
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPGraphsC10Utils.h>
#include <torch/extension.h>

#include <algorithm>
#include <cmath>
#include <functional>
#include <vector>

#include "../../../include/gsplat_amd.h"

namespace {

using torch::Tensor;

void check_rc(int rc, const char* what) { TORCH_CHECK(rc == GSR_OK, what, ": ", gsr_status_string(rc), " (", rc, ")"); }

void* stream_on(const c10::Device& dev) {
    return (void*)c10::hip::getCurrentHIPStreamMasqueradingAsCUDA(dev.index()).stream();
}

// What a kernel has written through a pointer counts as an in-place change for autograd.
void changed(const Tensor& t) {
    if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}

int norm_kind(double p, const char* what) {
    TORCH_CHECK(p == 1.0 || p == 2.0 || (std::isinf(p) && p > 0), what, ": norm_type must be 1, 2 or inf, got ", p);
    return std::isinf(p) ? 0 : (int)p;
}

int type_of(const Tensor& t, const char* what) {
    switch (t.scalar_type()) {
        case torch::kFloat32: return GSO_F32;
        case torch::kBFloat16: return GSO_BF16;
        case torch::kFloat16: return GSO_F16;
        default: TORCH_CHECK(false, what, ": gradients must be float32, bfloat16 or float16, got ", t.scalar_type());
    }
    return 0;
}

// The values that a tensor stands for in its memory (a lazy conjugate or negative has others there).
Tensor plain(const Tensor& t) { return t.is_conj() || t.is_neg() ? t.resolve_conj().resolve_neg() : t; }

// Memory that a call writes must not overlap any other that it uses: the kernels work on all tensors at once.
struct Spans {
    struct Span {
        uintptr_t begin, end;
        bool written;
    };
    std::vector<Span> all;
    void add(const void* p, int64_t bytes, bool written) {
        if (bytes > 0) all.push_back({(uintptr_t)p, (uintptr_t)p + (uintptr_t)bytes, written});
    }
    bool disjoint() {
        const auto before = [](const Span& a, const Span& b) { return a.begin < b.begin; };
        if (!std::is_sorted(all.begin(), all.end(), before)) std::sort(all.begin(), all.end(), before);
        uintptr_t end = 0, written_end = 0;
        for (const Span& s : all) {
            if (s.begin < (s.written ? end : written_end)) return false;
            end = std::max(end, s.end);
            if (s.written) written_end = std::max(written_end, s.end);
        }
        return true;
    }
};

// The gradients of a list of parameters as the C ABI takes them (the list outlives it).  A gradient whose elements do not
// fill a block of memory of their own (a slice of something wider) is worked on in a packed copy.
struct Grads {
    std::vector<const Tensor*> own;
    std::vector<Tensor> held;
    std::vector<c10::Storage> memory;
    std::vector<std::pair<size_t, Tensor>> packed;   // (index, copy)
    std::vector<void*> ptr;
    std::vector<int64_t> numel;
    std::vector<int> type;
    c10::Device device = c10::Device(c10::kCPU);
    int n() const { return (int)ptr.size(); }
    const void* const* cptr() const { return (const void* const*)ptr.data(); }
    // Before the host waits: other threads of the program run then, and may give the parameters other gradients, or a tensor
    // other memory.
    void hold() {
        held.reserve(own.size());
        for (const Tensor*& t : own) {
            held.push_back(*t);
            memory.push_back(t->storage());
            t = &held.back();
        }
    }
};

// A number that the device is still computing; other Python threads run while the host waits for it.
double wait_for(const Tensor& t) {
    pybind11::gil_scoped_release others;
    return t.item<double>();
}

Grads collect(const std::vector<Tensor>& params, const char* what) {
    torch::NoGradGuard no_grad;
    Grads g;
    const size_t n = params.size();
    g.own.reserve(n);
    g.ptr.reserve(n);
    g.numel.reserve(n);
    g.type.reserve(n);
    for (const Tensor& p : params) {
        TORCH_CHECK(p.defined(), what, ": expected tensors");
        const Tensor& t = p.grad();
        if (!t.defined()) continue;
        TORCH_CHECK(t.layout() == c10::kStrided, what, ": gradients must be dense, got layout ", t.layout());
        TORCH_CHECK(t.is_cuda(), what, ": gradients must be GPU tensors (there is no CPU path), got one on ", t.device());
        if (g.own.empty()) g.device = t.device();
        TORCH_CHECK(t.device() == g.device, what, ": gradients must be on one device, got ", g.device, " and ", t.device());
        g.type.push_back(type_of(t, what));
        if (!t.is_non_overlapping_and_dense() || t.is_neg()) {
            g.packed.emplace_back(g.own.size(), plain(t).contiguous());
            g.ptr.push_back(g.packed.back().second.data_ptr());
        } else {
            g.ptr.push_back(t.data_ptr());
        }
        g.own.push_back(&t);
        g.numel.push_back(t.numel());
    }
    return g;
}

// Whether x_0 * stride_0 + x_1 * stride_1 + ... = target has a solution in 0 <= x_k <= most_k.  Larger strides first; in the
// layouts of tensors each leaves the next a few values.  A search that takes too long counts as a solution.
struct Places {
    std::vector<std::pair<int64_t, int64_t>> terms;   // (stride > 0, most > 0)
    void add(int64_t stride, int64_t most) {
        if (most <= 0) return;
        for (auto& t : terms)
            if (t.first == stride) {
                t.second += most;
                return;
            }
        terms.emplace_back(stride, most);
    }
    bool reach(int64_t target) {
        std::sort(terms.begin(), terms.end(), std::greater<>());
        int64_t rest = 0;
        for (const auto& t : terms) rest += t.first * t.second;
        int64_t steps = 1 << 20;
        return search(0, target, rest, steps);
    }
    bool search(size_t k, int64_t target, int64_t rest, int64_t& steps) const {   // rest: the most that terms k and on can give
        if (target < 0 || target > rest) return false;
        if (target == 0 || --steps <= 0) return true;
        const int64_t stride = terms[k].first, after = rest - stride * terms[k].second;
        const int64_t low = target > after ? (target - after + stride - 1) / stride : 0;
        for (int64_t x = std::min(terms[k].second, target / stride); x >= low; --x)
            if (search(k + 1, target - x * stride, after, steps)) return true;
        return false;
    }
};

// Bytes from a tensor's first element to its last one.
int64_t bytes_to_last(const Tensor& t) {
    int64_t last = 0;
    for (int64_t d = 0; d < t.dim(); ++d) last += (t.size(d) - 1) * t.stride(d);
    return last * t.element_size();
}

// The tensor's bytes as a sum: element, and one term per dimension.
void add_bytes(Places& p, const Tensor& t) {
    if (t.is_non_overlapping_and_dense()) {
        p.add(1, t.numel() * t.element_size() - 1);
        return;
    }
    p.add(1, t.element_size() - 1);
    for (int64_t d = 0; d < t.dim(); ++d) p.add(t.stride(d) * t.element_size(), t.size(d) - 1);
}

// Byte i of a is byte j of b: with j counted from b's end all terms are positive.
bool share_bytes(const Tensor& a, const Tensor& b) {
    Places p;
    add_bytes(p, a);
    add_bytes(p, b);
    return p.reach((int64_t)((uintptr_t)b.data_ptr() - (uintptr_t)a.data_ptr()) + bytes_to_last(b) + b.element_size() - 1);
}

// Two indices of a tensor at one place: in the dimension of largest stride in which they differ they differ by x + 1, in those
// of smaller strides by anything, d_q = y_q - (size_q - 1).
bool meets_itself(const Tensor& t) {
    std::vector<std::pair<int64_t, int64_t>> dims;   // (stride, size - 1)
    for (int64_t d = 0; d < t.dim(); ++d) {
        if (t.size(d) <= 1) continue;
        if (t.stride(d) == 0) return true;
        dims.emplace_back(t.stride(d), t.size(d) - 1);
    }
    std::sort(dims.begin(), dims.end());
    for (size_t k = 0; k < dims.size(); ++k) {
        Places p;
        int64_t target = -dims[k].first;
        p.add(dims[k].first, dims[k].second - 1);
        for (size_t q = 0; q < k; ++q) {
            p.add(dims[q].first, 2 * dims[q].second);
            target += dims[q].first * dims[q].second;
        }
        if (p.reach(target)) return true;
    }
    return false;
}

// Scaling in place needs every element once: two gradients in the same memory would race, or count twice in the norm.
// Slices of one buffer may lie between each other.
void check_disjoint(const std::vector<Tensor>& params, const char* what) {
    struct Span {
        uintptr_t begin, end;
        const Tensor* t;
    };
    std::vector<Span> all;
    all.reserve(params.size());
    for (const Tensor& p : params) {
        if (!p.defined()) continue;
        const Tensor& t = p.grad();
        if (!t.defined() || t.layout() != c10::kStrided || t.numel() == 0) continue;
        const bool dense = t.is_non_overlapping_and_dense();
        TORCH_CHECK(dense || !meets_itself(t), what, ": a gradient has several elements in one place (an expanded tensor)");
        const uintptr_t begin = (uintptr_t)t.data_ptr();
        all.push_back({begin, begin + (uintptr_t)(dense ? (int64_t)t.nbytes() : bytes_to_last(t) + t.element_size()), &t});
    }
    const auto before = [](const Span& a, const Span& b) { return a.begin < b.begin; };
    if (!std::is_sorted(all.begin(), all.end(), before)) std::sort(all.begin(), all.end(), before);
    for (size_t i = 0; i < all.size(); ++i)
        for (size_t j = i + 1; j < all.size() && all[j].begin < all[i].end; ++j)
            TORCH_CHECK(!share_bytes(*all[i].t, *all[j].t), what, ": two gradients share memory (is a parameter listed twice?)");
}

bool capturing() { return c10::hip::currentStreamCaptureStatusMayInitCtx() != c10::hip::CaptureStatus::None; }

void check_may_wait(const char* what) {
    TORCH_CHECK(!capturing(), what,
                ": error_if_nonfinite makes the host wait, which a stream capture does not allow");
}

struct Norm {
    Tensor temp, value;
    size_t bytes;
    explicit Norm(const Grads& g) : bytes(gso_norm_temp_bytes(g.n())) {
        const auto opt = torch::TensorOptions().device(g.device);
        temp = torch::empty({(int64_t)bytes}, opt.dtype(torch::kUInt8));
        value = torch::empty({}, opt.dtype(torch::kFloat32));
    }
    float* out() const { return value.data_ptr<float>(); }
    void form(const Grads& g, int kind, void* st, const char* what) {
        check_rc(gso_grad_norm(g.n(), g.cptr(), g.numel.data(), g.type.data(), kind, temp.data_ptr(), bytes, out(), st), what);
    }
    // error_if_nonfinite: the norm before anything changes
    void look(Grads& g, int kind, void* st, const char* what) {
        form(g, kind, st, what);
        if (g.held.empty()) g.hold();
        const double norm = wait_for(value);
        TORCH_CHECK(std::isfinite(norm), what, ": the total norm of the gradients is ", norm,
                    " (error_if_nonfinite); nothing was changed");
    }
};

Tensor grad_norm(const std::vector<Tensor>& params, double norm_type) {
    const char* what = "grad_norm";
    const int kind = norm_kind(norm_type, what);
    const Grads g = collect(params, what);
    if (g.own.empty()) return torch::zeros({});
    c10::DeviceGuard guard(g.device);
    Norm r(g);
    r.form(g, kind, stream_on(g.device), what);
    return r.value;
}

Tensor clip_grad_norm(const std::vector<Tensor>& params, double max_norm, double norm_type, bool error_if_nonfinite) {
    const char* what = "clip_grad_norm_";
    const int kind = norm_kind(norm_type, what);
    TORCH_CHECK(max_norm >= 0.0, what, ": max_norm must not be negative or NaN, got ", max_norm);
    check_disjoint(params, what);
    Grads g = collect(params, what);
    if (g.own.empty()) return torch::zeros({});
    c10::DeviceGuard guard(g.device);
    if (error_if_nonfinite) check_may_wait(what);
    void* st = stream_on(g.device);
    Norm r(g);
    if (error_if_nonfinite) r.look(g, kind, st, what);
    check_rc(gso_clip_grads(g.n(), g.ptr.data(), g.numel.data(), g.type.data(), kind, max_norm, error_if_nonfinite,
                            r.temp.data_ptr(), r.bytes, r.out(), st),
             what);
    torch::NoGradGuard no_grad;
    for (const Tensor* t : g.own) changed(*t);
    for (const auto& copy : g.packed) g.own[copy.first]->copy_(copy.second);
    return r.value;
}

bool on_host(const Tensor& step) { return step.is_cpu() && step.scalar_type() == torch::kFloat32; }

// Parameters with gradients, their moments and step counts; scalars has four numbers per tensor, (lr, beta1, beta2, eps).
// Tensors marked `idle` count in the norm and are not updated.  The step counts go up once nothing can fail any more.
Tensor clipped_adam(const std::vector<Tensor>& params, const std::vector<Tensor>& exp_avg,
                    const std::vector<Tensor>& exp_avg_sq, const std::vector<Tensor>& steps,
                    const std::vector<double>& scalars, const std::vector<bool>& idle, const c10::optional<Tensor>& visibility,
                    double max_norm, double norm_type, bool error_if_nonfinite) {
    const char* what = "clipped_adam_step";
    const int kind = norm_kind(norm_type, what);
    const size_t n = params.size();
    TORCH_CHECK(exp_avg.size() == n && exp_avg_sq.size() == n && steps.size() == n && scalars.size() == 4 * n &&
                    idle.size() == n, what, ": inconsistent lists");
    // A gradient outlives `parameter.data = other`: the update would read as many elements as the parameter now has.
    const auto check_shape = [&](const Tensor& grad, size_t i) {
        TORCH_CHECK(idle[i] || grad.sizes() == params[i].sizes(), what, ": a gradient of shape ", grad.sizes(),
                    " does not have its parameter's shape ", params[i].sizes());
    };
    for (size_t i = 0; i < n; ++i)
        if (params[i].grad().defined()) check_shape(params[i].grad(), i);
    Grads g = collect(params, what);
    TORCH_CHECK(g.own.size() == n, what, ": inconsistent lists");
    if (n == 0) return torch::zeros({});
    torch::NoGradGuard no_grad;
    const c10::Device dev = g.device;
    c10::DeviceGuard guard(dev);
    TORCH_CHECK(!capturing(), what, " cannot be captured into a graph: its bias correction follows the step count, which lives "
                "on the host");
    Tensor visible;
    if (visibility) {
        TORCH_CHECK(visibility->device() == dev, what, ": visibility must be on ", dev, ", got ", visibility->device());
        visible = visibility->element_size() == 1 && !visibility->is_floating_point() ? visibility->contiguous()
                                                                                      : visibility->ne(0).contiguous();
    }
    // Counts that a checkpoint has brought to the GPU make the host wait, as they do in FusedGaussianAdam.step.  Addresses are
    // taken behind that.
    std::vector<double> count(n, 0.0);
    for (size_t i = 0; i < n; ++i) {
        TORCH_CHECK(steps[i].numel() == 1, what, ": a step count must be one number");
        if (idle[i] || visible.defined() || on_host(steps[i])) continue;
        if (g.held.empty()) g.hold();
        count[i] = wait_for(steps[i]);
    }
    std::vector<GsoAdamTensor> table;
    std::vector<Tensor> keep;
    std::vector<size_t> counted;
    Spans spans;
    table.reserve(n);
    for (size_t i = 0; i < n; ++i) {
        const Tensor& p = params[i];
        for (const Tensor* t : {&p, &exp_avg[i], &exp_avg_sq[i]})
            TORCH_CHECK(t->device() == dev && t->scalar_type() == torch::kFloat32 && t->is_contiguous() &&
                            t->sizes() == p.sizes(), what,
                        ": parameters and moments must be contiguous float32 tensors of one shape on the gradients' device");
        check_shape(*g.own[i], i);
        TORCH_CHECK(g.own[i]->scalar_type() == torch::kFloat32, what, ": gradients must be float32");
        if (idle[i]) continue;
        const int64_t rows = p.dim() > 0 ? p.size(0) : 1;
        TORCH_CHECK(!visible.defined() || visible.numel() == rows, what, ": visibility must have one entry per Gaussian");
        const double* s = &scalars[4 * i];
        GsoAdamTensor a;
        a.lr = s[0]; a.beta1 = s[1]; a.beta2 = s[2]; a.eps = s[3];
        a.bias_correction1 = a.bias_correction2_sqrt = 1.0;
        if (!visible.defined()) {
            const double t = (on_host(steps[i]) ? (double)*steps[i].data_ptr<float>() : count[i]) + 1.0;
            a.bias_correction1 = 1.0 - std::pow(a.beta1, t);
            a.bias_correction2_sqrt = std::sqrt(1.0 - std::pow(a.beta2, t));
            counted.push_back(i);
        }
        if (p.numel() == 0) continue;
        TORCH_CHECK(!p.is_neg() && !exp_avg[i].is_neg() && !exp_avg_sq[i].is_neg(), what, ": parameters and moments must hold "
                    "their own values");
        keep.push_back(plain(*g.own[i]).contiguous());
        a.param = p.data_ptr<float>();
        a.grad = keep.back().data_ptr<float>();
        a.exp_avg = exp_avg[i].data_ptr<float>();
        a.exp_avg_sq = exp_avg_sq[i].data_ptr<float>();
        a.rows = rows;
        a.width = p.numel() / rows;
        table.push_back(a);
        const int64_t bytes = p.numel() * (int64_t)sizeof(float);
        spans.add(a.param, bytes, true);
        spans.add(a.exp_avg, bytes, true);
        spans.add(a.exp_avg_sq, bytes, true);
        spans.add(a.grad, bytes, false);
    }
    TORCH_CHECK(spans.disjoint(), what, ": a parameter or moment shares memory with another tensor of the step");
    void* st = stream_on(dev);
    Norm r(g);
    std::vector<c10::Storage> memory;   // of what the update writes, over the wait
    if (error_if_nonfinite) {
        for (size_t i = 0; i < n; ++i)
            for (const Tensor* t : {&params[i], &exp_avg[i], &exp_avg_sq[i]}) memory.push_back(t->storage());
        r.look(g, kind, st, what);
    }
    check_rc(gso_adam_clipped(g.n(), g.cptr(), g.numel.data(), g.type.data(), (int)table.size(), table.data(),
                              visible.defined() ? (const uint8_t*)visible.data_ptr() : nullptr, kind, max_norm,
                              error_if_nonfinite, r.temp.data_ptr(), r.bytes, r.out(), st),
             what);
    for (size_t i : counted) {
        if (on_host(steps[i])) *steps[i].data_ptr<float>() += 1.0f;
        else steps[i].add_(1);
    }
    for (size_t i = 0; i < n; ++i) {
        if (idle[i]) continue;
        changed(params[i]);
        changed(exp_avg[i]);
        changed(exp_avg_sq[i]);
    }
    return r.value;
}

void accumulate_weights(const Tensor& weights, const std::vector<Tensor>& contributions, const c10::optional<Tensor>& opacity,
                        double decay) {
    const char* what = "accumulate_weights";
    torch::NoGradGuard no_grad;
    const int64_t N = weights.numel();
    std::vector<const float*> ptr;
    std::vector<Tensor> keep;
    auto take = [&](const Tensor& t, const char* name) {
        TORCH_CHECK(t.is_cuda() && t.device() == weights.device() && t.scalar_type() == torch::kFloat32 && t.numel() == N &&
                        t.dim() >= 1 && t.size(0) == N, what, ": ", name, " must be a float32 GPU tensor with one entry per "
                    "Gaussian (", N, ") on the weights' device, got ", t.sizes(), " ", t.scalar_type(), " on ", t.device());
        keep.push_back(plain(t).contiguous());
        return keep.back().data_ptr<float>();
    };
    take(weights, "weights");
    TORCH_CHECK(weights.is_contiguous() && !weights.is_neg(), what, ": weights are updated in place and must be contiguous");
    TORCH_CHECK(std::isfinite(decay), what, ": decay must be finite, got ", decay);
    for (const Tensor& c : contributions) ptr.push_back(take(c, "a contribution"));
    const float* o = opacity ? take(*opacity, "opacity") : nullptr;
    if (N == 0) return;
    Spans spans;
    for (size_t i = 0; i < keep.size(); ++i) spans.add(keep[i].data_ptr(), N * (int64_t)sizeof(float), i == 0);
    TORCH_CHECK(spans.disjoint(), what, ": weights must not share memory with what is added to them");
    c10::DeviceGuard guard(weights.device());
    check_rc(gso_accumulate_weights(N, weights.data_ptr<float>(), (int)ptr.size(), ptr.data(), o, decay,
                                    stream_on(weights.device())), what);
    changed(weights);
}

Tensor evict_select(const Tensor& weights, int64_t budget, int64_t recent) {
    torch::NoGradGuard no_grad;
    const char* what = "evict_rows";
    TORCH_CHECK(weights.is_cuda(), what, ": weights must be a GPU tensor (there is no CPU path)");
    const int64_t N = weights.numel();
    TORCH_CHECK(weights.scalar_type() == torch::kFloat32 && weights.dim() >= 1 && weights.size(0) == N, what,
                ": weights must be float32 with one entry per row, got ", weights.sizes(), " ", weights.scalar_type());
    TORCH_CHECK(budget >= 0, what, ": budget must not be negative, got ", budget);
    TORCH_CHECK(recent >= 0 && recent <= budget, what, ": recent must lie between 0 and the budget (", budget, "), got ",
                recent);
    c10::DeviceGuard guard(weights.device());
    const Tensor w = plain(weights).contiguous();
    Tensor rows = torch::empty({std::min(N, budget)}, w.options().dtype(torch::kInt32));
    if (rows.numel() == 0) return rows;
    const size_t bytes = gso_evict_temp_bytes(N);
    Tensor temp = torch::empty({(int64_t)bytes}, w.options().dtype(torch::kUInt8));
    check_rc(gso_evict_select(N, w.data_ptr<float>(), budget, recent, rows.data_ptr<int32_t>(), temp.data_ptr(), bytes,
                              stream_on(w.device())), what);
    return rows;
}

std::vector<Tensor> take_rows(const std::vector<Tensor>& tensors, const Tensor& rows, int64_t N) {
    const char* what = "evict_rows";
    const int64_t K = rows.numel();
    torch::NoGradGuard no_grad;
    std::vector<Tensor> out, keep;
    std::vector<GsoRowCopy> copies;
    out.reserve(tensors.size());
    for (const Tensor& own : tensors) {
        TORCH_CHECK(own.layout() == c10::kStrided && own.device() == rows.device() && own.dim() >= 1 && own.size(0) == N, what,
                    ": every tensor needs one row per weight (", N, ") on ", rows.device(), ", got ", own.sizes(), " on ",
                    own.device());
        const Tensor t = plain(own);
        // rows that are packed in themselves may lie any distance apart; others are packed first
        const Tensor s = t.is_contiguous() || (N > 0 && t.numel() > 0 && t.select(0, 0).is_contiguous()) ? t : t.contiguous();
        std::vector<int64_t> shape = s.sizes().vec();
        shape[0] = K;
        out.push_back(torch::empty(shape, s.options()));
        const int64_t row_bytes = t.numel() / std::max<int64_t>(N, 1) * t.element_size();
        if (K == 0 || row_bytes == 0) continue;
        keep.push_back(s);
        copies.push_back({s.data_ptr(), out.back().data_ptr(), row_bytes, (int64_t)(s.stride(0) * s.element_size())});
    }
    c10::DeviceGuard guard(rows.device());
    check_rc(gso_gather_rows_multi((int)copies.size(), copies.data(), rows.data_ptr<int32_t>(), K, stream_on(rows.device())), what);
    return out;
}

}  // namespace

void bind_optim(pybind11::module_& m) {
    namespace py = pybind11;
    m.def("grad_norm", &grad_norm);
    m.def("clip_grad_norm", &clip_grad_norm);
    m.def("clipped_adam", &clipped_adam);
    m.def("accumulate_weights", &accumulate_weights);
    m.def("evict_select", &evict_select);
    m.def("take_rows", &take_rows);
}
