// dense_torch.cpp -- fused_linear and fused_mlp as nodes of torch's autograd graph, and AdamW's calls: checks, allocations and the calls
// of the C entry points (dense_cuda.cu, adamw_cuda.cu) without the interpreter.  A backward that runs in Python is called by the engine's thread, which waits
// for the interpreter's lock: linear 128x367x512 with its backward, whose kernels take 20 us, took 115 us a pass that way.
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/jit/frontend/tracer.h>
#include <torch/extension.h>

#include "../../include/cafe_b200.h"

namespace {

using at::Tensor;
using torch::autograd::Node;
using torch::autograd::SavedVariable;
using torch::autograd::variable_list;
typedef std::optional<Tensor> Maybe;

int type_of(const Tensor& t) {
    switch (t.scalar_type()) {
        case at::kFloat: return CAFE_F32;
        case at::kBFloat16: return CAFE_BF16;
        case at::kHalf: return CAFE_F16;
        default: return -1;
    }
}
at::ScalarType slope_type(at::ScalarType t) { return t == at::kBFloat16 ? at::kShort : at::kFloat; }   // (codes of 16 bits, see the header)
void check_status(int status, const char* where) {
    if (status == CAFE_OK) return;
    TORCH_CHECK(status != CAFE_ERR_CUDA, where, ": ", cafe_last_error());
    TORCH_CHECK(false, where, status == CAFE_ERR_ARG ? ": invalid argument" : ": failed");
}

// t as rows of `cols` contiguous elements at one pitch; other layouts are copied, and views that carry a sign (the imaginary part of a
// conjugate) written out.  `repeated`: pitch 0 (a row that stands for all) is one.
struct Rows {
    Tensor t;
    int64_t m = 0, ld = 0;
    Rows() = default;
    Rows(const Tensor& given, int64_t cols, bool repeated = false) : t(given.resolve_neg()), m(1), ld(cols) {
        for (int64_t i = 0; i + 1 < given.dim(); ++i) m *= given.size(i);
        if (t.dim() != 2) t = t.reshape({m, cols});
        if (t.is_contiguous() || t.numel() == 0 || (m == 1 && t.stride(1) == 1)) return;
        if ((cols == 1 || t.stride(1) == 1) && (t.stride(0) >= cols || (repeated && t.stride(0) == 0))) ld = t.stride(0);
        else t = t.contiguous();
    }
    const void* ptr() const { return t.defined() ? t.const_data_ptr() : nullptr; }
};
Tensor plain(const Maybe& t) { return t && t->defined() ? t->contiguous().resolve_neg() : Tensor(); }
const void* ptr(const Tensor& t) { return t.defined() ? t.const_data_ptr() : nullptr; }
void* out(const Tensor& t) { return t.defined() ? t.mutable_data_ptr() : nullptr; }
// Workspace of one call, from torch's allocator: free again in the stream's order.
Tensor workspace(int64_t size, const Tensor& like) { return size > 0 ? at::empty({size}, like.options().dtype(at::kByte)) : Tensor(); }

// Outputs are allocated here and filled through pointers, which neither a forward derivative nor a recording of torch's calls sees:
// the one would read as zero, the other would replay the allocation alone.
void check_first_order_eager(const char* what, const Tensor& x, c10::ArrayRef<const Tensor*> others) {
    bool dual = x._fw_grad(0).defined();
    for (const Tensor* t : others) dual |= t && t->defined() && t->_fw_grad(0).defined();
    TORCH_CHECK_NOT_IMPLEMENTED(!dual, what, " has no forward-mode derivative");
    TORCH_CHECK_NOT_IMPLEMENTED(!torch::jit::tracer::isTracing() && !c10::impl::TorchDispatchModeTLS::get_mode(c10::impl::TorchDispatchModeKey::PROXY), what,
                                " cannot be recorded by a trace");
}
void check_tensors(const char* what, const Tensor& x, c10::ArrayRef<const Tensor*> others) {
    check_first_order_eager(what, x, others);
    TORCH_CHECK_VALUE(x.is_cuda() && type_of(x) >= 0, what, " needs CUDA tensors of fp32, bf16 or fp16");
    for (const Tensor* t : others)
        TORCH_CHECK_VALUE(!t || (t->is_cuda() && t->scalar_type() == x.scalar_type() && t->get_device() == x.get_device()), what,
                          ": all tensors must have one type and be on one device");
}
void check_layer(const char* what, int64_t cols, const Tensor& w, const Maybe& b) {
    TORCH_CHECK_VALUE(w.dim() == 2 && w.size(1) == cols, what, ": weight must be [out, ", cols, "], got ", w.sizes());
    TORCH_CHECK_VALUE(!b || (b->dim() == 1 && b->size(0) == w.size(0)), what, ": bias must be [", w.size(0), "], got ", b->sizes());
    TORCH_CHECK_VALUE(cols <= CAFE_LINEAR_MAX && w.size(0) <= CAFE_LINEAR_MAX, what, ": sizes up to ", CAFE_LINEAR_MAX);
}
std::vector<int64_t> out_shape(const Tensor& x, int64_t n) {
    std::vector<int64_t> shape(x.sizes().begin(), x.sizes().end());
    shape.back() = n;
    return shape;
}
// The gradients are those of first order: with create_graph they refuse to be differentiated again.
variable_list first_order(variable_list grads, const char* what) {
    if (!at::GradMode::is_enabled()) return grads;
    const std::string message = std::string(what) + ": its gradients cannot be differentiated again";
    auto refuse = std::make_shared<torch::autograd::DelayedError>(message, (int64_t)grads.size());
    // (a graph is made of what needs one)
    for (Tensor& g : grads)
        if (g.defined()) { g = g.detach(); g.set_requires_grad(true); }
    return (*refuse)(std::move(grads));
}
const char* const k_twice = "the saved tensors of fused_linear or fused_mlp have been freed: a second backward needs retain_graph=True";

// ---- one layer -------------------------------------------------------------------------------------------------------
struct LinearNode : Node {
    SavedVariable x, w, slope;
    int kind = CAFE_SLOPE_NONE;
    int64_t m = 0, n = 0, k = 0;
    std::vector<int64_t> shape;
    bool freed = false;

    std::string name() const override { return "FusedLinearBackward"; }
    void release_variables() override {
        std::lock_guard<std::mutex> lock(mutex_);
        x.reset_data(); w.reset_data(); slope.reset_data();
        freed = true;
    }
    variable_list apply(variable_list&& grads) override {
        std::lock_guard<std::mutex> lock(mutex_);
        TORCH_CHECK(!freed, k_twice);
        const Tensor& gy = grads[0];
        variable_list result(4);
        if (!gy.defined()) return result;
        const bool need_x = task_should_compute_output(0), need_w = task_should_compute_output(1), need_b = task_should_compute_output(2);
        if (need_x || need_w || need_b) {
            const auto self = shared_from_this();
            at::NoGradGuard plain_values;
            const c10::cuda::CUDAGuard device(gy.device());
            const Rows g(gy, n, true);
            // (what was saved need not come back at the pitch that it was saved with)
            Rows xs, ws;
            if (need_w) xs = Rows(x.unpack(self), k);
            if (need_x) ws = Rows(w.unpack(self), k);
            Tensor s;
            if (kind != CAFE_SLOPE_NONE) s = slope.unpack(self).contiguous();
            if (need_x) result[0] = at::empty(shape, gy.options());
            if (need_w) result[1] = at::empty({n, k}, gy.options());
            if (need_b) result[2] = at::empty({n}, gy.options());
            const int t = type_of(gy);
            const int64_t size = cafe_linear_backward_work(g.ptr(), g.ld, kind, xs.ptr(), xs.ld, ws.ptr(), ws.ld, m, n, k, t, need_x, need_w, need_b);
            const Tensor work = workspace(size, gy);
            check_status(cafe_linear_backward(g.ptr(), g.ld, ptr(s), n, kind, xs.ptr(), xs.ld, ws.ptr(), ws.ld, m, n, k, t, out(result[0]), k, out(result[1]), k,
                                              out(result[2]), out(work), size, c10::cuda::getCurrentCUDAStream().stream()), "cafe_linear_backward");
        }
        result = first_order(std::move(result), "fused_linear");
        if (task_should_compute_output(3)) result[3] = gy;
        return result;
    }
};

Tensor linear(const Tensor& x, const Tensor& w, const Maybe& b, const Maybe& r, int act) {
    static const char* const what = "fused_linear";
    check_tensors(what, x, {&w, b ? &*b : nullptr, r ? &*r : nullptr});
    TORCH_CHECK_VALUE(x.dim() >= 1, what, ": x must have a last dimension");
    check_layer(what, x.size(-1), w, b);
    const std::vector<int64_t> shape = out_shape(x, w.size(0));
    Tensor res = r ? *r : Tensor();
    if (res.defined() && res.sizes() != shape) res = res.expand(shape);   // (raises if it cannot)
    const bool grad = at::GradMode::is_enabled() && (x.requires_grad() || w.requires_grad() || (b && b->requires_grad()) || (res.defined() && res.requires_grad()));
    std::shared_ptr<LinearNode> node;
    if (grad) {
        node = std::shared_ptr<LinearNode>(new LinearNode(), torch::autograd::deleteNode);
        node->set_next_edges(torch::autograd::collect_next_edges(x, w, b ? *b : Tensor(), res));
    }
    Tensor y;
    {
        at::NoGradGuard plain_values;
        const c10::cuda::CUDAGuard device(x.device());
        const int64_t n = w.size(0), k = w.size(1);
        const Rows xs(x, k), ws(w, k), rs = res.defined() ? Rows(res, n, true) : Rows();
        TORCH_CHECK_VALUE(xs.m <= CAFE_LINEAR_MAX, what, ": up to ", CAFE_LINEAR_MAX, " rows");
        const Tensor bias = plain(b);
        y = at::empty(shape, x.options());
        Tensor slope;
        const bool output_tells = act == CAFE_ACT_RELU && !res.defined();
        if (grad && act != CAFE_ACT_NONE && !output_tells) slope = at::empty({xs.m, n}, x.options().dtype(slope_type(x.scalar_type())));
        const int t = type_of(x);
        const int64_t size = cafe_linear_forward_work(xs.ptr(), xs.ld, ws.ptr(), ws.ld, xs.m, n, k, t);
        const Tensor work = workspace(size, x);
        check_status(cafe_linear_forward(xs.ptr(), xs.ld, ws.ptr(), ws.ld, ptr(bias), rs.ptr(), rs.ld, xs.m, n, k, t, act,
                                         out(y), n, out(slope), n, out(work), size, c10::cuda::getCurrentCUDAStream().stream()), "cafe_linear_forward");
        if (grad) {
            node->m = xs.m; node->n = n; node->k = k;
            node->shape.assign(x.sizes().begin(), x.sizes().end());
            node->kind = act == CAFE_ACT_NONE ? CAFE_SLOPE_NONE : output_tells ? CAFE_SLOPE_OUTPUT : CAFE_SLOPE_VALUES;
            if (w.requires_grad()) node->x = SavedVariable(xs.t, false);
            if (x.requires_grad()) node->w = SavedVariable(ws.t, false);
            if (slope.defined()) node->slope = SavedVariable(slope, false);
        }
    }
    if (grad) {
        torch::autograd::set_history(y, node);
        if (node->kind == CAFE_SLOPE_OUTPUT) node->slope = SavedVariable(y, true);
    }
    return y;
}

// ---- a run of layers -------------------------------------------------------------------------------------------------
// Where the outputs between the layers and the slopes lie in one buffer: rows and starts on 16 bytes.
struct Plan {
    std::vector<int> widths, acts;
    std::vector<int64_t> pitch, y_at, slope_at;   // -1: no slope
    int64_t bytes = 0;
    Plan() = default;
    Plan(int64_t m, std::vector<int> w, std::vector<int> a, at::ScalarType type, bool keep) : widths(std::move(w)), acts(std::move(a)) {
        const int64_t size = c10::elementSize(type), slope_size = c10::elementSize(slope_type(type));
        const size_t n = acts.size();
        auto take = [&](int64_t row) { const int64_t at = bytes; bytes += (m * row + 255) / 256 * 256; return at; };
        for (size_t l = 0; l < n; ++l) pitch.push_back(l + 1 < n ? (widths[l + 1] + 7) / 8 * 8 : widths[l + 1]);
        for (size_t l = 0; l + 1 < n; ++l) y_at.push_back(take(pitch[l] * size));
        for (size_t l = 0; l < n; ++l) slope_at.push_back(keep && acts[l] != CAFE_ACT_NONE && acts[l] != CAFE_ACT_RELU ? take(pitch[l] * slope_size) : -1);
    }
    std::vector<void*> outputs(char* base, void* last) const {
        std::vector<void*> p;
        for (const int64_t a : y_at) p.push_back(base + a);
        p.push_back(last);
        return p;
    }
    std::vector<void*> slopes(char* base) const {
        std::vector<void*> p;
        for (const int64_t a : slope_at) p.push_back(a < 0 ? nullptr : base + a);
        return p;
    }
};
struct Weights {
    std::vector<Tensor> t;
    std::vector<const void*> p;
    std::vector<int64_t> ld;
    void add(const Tensor& w) {
        const Rows r = w.defined() ? Rows(w, w.size(1)) : Rows();
        t.push_back(r.t); p.push_back(r.ptr()); ld.push_back(r.ld);
    }
};

struct MlpNode : Node {
    // y: where the last layer is a ReLU, whose derivative it tells; x and each of w: where a gradient that can be asked for needs it
    SavedVariable x, y, between;
    std::vector<SavedVariable> w;
    std::vector<bool> has_w;
    bool has_x = false;
    Plan plan;
    int64_t m = 0;
    std::vector<int64_t> shape;
    bool freed = false;

    std::string name() const override { return "FusedMLPBackward"; }
    void release_variables() override {
        std::lock_guard<std::mutex> lock(mutex_);
        x.reset_data(); y.reset_data(); between.reset_data();
        for (SavedVariable& v : w) v.reset_data();
        freed = true;
    }
    variable_list apply(variable_list&& grads) override {
        std::lock_guard<std::mutex> lock(mutex_);
        TORCH_CHECK(!freed, k_twice);
        const Tensor& gy = grads[0];
        const int n = (int)plan.acts.size();
        variable_list result(1 + 2 * n);
        if (!gy.defined()) return result;
        {
            const auto self = shared_from_this();
            at::NoGradGuard plain_values;
            const c10::cuda::CUDAGuard device(gy.device());
            const Rows g(gy, plan.widths[n], true), xs = has_x ? Rows(x.unpack(self), plan.widths[0]) : Rows();
            Weights ws;
            for (int l = 0; l < n; ++l) ws.add(has_w[l] ? w[l].unpack(self) : Tensor());
            const Tensor held = between.unpack(self).contiguous(), ys = plan.acts[n - 1] == CAFE_ACT_RELU ? y.unpack(self).contiguous() : Tensor();
            std::vector<void*> gw(n, nullptr), gb(n, nullptr);
            if (task_should_compute_output(0)) result[0] = at::empty(shape, gy.options());
            for (int l = 0; l < n; ++l) {
                if (task_should_compute_output(1 + l)) gw[l] = out(result[1 + l] = at::empty({plan.widths[l + 1], plan.widths[l]}, gy.options()));
                if (task_should_compute_output(1 + n + l)) gb[l] = out(result[1 + n + l] = at::empty({plan.widths[l + 1]}, gy.options()));
            }
            char* const base = static_cast<char*>(const_cast<void*>(held.const_data_ptr()));
            const std::vector<void*> outputs = plan.outputs(base, const_cast<void*>(ptr(ys))), slopes = plan.slopes(base);
            const int t = type_of(gy);
            const int64_t size = cafe_mlp_backward_work(n, plan.widths.data(), m, g.ptr(), g.ld, xs.ptr(), xs.ld, ws.p.data(), ws.ld.data(), t);
            const Tensor work = workspace(size, gy);
            check_status(cafe_mlp_backward(n, plan.widths.data(), m, g.ptr(), g.ld, xs.ptr(), xs.ld, ws.p.data(), ws.ld.data(), plan.acts.data(), t, outputs.data(),
                                           plan.pitch.data(), slopes.data(), out(result[0]), plan.widths[0], gw.data(), gb.data(), out(work), size,
                                           c10::cuda::getCurrentCUDAStream().stream()), "cafe_mlp_backward");
        }
        return first_order(std::move(result), "fused_mlp");
    }
};

Tensor mlp(const Tensor& x, const std::vector<Tensor>& w, const std::vector<Maybe>& b, const std::vector<int>& acts) {
    static const char* const what = "fused_mlp";
    const int n = (int)w.size();
    TORCH_CHECK_VALUE(n >= 1 && n <= CAFE_MLP_MAX_LAYERS && (int)b.size() == n && (int)acts.size() == n, what,
                      ": one bias (or None) and one activation for each of 1 to ", CAFE_MLP_MAX_LAYERS, " weights");
    std::vector<const Tensor*> all;
    for (int l = 0; l < n; ++l) { all.push_back(&w[l]); all.push_back(b[l] ? &*b[l] : nullptr); }
    check_tensors(what, x, all);
    TORCH_CHECK_VALUE(x.dim() >= 1, what, ": x must have a last dimension");
    std::vector<int> widths;
    int64_t cols = x.size(-1);
    bool grad = x.requires_grad();
    for (int l = 0; l < n; ++l) {
        check_layer(what, cols, w[l], b[l]);
        widths.push_back((int)cols);
        cols = w[l].size(0);
        grad |= w[l].requires_grad() || (b[l] && b[l]->requires_grad());
    }
    widths.push_back((int)cols);
    grad &= at::GradMode::is_enabled();
    std::shared_ptr<MlpNode> node;
    if (grad) {
        node = std::shared_ptr<MlpNode>(new MlpNode(), torch::autograd::deleteNode);
        torch::autograd::edge_list edges;
        auto edge = [&](const Tensor& t) {
            const auto e = torch::autograd::collect_next_edges(t);
            edges.push_back(e.empty() ? torch::autograd::Edge() : e[0]);
        };
        edge(x);
        for (const Tensor& t : w) edge(t);
        for (const Maybe& t : b) edge(t ? *t : Tensor());
        node->set_next_edges(std::move(edges));
    }
    Tensor y;
    {
        at::NoGradGuard plain_values;
        const c10::cuda::CUDAGuard device(x.device());
        const Rows xs(x, widths[0]);
        TORCH_CHECK_VALUE(xs.m <= CAFE_LINEAR_MAX, what, ": up to ", CAFE_LINEAR_MAX, " rows");
        const Plan plan(xs.m, widths, acts, x.scalar_type(), grad);
        Weights ws;
        std::vector<Tensor> bs;
        std::vector<const void*> bias;
        for (int l = 0; l < n; ++l) {
            ws.add(w[l]);
            bs.push_back(plain(b[l]));
            bias.push_back(ptr(bs[l]));
        }
        y = at::empty(out_shape(x, cols), x.options());
        const Tensor between = at::empty({plan.bytes}, x.options().dtype(at::kByte));
        char* const base = static_cast<char*>(between.mutable_data_ptr());
        const std::vector<void*> outputs = plan.outputs(base, out(y)), slopes = plan.slopes(base);
        const int t = type_of(x);
        const int64_t size = cafe_mlp_forward_work(n, widths.data(), xs.m, xs.ptr(), xs.ld, ws.p.data(), ws.ld.data(), t);
        const Tensor work = workspace(size, x);
        check_status(cafe_mlp_forward(n, widths.data(), xs.m, xs.ptr(), xs.ld, ws.p.data(), ws.ld.data(), bias.data(), acts.data(), t, outputs.data(), plan.pitch.data(),
                                      grad ? slopes.data() : nullptr, out(work), size, c10::cuda::getCurrentCUDAStream().stream()), "cafe_mlp_forward");
        if (grad) {
            node->plan = plan;
            node->m = xs.m;
            node->shape.assign(x.sizes().begin(), x.sizes().end());
            node->between = SavedVariable(between, false);
            node->has_x = w[0].requires_grad();
            if (node->has_x) node->x = SavedVariable(xs.t, false);
            bool below = x.requires_grad();   // (a layer's weight carries the gradient on to what lies below it)
            for (int l = 0; l < n; ++l) {
                node->has_w.push_back(below);
                node->w.push_back(below ? SavedVariable(ws.t[l], false) : SavedVariable());
                below |= w[l].requires_grad() || (b[l] && b[l]->requires_grad());
            }
        }
    }
    if (grad) {
        torch::autograd::set_history(y, node);
        if (acts[n - 1] == CAFE_ACT_RELU) node->y = SavedVariable(y, true);
    }
    return y;
}

// ---- AdamW -----------------------------------------------------------------------------------------------------------
std::vector<void*> pointers(const std::vector<Tensor>& t) {
    std::vector<void*> p;
    p.reserve(t.size());
    for (const Tensor& x : t) p.push_back(const_cast<void*>(x.const_data_ptr()));
    return p;
}
// Whether elements of these sizes and strides lie one behind the other in the order of their indexes.
bool row_major(at::IntArrayRef sizes, at::IntArrayRef strides) {
    int64_t at = 1;
    for (const int64_t n : sizes) if (n == 0) return true;
    for (size_t i = sizes.size(); i-- > 0;) {
        if (sizes[i] == 1) continue;
        if (strides[i] != at) return false;
        at *= sizes[i];
    }
    return true;
}
// Whether p's k-th element in memory is also the k-th of these: both row-major, or the same axes (but for those of one element).
bool same_order(const Tensor& p, at::IntArrayRef sizes, at::IntArrayRef strides) {
    if (row_major(p.sizes(), p.strides())) return row_major(sizes, strides);
    size_t j = 0;
    for (int64_t i = 0; i < p.dim(); ++i) {
        if (p.size(i) == 1) continue;
        while (j < sizes.size() && sizes[j] == 1) ++j;
        if (j == sizes.size() || sizes[j] != p.size(i) || strides[j] != p.stride(i)) return false;
        ++j;
    }
    while (j < sizes.size() && sizes[j] == 1) ++j;
    return j == sizes.size();
}
// A parameter's memory may have been exchanged since its moments were made.  `layout`: of 8-bit moments, whose codes lie flat, the
// parameter's sizes and strides then (host, [2, axes]); 32-bit moments have their own.
void check_moments(const Tensor& p, const Tensor& m, const Tensor* layout) {
    TORCH_CHECK(p.is_cuda() && type_of(p) >= 0, "AdamW: a parameter has become ", p.scalar_type(), " on ", p.device());
    TORCH_CHECK(m.numel() == p.numel() && m.device() == p.device() && p.is_non_overlapping_and_dense(),
                "AdamW: a parameter has changed its size, device or layout since its moments were made");
    bool same;
    if (layout) {
        TORCH_CHECK(layout->device().is_cpu() && layout->scalar_type() == at::kLong && layout->dim() == 2 && layout->size(0) == 2 && layout->is_contiguous(),
                    "AdamW: the layout of a state is not what it was made as");
        const int64_t* const at = layout->const_data_ptr<int64_t>();
        const size_t axes = (size_t)layout->size(1);
        same = same_order(p, {at, axes}, {at + axes, axes});
    } else same = same_order(p, m.sizes(), m.strides());
    TORCH_CHECK(same, "AdamW: a parameter's elements lie in another order than when its moments were made",
                layout ? "" : " (load_state_dict(state_dict()) lays the moments out anew)");
}
// An array of the state is what the kernels read and write: `n` elements of a type, on p's device.
void check_state(const Tensor& p, const Tensor& s, int64_t n, at::ScalarType type) {
    TORCH_CHECK(s.numel() == n && s.scalar_type() == type && s.device() == p.device() && s.is_non_overlapping_and_dense(),
                "AdamW: the moments or the step of a parameter are not what they were made as");
}
// one step of parameters of one type on one device; mtop, vtop and layout are empty with 32-bit moments
void adamw_step(const std::vector<Tensor>& p, std::vector<Tensor> g, const std::vector<Tensor>& m, const std::vector<Tensor>& v, const std::vector<Tensor>& mtop,
                const std::vector<Tensor>& vtop, const std::vector<Tensor>& layout, const std::vector<Tensor>& step, const std::vector<int>& index, double lr, double beta1, double beta2, double eps,
                double weight_decay, uint32_t seed, const Tensor& ticket) {
    at::NoGradGuard plain_values;
    const c10::cuda::CUDAGuard device(ticket.device());
    const size_t n = p.size();
    const bool packed = !mtop.empty();
    std::vector<int64_t> numel(n);
    for (size_t i = 0; i < n; ++i) {
        check_moments(p[i], m[i], layout.empty() ? nullptr : &layout[i]);
        numel[i] = p[i].numel();
        check_state(p[i], m[i], numel[i], packed ? at::kByte : at::kFloat);
        check_state(p[i], v[i], numel[i], packed ? at::kByte : at::kFloat);
        check_state(p[i], step[i], 1, at::kLong);
        if (packed) {
            check_state(p[i], mtop[i], (numel[i] + 255) / 256, at::kByte);
            check_state(p[i], vtop[i], (numel[i] + 255) / 256, at::kByte);
        } else check_moments(p[i], v[i], nullptr);
        TORCH_CHECK(g[i].scalar_type() == p[i].scalar_type(), "AdamW: a gradient of ", g[i].scalar_type(), " for a parameter of ", p[i].scalar_type());
        TORCH_CHECK(g[i].sizes() == p[i].sizes() && g[i].device() == p[i].device(), "AdamW: a gradient of ", g[i].sizes(), " on ", g[i].device(),
                    " for a parameter of ", p[i].sizes(), " on ", p[i].device());
        TORCH_CHECK(!p[i].is_neg(), "AdamW: a parameter has become a view that carries a sign");
        g[i] = g[i].resolve_neg();
        if (!(g[i].is_contiguous() && p[i].is_contiguous()) && g[i].strides() != p[i].strides()) {
            const Tensor same = at::empty_like(p[i]);
            same.copy_(g[i]);
            g[i] = same;
        }
    }
    const std::vector<void*> gs = pointers(g), ms = pointers(mtop), vs = pointers(vtop), steps = pointers(step);
    check_status(cafe_adamw_step((int)n, pointers(p).data(), gs.data(), pointers(m).data(), pointers(v).data(), packed ? (uint8_t* const*)ms.data() : nullptr,
                                 packed ? (uint8_t* const*)vs.data() : nullptr, (int64_t* const*)steps.data(), numel.data(), index.data(), type_of(p[0]), packed ? 8 : 32,
                                 lr, beta1, beta2, eps, weight_decay, seed, static_cast<int*>(ticket.mutable_data_ptr()), c10::cuda::getCurrentCUDAStream().stream()),
                 "cafe_adamw_step");
    for (const Tensor& t : p)   // (a backward that has saved one of them must say so)
        if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();
}
// the values of 8-bit moments of parameters on one device, (m, root of v) of each
std::vector<std::pair<Tensor, Tensor>> adamw_moments(const std::vector<Tensor>& p, const std::vector<Tensor>& m, const std::vector<Tensor>& mtop, const std::vector<Tensor>& r,
                                                     const std::vector<Tensor>& rtop, const std::vector<Tensor>& layout) {
    at::NoGradGuard plain_values;
    const c10::cuda::CUDAGuard device(p[0].device());
    const size_t n = p.size();
    std::vector<int64_t> numel(n);
    int64_t all = 0;
    bool together = true;   // one allocation, every tensor on 16 bytes
    for (size_t i = 0; i < n; ++i) {
        check_moments(p[i], m[i], &layout[i]);
        for (const Tensor* c : {&m[i], &r[i]}) check_state(p[i], *c, p[i].numel(), at::kByte);
        for (const Tensor* c : {&mtop[i], &rtop[i]}) check_state(p[i], *c, (p[i].numel() + 255) / 256, at::kByte);
        together &= p[i].is_contiguous() && all % 8 == 0;
        all += numel[i] = p[i].numel();
    }
    const auto options = p[0].options().dtype(at::kBFloat16);
    std::vector<std::pair<Tensor, Tensor>> out(n);
    std::vector<void*> mo(n), ro(n);
    Tensor flat_m, flat_r;
    if (together) { flat_m = at::empty({all}, options); flat_r = at::empty({all}, options); }
    int64_t at = 0;
    for (size_t i = 0; i < n; ++i) {
        if (together) out[i] = {flat_m.as_strided(p[i].sizes(), p[i].strides(), at), flat_r.as_strided(p[i].sizes(), p[i].strides(), at)};
        else out[i] = {at::empty_like(p[i], options), at::empty_like(p[i], options)};
        at += numel[i];
        mo[i] = out[i].first.mutable_data_ptr();
        ro[i] = out[i].second.mutable_data_ptr();
    }
    const std::vector<void*> mc = pointers(m), mt = pointers(mtop), rc = pointers(r), rt = pointers(rtop);
    check_status(cafe_adamw_moments((int)n, (const uint8_t* const*)mc.data(), (const uint8_t* const*)mt.data(), (const uint8_t* const*)rc.data(), (const uint8_t* const*)rt.data(),
                                    numel.data(), mo.data(), ro.data(), c10::cuda::getCurrentCUDAStream().stream()), "cafe_adamw_moments");
    return out;
}

}  // namespace

PYBIND11_MODULE(_dense_torch, m) {
    m.def("linear", &linear, pybind11::call_guard<pybind11::gil_scoped_release>());
    m.def("mlp", &mlp, pybind11::call_guard<pybind11::gil_scoped_release>());
    m.def("adamw_step", &adamw_step, pybind11::call_guard<pybind11::gil_scoped_release>());
    m.def("adamw_moments", &adamw_moments, pybind11::call_guard<pybind11::gil_scoped_release>());
}
