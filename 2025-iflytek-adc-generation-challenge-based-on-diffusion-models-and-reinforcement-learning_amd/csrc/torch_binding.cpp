// The operators around a residual block as PyTorch operators (torch.ops.adcdiff.*) over the C ABI (include/adcdiff.h): argument checks,
// allocation, streams and autograd.  In C++ because at small sizes the host is what a call costs: the same operators bound in Python took
// 13-16 us a call and 170 us for a training call, whose backward pass runs in autograd's own thread.
// The C functions are resolved from libadcdiff.so, which the package loads first.
#include <ATen/ATen.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/library.h>

#include <array>
#include <functional>
#include <vector>

#include "../../include/adcdiff.h"

namespace {

using at::Tensor;
using OptTensor = std::optional<Tensor>;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

void check(int rc) { TORCH_CHECK(rc == ADCDIFF_OK, "adcdiff error ", rc, ": ", adcdiff_last_error()); }

void need_gpu(const Tensor& t) {
    TORCH_CHECK(t.is_cuda(), "adcdiff kernels run on an MI355X only; got a ", t.device(), " tensor (no CPU fallback exists)");
}

// All tensors on one GPU: that GPU
c10::Device one_device(std::initializer_list<const Tensor*> tensors) {
    const Tensor* first = nullptr;
    for (const Tensor* t : tensors) {
        if (!t || !t->defined()) continue;
        need_gpu(*t);
        if (!first) first = t;
        TORCH_CHECK_VALUE(t->device() == first->device(), "tensors on different devices: ", first->device(), " and ", t->device());
    }
    return first->device();
}

const Tensor* ptr(const OptTensor& t) { return t.has_value() ? &*t : nullptr; }
bool given(const OptTensor& t) { return t.has_value() && t->defined(); }

adcdiff_stream_t stream_of(c10::Device d) { return c10::hip::getCurrentHIPStream(d.index()).stream(); }

int code_of(const Tensor& t, const char* what) {
    if (t.scalar_type() == at::kFloat) return ADCDIFF_F32;
    TORCH_CHECK_VALUE(t.scalar_type() == at::kBFloat16, what, " must be float32 or bfloat16, got ", t.scalar_type());
    return ADCDIFF_BF16;
}

at::ScalarType type_of(int64_t code) {
    TORCH_CHECK_VALUE(code == ADCDIFF_F32 || code == ADCDIFF_BF16, "type code ", code);
    return code == ADCDIFF_BF16 ? at::kBFloat16 : at::kFloat;
}

int narrow(int64_t v, const char* what) {
    TORCH_CHECK_VALUE(v >= 0 && v <= 0x7fffffff, what, " of ", v);
    return (int)v;
}

// Row pitch in elements of a 2-D tensor whose rows are contiguous and do not overlap
int64_t pitch_of(const Tensor& t, const char* what) {
    TORCH_CHECK_VALUE(t.dim() == 2, what, " must be two-dimensional, got shape ", t.sizes());
    const int64_t rows = t.size(0), cols = t.size(1);
    TORCH_CHECK_VALUE(cols <= 1 || t.stride(1) == 1, "the rows of ", what, " must be contiguous, got strides ", t.strides());
    if (rows <= 1) return cols;
    TORCH_CHECK_VALUE(t.stride(0) >= cols, "the rows of ", what, " overlap: strides ", t.strides());
    return t.stride(0);
}

// An optional contiguous float32 vector
const float* vector_of(const OptTensor& t, int64_t n, const char* what) {
    if (!given(t)) return nullptr;
    TORCH_CHECK_VALUE(t->scalar_type() == at::kFloat && t->dim() == 1 && t->size(0) == n && t->is_contiguous(), what,
                      " must be a contiguous float32 vector of ", n, " elements, got ", t->scalar_type(), " ", t->sizes());
    return t->const_data_ptr<float>();
}

// ------------------------------------------------------------------ gated residual norms
adcdiff_residual_norm_args norm_args(const OptTensor& h, const Tensor& x, const OptTensor& gate, const OptTensor& post_weight, const OptTensor& post_bias,
                                     const OptTensor& pre_weight, const OptTensor& pre_bias, int64_t post_norm, int64_t pre_norm, double residual_scale,
                                     double eps) {
    adcdiff_residual_norm_args a{};
    a.ldx = pitch_of(x, "x");
    a.stream_dtype = a.dtype = code_of(x, "x");
    a.x = x.const_data_ptr();
    const int64_t M = x.size(0), D = x.size(1);
    a.M = narrow(M, "rows");
    a.D = narrow(D, "columns");
    a.residual_scale = (float)residual_scale;
    a.eps = (float)eps;
    if (given(h)) {
        TORCH_CHECK_VALUE(h->sizes() == x.sizes(), "h ", h->sizes(), " and x ", x.sizes(), " differ in shape");
        a.h = h->const_data_ptr();
        a.ldh = pitch_of(*h, "h");
        a.dtype = code_of(*h, "h");
    } else {
        TORCH_CHECK_VALUE(!given(gate) && !post_norm && residual_scale == 1.0, "a gate, a post norm or a residual scale needs h");
    }
    if (given(gate)) {
        const int64_t G = gate->dim() == 2 ? gate->size(0) : 0;
        TORCH_CHECK_VALUE(gate->dim() == 2 && gate->size(1) == D && (M == 0 || (G > 0 && M % G == 0)), "gate must be [G, ", D, "] with G dividing ", M,
                          " rows, got ", gate->sizes());
        a.gate = gate->const_data_ptr();
        a.gate_dtype = code_of(*gate, "gate");
        a.gate_rows = narrow(G, "gate rows");
        const bool expanded = G > 1 && gate->stride(0) == 0 && (D <= 1 || gate->stride(1) == 1);   // one row for all groups
        a.ldg = expanded ? 0 : pitch_of(*gate, "gate");
    }
    TORCH_CHECK_VALUE(post_norm || (!given(post_weight) && !given(post_bias)), "post_weight / post_bias without a post norm");
    TORCH_CHECK_VALUE(pre_norm || (!given(pre_weight) && !given(pre_bias)), "pre_weight / pre_bias without a pre norm");
    a.post_norm = (int)post_norm;
    a.pre_norm = (int)pre_norm;
    a.post_weight = vector_of(post_weight, D, "post_weight");
    a.post_bias = vector_of(post_bias, D, "post_bias");
    a.pre_weight = vector_of(pre_weight, D, "pre_weight");
    a.pre_bias = vector_of(pre_bias, D, "pre_bias");
    return a;
}

// [x_new where with_x] + [y where there is a pre norm] + [stats [M, 4] where with_stats]
std::vector<Tensor> residual_norm(const OptTensor& h, const Tensor& x, const OptTensor& gate, const OptTensor& post_weight, const OptTensor& post_bias,
                                  const OptTensor& pre_weight, const OptTensor& pre_bias, int64_t post_norm, int64_t pre_norm, double residual_scale,
                                  double eps, bool with_x, bool with_stats) {
    const c10::Device dev = one_device({&x, ptr(h), ptr(gate), ptr(post_weight), ptr(post_bias), ptr(pre_weight), ptr(pre_bias)});
    adcdiff_residual_norm_args a = norm_args(h, x, gate, post_weight, post_bias, pre_weight, pre_bias, post_norm, pre_norm, residual_scale, eps);
    const c10::DeviceGuard guard(dev);
    std::vector<Tensor> outs;
    outs.reserve(3);
    if (with_x) {
        outs.push_back(at::empty(x.sizes(), x.options()));
        a.x_new = outs.back().mutable_data_ptr();
        a.ldx_new = a.D;
    }
    if (pre_norm) {
        outs.push_back(at::empty(x.sizes(), x.options().dtype(type_of(a.dtype))));
        a.y = outs.back().mutable_data_ptr();
        a.ldy = a.D;
    }
    if (with_stats) {
        outs.push_back(at::empty({x.size(0), 4}, x.options().dtype(at::kFloat)));
        a.stats = outs.back().mutable_data_ptr<float>();
    }
    check(adcdiff_residual_norm(&a, stream_of(dev)));
    return outs;
}

// An incoming gradient with contiguous rows that do not overlap (it may arrive expanded)
Tensor gradient_rows(const OptTensor& t, const Tensor& x, at::ScalarType type, const char* what) {
    if (!given(t)) return Tensor();
    TORCH_CHECK_VALUE(t->sizes() == x.sizes() && t->scalar_type() == type, what, " must be ", type, " ", x.sizes(), ", got ", t->scalar_type(), " ", t->sizes());
    const int64_t rows = t->size(0), cols = t->size(1);
    if ((cols > 1 && t->stride(1) != 1) || (rows > 1 && t->stride(0) < cols)) return t->contiguous();
    return *t;
}

// The gradients of (h, x, gate, post_weight, post_bias, pre_weight, pre_bias) that `need` asks for, in that order
std::vector<Tensor> residual_norm_backward(const OptTensor& h, const Tensor& x, const OptTensor& gate, const OptTensor& post_weight,
                                           const OptTensor& post_bias, const OptTensor& pre_weight, const OptTensor& pre_bias, const OptTensor& stats,
                                           const OptTensor& d_x_new, const OptTensor& d_y, int64_t post_norm, int64_t pre_norm, double residual_scale,
                                           double eps, std::array<bool, 7> need) {
    const c10::Device dev = one_device({&x, ptr(h), ptr(gate), ptr(post_weight), ptr(post_bias), ptr(pre_weight), ptr(pre_bias), ptr(stats), ptr(d_x_new), ptr(d_y)});
    adcdiff_residual_norm_args a = norm_args(h, x, gate, post_weight, post_bias, pre_weight, pre_bias, post_norm, pre_norm, residual_scale, eps);
    if (post_norm || pre_norm) {
        TORCH_CHECK_VALUE(given(stats) && stats->scalar_type() == at::kFloat && stats->dim() == 2 && stats->size(0) == x.size(0) && stats->size(1) == 4 &&
                              stats->is_contiguous(), "stats must be the contiguous float32 [", x.size(0), ", 4] tensor of the forward pass");
        a.stats = const_cast<float*>(stats->const_data_ptr<float>());
    }
    const c10::DeviceGuard guard(dev);
    adcdiff_residual_norm_grads g{};
    const Tensor in_x = gradient_rows(d_x_new, x, x.scalar_type(), "d_x_new"), in_y = gradient_rows(d_y, x, type_of(a.dtype), "d_y");
    if (in_x.defined()) {
        g.d_x_new = in_x.const_data_ptr();
        g.ld_d_x_new = pitch_of(in_x, "d_x_new");
    }
    if (in_y.defined()) {
        g.d_y = in_y.const_data_ptr();
        g.ld_d_y = pitch_of(in_y, "d_y");
    }
    std::vector<Tensor> outs;
    outs.reserve(7);
    const Tensor* inputs[7] = {ptr(h), &x, ptr(gate), ptr(post_weight), ptr(post_bias), ptr(pre_weight), ptr(pre_bias)};
    void* at_[7] = {};
    for (int i = 0; i < 7; ++i) {
        if (!need[i]) continue;
        TORCH_CHECK_VALUE(inputs[i] && inputs[i]->defined(), "need asks for the gradient of an input that is not there");
        outs.push_back(at::empty(inputs[i]->sizes(), inputs[i]->options()));
        at_[i] = outs.back().mutable_data_ptr();
    }
    g.h = at_[0]; g.x = at_[1]; g.gate = at_[2];
    g.ld_h = g.ld_x = g.ld_gate = a.D;
    g.post_weight = static_cast<float*>(at_[3]); g.post_bias = static_cast<float*>(at_[4]);
    g.pre_weight = static_cast<float*>(at_[5]); g.pre_bias = static_cast<float*>(at_[6]);
    const size_t bytes = adcdiff_residual_norm_backward_workspace_bytes(&a, &g);
    Tensor ws = at::empty({(int64_t)bytes}, x.options().dtype(at::kByte));
    check(adcdiff_residual_norm_backward(&a, &g, ws.mutable_data_ptr(), bytes, stream_of(dev)));
    return outs;
}

// ------------------------------------------------------------------ gradient norm
std::vector<adcdiff_grad_tensor> grad_table(at::TensorList grads, const at::TensorList* out) {
    TORCH_CHECK_VALUE(!grads.empty(), "no gradients");
    std::vector<adcdiff_grad_tensor> table(grads.size());
    for (size_t i = 0; i < grads.size(); ++i) {
        const Tensor& g = grads[i];
        need_gpu(g);
        TORCH_CHECK_VALUE(g.device() == grads[0].device(), "gradients on different devices: ", grads[0].device(), " and ", g.device());
        TORCH_CHECK_VALUE(g.layout() == at::kStrided && (g.is_contiguous() || g.is_non_overlapping_and_dense()), "gradient ", i,
                          " has gaps or overlaps in memory: shape ", g.sizes());
        adcdiff_grad_tensor& e = table[i];
        e.grad = g.const_data_ptr();
        e.numel = g.numel();
        e.dtype = e.out_dtype = code_of(g, "gradients");
        e.out = const_cast<void*>(e.grad);
        if (out) {
            const Tensor& o = (*out)[i];
            need_gpu(o);
            TORCH_CHECK_VALUE(o.device() == g.device() && o.sizes() == g.sizes() && ((o.is_contiguous() && g.is_contiguous()) || o.strides() == g.strides()),
                              "output ", i, " must be like its gradient in device, shape and strides");
            e.out = o.mutable_data_ptr();
            e.out_dtype = code_of(o, "outputs");
        }
    }
    return table;
}

Tensor norm_call(at::TensorList grads, int64_t norm_type, const double* max_norm, const at::TensorList* out) {
    if (out) TORCH_CHECK_VALUE(out->size() == grads.size(), out->size(), " outputs for ", grads.size(), " gradients");
    const std::vector<adcdiff_grad_tensor> table = grad_table(grads, out);
    const c10::Device dev = grads[0].device();
    const c10::DeviceGuard guard(dev);
    const int n = (int)table.size();
    const size_t bytes = adcdiff_grad_norm_workspace_bytes(table.data(), n);
    Tensor norm = at::empty({}, grads[0].options().dtype(at::kFloat)), ws = at::empty({(int64_t)bytes}, grads[0].options().dtype(at::kByte));
    float* value = norm.mutable_data_ptr<float>();
    if (!max_norm) {
        check(adcdiff_grad_norm(table.data(), n, (int)norm_type, value, ws.mutable_data_ptr(), bytes, stream_of(dev)));
    } else {
        check(adcdiff_clip_grad_norm(table.data(), n, (int)norm_type, *max_norm, value, ws.mutable_data_ptr(), bytes, stream_of(dev)));
        for (const Tensor& t : out ? *out : grads)
            if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version();   // written behind autograd's back
    }
    return norm;
}

Tensor grad_norm(at::TensorList grads, int64_t norm_type) { return norm_call(grads, norm_type, nullptr, nullptr); }
Tensor clip_grad_norm_(at::TensorList grads, double max_norm, int64_t norm_type) { return norm_call(grads, norm_type, &max_norm, nullptr); }
Tensor clip_grad_norm_out(at::TensorList grads, double max_norm, int64_t norm_type, at::TensorList out) { return norm_call(grads, norm_type, &max_norm, &out); }

// ------------------------------------------------------------------ 8-bit integer layer
int64_t pitch16(int64_t K) { return (K + 15) / 16 * 16; }

std::tuple<Tensor, Tensor> quantize_rows(const Tensor& x) {
    const c10::Device dev = one_device({&x});
    const int code = code_of(x, "x");
    const int64_t ldx = pitch_of(x, "x"), M = x.size(0), K = x.size(1);
    TORCH_CHECK_VALUE(K > 0, "rows of no columns have no scale");
    const c10::DeviceGuard guard(dev);
    Tensor q = at::empty({M, pitch16(K)}, x.options().dtype(at::kChar)), scale = at::empty({M}, x.options().dtype(at::kFloat));
    check(adcdiff_quantize_rows(x.const_data_ptr(), ldx, code, narrow(M, "rows"), narrow(K, "columns"), q.mutable_data_ptr<int8_t>(), pitch16(K),
                                scale.mutable_data_ptr<float>(), stream_of(dev)));
    return {K == pitch16(K) ? q : q.narrow(1, 0, K), scale};
}

// Codes as the product reads them: rows on 16-byte boundaries.  Those that are not are copied, all of a call in one launch.
struct Rows16 {
    adcdiff_i8_copy copies[2];
    int n = 0;
    // t itself, or the copy it will be; *ld: its pitch
    Tensor add(const Tensor& t, const char* what, long long* ld) {
        TORCH_CHECK_VALUE(t.scalar_type() == at::kChar, what, " must be int8, got ", t.scalar_type());
        const int64_t pitch = pitch_of(t, what), M = t.size(0), K = t.size(1);
        *ld = M > 1 ? pitch : pitch16(K);
        if (reinterpret_cast<uintptr_t>(t.const_data_ptr()) % 16 == 0 && *ld % 16 == 0) return t;
        Tensor o = at::empty({M, pitch16(K)}, t.options());
        *ld = pitch16(K);
        copies[n++] = adcdiff_i8_copy{t.const_data_ptr<int8_t>(), pitch, o.mutable_data_ptr<int8_t>(), pitch16(K), narrow(M, "rows"), narrow(K, "columns")};
        return o;
    }
    void run(c10::Device dev) {
        if (n) check(adcdiff_pitch_rows_i8(copies, n, stream_of(dev)));
    }
};

// The arguments that both forms of the layer share; fills `out` and `held` (what has to live until the launch)
adcdiff_gemm_i8_args layer_args(const Tensor& left, const Tensor& w, const Tensor& w_scale, const OptTensor& bias, const OptTensor& residual, int64_t act,
                                int64_t out_dtype, Rows16* rows, Tensor* out, Tensor* held) {
    TORCH_CHECK_VALUE(left.dim() == 2 && w.dim() == 2 && left.size(1) == w.size(1), "rows ", left.sizes(), " and weights ", w.sizes(), " do not fit");
    const int64_t M = left.size(0), K = left.size(1), N = w.size(0);
    TORCH_CHECK_VALUE(K > 0 && N > 0, "no columns: K ", K, ", N ", N);
    adcdiff_gemm_i8_args p{};
    p.M = narrow(M, "rows");
    p.N = narrow(N, "outputs");
    p.K = narrow(K, "columns");
    p.act = (int)act;
    p.out_dtype = (int)out_dtype;
    p.w_scale = vector_of(w_scale, N, "w_scale");
    p.bias = vector_of(bias, N, "bias");
    *out = at::empty({M, N}, left.options().dtype(type_of(out_dtype)));
    if (given(residual)) {
        TORCH_CHECK_VALUE(residual->sizes() == out->sizes() && residual->scalar_type() == out->scalar_type(), "residual must be ", out->scalar_type(), " ",
                          out->sizes(), ", got ", residual->scalar_type(), " ", residual->sizes());
        p.residual = residual->const_data_ptr();
        p.ldr = pitch_of(*residual, "residual");
    }
    *held = rows->add(w, "w", &p.ldw);
    p.w = held->const_data_ptr<int8_t>();
    p.out = out->mutable_data_ptr();
    p.ldo = N;
    return p;
}

Tensor gemm_int8(const Tensor& a, const Tensor& a_scale, const Tensor& w, const Tensor& w_scale, const OptTensor& bias, const OptTensor& residual, int64_t act,
                 int64_t out_dtype) {
    const c10::Device dev = one_device({&a, &a_scale, &w, &w_scale, ptr(bias), ptr(residual)});
    const c10::DeviceGuard guard(dev);
    Tensor out, held_w;
    Rows16 rows;
    adcdiff_gemm_i8_args p = layer_args(a, w, w_scale, bias, residual, act, out_dtype, &rows, &out, &held_w);
    p.a_scale = vector_of(a_scale, a.size(0), "a_scale");
    const Tensor held_a = rows.add(a, "a", &p.lda);
    p.a = held_a.const_data_ptr<int8_t>();
    rows.run(dev);
    check(adcdiff_gemm_i8(&p, stream_of(dev)));
    return out;
}

Tensor linear_int8(const Tensor& x, const Tensor& w, const Tensor& w_scale, const OptTensor& bias, const OptTensor& residual, int64_t act, int64_t out_dtype) {
    const c10::Device dev = one_device({&x, &w, &w_scale, ptr(bias), ptr(residual)});
    const int code = code_of(x, "x");
    const int64_t ldx = pitch_of(x, "x");
    const c10::DeviceGuard guard(dev);
    Tensor out, held_w;
    Rows16 rows;
    const adcdiff_gemm_i8_args p = layer_args(x, w, w_scale, bias, residual, act, out_dtype, &rows, &out, &held_w);
    rows.run(dev);
    const size_t bytes = adcdiff_linear_i8_workspace_bytes(p.M, p.K);
    Tensor ws = at::empty({(int64_t)bytes}, x.options().dtype(at::kByte));
    check(adcdiff_linear_i8(x.const_data_ptr(), ldx, code, &p, ws.mutable_data_ptr(), bytes, stream_of(dev)));
    return out;
}

// ------------------------------------------------------------------ autograd
template <typename F>
auto below_autograd(const char* name, F*) {
    return c10::Dispatcher::singleton().findSchemaOrThrow(name, "").typed<std::remove_pointer_t<F>>();
}

bool wants_grad(std::initializer_list<const Tensor*> tensors) {
    if (!at::GradMode::is_enabled()) return false;
    for (const Tensor* t : tensors)
        if (t && t->defined() && t->requires_grad()) return true;
    return false;
}

// No operator here has a forward-mode derivative.  A tangent is refused: below autograd it would be dropped, and a result without one counts as constant.
void no_tangent(const char* name, const Tensor& t) {
    TORCH_CHECK_NOT_IMPLEMENTED(!t.defined() || !t._fw_grad(/*level=*/0).defined(), name, " has no forward-mode derivative");
}
void no_tangents(const char* name, std::initializer_list<const Tensor*> tensors) {
    for (const Tensor* t : tensors)
        if (t) no_tangent(name, *t);
}
void no_tangents(const char* name, at::TensorList tensors) {
    for (const Tensor& t : tensors) no_tangent(name, t);
}

// A result without a gradient of its own: asking for one raises instead of leaving it out.  `call` makes the outputs.
struct Ungraded : torch::autograd::Function<Ungraded> {
    static variable_list forward(AutogradContext* ctx, at::TensorList inputs, const std::function<variable_list()>& call, const std::string& message) {
        ctx->saved_data["message"] = message;
        at::AutoDispatchBelowADInplaceOrView below;
        variable_list outs = call();
        variable_list codes;
        for (const Tensor& t : outs)
            if (!t.is_floating_point()) codes.push_back(t);
        ctx->mark_non_differentiable(codes);
        return outs;
    }
    static variable_list backward(AutogradContext* ctx, const variable_list&) {
        TORCH_CHECK(false, ctx->saved_data["message"].toStringRef());
    }
};

variable_list ungraded(std::initializer_list<const Tensor*> tensors, const std::function<variable_list()>& call, const char* message) {
    variable_list inputs;
    for (const Tensor* t : tensors)
        if (t && t->defined()) inputs.push_back(*t);
    return Ungraded::apply(at::TensorList(inputs), call, std::string(message));
}

constexpr const char* kNoLayerGradient = "the 8-bit integer layer has no gradient: it serves trained weights";

std::vector<Tensor> residual_norm_backward_autograd(const OptTensor& h, const Tensor& x, const OptTensor& gate, const OptTensor& post_weight,
                                                    const OptTensor& post_bias, const OptTensor& pre_weight, const OptTensor& pre_bias,
                                                    const OptTensor& stats, const OptTensor& d_x_new, const OptTensor& d_y, int64_t post_norm,
                                                    int64_t pre_norm, double residual_scale, double eps, std::array<bool, 7> need) {
    static const auto op = below_autograd("adcdiff::residual_norm_backward", &residual_norm_backward);
    auto call = [&] { return op.call(h, x, gate, post_weight, post_bias, pre_weight, pre_bias, stats, d_x_new, d_y, post_norm, pre_norm, residual_scale, eps, need); };
    const std::initializer_list<const Tensor*> inputs = {&x, ptr(h), ptr(gate), ptr(post_weight), ptr(post_bias), ptr(pre_weight), ptr(pre_bias), ptr(d_x_new), ptr(d_y)};
    no_tangents("residual_norm_backward", inputs);
    if (wants_grad(inputs)) return ungraded(inputs, call, "residual_norm is differentiable once");
    at::AutoDispatchBelowADInplaceOrView below;
    return call();
}

struct ResidualNorm : torch::autograd::Function<ResidualNorm> {
    static variable_list forward(AutogradContext* ctx, const OptTensor& h, const Tensor& x, const OptTensor& gate, const OptTensor& post_weight,
                                 const OptTensor& post_bias, const OptTensor& pre_weight, const OptTensor& pre_bias, int64_t post_norm, int64_t pre_norm,
                                 double residual_scale, double eps, bool with_x, bool with_stats) {
        static const auto op = below_autograd("adcdiff::residual_norm", &residual_norm);
        variable_list outs;
        {
            at::AutoDispatchBelowADInplaceOrView below;
            outs = op.call(h, x, gate, post_weight, post_bias, pre_weight, pre_bias, post_norm, pre_norm, residual_scale, eps, with_x, true);
        }
        auto plain = [](const OptTensor& t) { return given(t) ? *t : Tensor(); };
        ctx->save_for_backward({plain(h), x, plain(gate), plain(post_weight), plain(post_bias), plain(pre_weight), plain(pre_bias), outs.back()});
        ctx->saved_data["args"] = std::vector<double>{(double)post_norm, (double)pre_norm, residual_scale, eps, with_x ? 1.0 : 0.0};
        ctx->set_materialize_grads(false);
        if (with_stats) ctx->mark_non_differentiable({outs.back()});
        else outs.pop_back();
        return outs;
    }
    static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
        static const auto op = below_autograd("adcdiff::residual_norm_backward", &residual_norm_backward);
        const std::vector<double> args = ctx->saved_data["args"].toDoubleVector();
        const int64_t post_norm = (int64_t)args[0], pre_norm = (int64_t)args[1];
        const bool with_x = args[4] != 0.0;
        const variable_list s = ctx->get_saved_variables();
        const Tensor d_x = with_x ? grads[0] : Tensor(), d_y = pre_norm ? grads[with_x ? 1 : 0] : Tensor();
        variable_list result(13);
        if (!d_x.defined() && !d_y.defined()) return result;
        std::array<bool, 7> need{};
        size_t edge = 0;   // autograd counts the inputs that are there
        for (int i = 0; i < 7; ++i) need[i] = s[i].defined() && ctx->needs_input_grad(edge++);
        auto opt = [](const Tensor& t) { return t.defined() ? OptTensor(t) : OptTensor(); };
        const std::vector<Tensor> outs = op.call(opt(s[0]), s[1], opt(s[2]), opt(s[3]), opt(s[4]), opt(s[5]), opt(s[6]), opt(s[7]), opt(d_x), opt(d_y), post_norm,
                                                 pre_norm, args[2], args[3], need);
        size_t k = 0;
        for (int i = 0; i < 7; ++i)
            if (need[i]) result[i] = outs[k++];
        return result;
    }
};

std::vector<Tensor> residual_norm_autograd(const OptTensor& h, const Tensor& x, const OptTensor& gate, const OptTensor& post_weight, const OptTensor& post_bias,
                                           const OptTensor& pre_weight, const OptTensor& pre_bias, int64_t post_norm, int64_t pre_norm,
                                           double residual_scale, double eps, bool with_x, bool with_stats) {
    const std::initializer_list<const Tensor*> inputs = {&x, ptr(h), ptr(gate), ptr(post_weight), ptr(post_bias), ptr(pre_weight), ptr(pre_bias)};
    no_tangents("residual_norm", inputs);
    if (wants_grad(inputs))
        return ResidualNorm::apply(h, x, gate, post_weight, post_bias, pre_weight, pre_bias, post_norm, pre_norm, residual_scale, eps, with_x, with_stats);
    static const auto op = below_autograd("adcdiff::residual_norm", &residual_norm);
    at::AutoDispatchBelowADInplaceOrView below;
    return op.call(h, x, gate, post_weight, post_bias, pre_weight, pre_bias, post_norm, pre_norm, residual_scale, eps, with_x, with_stats);
}

// Gradients that themselves require one (create_graph): the norm is a constant, as torch.nn.utils' total norm is, and the clipping is not recorded
Tensor grad_norm_autograd(at::TensorList grads, int64_t norm_type) {
    static const auto op = below_autograd("adcdiff::grad_norm", &grad_norm);
    no_tangents("grad_norm", grads);
    at::AutoDispatchBelowADInplaceOrView below;
    return op.call(grads, norm_type);
}
Tensor clip_grad_norm_autograd_(at::TensorList grads, double max_norm, int64_t norm_type) {
    static const auto op = below_autograd("adcdiff::clip_grad_norm_", &clip_grad_norm_);
    no_tangents("clip_grad_norm_", grads);
    at::AutoDispatchBelowADInplaceOrView below;
    return op.call(grads, max_norm, norm_type);
}
Tensor clip_grad_norm_out_autograd(at::TensorList grads, double max_norm, int64_t norm_type, at::TensorList out) {
    static const auto op = below_autograd("adcdiff::clip_grad_norm_out", &clip_grad_norm_out);
    no_tangents("clip_grad_norm_out", grads);
    no_tangents("clip_grad_norm_out", out);
    at::AutoDispatchBelowADInplaceOrView below;
    return op.call(grads, max_norm, norm_type, out);
}

std::tuple<Tensor, Tensor> quantize_rows_autograd(const Tensor& x) {
    static const auto op = below_autograd("adcdiff::quantize_rows", &quantize_rows);
    no_tangents("quantize_rows", {&x});
    if (wants_grad({&x})) {
        const variable_list outs = ungraded({&x}, [&] { auto r = op.call(x); return variable_list{std::get<0>(r), std::get<1>(r)}; }, kNoLayerGradient);
        return {outs[0], outs[1]};
    }
    at::AutoDispatchBelowADInplaceOrView below;
    return op.call(x);
}
Tensor gemm_int8_autograd(const Tensor& a, const Tensor& a_scale, const Tensor& w, const Tensor& w_scale, const OptTensor& bias, const OptTensor& residual,
                          int64_t act, int64_t out_dtype) {
    static const auto op = below_autograd("adcdiff::gemm_int8", &gemm_int8);
    const std::initializer_list<const Tensor*> inputs = {&a_scale, &w_scale, ptr(bias), ptr(residual)};
    no_tangents("gemm_int8", inputs);
    if (wants_grad(inputs))
        return ungraded(inputs, [&] { return variable_list{op.call(a, a_scale, w, w_scale, bias, residual, act, out_dtype)}; }, kNoLayerGradient)[0];
    at::AutoDispatchBelowADInplaceOrView below;
    return op.call(a, a_scale, w, w_scale, bias, residual, act, out_dtype);
}
Tensor linear_int8_autograd(const Tensor& x, const Tensor& w, const Tensor& w_scale, const OptTensor& bias, const OptTensor& residual, int64_t act,
                            int64_t out_dtype) {
    static const auto op = below_autograd("adcdiff::linear_int8", &linear_int8);
    const std::initializer_list<const Tensor*> inputs = {&x, &w_scale, ptr(bias), ptr(residual)};
    no_tangents("linear_int8", inputs);
    if (wants_grad(inputs))
        return ungraded(inputs, [&] { return variable_list{op.call(x, w, w_scale, bias, residual, act, out_dtype)}; }, kNoLayerGradient)[0];
    at::AutoDispatchBelowADInplaceOrView below;
    return op.call(x, w, w_scale, bias, residual, act, out_dtype);
}

}  // namespace

TORCH_LIBRARY_FRAGMENT(adcdiff, m) {
    const std::vector<at::Tag> tags = {at::Tag::pt2_compliant_tag};
    m.def("residual_norm(Tensor? h, Tensor x, Tensor? gate, Tensor? post_weight, Tensor? post_bias, Tensor? pre_weight, Tensor? pre_bias, int post_norm, "
          "int pre_norm, float residual_scale, float eps, bool with_x, bool with_stats) -> Tensor[]", tags);
    m.def("residual_norm_backward(Tensor? h, Tensor x, Tensor? gate, Tensor? post_weight, Tensor? post_bias, Tensor? pre_weight, Tensor? pre_bias, "
          "Tensor? stats, Tensor? d_x_new, Tensor? d_y, int post_norm, int pre_norm, float residual_scale, float eps, bool[7] need) -> Tensor[]", tags);
    m.def("grad_norm(Tensor[] grads, int norm_type) -> Tensor", tags);
    m.def("clip_grad_norm_(Tensor(a!)[] grads, float max_norm, int norm_type) -> Tensor", tags);
    m.def("clip_grad_norm_out(Tensor[] grads, float max_norm, int norm_type, Tensor(a!)[] out) -> Tensor", tags);
    m.def("quantize_rows(Tensor x) -> (Tensor, Tensor)", tags);
    m.def("gemm_int8(Tensor a, Tensor a_scale, Tensor w, Tensor w_scale, Tensor? bias, Tensor? residual, int act, int out_dtype) -> Tensor", tags);
    m.def("linear_int8(Tensor x, Tensor w, Tensor w_scale, Tensor? bias, Tensor? residual, int act, int out_dtype) -> Tensor", tags);
}

// The CPU entries refuse: every implementation asks for tensors on a GPU.
#define ADCDIFF_IMPLS(m)                                    \
    m.impl("residual_norm", &residual_norm);                \
    m.impl("residual_norm_backward", &residual_norm_backward); \
    m.impl("grad_norm", &grad_norm);                        \
    m.impl("clip_grad_norm_", &clip_grad_norm_);            \
    m.impl("clip_grad_norm_out", &clip_grad_norm_out);      \
    m.impl("quantize_rows", &quantize_rows);                \
    m.impl("gemm_int8", &gemm_int8);                        \
    m.impl("linear_int8", &linear_int8);
TORCH_LIBRARY_IMPL(adcdiff, CUDA, m) { ADCDIFF_IMPLS(m) }
TORCH_LIBRARY_IMPL(adcdiff, CPU, m) { ADCDIFF_IMPLS(m) }

TORCH_LIBRARY_IMPL(adcdiff, Autograd, m) {
    m.impl("residual_norm", &residual_norm_autograd);
    m.impl("residual_norm_backward", &residual_norm_backward_autograd);
    m.impl("grad_norm", &grad_norm_autograd);
    m.impl("clip_grad_norm_", &clip_grad_norm_autograd_);
    m.impl("clip_grad_norm_out", &clip_grad_norm_out_autograd);
    m.impl("quantize_rows", &quantize_rows_autograd);
    m.impl("gemm_int8", &gemm_int8_autograd);
    m.impl("linear_int8", &linear_int8_autograd);
}
