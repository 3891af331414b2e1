// The host side of one call of group norm or of the 8-bit product: outputs and workspace from torch's allocator, the descriptor, the
// entry point of liby5hip.so on the current stream, and the node of the gradient.  The kernels of a small map take a few
// microseconds; the same steps in Python take ten (and sixty for the gradient, whose thread has to wait for the interpreter).
// Arguments arrive checked (yolo_amd/groupnorm.py, yolo_amd/int8.py).
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPGraphsC10Utils.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/variable.h>
#include <torch/extension.h>

#include <optional>
#include <stdexcept>
#include <string>

#include "../../include/y5hip.h"

namespace {

using at::Tensor;
typedef const std::optional<Tensor>& Maybe;

struct Error : std::runtime_error {
    using std::runtime_error::runtime_error;
};

void check(int rc) {
    if (rc) throw Error("liby5hip error " + std::to_string(rc) + ": " + y5_last_error());
}

int code(at::ScalarType t) {
    if (t == at::kHalf) return Y5_F16;
    if (t == at::kBFloat16) return Y5_BF16;
    TORCH_CHECK_TYPE(t == at::kFloat, "fp16, bf16 or fp32 expected, got ", t);
    return Y5_F32;
}

void* stream_of(const Tensor& t) { return c10::hip::getCurrentHIPStream(t.get_device()).stream(); }
void* ptr(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
Tensor or_none(Maybe t) { return t.has_value() ? *t : Tensor(); }

Tensor bytes(size_t n, const Tensor& like) {
    return n ? at::empty({(int64_t)n}, like.options().dtype(at::kByte)) : Tensor();
}

// x's shape in dense channels-last memory
Tensor empty_channels_last(const Tensor& x) {
    c10::SmallVector<int64_t, 6> strides(x.dim());
    int64_t at = x.size(1);
    strides[1] = 1;
    for (int64_t d = x.dim() - 1; d >= 2; --d) {
        strides[d] = at;
        at *= x.size(d);
    }
    strides[0] = at;
    return at::empty_strided(x.sizes(), strides, x.options());
}

struct Norm {
    int64_t pitch, groups, act;
    double eps, slope;
};

y5_group_norm_desc describe(const Tensor& x, const Norm& n, const Tensor& weight, const Tensor& bias) {
    y5_group_norm_desc d{};
    d.x = x.data_ptr();
    d.weight = ptr(weight);
    d.bias = ptr(bias);
    d.batch = (int32_t)x.size(0);
    d.c = (int32_t)x.size(1);
    d.pixels = (int32_t)std::min<int64_t>(x.numel() / (x.size(0) * x.size(1)), INT32_MAX);  // too many are refused there
    d.groups = (int32_t)n.groups;
    d.x_ld = (int32_t)n.pitch;
    d.y_ld = d.dy_ld = d.dx_ld = d.c;
    d.dtype = code(x.scalar_type());
    d.param_dtype = weight.defined() ? code(weight.scalar_type()) : bias.defined() ? code(bias.scalar_type()) : Y5_F32;
    d.act = (int32_t)n.act;
    d.slope = (float)n.slope;
    d.eps = (float)n.eps;
    TORCH_CHECK_VALUE(x.size(0) <= INT32_MAX && x.size(1) <= INT32_MAX && n.pitch <= INT32_MAX, "group_norm: shape ", x.sizes(), " with pitch ", n.pitch);
    return d;
}

Tensor give_workspace(y5_group_norm_desc& d, int what, const Tensor& like) {
    size_t n = 0;
    check(y5_group_norm_workspace(&d, what, &n));
    Tensor ws = bytes(n, like);
    d.workspace = ptr(ws);
    d.workspace_bytes = n;
    return ws;
}

Tensor run_forward(const Tensor& x, const Norm& n, const Tensor& weight, const Tensor& bias, const Tensor& stats) {
    const c10::DeviceGuard guard(x.device());
    y5_group_norm_desc d = describe(x, n, weight, bias);
    const Tensor ws = give_workspace(d, Y5_GN_FORWARD, x), y = empty_channels_last(x);
    d.y = y.data_ptr();
    if (stats.defined()) {
        d.mean = stats.data_ptr<float>();
        d.rstd = d.mean + stats.numel() / 2;
    }
    check(y5_group_norm(&d, stream_of(x)));
    return y;
}

// torch keeps one accumulation node a leaf as long as any graph of it lives, on the stream of the first.  The default stream cannot
// join a capture: the captured gradient of a leaf whose node lives there ends the process.  Under capture the forward pass looks for
// such leaves (the node would otherwise be made with this call's own), and the gradient is refused.
bool lives_elsewhere(const Tensor& t) {
    if (!t.defined() || !t.requires_grad() || !t.is_leaf()) return false;
    const auto node = torch::autograd::impl::try_get_grad_accumulator(t);
    if (!node) return false;
    const auto stream = node->stream();
    return stream && stream->id() == c10::hip::getDefaultHIPStream(t.get_device()).id();
}

struct GroupNorm : torch::autograd::Function<GroupNorm> {
    static Tensor forward(torch::autograd::AutogradContext* ctx, const Tensor& x, Maybe weight, Maybe bias, int64_t pitch, int64_t groups, double eps,
                          int64_t act, double slope, bool refused) {
        const Tensor w = or_none(weight), b = or_none(bias);
        const Tensor stats = at::empty({2, x.size(0), groups}, x.options().dtype(at::kFloat));  // mean and 1 / deviation
        const Tensor y = run_forward(x, Norm{pitch, groups, act, eps, slope}, w, b, stats);
        ctx->save_for_backward({x, w, b, stats});
        ctx->saved_data["pitch"] = pitch;
        ctx->saved_data["groups"] = groups;
        ctx->saved_data["act"] = act;
        ctx->saved_data["eps"] = eps;
        ctx->saved_data["slope"] = slope;
        ctx->saved_data["refused"] = refused;
        return y;
    }

    static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list grads) {
        const auto saved = ctx->get_saved_variables();
        const Tensor &x = saved[0], &w = saved[1], &b = saved[2], &stats = saved[3];
        auto& kept = ctx->saved_data;
        TORCH_CHECK(!kept["refused"].toBool(), "group_norm: a live graph on the default stream holds x, weight or bias, and their captured gradient would have to wait "
                                               "for that stream: drop the graph before the capture");
        const Norm n{kept["pitch"].toInt(), kept["groups"].toInt(), kept["act"].toInt(), kept["eps"].toDouble(), kept["slope"].toDouble()};
        Tensor dx, dw, db;
        {
            const at::AutoGradMode off(false);
            const c10::DeviceGuard guard(x.device());
            const Tensor dy = grads[0].movedim(1, -1).contiguous();  // (batch, *spatial, channels): itself where it is channels-last
            if (ctx->needs_input_grad(0)) dx = empty_channels_last(x);
            if (w.defined() && ctx->needs_input_grad(1)) dw = at::empty_like(w);
            if (b.defined() && ctx->needs_input_grad(w.defined() ? 2 : 1)) db = at::empty_like(b);
            y5_group_norm_desc d = describe(x, n, w, b);
            const Tensor ws = give_workspace(d, Y5_GN_BACKWARD, x);
            d.dy = dy.data_ptr();
            d.dx = ptr(dx);
            d.dweight = ptr(dw);
            d.dbias = ptr(db);
            d.mean = stats.data_ptr<float>();
            d.rstd = d.mean + stats.numel() / 2;
            check(y5_group_norm_backward(&d, stream_of(x)));
        }
        if (at::GradMode::is_enabled()) {  // create_graph: an error for whoever differentiates these in turn
            torch::autograd::variable_list out;
            for (Tensor* t : {&dx, &dw, &db})
                if (t->defined()) out.push_back(t->detach().requires_grad_(true));
            const auto once = std::make_shared<torch::autograd::DelayedError>("group_norm is differentiable once", (int64_t)out.size());
            out = (*once)(std::move(out));
            size_t i = 0;
            for (Tensor* t : {&dx, &dw, &db})
                if (t->defined()) *t = out[i++];
        }
        return {dx, dw, db, Tensor(), Tensor(), Tensor(), Tensor(), Tensor(), Tensor()};
    }
};

Tensor group_norm(const Tensor& x, int64_t pitch, int64_t groups, Maybe weight, Maybe bias, double eps, int64_t act, double slope) {
    const Tensor w = or_none(weight), b = or_none(bias);
    if (at::GradMode::is_enabled() && (x.requires_grad() || (w.defined() && w.requires_grad()) || (b.defined() && b.requires_grad()))) {
        const bool refused = c10::hip::currentStreamCaptureStatusMayInitCtx() != c10::hip::CaptureStatus::None &&
                             (lives_elsewhere(x) || lives_elsewhere(w) || lives_elsewhere(b));
        return GroupNorm::apply(x, weight, bias, pitch, groups, eps, act, slope, refused);
    }
    return run_forward(x, Norm{pitch, groups, act, eps, slope}, w, b, Tensor());
}

int64_t row_bytes(int64_t k) { return (k + 15) / 16 * 16; }

std::tuple<Tensor, Tensor> group_norm_rows(const Tensor& x, int64_t pitch, int64_t groups, Maybe weight, Maybe bias, double eps, int64_t act, double slope) {
    const c10::DeviceGuard guard(x.device());
    const Tensor w = or_none(weight), b = or_none(bias);
    y5_group_norm_desc d = describe(x, Norm{pitch, groups, act, eps, slope}, w, b);
    const Tensor ws = give_workspace(d, Y5_GN_ROWS, x);
    const int64_t rows = x.numel() / x.size(1), ld = row_bytes(x.size(1));
    Tensor q = at::empty({rows, ld}, x.options().dtype(at::kChar)), scale = at::empty({rows}, x.options().dtype(at::kFloat));
    check(y5_group_norm_rows_i8(&d, q.data_ptr(), (int)ld, scale.data_ptr<float>(), stream_of(x)));
    return {q, scale};
}

std::tuple<Tensor, Tensor> quantize_rows(const Tensor& x, int64_t pitch, int64_t rows, int64_t k) {
    const c10::DeviceGuard guard(x.device());
    const int64_t ld = row_bytes(k);
    Tensor q = at::empty({rows, ld}, x.options().dtype(at::kChar)), scale = at::empty({rows}, x.options().dtype(at::kFloat));
    check(y5_quantize_rows_i8(x.data_ptr(), pitch, code(x.scalar_type()), rows, (int)k, q.data_ptr(), (int)ld, scale.data_ptr<float>(), stream_of(x)));
    return {q, scale};
}

y5_gemm_i8_desc describe(const Tensor& wq, const Tensor& wscale, int64_t k, Maybe bias, int64_t act, double slope, int64_t m, const Tensor& y) {
    y5_gemm_i8_desc d{};
    d.w = wq.data_ptr();
    d.w_scale = wscale.data_ptr<float>();
    d.bias = bias.has_value() ? bias->data_ptr<float>() : nullptr;
    d.y = y.data_ptr();
    d.m = m;
    d.n = (int32_t)wq.size(0);
    d.y_ld = d.n;
    d.k = (int32_t)k;
    d.ld = (int32_t)wq.size(1);
    d.dtype = code(y.scalar_type());
    d.act = (int32_t)act;
    d.slope = (float)slope;
    return d;
}

// sizes: of the result, (*lead, n)
Tensor product(const Tensor& q, const Tensor& scale, const Tensor& wq, const Tensor& wscale, int64_t k, Maybe bias, int64_t act, double slope,
               at::ScalarType dtype, const std::vector<int64_t>& sizes) {
    const c10::DeviceGuard guard(q.device());
    Tensor y = at::empty(sizes, q.options().dtype(dtype));
    y5_gemm_i8_desc d = describe(wq, wscale, k, bias, act, slope, q.size(0), y);
    d.a = q.data_ptr();
    d.a_scale = scale.data_ptr<float>();
    check(y5_gemm_i8(&d, stream_of(q)));
    return y;
}

// m rows of k values `pitch` elements apart
Tensor linear(const Tensor& x, int64_t pitch, int64_t m, const Tensor& wq, const Tensor& wscale, int64_t k, Maybe bias, int64_t act, double slope,
              at::ScalarType dtype, const std::vector<int64_t>& sizes) {
    const c10::DeviceGuard guard(x.device());
    Tensor y = at::empty(sizes, x.options().dtype(dtype));
    const y5_gemm_i8_desc d = describe(wq, wscale, k, bias, act, slope, m, y);
    const int x_dtype = code(x.scalar_type());
    size_t n = 0;
    check(y5_linear_i8_workspace(&d, x_dtype, &n));
    const Tensor ws = bytes(n, x);
    check(y5_linear_i8(&d, x.data_ptr(), pitch, x_dtype, ptr(ws), n, stream_of(x)));
    return y;
}

}  // namespace

PYBIND11_MODULE(_calls, m) {
    m.doc() = "Per-call host side of yolo_amd.groupnorm and yolo_amd.int8 (arguments checked there)";
    // errors of the library surface as the class that yolo_amd._lib raises
    m.def("raise_as", [](py::object error) {
        static py::object* cls = nullptr;
        if (!cls) {
            cls = new py::object(error);
            py::register_exception_translator([](std::exception_ptr p) {
                try {
                    if (p) std::rethrow_exception(p);
                } catch (const Error& e) {
                    PyErr_SetString(cls->ptr(), e.what());
                }
            });
        }
    });
    m.def("group_norm", &group_norm);
    m.def("group_norm_rows", &group_norm_rows);
    m.def("quantize_rows", &quantize_rows);
    m.def("product", &product);
    m.def("linear", &linear);
}
