// layers_torch.cpp -- the autograd side of nerf_loam_amd.layers over the C ABI of libnerfloam_hip.so (include/nerfloam_hip.h nl_linear_*, nl_mx8_*, nl_embedding_*).
// Host code only: argument checks, output and workspace tensors, the autograd nodes.  A small layer's kernels take a few microseconds, so what surrounds them is
// C++: a call from Python costs about as much here as one torch operation, and the backward pass never takes the interpreter lock.
// The C functions are bound by address (bind), so that the library the Python side loaded is the one that runs.
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPGraphsC10Utils.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/extension.h>

#include <sstream>

#include "nerfloam_hip.h"

namespace {

using at::Tensor;
using OptTensor = std::optional<Tensor>;
namespace py = pybind11;

struct NlError : std::runtime_error { using std::runtime_error::runtime_error; };        // -> nerf_loam_amd._lib.NerfLoamHipError
py::object& error_class() { static py::object* o = new py::object(); return *o; }

decltype(&nl_linear_forward) f_forward = nullptr;
decltype(&nl_linear_backward) f_backward = nullptr;
decltype(&nl_linear_workspace) f_workspace = nullptr;
decltype(&nl_mx8_encode) f_encode = nullptr;
decltype(&nl_mx8_decode) f_decode = nullptr;
decltype(&nl_embedding_forward) f_emb_forward = nullptr;
decltype(&nl_embedding_backward) f_emb_backward = nullptr;
decltype(&nl_embedding_workspace) f_emb_workspace = nullptr;

template <class... A> std::string cat(const A&... a) { std::ostringstream s; (s << ... << a); return s.str(); }
[[noreturn]] void fail(const std::string& s) { throw NlError(s); }
void check(int rc, const char* what)
{
    if (rc == NL_OK) return;
    fail(cat(what, " failed: ", rc == NL_ERR_INVALID_ARG ? "invalid argument" : rc == NL_ERR_LAUNCH ? "kernel launch failed" : rc == NL_ERR_NO_DEVICE ? "no HIP device" : "capacity exceeded"));
}

int dtype_of(const Tensor& t, const char* name)
{
    switch (t.scalar_type()) {
        case at::kFloat: return NL_DT_F32;
        case at::kBFloat16: return NL_DT_BF16;
        case at::kHalf: return NL_DT_F16;
        default: fail(cat(name, " must be float32, bfloat16 or float16, got ", t.scalar_type()));
    }
}
void on_gpu(const Tensor& t, const char* name)
{
    if (!t.is_cuda()) fail(cat(name, ": the layer operators run on the GPU only - no CPU path"));
}
void same_kind(const Tensor& t, const Tensor& like, const char* name)
{
    if (t.device() != like.device() || t.scalar_type() != like.scalar_type())
        fail(cat(name, " must be ", like.scalar_type(), " on ", like.device(), ", got ", t.scalar_type(), " on ", t.device()));
}
void* stream_of(const Tensor& t) { return (void*)c10::hip::getCurrentHIPStream(t.device().index()).stream(); }
// a result would come without the tangent, and nobody would notice
void no_tangent(const char* what, std::initializer_list<const Tensor*> in)
{
    for (const Tensor* t : in)
        if (t && t->defined() && t->_fw_grad(0).defined()) fail(cat(what, ": forward-mode derivatives are not provided"));
}
const Tensor* opt(const OptTensor& t) { return t ? &*t : nullptr; }
void no_capture(const char* what)
{
    if (c10::hip::currentStreamCaptureStatusMayInitCtx() != c10::hip::CaptureStatus::None)
        fail(cat(what, ": the backward pass cannot run through autograd while a stream is being captured; capture the functions of ops instead"));
}

// [..., cols] -> [rows, cols] with adjacent elements in a row; a copy only where the strides allow nothing else
Tensor rows2d(const Tensor& t, int64_t cols)
{
    Tensor r = t.dim() == 2 && t.size(1) == cols ? t : t.reshape({cols ? t.numel() / cols : 0, cols});
    if ((cols > 1 && r.stride(1) != 1) || (r.size(0) > 1 && r.stride(0) < cols)) r = r.contiguous();
    return r;
}
int64_t row_stride(const Tensor& t) { return t.size(0) > 1 ? t.stride(0) : t.size(1); }
void* ptr(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }

Tensor workspace(int64_t need, const Tensor& like, const char* what)
{
    if (need < 0) fail(cat(what, " failed: invalid argument"));
    return need == 0 ? Tensor() : at::empty({need}, like.options().dtype(at::kByte));
}
// Gradients of gradients are not provided: a gradient that depends on a tensor somebody differentiates by (`depends`) carries an error that comes when it is
// differentiated itself; one that does not is a constant
void once_differentiable(Tensor& t, bool depends)
{
    if (!at::GradMode::is_enabled() || !t.defined() || !depends) return;
    t = (*std::make_shared<torch::autograd::DelayedError>("gradients of gradients of the layer operators are not provided", 1))({t.detach().requires_grad_(true)})[0];
}

struct Kept { Tensor z, bits, z8, z8e, x8, x8e; };

Tensor linear_forward(const Tensor& x, const Tensor& w, const Tensor& b, const Tensor& r, int act, bool mx8, bool keep, bool keep_x, Kept* kept)
{
    const int64_t M = x.size(0), K = x.size(1), N = w.size(0);
    c10::DeviceGuard guard(x.device());
    const auto bytes = x.options().dtype(at::kByte);
    if (keep && act != NL_ACT_NONE) {
        const int64_t nb = (N + 31) / 32;
        if (act == NL_ACT_RELU) kept->bits = at::empty({M, nb}, x.options().dtype(at::kInt));
        else if (mx8) { kept->z8 = at::empty({M, 32 * nb}, bytes); kept->z8e = at::empty({M, nb}, bytes); }
        else kept->z = at::empty({M, N}, x.options());
    }
    if (keep_x && mx8) { kept->x8 = at::empty({M, (K + 31) / 32 * 32}, bytes); kept->x8e = at::empty({M, (K + 31) / 32}, bytes); }
    Tensor y = at::empty({M, N}, x.options());
    NlLinear d = {};
    d.struct_size = (int)sizeof d; d.dtype = dtype_of(x, "x"); d.act = act; d.M = M;
    if (K < 1 || N < 1 || K > INT32_MAX || N > INT32_MAX) fail("linear_act failed: invalid argument");
    d.K = (int)K; d.N = (int)N;
    d.x = ptr(x); d.ldx = row_stride(x); d.w = ptr(w); d.ldw = row_stride(w); d.b = ptr(b);
    if (r.defined()) { d.r = ptr(r); d.ldr = row_stride(r); }
    d.y = ptr(y); d.ldy = N;
    d.z = ptr(kept->z); d.bits = (unsigned*)ptr(kept->bits); d.z8 = (unsigned char*)ptr(kept->z8); d.z8e = (unsigned char*)ptr(kept->z8e);
    d.x8 = (unsigned char*)ptr(kept->x8); d.x8e = (unsigned char*)ptr(kept->x8e);
    const Tensor ws = workspace(f_workspace(&d, 0), x, "nl_linear_forward");
    d.ws = ptr(ws); d.ws_bytes = ws.defined() ? ws.numel() : 0;
    check(f_forward(&d, stream_of(x)), "nl_linear_forward");
    return y;
}

void encode(const Tensor& x, Tensor& codes, Tensor& exps)
{
    const int64_t M = x.size(0), K = x.size(1), kb = (K + 31) / 32;
    c10::DeviceGuard guard(x.device());
    codes = at::empty({M, 32 * kb}, x.options().dtype(at::kByte));
    exps = at::empty({M, kb}, x.options().dtype(at::kByte));
    if (K > INT32_MAX) fail("nl_mx8_encode failed: invalid argument");
    check(f_encode(ptr(x), row_stride(x), M, (int)K, dtype_of(x, "x"), (unsigned char*)ptr(codes), (unsigned char*)ptr(exps), stream_of(x)), "nl_mx8_encode");
}

struct LinearFn : torch::autograd::Function<LinearFn> {
    static Tensor forward(torch::autograd::AutogradContext* ctx, const Tensor& x, const Tensor& w, const OptTensor& b, const OptTensor& r, int64_t act, bool mx8)
    {
        const bool gx = x.requires_grad(), gw = w.requires_grad(), gb = b && b->requires_grad(), gr = r && r->requires_grad();
        Kept kept;
        Tensor y = linear_forward(x, w, b ? *b : Tensor(), r ? *r : Tensor(), (int)act, mx8, gx || gw || gb, gw, &kept);
        // only what a gradient holds: what is not saved may be written before the backward pass
        ctx->save_for_backward({gw && !mx8 ? x : Tensor(), gx ? w : Tensor(), kept.x8, kept.x8e, kept.z, kept.bits, kept.z8, kept.z8e});
        ctx->saved_data["c"] = std::vector<int64_t>{act, gx, gw, gb, gr, b.has_value(), r.has_value(), w.size(0), w.size(1)};
        return y;
    }
    static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list grads)
    {
        no_capture("linear_act");
        const auto saved = ctx->get_saved_variables();
        const auto c = ctx->saved_data["c"].toIntVector();
        const Tensor &w = saved[1], &g = grads[0];
        torch::autograd::variable_list out(6);
        if (!g.defined()) return out;
        // edges: x, w, then bias and residual where given
        const bool gx = c[1] && ctx->needs_input_grad(0), gw = c[2] && ctx->needs_input_grad(1), gb = c[3] && ctx->needs_input_grad(2), gr = c[4] && ctx->needs_input_grad(2 + c[5]);
        const int64_t N = c[7], K = c[8];
        const Tensor g2 = rows2d(g, N);
        const int64_t M = g2.size(0);
        if (gx || gw || gb) {
            c10::DeviceGuard guard(g.device());
            if (gx) out[0] = at::empty({M, K}, g.options());
            if (gw) out[1] = at::empty({N, K}, g.options());
            if (gb) out[2] = at::empty({N}, g.options());
            NlLinear d = {};
            d.struct_size = (int)sizeof d; d.dtype = dtype_of(g2, "gy"); d.act = (int)c[0]; d.M = M; d.K = (int)K; d.N = (int)N;
            d.gy = ptr(g2); d.ldgy = row_stride(g2);
            if (w.defined()) { d.w = ptr(w); d.ldw = row_stride(w); }
            if (saved[0].defined()) { d.x = ptr(saved[0]); d.ldx = row_stride(saved[0]); }
            d.x8 = (unsigned char*)ptr(saved[2]); d.x8e = (unsigned char*)ptr(saved[3]);
            d.z = ptr(saved[4]); d.bits = (unsigned*)ptr(saved[5]); d.z8 = (unsigned char*)ptr(saved[6]); d.z8e = (unsigned char*)ptr(saved[7]);
            d.gx = ptr(out[0]); d.gw = ptr(out[1]); d.gb = ptr(out[2]);
            const Tensor ws = workspace(f_workspace(&d, 1), g2, "nl_linear_backward");
            d.ws = ptr(ws); d.ws_bytes = ws.defined() ? ws.numel() : 0;
            check(f_backward(&d, stream_of(g2)), "nl_linear_backward");
        }
        // gx = dz w, gw = dz^T x, gb = sum of dz with dz = gy act'(x w^T + b); act' of none and relu is constant almost everywhere
        const bool dz = g.requires_grad() || ((c[0] == NL_ACT_GELU || c[0] == NL_ACT_SILU) && (c[1] || c[2] || c[3]));
        once_differentiable(out[0], dz || c[2]);
        once_differentiable(out[1], dz || c[1]);
        once_differentiable(out[2], dz);
        if (gr) out[3] = g;
        return out;
    }
};

Tensor linear_act(const Tensor& x, const Tensor& weight, const OptTensor& bias, int64_t act, const OptTensor& residual, bool mx8)
{
    no_tangent("linear_act", {&x, &weight, opt(bias), opt(residual)});
    on_gpu(x, "linear_act");
    if (weight.dim() != 2 || x.dim() < 1 || x.size(-1) != weight.size(1)) throw py::value_error(cat("linear_act: x ", x.sizes(), " must be [..., K] and weight ", weight.sizes(), " [N, K]"));
    const int64_t K = weight.size(1), N = weight.size(0);
    auto shape = x.sizes().vec();
    shape.back() = N;
    if (bias && (bias->dim() != 1 || bias->size(0) != N)) throw py::value_error(cat("linear_act: bias ", bias->sizes(), " must be [", N, "]"));
    if (residual && residual->sizes() != at::IntArrayRef(shape)) throw py::value_error(cat("linear_act: residual ", residual->sizes(), " must be ", at::IntArrayRef(shape)));
    if (K < 1 || N < 1) throw py::value_error(cat("linear_act: weight ", weight.sizes(), " must have elements"));
    dtype_of(x, "x");
    same_kind(weight, x, "weight");
    const Tensor x2 = rows2d(x, K), w2 = rows2d(weight, K);
    OptTensor b, r;
    if (bias) { same_kind(*bias, x, "bias"); b = bias->contiguous(); }
    if (residual) { same_kind(*residual, x, "residual"); r = rows2d(*residual, N); }
    Tensor y;
    if (at::GradMode::is_enabled() && (x2.requires_grad() || w2.requires_grad() || (b && b->requires_grad()) || (r && r->requires_grad()))) y = LinearFn::apply(x2, w2, b, r, act, mx8);
    else {
        Kept kept;
        y = linear_forward(x2, w2, b ? *b : Tensor(), r ? *r : Tensor(), (int)act, mx8, false, false, &kept);
    }
    return shape.size() == 2 ? y : y.view(shape);
}

std::tuple<Tensor, Tensor> checkpoint_encode(const Tensor& x)
{
    on_gpu(x, "checkpoint_encode");
    if (x.dim() < 1 || x.size(-1) < 1) throw py::value_error(cat("checkpoint_encode: x ", x.sizes(), " must be [..., K], K >= 1"));
    Tensor codes, exps;
    encode(rows2d(x.detach(), x.size(-1)), codes, exps);
    return {codes, exps};
}
Tensor checkpoint_decode(const Tensor& codes, const Tensor& exps, std::vector<int64_t> shape, at::ScalarType dtype)
{
    on_gpu(codes, "checkpoint_decode");
    if (shape.empty() || shape.back() < 1 || shape.back() > INT32_MAX) throw py::value_error("checkpoint_decode: the shape must be [..., K], K >= 1");
    const int64_t K = shape.back(), kb = (K + 31) / 32;
    int64_t M = 1;
    for (size_t i = 0; i + 1 < shape.size(); i++) M *= shape[i];
    for (const Tensor* t : {&codes, &exps})
        if (t->device() != codes.device() || t->scalar_type() != at::kByte || !t->is_contiguous() || t->dim() != 2 || t->size(0) != M || t->size(1) != (t == &codes ? 32 * kb : kb))
            fail(cat("checkpoint_decode: codes and exps must be contiguous uint8 [", M, ", ", 32 * kb, "] and [", M, ", ", kb, "], got ", codes.sizes(), " and ", exps.sizes()));
    c10::DeviceGuard guard(codes.device());
    Tensor out = at::empty(shape, codes.options().dtype(dtype));
    check(f_decode((const unsigned char*)ptr(codes), (const unsigned char*)ptr(exps), M, (int)K, dtype_of(out, "out"), ptr(out), stream_of(codes)), "nl_mx8_decode");
    return out;
}

Tensor emb_forward(const Tensor& table, const Tensor& ids, const Tensor& w, double scale)
{
    const int64_t M = ids.size(0), D = table.size(1);
    c10::DeviceGuard guard(table.device());
    Tensor y = at::empty({M, D}, table.options());
    if (D > INT32_MAX || ids.size(1) > INT32_MAX) fail("nl_embedding_forward failed: invalid argument");
    check(f_emb_forward(ptr(table), table.size(0), (int)D, dtype_of(table, "table"), ptr(ids), ids.scalar_type() == at::kLong, (const float*)ptr(w), M, (int)ids.size(1), (float)scale, ptr(y),
                        stream_of(table)), "nl_embedding_forward");
    return y;
}

struct EmbeddingFn : torch::autograd::Function<EmbeddingFn> {
    static Tensor forward(torch::autograd::AutogradContext* ctx, const Tensor& table, const Tensor& ids, const OptTensor& w, double scale)
    {
        const bool gt = table.requires_grad(), gw = w && w->requires_grad();
        // g_table holds the weights, g_weights the table: what is not saved may be written before the backward pass
        ctx->save_for_backward({gw ? table : Tensor(), ids, gt && w ? *w : Tensor()});
        ctx->saved_data["scale"] = scale;
        ctx->saved_data["c"] = std::vector<int64_t>{gt, gw, table.size(0), table.size(1)};
        return emb_forward(table, ids, w ? *w : Tensor(), scale);
    }
    static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list grads)
    {
        no_capture("embedding_lookup");
        const auto saved = ctx->get_saved_variables();
        const auto c = ctx->saved_data["c"].toIntVector();
        const Tensor &table = saved[0], &ids = saved[1], &w = saved[2];
        torch::autograd::variable_list out(4);
        if (!grads[0].defined()) return out;
        const Tensor g = grads[0].contiguous();
        c10::DeviceGuard guard(g.device());
        const int64_t V = c[2], D = c[3];
        if (c[0] && ctx->needs_input_grad(0)) out[0] = at::empty({V, D}, g.options());
        if (c[1] && ctx->needs_input_grad(2)) out[2] = at::empty(ids.sizes(), g.options().dtype(at::kFloat));
        if (out[0].defined() || out[2].defined()) {
            const Tensor ws = workspace(out[0].defined() ? f_emb_workspace(V, (int)D, ids.size(0), (int)ids.size(1)) : 0, g, "nl_embedding_backward");
            check(f_emb_backward(ptr(table), V, (int)D, dtype_of(g, "g"), ptr(ids), ids.scalar_type() == at::kLong, (const float*)ptr(w), ids.size(0), (int)ids.size(1),
                                 (float)ctx->saved_data["scale"].toDouble(), ptr(g), ptr(out[0]), (float*)ptr(out[2]), ptr(ws), ws.defined() ? ws.numel() : 0, stream_of(g)), "nl_embedding_backward");
        }
        once_differentiable(out[0], grads[0].requires_grad() || c[1]);        // sums of w g
        once_differentiable(out[2], grads[0].requires_grad() || c[0]);        // <g, table>
        return out;
    }
};

Tensor embedding_lookup(const Tensor& table, const Tensor& ids, double scale, const OptTensor& weights)
{
    no_tangent("embedding_lookup", {&table, opt(weights)});
    on_gpu(table, "embedding_lookup");
    if (table.dim() != 2) throw py::value_error(cat("embedding_lookup: table ", table.sizes(), " must be [V, D]"));
    if (weights && (weights->sizes() != ids.sizes() || ids.dim() < 1 || ids.size(-1) < 1))
        throw py::value_error(cat("embedding_lookup: weights ", weights->sizes(), " must have the shape of ids ", ids.sizes(), ", [..., bag]"));
    dtype_of(table, "table");
    if (ids.device() != table.device() || (ids.scalar_type() != at::kInt && ids.scalar_type() != at::kLong))
        fail(cat("embedding_lookup: ids must be int32 or int64 on ", table.device(), ", got ", ids.scalar_type(), " on ", ids.device()));
    if (weights && (weights->device() != table.device() || weights->scalar_type() != at::kFloat))
        fail(cat("embedding_lookup: weights must be float32 on ", table.device(), ", got ", weights->scalar_type(), " on ", weights->device()));
    auto shape = ids.sizes().vec();
    const int64_t bag = weights ? shape.back() : 1;
    if (weights) shape.pop_back();
    const Tensor t = table.contiguous(), i2 = ids.reshape({ids.numel() / bag, bag}).contiguous();
    OptTensor w;
    if (weights) w = weights->reshape({ids.numel() / bag, bag}).contiguous();
    const Tensor y = at::GradMode::is_enabled() && (t.requires_grad() || (w && w->requires_grad())) ? EmbeddingFn::apply(t, i2, w, scale) : emb_forward(t, i2, w ? *w : Tensor(), scale);
    if (shape.size() == 1) return y;
    shape.push_back(table.size(1));
    return y.view(shape);
}

template <class F> void set(F& f, const py::dict& d, const char* name) { f = reinterpret_cast<F>(d[name].cast<uintptr_t>()); }

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m)
{
    m.def("bind", [](py::object cls, py::dict d) {
        error_class() = cls;
        set(f_forward, d, "nl_linear_forward"); set(f_backward, d, "nl_linear_backward"); set(f_workspace, d, "nl_linear_workspace");
        set(f_encode, d, "nl_mx8_encode"); set(f_decode, d, "nl_mx8_decode");
        set(f_emb_forward, d, "nl_embedding_forward"); set(f_emb_backward, d, "nl_embedding_backward"); set(f_emb_workspace, d, "nl_embedding_workspace");
    });
    py::register_exception_translator([](std::exception_ptr p) {
        try {
            if (p) std::rethrow_exception(p);
        } catch (const NlError& e) {
            PyErr_SetString(error_class().ptr() ? error_class().ptr() : PyExc_RuntimeError, e.what());
        }
    });
    m.def("linear_act", &linear_act);
    m.def("checkpoint_encode", &checkpoint_encode);
    m.def("checkpoint_decode", &checkpoint_decode);
    m.def("embedding_lookup", &embedding_lookup);
}
