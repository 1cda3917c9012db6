// Short way from Python to the calls of the dense operators.  A one-token call is bound by the host: through ctypes and torch's Python it takes 13 us, of
// which the launch is 3; from here 4.4 (a projection) to 6.4 (a norm in 8 bits with its three outputs), calls in a row.  A training step of one
// 32 x 64 x 64 projection with silu takes 125 us with autograd functions in Python and 68 with the ones here (torch's own linear: 83, with silu 104).  Each function takes the plain case only (CUDA tensors of one device, the current one; contiguous;
// shapes and types that fit) and answers None to everything else, which dense.py then checks, refuses or lays out.  The kernels are the same
// entry points of libb200moe.so; their addresses are handed in once by dense.py.
#include <ATen/ATen.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <c10/core/GradMode.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/utils/pybind.h>

#include <map>
#include <optional>
#include <stdexcept>
#include <string>

namespace py = pybind11;
using at::Tensor;
using OptTensor = std::optional<Tensor>;

namespace {

int (*f_norm)(const void*, long long, const void*, long long, const void*, int, int, long long, int, float, void*, void*, void*, void*, void*) = nullptr;
int (*f_linear)(const void*, long long, const void*, long long, int, int, int, int, const void*, int, const void*, long long, void*, long long, float*, long long, void*) = nullptr;
int (*f_gated)(const void*, long long, const void*, long long, int, int, int, int, int, float, void*, long long, float*, long long, void*) = nullptr;
int (*f_q8)(const void*, const void*, const void*, const void*, int, int, int, int, const void*, int, const void*, long long, void*, long long, void*, size_t, void*) = nullptr;
size_t (*f_q8_ws)(int, int, int) = nullptr;
size_t (*f_norm_bwd_ws)(long long, int) = nullptr;
int (*f_norm_bwd)(const void*, long long, const void*, long long, const void*, int, int, long long, int, float, const void*, const void*, void*, void*, void*, size_t, void*) = nullptr;
size_t (*f_linear_bwd_ws)(int, int) = nullptr;
int (*f_linear_bwd)(const void*, long long, const float*, long long, int, int, int, int, void*, long long, void*, void*, size_t, void*) = nullptr;
int (*f_gated_bwd)(const void*, long long, const float*, long long, int, float, int, int, int, void*, long long, void*) = nullptr;
int (*f_align)(const void*, long long, void*, long long, const void*, long long, void*, long long, int, long long, void*) = nullptr;
int (*f_product)(const void*, long long, int, const void*, long long, int, int, int, int, int, void*, long long, void*) = nullptr;
const char* (*f_error)(int) = nullptr;

void bind(const std::map<std::string, uintptr_t>& a) {
    f_norm = reinterpret_cast<decltype(f_norm)>(a.at("b200_add_rms_norm"));
    f_linear = reinterpret_cast<decltype(f_linear)>(a.at("b200_linear_act"));
    f_gated = reinterpret_cast<decltype(f_gated)>(a.at("b200_gated_linear"));
    f_q8 = reinterpret_cast<decltype(f_q8)>(a.at("b200_linear_act_q8"));
    f_q8_ws = reinterpret_cast<decltype(f_q8_ws)>(a.at("b200_linear_act_q8_workspace_bytes"));
    f_norm_bwd_ws = reinterpret_cast<decltype(f_norm_bwd_ws)>(a.at("b200_add_rms_norm_bwd_workspace_bytes"));
    f_norm_bwd = reinterpret_cast<decltype(f_norm_bwd)>(a.at("b200_add_rms_norm_bwd"));
    f_linear_bwd_ws = reinterpret_cast<decltype(f_linear_bwd_ws)>(a.at("b200_linear_act_bwd_workspace_bytes"));
    f_linear_bwd = reinterpret_cast<decltype(f_linear_bwd)>(a.at("b200_linear_act_bwd"));
    f_gated_bwd = reinterpret_cast<decltype(f_gated_bwd)>(a.at("b200_gated_linear_bwd"));
    f_align = reinterpret_cast<decltype(f_align)>(a.at("b200_align_rows"));
    f_product = reinterpret_cast<decltype(f_product)>(a.at("b200_dense_product"));
    f_error = reinterpret_cast<decltype(f_error)>(a.at("b200_error_string"));
}

void check(int rc, const char* what) {
    if (rc) throw std::runtime_error(std::string(what) + " failed with CUDA error " + std::to_string(rc) + " (" + f_error(rc) + ")");
}

// contiguous, on the given device, of the given type
bool plain(const Tensor& t, int dev, at::ScalarType type) { return t.is_cuda() && t.get_device() == dev && t.scalar_type() == type && t.is_contiguous(); }
bool wants(const Tensor& t) { return t.requires_grad(); }
bool wants(const OptTensor& t) { return t && t->requires_grad(); }
template <typename... Ts>
bool wants_grad(const Ts&... ts) { return c10::GradMode::is_enabled() && (... || wants(ts)); }
// a forward-mode tangent: dense.py refuses the call
bool dual(const Tensor& t) { return t._fw_grad(0).defined(); }
bool dual(const OptTensor& t) { return t && t->_fw_grad(0).defined(); }
template <typename... Ts>
bool any_dual(const Ts&... ts) { return (... || dual(ts)); }
bool fits16(const Tensor& t) { return (reinterpret_cast<uintptr_t>(t.data_ptr()) & 15) == 0; }
void* ptr(const OptTensor& t) { return t ? t->data_ptr() : nullptr; }
void* stream(int dev) { return c10::cuda::getCurrentCUDAStream((c10::DeviceIndex)dev).stream(); }

// the device that a plain call runs on, or -1
int plain_device(const Tensor& x) {
    if (!x.is_cuda() || x.dim() < 1 || x.numel() == 0) return -1;
    const int dev = x.get_device();
    return dev == c10::cuda::current_device() ? dev : -1;
}
int half_type(const Tensor& x) { return x.scalar_type() == at::kBFloat16 ? 0 : x.scalar_type() == at::kHalf ? 1 : -1; }

// rows [.., K] against w [N, K]
bool product_fits(const Tensor& x, const Tensor& w, int dev) {
    if (w.dim() != 2 || half_type(x) < 0 || !plain(x, dev, x.scalar_type()) || !plain(w, dev, x.scalar_type())) return false;
    const int64_t K = w.size(1), rows = x.numel() / x.size(-1);
    return x.size(-1) == K && K > 0 && w.size(0) > 0 && rows <= (1 << 30) && w.size(0) <= (1 << 30) && K <= (1 << 30);
}
bool same_but_last(const Tensor& a, const Tensor& b, int64_t last) {
    if (a.dim() != b.dim() || a.size(-1) != last) return false;
    for (int64_t i = 0; i + 1 < a.dim(); ++i)
        if (a.size(i) != b.size(i)) return false;
    return true;
}
Tensor like_rows(const Tensor& x, int64_t width) {
    auto shape = x.sizes().vec();
    shape.back() = width;
    return at::empty(shape, x.options().requires_grad(false));
}

int64_t pitch(int64_t n) { return (n + 7) / 8 * 8; }

// x [.., K] and w [N, K] as the kernels fetch them: themselves, or one copy of both with rows that start on 16 bytes (x's rows, then w's)
struct Operands {
    Tensor copy;     // defined: holds both
    Tensor kx, kw;   // of a backward pass: keep the memory of x and w where the copy does not
    const void *x, *w;
    int64_t M, N, K, ld;
};
Operands operands(const Tensor& x, const Tensor& w) {
    Operands o{Tensor(), Tensor(), Tensor(), x.data_ptr(), w.data_ptr(), x.numel() / w.size(1), w.size(0), w.size(1), w.size(1)};
    if (o.K % 8 == 0 && fits16(x) && fits16(w)) return o;
    o.ld = pitch(o.K);
    o.copy = at::empty({o.M + o.N, o.ld}, x.options().requires_grad(false));
    char* p = static_cast<char*>(o.copy.data_ptr());
    check(f_align(o.x, o.K, p, o.M, o.w, o.K, p + 2 * o.M * o.ld, o.N, (int)o.K, o.ld, stream(x.get_device())), "b200_align_rows");
    o.x = p;
    o.w = p + 2 * o.M * o.ld;
    return o;
}
// what a backward pass keeps of them, and the way back
void keep(torch::autograd::AutogradContext* ctx, const Operands& o, const Tensor& x, const Tensor& w, const Tensor& z) {
    if (o.copy.defined()) ctx->save_for_backward({o.copy, Tensor(), z});
    else ctx->save_for_backward({x, w, z});
    ctx->saved_data["M"] = o.M;
    ctx->saved_data["N"] = o.N;
    ctx->saved_data["K"] = o.K;
}
// A saved tensor as the backward pass gets it.  A saved-tensor hook (save_on_cpu) may hand back other strides and another address than were saved: laid out
// again here; not other sizes, type or device.
Tensor restored(const Tensor& t, at::IntArrayRef sizes, at::ScalarType type, int dev) {
    if (!t.defined() || !t.is_cuda() || t.get_device() != dev || t.scalar_type() != type || !t.sizes().equals(sizes))
        throw std::runtime_error("a saved-tensor hook returned a tensor of other sizes, type or device than it was given");
    Tensor d = t.contiguous();
    return fits16(d) ? d : d.clone();
}
Operands kept(torch::autograd::AutogradContext* ctx, const std::vector<Tensor>& saved, at::ScalarType type, int dev) {
    Operands o{};
    o.M = ctx->saved_data["M"].toInt();
    o.N = ctx->saved_data["N"].toInt();
    o.K = ctx->saved_data["K"].toInt();
    if (saved[1].defined()) {
        o.ld = o.K;
        o.kx = restored(saved[0], ctx->saved_data["x"].toIntVector(), type, dev);
        o.kw = restored(saved[1], {o.N, o.K}, type, dev);
        o.x = o.kx.data_ptr();
        o.w = o.kw.data_ptr();
    } else {
        o.ld = pitch(o.K);
        o.copy = restored(saved[0], {o.M + o.N, o.ld}, type, dev);
        o.x = o.copy.data_ptr();
        o.w = static_cast<const char*>(o.x) + 2 * o.M * o.ld;
    }
    return o;
}

// ------------------------------------------------------------------ launches
void launch_norm(const Tensor& x, const OptTensor& res, const OptTensor& w, double eps, const Tensor& y, const Tensor& s, const Tensor& q8, const Tensor& sf) {
    const int dev = x.get_device();
    const int64_t D = x.size(-1);
    auto p = [](const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; };
    check(f_norm(x.data_ptr(), D, ptr(res), D, ptr(w), w && w->scalar_type() == at::kFloat, x.scalar_type() == at::kFloat ? 2 : half_type(x), x.numel() / D, (int)D, (float)eps, p(y),
                 p(s), p(q8), p(sf), stream(dev)),
          "b200_add_rms_norm");
}
void launch_linear(const Operands& o, const Tensor& like, const OptTensor& bias, int act, const OptTensor& res, const Tensor& out, float* z) {
    check(f_linear(o.x, o.ld, o.w, o.ld, half_type(like), (int)o.M, (int)o.N, (int)o.K, ptr(bias), act, ptr(res), o.N, out.data_ptr(), o.N, z, pitch(o.N), stream(like.get_device())),
          "b200_linear_act");
}
void launch_gated(const Operands& o, const Tensor& like, int act, double limit, const Tensor& out, float* gu) {
    check(f_gated(o.x, o.ld, o.w, o.ld, half_type(like), (int)o.M, (int)(o.N / 2), (int)o.K, act, (float)limit, out.data_ptr(), o.N / 2, gu, pitch(o.N), stream(like.get_device())),
          "b200_gated_linear");
}
// [M, N] = A B^T over K: element (i, k) of A at a[i * a_ld + k] or, with a_mn, a[k * a_ld + i]; of B at b[k * b_ld + i]
Tensor product(const Tensor& like, const void* a, int64_t a_ld, int a_mn, const void* b, int64_t b_ld, int64_t M, int64_t N, int64_t K, at::IntArrayRef shape) {
    Tensor out = at::empty(shape, like.options().requires_grad(false));
    check(f_product(a, a_ld, a_mn, b, b_ld, 1, half_type(like), (int)M, (int)N, (int)K, out.data_ptr(), N, stream(like.get_device())), "b200_dense_product");
    return out;
}

// ------------------------------------------------------------------ gradients
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

// The gradients of a backward pass that records its graph (create_graph).  They cannot be differentiated again; a node that raises when that is tried stands
// behind each, with edges to what the gradient depends on: `inputs[i]`, positions among this function's tensor inputs, and the incoming gradients.  So it is
// met on the way to any of these, whichever leaves are asked for and whether the incoming gradients are constants or not; a gradient that depends on
// nothing that wants one stays a plain tensor.
using Inputs = std::vector<int>;
std::vector<Tensor> once(std::vector<Tensor> out, const std::vector<Inputs>& inputs, const std::vector<Tensor>& incoming) {
    namespace ag = torch::autograd;
    if (!c10::GradMode::is_enabled()) return out;
    const auto self = ag::get_current_node();
    for (size_t i = 0; i < out.size(); ++i) {
        if (!out[i].defined() || !out[i].is_floating_point()) continue;
        ag::edge_list edges;
        for (int j : inputs[i])
            if (j < (int)self->num_outputs() && self->next_edge(j).is_valid()) edges.push_back(self->next_edge(j));
        for (const Tensor& g : incoming)
            if (g.defined() && g.requires_grad()) edges.push_back(ag::impl::gradient_edge(g));
        if (edges.empty()) continue;
        out[i] = out[i].detach();
        ag::set_history(out[i], std::make_shared<ag::Error>("trying to differentiate twice a function that was marked with @once_differentiable", std::move(edges)));
    }
    return out;
}
// incoming gradients as dense rows the kernels can fetch
Tensor dense(const Tensor& g) {
    Tensor d = g.contiguous();
    return fits16(d) ? d : d.clone();
}

struct NormFn : torch::autograd::Function<NormFn> {
    static variable_list forward(AutogradContext* ctx, const Tensor& x, const OptTensor& res, const OptTensor& w, double eps) {
        const auto opt = x.options().requires_grad(false);
        Tensor y = at::empty(x.sizes(), opt), s;
        if (res) s = at::empty(x.sizes(), opt);
        launch_norm(x, res, w, eps, y, s, Tensor(), Tensor());
        ctx->set_materialize_grads(false);
        ctx->save_for_backward({x, res ? *res : Tensor(), w ? *w : Tensor()});
        ctx->saved_data["eps"] = eps;
        ctx->saved_data["w_f32"] = w && w->scalar_type() == at::kFloat;
        return res ? variable_list{y, s} : variable_list{y};
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        const auto saved = ctx->get_saved_variables();
        Tensor x = saved[0], r = saved[1], w = saved[2];
        const bool need_x = ctx->needs_input_grad(0), need_r = r.defined() && ctx->needs_input_grad(1), need_w = w.defined() && ctx->needs_input_grad(r.defined() ? 2 : 1);
        const Tensor gs_in = grads.size() > 1 ? grads[1] : Tensor();
        if (!grads[0].defined())  // the normed output was not used
            return {need_x ? gs_in : Tensor(), need_r ? gs_in : Tensor(), need_w ? at::zeros(w.sizes(), w.options().requires_grad(false)) : Tensor(), Tensor()};
        const Tensor gy = dense(grads[0]), gs = gs_in.defined() ? dense(gs_in) : gs_in;
        const int dev = gy.get_device();
        x = restored(x, gy.sizes(), gy.scalar_type(), dev);
        if (r.defined()) r = restored(r, gy.sizes(), gy.scalar_type(), dev);
        if (w.defined()) w = restored(w, {gy.size(-1)}, ctx->saved_data["w_f32"].toBool() ? at::kFloat : gy.scalar_type(), dev);
        const int64_t D = x.size(-1), rows = x.numel() / D;
        const size_t nb = need_w ? f_norm_bwd_ws(rows, (int)D) : 0;
        Tensor ds = at::empty(x.sizes(), x.options().requires_grad(false)), dw, ws;
        if (need_w) {
            dw = at::empty(w.sizes(), w.options().requires_grad(false));
            ws = at::empty({(int64_t)nb}, x.options().dtype(at::kByte).requires_grad(false));
        }
        check(f_norm_bwd(x.data_ptr(), D, r.defined() ? r.data_ptr() : nullptr, D, w.defined() ? w.data_ptr() : nullptr, w.defined() && w.scalar_type() == at::kFloat,
                         x.scalar_type() == at::kFloat ? 2 : half_type(x), rows, (int)D, (float)ctx->saved_data["eps"].toDouble(), gy.data_ptr(), gs.defined() ? gs.data_ptr() : nullptr,
                         ds.data_ptr(), need_w ? dw.data_ptr() : nullptr, need_w ? ws.data_ptr() : nullptr, nb, stream(x.get_device())),
              "b200_add_rms_norm_bwd");
        const bool has_r = r.defined(), has_w = w.defined();
        const Inputs stream_in = has_r ? Inputs{0, 1} : Inputs{0};
        Inputs all = stream_in;
        if (has_w) all.push_back(has_r ? 2 : 1);
        return once({need_x ? ds : Tensor(), need_r ? ds : Tensor(), dw, Tensor()}, {all, all, stream_in, {}}, grads);
    }
};

struct LinearFn : torch::autograd::Function<LinearFn> {
    static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& w, const OptTensor& bias, const OptTensor& res, int64_t act) {
        const Operands o = operands(x, w);
        Tensor out = like_rows(x, o.N), z;
        if (act) z = at::empty({o.M, pitch(o.N)}, x.options().dtype(at::kFloat).requires_grad(false));
        launch_linear(o, x, bias, (int)act, res, out, act ? z.data_ptr<float>() : nullptr);
        keep(ctx, o, x, w, z);
        ctx->saved_data["x"] = x.sizes().vec();
        ctx->saved_data["act"] = act;
        ctx->saved_data["bias"] = bias.has_value();
        ctx->saved_data["res"] = res.has_value();
        return out;
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        const auto saved = ctx->get_saved_variables();
        const Tensor gy = dense(grads[0]), &like = gy;
        const int act = (int)ctx->saved_data["act"].toInt(), dev = gy.get_device();
        const Operands o = kept(ctx, saved, gy.scalar_type(), dev);
        const Tensor z = act ? restored(saved[2], {o.M, pitch(o.N)}, at::kFloat, dev) : Tensor();
        const bool has_b = ctx->saved_data["bias"].toBool(), has_r = ctx->saved_data["res"].toBool();
        const bool need_x = ctx->needs_input_grad(0), need_w = ctx->needs_input_grad(1), need_b = has_b && ctx->needs_input_grad(2),
                   need_r = has_r && ctx->needs_input_grad(has_b ? 3 : 2);
        const auto opt = like.options().requires_grad(false);
        const bool own_dz = (act || o.N % 8) && (need_x || need_w);
        const int64_t dz_ld = own_dz ? pitch(o.N) : o.N;
        Tensor dz = own_dz ? at::empty({o.M, dz_ld}, opt) : gy, db, ws, dx, dw;
        if (need_b) db = at::empty({o.N}, opt);
        if (own_dz || need_b) {
            const size_t nb = need_b ? f_linear_bwd_ws((int)o.M, (int)o.N) : 0;
            if (nb) ws = at::empty({(int64_t)nb}, opt.dtype(at::kByte));
            check(f_linear_bwd(gy.data_ptr(), o.N, act ? z.data_ptr<float>() : nullptr, pitch(o.N), act, half_type(like), (int)o.M, (int)o.N, own_dz ? dz.data_ptr() : nullptr, dz_ld,
                               need_b ? db.data_ptr() : nullptr, nb ? ws.data_ptr() : nullptr, nb, stream(dev)),
                  "b200_linear_act_bwd");
        }
        if (need_x) dx = product(like, dz.data_ptr(), dz_ld, 0, o.w, o.ld, o.M, o.K, o.N, ctx->saved_data["x"].toIntVector());
        if (need_w) dw = product(like, dz.data_ptr(), dz_ld, 1, o.x, o.ld, o.N, o.K, o.M, {o.N, o.K});
        const bool curved = act > 1;  // without an activation, and with relu but for its corner, the slope does not depend on z
        const Inputs of_z = curved ? (has_b ? Inputs{0, 1, 2} : Inputs{0, 1}) : Inputs{};
        variable_list out = once({dx, dw, db}, {curved ? of_z : Inputs{1}, curved ? of_z : Inputs{0}, of_z}, grads);
        return {out[0], out[1], out[2], need_r ? grads[0] : Tensor(), Tensor()};
    }
};

struct GatedFn : torch::autograd::Function<GatedFn> {
    static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& w13, int64_t act, double limit) {
        const Operands o = operands(x, w13);
        Tensor out = like_rows(x, o.N / 2), gu = at::empty({o.M, pitch(o.N)}, x.options().dtype(at::kFloat).requires_grad(false));
        launch_gated(o, x, (int)act, limit, out, gu.data_ptr<float>());
        keep(ctx, o, x, w13, gu);
        ctx->saved_data["x"] = x.sizes().vec();
        ctx->saved_data["act"] = act;
        ctx->saved_data["limit"] = limit;
        return out;
    }
    static variable_list backward(AutogradContext* ctx, variable_list grads) {
        const auto saved = ctx->get_saved_variables();
        const Tensor gy = dense(grads[0]), &like = gy;
        const int dev = gy.get_device();
        const Operands o = kept(ctx, saved, gy.scalar_type(), dev);
        const int64_t ld = pitch(o.N);
        const Tensor gu = restored(saved[2], {o.M, ld}, at::kFloat, dev);
        Tensor dgu = at::empty({o.M, ld}, like.options().requires_grad(false)), dx, dw;
        check(f_gated_bwd(gy.data_ptr(), o.N / 2, gu.data_ptr<float>(), ld, (int)ctx->saved_data["act"].toInt(), (float)ctx->saved_data["limit"].toDouble(), half_type(like), (int)o.M,
                          (int)(o.N / 2), dgu.data_ptr(), ld, stream(dev)),
              "b200_gated_linear_bwd");
        if (ctx->needs_input_grad(0)) dx = product(like, dgu.data_ptr(), ld, 0, o.w, o.ld, o.M, o.K, o.N, ctx->saved_data["x"].toIntVector());
        if (ctx->needs_input_grad(1)) dw = product(like, dgu.data_ptr(), ld, 1, o.x, o.ld, o.N, o.K, o.M, {o.N, o.K});
        return once({dx, dw, Tensor(), Tensor()}, {{0, 1}, {0, 1}, {}, {}}, grads);
    }
};

// ------------------------------------------------------------------ calls
py::object norm(const Tensor& x, const OptTensor& res, const OptTensor& w, double eps, bool quant, bool want_y) {
    const int dev = plain_device(x);
    if (dev < 0) return py::none();
    const auto type = x.scalar_type();
    const int64_t D = x.size(-1);
    if ((type != at::kFloat && half_type(x) < 0) || D > 16384 || !(eps >= 0) || !plain(x, dev, type) || any_dual(x, res, w)) return py::none();
    if (res && (!plain(*res, dev, type) || !res->sizes().equals(x.sizes()))) return py::none();
    if (w && (w->dim() != 1 || w->size(0) != D || !(plain(*w, dev, type) || plain(*w, dev, at::kFloat)))) return py::none();
    const auto opt = x.options().requires_grad(false);
    if (wants_grad(x, res, w)) {
        if (quant) return py::none();
        variable_list out = NormFn::apply(x, res, w, eps);
        return py::make_tuple(out[0], res ? out[1] : x);
    }
    const int64_t rows = x.numel() / D;
    Tensor y, s, q8, sf;
    if (want_y) y = at::empty(x.sizes(), opt);
    if (res) s = at::empty(x.sizes(), opt);
    if (quant) {
        if (D % 32) return py::none();
        q8 = at::empty({rows, D}, opt.dtype(at::kByte));
        sf = at::empty({rows, D / 32}, opt.dtype(at::kByte));
    }
    launch_norm(x, res, w, eps, y, s, q8, sf);
    if (!res) s = x;
    if (!quant) return py::make_tuple(y, s);
    return want_y ? py::make_tuple(q8, sf, s, y) : py::make_tuple(q8, sf, s);
}

py::object linear(const Tensor& x, const Tensor& w, const OptTensor& bias, int act, const OptTensor& res) {
    const int dev = plain_device(x);
    if (dev < 0 || act < 0 || !product_fits(x, w, dev) || any_dual(x, w, bias, res)) return py::none();
    const auto type = x.scalar_type();
    const int64_t N = w.size(0);
    if (bias && (bias->dim() != 1 || bias->size(0) != N || !plain(*bias, dev, type))) return py::none();
    if (res && (!plain(*res, dev, type) || !same_but_last(*res, x, N))) return py::none();
    if (wants_grad(x, w, bias, res)) return py::cast(Tensor(LinearFn::apply(x, w, bias, res, (int64_t)act)));
    Tensor out = like_rows(x, N);
    launch_linear(operands(x, w), x, bias, act, res, out, nullptr);
    return py::cast(out);
}

py::object gated(const Tensor& x, const Tensor& w13, int act, double limit) {
    const int dev = plain_device(x);
    if (dev < 0 || act < 0 || !(limit >= 0) || !product_fits(x, w13, dev) || w13.size(0) % 2 || any_dual(x, w13)) return py::none();
    if (wants_grad(x, w13)) return py::cast(Tensor(GatedFn::apply(x, w13, (int64_t)act, limit)));
    Tensor out = like_rows(x, w13.size(0) / 2);
    launch_gated(operands(x, w13), x, act, limit, out, nullptr);
    return py::cast(out);
}

py::object q8(const Tensor& x8, const Tensor& xsf, const Tensor& w8, const Tensor& s8, const OptTensor& bias, int act, const OptTensor& res) {
    const int dev = plain_device(x8);
    if (dev < 0 || act < 0 || x8.dim() != 2 || xsf.dim() != 2 || w8.dim() != 2 || s8.dim() != 2) return py::none();
    for (const Tensor* t : {&x8, &xsf, &w8, &s8})
        if (!plain(*t, dev, at::kByte)) return py::none();
    const int64_t M = x8.size(0), K = x8.size(1), N = w8.size(0);
    if (K % 128 || w8.size(1) != K || N < 1 || xsf.size(0) != M || xsf.size(1) != K / 32 || s8.size(0) != (N + 31) / 32 || s8.size(1) < K / 32) return py::none();
    if (!fits16(x8) || !fits16(w8) || (reinterpret_cast<uintptr_t>(xsf.data_ptr()) & 3) || M > (1 << 30) || N > (1 << 30) || K > (1 << 30) || s8.size(1) > INT32_MAX) return py::none();
    if (bias && (bias->dim() != 1 || bias->size(0) != N || !plain(*bias, dev, at::kBFloat16))) return py::none();
    if (wants_grad(bias, res) || any_dual(bias, res)) return py::none();
    if (res && (!plain(*res, dev, at::kBFloat16) || res->dim() != 2 || res->size(0) != M || res->size(1) != N)) return py::none();
    Tensor out = at::empty({M, N}, x8.options().dtype(at::kBFloat16)), ws;
    const size_t nb = f_q8_ws((int)M, (int)N, (int)K);
    if (nb) ws = at::empty({(int64_t)nb}, x8.options());
    check(f_q8(x8.data_ptr(), xsf.data_ptr(), w8.data_ptr(), s8.data_ptr(), (int)s8.size(1), (int)M, (int)N, (int)K, ptr(bias), act, ptr(res), N, out.data_ptr(), N,
               nb ? ws.data_ptr() : nullptr, nb, stream(dev)),
          "b200_linear_act_q8");
    return py::cast(out);
}

}  // namespace

PYBIND11_MODULE(_fastcall, m) {
    m.def("bind", &bind);
    m.def("norm", &norm);
    m.def("linear", &linear);
    m.def("gated", &gated);
    m.def("q8", &q8);
    m.def("tangents", [](const std::vector<OptTensor>& ts) {
        for (const OptTensor& t : ts)
            if (dual(t)) return true;
        return false;
    });
    m.def("once", [](const std::vector<OptTensor>& out, const std::vector<Inputs>& inputs, const std::vector<OptTensor>& incoming) {
        auto defined = [](const std::vector<OptTensor>& v) {
            std::vector<Tensor> t;
            for (const OptTensor& o : v) t.push_back(o ? *o : Tensor());
            return t;
        };
        std::vector<OptTensor> back;
        for (const Tensor& t : once(defined(out), inputs, defined(incoming))) back.push_back(t.defined() ? OptTensor(t) : std::nullopt);
        return back;
    });
}
