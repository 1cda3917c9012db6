// Short way from Python to the forward calls of the dense operators.  A one-token call is bound by the host: through ctypes and torch's Python it takes
// 10 to 14 us, of which the launch is 3; from here 5 to 8.  Each function takes the plain case only (CUDA tensors of one device, the current one;
// contiguous, fetchable rows; no gradient wanted; shapes and types that fit) and answers None to everything else, which dense.py then checks, refuses or
// lays out.  The kernels are the same entry points of libb200moe.so; their addresses are handed in once by dense.py.
#include <ATen/ATen.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <c10/core/GradMode.h>
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
const char* (*f_error)(int) = nullptr;

void bind(const std::map<std::string, uintptr_t>& a) {
    f_norm = reinterpret_cast<decltype(f_norm)>(a.at("b200_add_rms_norm"));
    f_linear = reinterpret_cast<decltype(f_linear)>(a.at("b200_linear_act"));
    f_gated = reinterpret_cast<decltype(f_gated)>(a.at("b200_gated_linear"));
    f_q8 = reinterpret_cast<decltype(f_q8)>(a.at("b200_linear_act_q8"));
    f_q8_ws = reinterpret_cast<decltype(f_q8_ws)>(a.at("b200_linear_act_q8_workspace_bytes"));
    f_error = reinterpret_cast<decltype(f_error)>(a.at("b200_error_string"));
}

void check(int rc, const char* what) {
    if (rc) throw std::runtime_error(std::string(what) + " failed with CUDA error " + std::to_string(rc) + " (" + f_error(rc) + ")");
}

// contiguous, on the given device, of the given type, no gradient wanted
bool plain(const Tensor& t, int dev, at::ScalarType type) {
    return t.is_cuda() && t.get_device() == dev && t.scalar_type() == type && t.is_contiguous() && !(t.requires_grad() && c10::GradMode::is_enabled());
}
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
    return x.size(-1) == K && K % 8 == 0 && w.size(0) > 0 && fits16(x) && fits16(w) && rows <= INT32_MAX && w.size(0) <= (1 << 30) && K <= (1 << 30);
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

py::object norm(const Tensor& x, const OptTensor& res, const OptTensor& w, double eps, bool quant, bool want_y) {
    const int dev = plain_device(x);
    if (dev < 0) return py::none();
    const auto type = x.scalar_type();
    const int64_t D = x.size(-1);
    const int code = type == at::kFloat ? 2 : half_type(x);
    if (code < 0 || D > 16384 || !(eps >= 0) || !plain(x, dev, type)) return py::none();
    if (res && (!plain(*res, dev, type) || !res->sizes().equals(x.sizes()))) return py::none();
    if (w && (w->dim() != 1 || w->size(0) != D || !(plain(*w, dev, type) || plain(*w, dev, at::kFloat)))) return py::none();
    if (quant && D % 32) return py::none();
    const int64_t rows = x.numel() / D;
    Tensor y, s, q8, sf;
    const auto opt = x.options().requires_grad(false);
    if (want_y) y = at::empty(x.sizes(), opt);
    if (res) s = at::empty(x.sizes(), opt);
    if (quant) {
        q8 = at::empty({rows, D}, opt.dtype(at::kByte));
        sf = at::empty({rows, D / 32}, opt.dtype(at::kByte));
    }
    check(f_norm(x.data_ptr(), D, ptr(res), D, ptr(w), w && w->scalar_type() == at::kFloat, code, rows, (int)D, (float)eps, want_y ? y.data_ptr() : nullptr,
                 res ? s.data_ptr() : nullptr, quant ? q8.data_ptr() : nullptr, quant ? sf.data_ptr() : nullptr, stream(dev)),
          "b200_add_rms_norm");
    if (!res) s = x;
    if (!quant) return py::make_tuple(y, s);
    return want_y ? py::make_tuple(q8, sf, s, y) : py::make_tuple(q8, sf, s);
}

py::object linear(const Tensor& x, const Tensor& w, const OptTensor& bias, int act, const OptTensor& res) {
    const int dev = plain_device(x);
    if (dev < 0 || act < 0 || !product_fits(x, w, dev)) return py::none();
    const auto type = x.scalar_type();
    const int64_t N = w.size(0), K = w.size(1);
    if (bias && (bias->dim() != 1 || bias->size(0) != N || !plain(*bias, dev, type))) return py::none();
    if (res && (!plain(*res, dev, type) || !same_but_last(*res, x, N))) return py::none();
    Tensor out = like_rows(x, N);
    check(f_linear(x.data_ptr(), K, w.data_ptr(), K, half_type(x), (int)(x.numel() / K), (int)N, (int)K, ptr(bias), act, ptr(res), N, out.data_ptr(), N, nullptr, 0, stream(dev)),
          "b200_linear_act");
    return py::cast(out);
}

py::object gated(const Tensor& x, const Tensor& w13, int act, double limit) {
    const int dev = plain_device(x);
    if (dev < 0 || act < 0 || !(limit >= 0) || !product_fits(x, w13, dev) || w13.size(0) % 2) return py::none();
    const int64_t inter = w13.size(0) / 2, K = w13.size(1);
    Tensor out = like_rows(x, inter);
    check(f_gated(x.data_ptr(), K, w13.data_ptr(), K, half_type(x), (int)(x.numel() / K), (int)inter, (int)K, act, (float)limit, out.data_ptr(), inter, nullptr, 0, stream(dev)),
          "b200_gated_linear");
    return py::cast(out);
}

py::object q8(const Tensor& x8, const Tensor& xsf, const Tensor& w8, const Tensor& s8, const OptTensor& bias, int act, const OptTensor& res) {
    const int dev = plain_device(x8);
    if (dev < 0 || act < 0 || x8.dim() != 2 || xsf.dim() != 2 || w8.dim() != 2 || s8.dim() != 2) return py::none();
    for (const Tensor* t : {&x8, &xsf, &w8, &s8})
        if (!plain(*t, dev, at::kByte)) return py::none();
    const int64_t M = x8.size(0), K = x8.size(1), N = w8.size(0);
    if (K % 128 || w8.size(1) != K || N < 1 || xsf.size(0) != M || xsf.size(1) != K / 32 || s8.size(0) != (N + 31) / 32 || s8.size(1) < K / 32) return py::none();
    if (!fits16(x8) || !fits16(w8) || (reinterpret_cast<uintptr_t>(xsf.data_ptr()) & 3) || M > INT32_MAX || N > (1 << 30) || K > (1 << 30) || s8.size(1) > INT32_MAX) return py::none();
    if (bias && (bias->dim() != 1 || bias->size(0) != N || !plain(*bias, dev, at::kBFloat16))) return py::none();
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
}
