// The residual path of an mHC layer in mhc_proj.torch: layer_norm, dropout,
// stream_norm_n4 and stream_mix_n4 with their backward functions (no reference
// counterparts).  The conventions are the other functions': dict results,
// RuntimeError for shapes, ValueError for numbers out of range, the current
// stream of the first tensor's device.  fp32/bf16/fp16 CUDA tensors whose rows
// are contiguous are read in place at any stride (other layouts are copied in
// their own type); tensors of other types or devices are converted to fp32 on
// that device and the results converted back.  Tensors beside the first one
// move to its device.
#include <optional>
#include <utility>

#include <ATen/cuda/EmptyTensor.h>

#include "torch_binding.h"

namespace mhcp_torch {

namespace {

using Opt = std::optional<torch::Tensor>;

[[noreturn]] void bad_shape(const char* name, const char* size)
{
    throw std::runtime_error(std::string(name) + " must be a tensor of size " + size);
}

void check_rows(const torch::Tensor& x, const char* name)
{
    if (x.dim() != 2 || x.size(1) < 1) bad_shape(name, "B x C");
}

void check_streams(const torch::Tensor& x, const char* name)
{
    if (x.dim() != 3 || x.size(1) != 4 || x.size(2) < 1) bad_shape(name, "B x 4 x C");
}

void check_like(const torch::Tensor& x, torch::IntArrayRef sizes, const char* name, const char* size)
{
    if (x.sizes() != sizes) bad_shape(name, size);
}

void check_real(const torch::Tensor& x, const char* name)
{
    if (!x.is_floating_point()) throw std::runtime_error(std::string(name) + " must be a floating-point tensor");
}

void check_p(double p)
{
    if (!(p >= 0.0 && p <= 1.0)) throw std::invalid_argument("p must be between 0 and 1");
}

// The type and device an operator computes on: the tensors' own type when
// all of them are `x`'s and the kernels take it, else fp32.
torch::TensorOptions compute_options(const torch::Tensor& x, std::initializer_list<const torch::Tensor*> others = {})
{
    auto opts = target_options(x);
    if (!x.is_cuda() || dtype_code(x) < 0) return opts;
    for (const torch::Tensor* o : others)
        if (o->scalar_type() != x.scalar_type()) return opts;
    return opts.dtype(x.scalar_type());
}

// x of opts' device and type.  A call on a few tokens takes little longer than
// its trips through the dispatcher, so nothing is asked of it that is so already.
torch::Tensor on(const torch::Tensor& x, const torch::TensorOptions& opts)
{
    return x.device() == opts.device() && x.scalar_type() == opts.dtype() ? x : x.to(opts);
}

torch::Tensor whole(const torch::Tensor& x) { return x.is_contiguous() ? x : x.contiguous(); }

// An uninitialised contiguous tensor of opts' device.
torch::Tensor fresh(at::IntArrayRef sizes, const torch::TensorOptions& opts, torch::ScalarType type)
{
    return at::detail::empty_cuda(sizes, type, opts.device(), std::nullopt);
}

torch::Tensor fresh(at::IntArrayRef sizes, const torch::TensorOptions& opts)
{
    return fresh(sizes, opts, c10::typeMetaToScalarType(opts.dtype()));
}

// The rows' mean and rstd, from one allocation (layer_norm of 8 rows takes 5.4 us
// of the caller's time with it, 6.0 with two).
std::pair<torch::Tensor, torch::Tensor> fresh_stats(int64_t n, const torch::TensorOptions& opts)
{
    const torch::Tensor mean = fresh({2 * n}, opts, torch::kFloat32);
    torch::Tensor rstd = at::detail::make_tensor<c10::TensorImpl>(c10::Storage(mean.storage()), mean.key_set(), mean.dtype());
    rstd.unsafeGetTensorImpl()->set_storage_offset(n);
    rstd.unsafeGetTensorImpl()->set_sizes_contiguous({n});
    mean.unsafeGetTensorImpl()->set_sizes_contiguous({n});
    return {mean, rstd};
}

// A result in the type and on the device that the caller's tensor has.
torch::Tensor as(const torch::Tensor& x, const torch::TensorOptions& src) { return on(x, src); }

// x on opts with its last dimension contiguous (a copy only where needed).
torch::Tensor rows_on(const torch::Tensor& x, const torch::TensorOptions& opts)
{
    torch::Tensor t = on(x, opts);
    return t.size(-1) == 1 || t.stride(-1) == 1 ? t : t.contiguous();
}

// A small operand (coefficients, a weight): contiguous on opts' device, in its
// own type when the kernels take it, else fp32.
torch::Tensor small_on(const torch::Tensor& x, const torch::TensorOptions& opts)
{
    return whole(on(x, opts.dtype(dtype_code(x) >= 0 ? x.scalar_type() : torch::kFloat32)));
}

void check_affine(const Opt& weight, const Opt& bias, int64_t width)
{
    if (weight) {
        check_like(*weight, {width}, "weight", "C");
        check_real(*weight, "weight");
    }
    if (bias) {
        check_like(*bias, {width}, "bias", "C");
        check_real(*bias, "bias");
    }
}

struct Affine {
    torch::Tensor w, b;
    int dtype = MHC_DTYPE_F32;

    Affine(const Opt& weight, const Opt& bias, const torch::TensorOptions& opts)
    {
        if (weight) w = small_on(*weight, opts);
        if (bias) b = small_on(*bias, opts);
        if (weight && bias && w.scalar_type() != b.scalar_type()) {
            w = w.to(torch::kFloat32);
            b = b.to(torch::kFloat32);
        }
        if (weight || bias) dtype = dtype_code(weight ? w : b);
    }

    const void* weight() const { return w.defined() ? w.data_ptr() : nullptr; }
    const void* bias() const { return b.defined() ? b.data_ptr() : nullptr; }
    // Somewhere to write the gradient of a given parameter, in the pair's type.
    torch::Tensor grad_of(const torch::Tensor& of) const { return of.defined() ? fresh(of.sizes(), of.options()) : torch::Tensor(); }
};

void* ptr(const torch::Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }

void check_eps(double eps)
{
    if (!(eps >= 0.0)) throw std::invalid_argument("eps must not be negative");
}

py::dict layer_norm(torch::Tensor x, const Opt& weight, const Opt& bias, double eps)
{
    check_rows(x, "x");
    check_real(x, "x");
    check_affine(weight, bias, x.size(1));
    check_eps(eps);
    const auto src = x.options();
    const auto opts = compute_options(x);
    const int64_t n = x.size(0), c = x.size(1);
    const Affine a(weight, bias, opts);
    x = rows_on(x, opts);
    const c10::cuda::CUDAGuard guard(x.device());
    torch::Tensor y = fresh({n, c}, opts);
    const auto [mean, rstd] = fresh_stats(n, opts);
    check_status(mhc_layer_norm(x.data_ptr(), x.stride(0), dtype_code(x), a.weight(), a.bias(), a.dtype, y.data_ptr(),
                                mean.data_ptr<float>(), rstd.data_ptr<float>(), static_cast<float>(eps), n, c,
                                current_stream()),
                 "layer_norm");
    py::dict out;
    out["y"] = as(y, src);
    out["mean"] = mean;
    out["rstd"] = rstd;
    return out;
}

// The statistics of a forward pass.
void check_stats(const torch::Tensor& mean, const torch::Tensor& rstd, int64_t n)
{
    check_like(mean, {n}, "mean", "B");
    check_like(rstd, {n}, "rstd", "B");
}

torch::Tensor stats_on(const torch::Tensor& s, const torch::TensorOptions& opts)
{
    return whole(on(s, opts.dtype(torch::kFloat32)));
}

void put_affine_grads(py::dict& out, const torch::Tensor& dw, const torch::Tensor& db, const Opt& weight,
                      const Opt& bias)
{
    if (weight) out["d_weight"] = as(dw, weight->options());
    if (bias) out["d_bias"] = as(db, bias->options());
}

py::dict layer_norm_backward(torch::Tensor G, torch::Tensor x, torch::Tensor mean, torch::Tensor rstd,
                             const Opt& weight, const Opt& bias)
{
    check_rows(x, "x");
    check_real(x, "x");
    check_like(G, x.sizes(), "G", "B x C");
    check_real(G, "G");
    check_stats(mean, rstd, x.size(0));
    check_affine(weight, bias, x.size(1));
    const auto src = x.options();
    const auto opts = compute_options(x, {&G});
    const int64_t n = x.size(0), c = x.size(1);
    const Affine a(weight, bias, opts);
    mean = stats_on(mean, opts);
    rstd = stats_on(rstd, opts);
    x = rows_on(x, opts);
    G = rows_on(G, opts);
    const c10::cuda::CUDAGuard guard(x.device());
    torch::Tensor dx = fresh({n, c}, opts);
    torch::Tensor dw = a.grad_of(a.w), db = a.grad_of(a.b), ws;
    int64_t bytes = 0;
    if (weight || bias) {
        check_status(mhc_layer_norm_backward_workspace(n, c, &bytes), "layer_norm_backward");
        ws = fresh({bytes}, opts, torch::kUInt8);
    }
    check_status(mhc_layer_norm_backward(G.data_ptr(), G.stride(0), x.data_ptr(), x.stride(0), dtype_code(x),
                                         mean.data_ptr<float>(), rstd.data_ptr<float>(), a.weight(), a.dtype,
                                         dx.data_ptr(), ptr(dw), ptr(db), n, c, ptr(ws), bytes, current_stream()),
                 "layer_norm_backward");
    py::dict out;
    out["d_x"] = as(dx, src);
    put_affine_grads(out, dw, db, weight, bias);
    return out;
}

// Dropout's key: a number (host), or a one-element int64 tensor that the kernel
// reads when it is on the GPU.
[[noreturn]] void bad_seed() { throw std::runtime_error("seed must be a whole number or a one-element int64 tensor"); }

// The 64 bits of a whole number, signed or not (torch.initial_seed() is unsigned).
int64_t seed_bits(const py::object& seed)
{
    const py::object number = py::reinterpret_steal<py::object>(PyNumber_Index(seed.ptr()));
    if (!number) {
        PyErr_Clear();
        bad_seed();
    }
    int over = 0;
    const long long bits = PyLong_AsLongLongAndOverflow(number.ptr(), &over);
    if (!over) return bits;
    const unsigned long long wide = over > 0 ? PyLong_AsUnsignedLongLong(number.ptr()) : 0;
    if (over < 0 || PyErr_Occurred()) {
        PyErr_Clear();
        throw std::invalid_argument("seed must be between -2^63 and 2^64 - 1");
    }
    return static_cast<int64_t>(wide);
}

void check_seed(const py::object& seed)
{
    if (!THPVariable_Check(seed.ptr())) {
        seed_bits(seed);
    } else {
        const torch::Tensor t = py::cast<torch::Tensor>(seed);
        if (t.scalar_type() != torch::kInt64 || t.numel() != 1) bad_seed();
    }
}

struct Seed {
    int64_t value = 0;
    torch::Tensor held;

    Seed(const py::object& seed, const torch::TensorOptions& opts)
    {
        if (!THPVariable_Check(seed.ptr())) {
            value = seed_bits(seed);
            return;
        }
        held = py::cast<torch::Tensor>(seed);
        if (held.is_cuda()) {
            held = held.to(opts.dtype(torch::kInt64));
        } else {
            value = held.item<int64_t>();
            held = torch::Tensor();
        }
    }

    const int64_t* device() const { return held.defined() ? held.data_ptr<int64_t>() : nullptr; }
};

torch::Tensor dropped(torch::Tensor x, double p, const py::object& seed, int64_t offset, const char* name,
                      const char* what)
{
    check_real(x, name);
    check_p(p);
    check_seed(seed);
    const auto src = x.options();
    const auto opts = compute_options(x);
    const Seed key(seed, opts);
    x = whole(on(x, opts));
    const c10::cuda::CUDAGuard guard(x.device());
    torch::Tensor y = fresh(x.sizes(), opts);
    check_status(mhc_dropout(x.data_ptr(), y.data_ptr(), dtype_code(x), x.numel(), p, key.value, key.device(), offset,
                             current_stream()),
                 what);
    return as(y, src);
}

py::dict dropout(torch::Tensor x, double p, py::object seed, int64_t offset)
{
    py::dict out;
    out["y"] = dropped(x, p, seed, offset, "x", "dropout");
    return out;
}

py::dict dropout_backward(torch::Tensor G, double p, py::object seed, int64_t offset)
{
    py::dict out;
    out["d_x"] = dropped(G, p, seed, offset, "G", "dropout_backward");
    return out;
}

py::dict stream_norm_n4(torch::Tensor X, torch::Tensor h_pre, const Opt& weight, const Opt& bias, double eps)
{
    check_streams(X, "X");
    check_real(X, "X");
    const int64_t n = X.size(0), c = X.size(2);
    check_like(h_pre, {n, 4}, "h_pre", "B x 4");
    check_real(h_pre, "h_pre");
    check_affine(weight, bias, c);
    check_eps(eps);
    const auto src = X.options();
    const auto opts = compute_options(X);
    const Affine a(weight, bias, opts);
    X = rows_on(X, opts);
    const torch::Tensor h = small_on(h_pre, opts);
    const c10::cuda::CUDAGuard guard(X.device());
    torch::Tensor y = fresh({n, c}, opts);
    const auto [mean, rstd] = fresh_stats(n, opts);
    check_status(mhc_stream_norm_n4(X.data_ptr(), X.stride(0), X.stride(1), dtype_code(X), h.data_ptr(), dtype_code(h),
                                    a.weight(), a.bias(), a.dtype, y.data_ptr(), mean.data_ptr<float>(),
                                    rstd.data_ptr<float>(), static_cast<float>(eps), n, c, current_stream()),
                 "stream_norm_n4");
    py::dict out;
    out["y"] = as(y, src);
    out["mean"] = mean;
    out["rstd"] = rstd;
    return out;
}

py::dict stream_norm_n4_backward(torch::Tensor G, torch::Tensor X, torch::Tensor h_pre, torch::Tensor mean,
                                 torch::Tensor rstd, const Opt& weight, const Opt& bias)
{
    check_streams(X, "X");
    check_real(X, "X");
    const int64_t n = X.size(0), c = X.size(2);
    check_like(G, {n, c}, "G", "B x C");
    check_real(G, "G");
    check_like(h_pre, {n, 4}, "h_pre", "B x 4");
    check_real(h_pre, "h_pre");
    check_stats(mean, rstd, n);
    check_affine(weight, bias, c);
    const auto src = X.options();
    const auto opts = compute_options(X, {&G});
    const Affine a(weight, bias, opts);
    mean = stats_on(mean, opts);
    rstd = stats_on(rstd, opts);
    X = rows_on(X, opts);
    G = rows_on(G, opts);
    const torch::Tensor h = small_on(h_pre, opts);
    const c10::cuda::CUDAGuard guard(X.device());
    torch::Tensor dX = fresh({n, 4, c}, opts);
    torch::Tensor dh = fresh(h.sizes(), h.options());
    torch::Tensor dw = a.grad_of(a.w), db = a.grad_of(a.b), ws;
    int64_t bytes = 0;
    if (weight || bias) {
        check_status(mhc_stream_norm_n4_backward_workspace(n, c, &bytes), "stream_norm_n4_backward");
        ws = fresh({bytes}, opts, torch::kUInt8);
    }
    check_status(mhc_stream_norm_n4_backward(G.data_ptr(), G.stride(0), X.data_ptr(), X.stride(0), X.stride(1),
                                             dtype_code(X), h.data_ptr(), dtype_code(h), mean.data_ptr<float>(),
                                             rstd.data_ptr<float>(), a.weight(), a.dtype, dX.data_ptr(), dh.data_ptr(),
                                             ptr(dw), ptr(db), n, c, ptr(ws), bytes, current_stream()),
                 "stream_norm_n4_backward");
    py::dict out;
    out["d_X"] = as(dX, src);
    out["d_h_pre"] = as(dh, h_pre.options());
    put_affine_grads(out, dw, db, weight, bias);
    return out;
}

void check_mix(const torch::Tensor& X, const torch::Tensor& T, const torch::Tensor& y, const torch::Tensor& h_post,
               double p, const py::object& seed)
{
    check_streams(X, "X");
    check_real(X, "X");
    const int64_t n = X.size(0), c = X.size(2);
    check_like(T, {n, 4, 4}, "T", "B x 4 x 4");
    check_real(T, "T");
    check_like(y, {n, c}, "y", "B x C");
    check_real(y, "y");
    check_like(h_post, {n, 4}, "h_post", "B x 4");
    check_real(h_post, "h_post");
    check_p(p);
    check_seed(seed);
}

py::dict stream_mix_n4(torch::Tensor X, torch::Tensor T, torch::Tensor y, torch::Tensor h_post, double p,
                       py::object seed, int64_t offset)
{
    check_mix(X, T, y, h_post, p, seed);
    const int64_t n = X.size(0), c = X.size(2);
    const auto src = X.options();
    const auto opts = compute_options(X, {&y});
    const Seed key(seed, opts);
    X = rows_on(X, opts);
    y = rows_on(y, opts);
    const torch::Tensor t = small_on(T, opts), h = small_on(h_post, opts);
    const c10::cuda::CUDAGuard guard(X.device());
    torch::Tensor out_x = fresh({n, 4, c}, opts);
    check_status(mhc_stream_mix_n4(X.data_ptr(), X.stride(0), X.stride(1), y.data_ptr(), y.stride(0), dtype_code(X),
                                   t.data_ptr(), dtype_code(t), h.data_ptr(), dtype_code(h), out_x.data_ptr(), p,
                                   key.value, key.device(), offset, n, c, current_stream()),
                 "stream_mix_n4");
    py::dict out;
    out["X"] = as(out_x, src);
    return out;
}

py::dict stream_mix_n4_backward(torch::Tensor G, torch::Tensor X, torch::Tensor T, torch::Tensor y,
                                torch::Tensor h_post, double p, py::object seed, int64_t offset)
{
    check_mix(X, T, y, h_post, p, seed);
    check_like(G, X.sizes(), "G", "B x 4 x C");
    check_real(G, "G");
    const int64_t n = X.size(0), c = X.size(2);
    const auto src = X.options(), y_src = y.options();
    const auto opts = compute_options(X, {&y, &G});
    const Seed key(seed, opts);
    X = rows_on(X, opts);
    y = rows_on(y, opts);
    G = rows_on(G, opts);
    const torch::Tensor t = small_on(T, opts), h = small_on(h_post, opts);
    const c10::cuda::CUDAGuard guard(X.device());
    torch::Tensor dX = fresh({n, 4, c}, opts), dT = fresh(t.sizes(), t.options());
    torch::Tensor dy = fresh({n, c}, opts), dh = fresh(h.sizes(), h.options());
    check_status(mhc_stream_mix_n4_backward(G.data_ptr(), G.stride(0), G.stride(1), X.data_ptr(), X.stride(0),
                                            X.stride(1), y.data_ptr(), y.stride(0), dtype_code(X), t.data_ptr(),
                                            dtype_code(t), h.data_ptr(), dtype_code(h), dX.data_ptr(), dT.data_ptr(),
                                            dy.data_ptr(), dh.data_ptr(), p, key.value, key.device(), offset, n, c,
                                            current_stream()),
                 "stream_mix_n4_backward");
    py::dict out;
    out["d_X"] = as(dX, src);
    out["d_T"] = as(dT, T.options());
    out["d_y"] = as(dy, y_src);
    out["d_h_post"] = as(dh, h_post.options());
    return out;
}

}  // namespace

void bind_residual_path(py::module& m)
{
    const py::object none = py::none();
    m.def("layer_norm", &layer_norm, py::arg("x"), py::arg("weight") = none, py::arg("bias") = none,
          py::arg("eps") = 1e-5, "Layer norm of the rows of x (B x C): y, and the mean and rstd its backward takes");
    m.def("layer_norm_backward", &layer_norm_backward, py::arg("G"), py::arg("x"), py::arg("mean"), py::arg("rstd"),
          py::arg("weight") = none, py::arg("bias") = none,
          "Gradients of layer_norm: d_x, and d_weight and d_bias for those given");
    m.def("dropout", &dropout, py::arg("x"), py::arg("p"), py::arg("seed"), py::arg("offset") = 0,
          "Dropout with the mask of (seed, offset) from a counter-based generator (Philox4x32-10, 16 bits an element)");
    m.def("dropout_backward", &dropout_backward, py::arg("G"), py::arg("p"), py::arg("seed"), py::arg("offset") = 0,
          "Gradient of dropout: the same mask, formed again, on G");
    m.def("stream_norm_n4", &stream_norm_n4, py::arg("X"), py::arg("h_pre"), py::arg("weight") = none,
          py::arg("bias") = none, py::arg("eps") = 1e-5,
          "Layer norm of sum_i h_pre[:, i] * X[:, i] for four residual streams X (B x 4 x C)");
    m.def("stream_norm_n4_backward", &stream_norm_n4_backward, py::arg("G"), py::arg("X"), py::arg("h_pre"),
          py::arg("mean"), py::arg("rstd"), py::arg("weight") = none, py::arg("bias") = none,
          "Gradients of stream_norm_n4: d_X, d_h_pre, and d_weight and d_bias for those given");
    m.def("stream_mix_n4", &stream_mix_n4, py::arg("X"), py::arg("T"), py::arg("y"), py::arg("h_post"),
          py::arg("p") = 0.0, py::arg("seed") = 0, py::arg("offset") = 0,
          "The residual update T X + h_post (x) dropout(y) of four streams X (B x 4 x C)");
    m.def("stream_mix_n4_backward", &stream_mix_n4_backward, py::arg("G"), py::arg("X"), py::arg("T"), py::arg("y"),
          py::arg("h_post"), py::arg("p") = 0.0, py::arg("seed") = 0, py::arg("offset") = 0,
          "Gradients of stream_mix_n4: d_X, d_T, d_y and d_h_post");
}

}  // namespace mhcp_torch
