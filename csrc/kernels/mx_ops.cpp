// Torch wrappers of the microscaled formats, their products and the RMS norm.
#include <ATen/cuda/CUDAContext.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDACachingAllocator.h>
#include <c10/cuda/CUDAGraphsC10Utils.h>
#include <c10/cuda/CUDAGuard.h>

#include <atomic>
#include <limits>
#include <mutex>
#include <vector>

#include "microscale.h"
#include "torch_ops.h"

namespace mmltk {

namespace {

using OptTensor = c10::optional<torch::Tensor>;

bool has(const OptTensor& t) { return t.has_value() && t->defined(); }

Elt elt_of(const torch::Tensor& t, const char* what) {
    switch (t.scalar_type()) {
        case torch::kFloat32: return Elt::kF32;
        case torch::kBFloat16: return Elt::kBF16;
        case torch::kFloat16: return Elt::kF16;
        default: TORCH_CHECK(false, what, ": bf16, fp16 or fp32 expected, got ", t.scalar_type());
    }
}

MxFormat format_of(int64_t f) {
    TORCH_CHECK(f >= 0 && f <= 2, "microscale: unknown format ", f);
    return static_cast<MxFormat>(f);
}

// A new tensor without a trip through the dispatcher (half of torch::empty's 1.7 us, and a small call makes three).
torch::Tensor fresh(at::IntArrayRef sizes, torch::ScalarType dtype, const torch::Tensor& like) {
    return at::detail::empty_cuda(sizes, dtype, like.device(), c10::nullopt);
}
// Work space of the current stream, given back to the allocator at the end of the scope.
struct WorkSpace {
    explicit WorkSpace(int64_t bytes) : block(c10::cuda::CUDACachingAllocator::get()->allocate(static_cast<size_t>(bytes))) {}
    void* at(int64_t offset) const { return static_cast<char*>(block.get()) + offset; }
    c10::DataPtr block;
};

bool aligned16(const torch::Tensor& t) { return reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0; }

// x [..., K] as rows of K elements, a view where its strides allow one
torch::Tensor as_rows(const torch::Tensor& x) {
    torch::Tensor r = x.dim() == 2 ? x : x.reshape({-1, x.size(-1)});
    if (r.size(1) > 1 && r.stride(1) != 1) r = r.contiguous();
    if (r.size(1) == 1 && r.stride(1) != 1) r = r.contiguous();
    return r;
}
int64_t row_pitch(const torch::Tensor& r) { return r.size(0) > 1 ? r.stride(0) : r.size(1); }

void check_input(const torch::Tensor& x, const char* what) {
    TORCH_CHECK(x.is_cuda(), what, ": CUDA tensor expected");
    TORCH_CHECK(x.dim() >= 1 && x.size(-1) > 0, what, ": needs a last dimension of at least one element");
}

void check_scalar(const torch::Tensor& g, const torch::Tensor& like, const char* what) {
    TORCH_CHECK(g.scalar_type() == torch::kFloat32 && g.numel() == 1 && g.device() == like.device(), what,
                ": the tensor scale is one fp32 value on the same device");
}

torch::ScalarType code_type(MxFormat f) {
    return f == MxFormat::kMxFp8 ? torch::ScalarType::Float8_e4m3fn : torch::kUInt8;
}
torch::Tensor new_codes(MxFormat f, int64_t rows, int64_t dim, const torch::Tensor& like) {
    return fresh({rows, mx_pitch(f, dim)}, code_type(f), like);
}
torch::Tensor new_scales(MxFormat f, int64_t rows, int64_t dim, const torch::Tensor& like) {
    return fresh({(rows + 127) / 128, mx_scale_tiles(f, dim), 32, 4, 4}, torch::kUInt8, like);
}
void check_coded(MxFormat f, const torch::Tensor& codes, const torch::Tensor& scales, int64_t rows, int64_t dim,
                 const char* what) {
    TORCH_CHECK(rows >= 0 && dim > 0, what, ": bad shape");
    TORCH_CHECK(codes.is_cuda() && scales.device() == codes.device(), what, ": codes and scales on one CUDA device");
    TORCH_CHECK(codes.scalar_type() == code_type(f) && codes.dim() == 2 && codes.is_contiguous() &&
                    codes.size(0) == rows && codes.size(1) == mx_pitch(f, dim),
                what, ": codes must be contiguous ", code_type(f), " [", rows, ", ", mx_pitch(f, dim), "]");
    TORCH_CHECK(scales.scalar_type() == torch::kUInt8 && scales.is_contiguous() &&
                    scales.numel() == (rows + 127) / 128 * mx_scale_tiles(f, dim) * 512,
                what, ": scales must be contiguous uint8 [", (rows + 127) / 128, ", ", mx_scale_tiles(f, dim),
                ", 32, 4, 4]");
    TORCH_CHECK(aligned16(codes) && aligned16(scales), what, ": codes and scales must start on 16 bytes");
}

void no_grad_here(const torch::Tensor& t, const char* what) {
    TORCH_CHECK(!(at::GradMode::is_enabled() && t.requires_grad()), what,
                ": has no gradient (a serving operator); call it under torch.no_grad() or on detached tensors");
}

// The current device's status word: allocated and cleared before the first call that takes it returns, on a stream of its
// own, so that a first call under graph capture leaves no clear in the graph (its replays would erase what they record).
int* mx_status_word(const torch::Device& dev) {
    static std::mutex mu;
    static std::vector<int*> words(64);
    std::lock_guard<std::mutex> lk(mu);
    int*& word = words.at(dev.index());
    if (!word) {
        c10::cuda::CUDAStreamCaptureModeGuard relaxed(cudaStreamCaptureModeRelaxed);
        int* p = nullptr;
        cudaStream_t own = nullptr;
        check_cuda(cudaMalloc(reinterpret_cast<void**>(&p), sizeof(int)), "mx_status");
        cudaError_t e = cudaStreamCreateWithFlags(&own, cudaStreamNonBlocking);
        if (e == cudaSuccess) {
            e = cudaMemsetAsync(p, 0, sizeof(int), own);
            if (e == cudaSuccess) e = cudaStreamSynchronize(own);
            cudaStreamDestroy(own);
        }
        if (e != cudaSuccess) cudaFree(p);
        check_cuda(e, "mx_status");
        word = p;
    }
    return word;
}

// Tries that a wait for loaded data makes before the kernel gives up; 0: none (tests of the status word).
std::atomic<int> wait_limit{kMxWaitLimit};
int64_t mx_wait_limit(int64_t tries) {
    TORCH_CHECK(tries >= 0 && tries <= kMxWaitLimit, "mx_wait_limit: 0 to ", kMxWaitLimit, " tries");
    return wait_limit.exchange(static_cast<int>(tries));
}

// Non-zero when a kernel on this device gave up a bounded wait (products: 1 loads, 2 MMA, 3 epilogue; 4 norm
// backward); waits for all work on the device, and clears it.
int64_t mx_status(int64_t device) {
    const torch::Device dev(torch::kCUDA, static_cast<c10::DeviceIndex>(device));
    at::cuda::CUDAGuard guard(dev);
    int* w = mx_status_word(dev);
    const int zero = 0;
    int v = 0;
    check_cuda(cudaDeviceSynchronize(), "mx_status");
    check_cuda(cudaMemcpy(&v, w, sizeof(v), cudaMemcpyDeviceToHost), "mx_status");
    if (v) check_cuda(cudaMemcpy(w, &zero, sizeof(v), cudaMemcpyHostToDevice), "mx_status");
    return v;
}

// ---------------------------------------------------------------- formats
// -> codes, scales, g (undefined but for nvfp4)
std::vector<OptTensor> mx_quantize(torch::Tensor x, int64_t fmt, OptTensor g) {
    check_input(x, "mx_quantize");
    no_grad_here(x, "mx_quantize");
    const MxFormat f = format_of(fmt);
    const Elt et = elt_of(x, "mx_quantize");
    at::cuda::CUDAGuard guard(x.device());
    const torch::Tensor r = as_rows(x);
    const int64_t rows = r.size(0), dim = r.size(1);
    auto codes = new_codes(f, rows, dim, x), scales = new_scales(f, rows, dim, x);
    torch::Tensor gt;
    c10::optional<WorkSpace> work;
    if (f == MxFormat::kNvFp4) {
        if (has(g)) {
            check_scalar(*g, x, "mx_quantize");
            gt = *g;
        } else {
            gt = rows ? fresh({1}, torch::kFloat32, x)
                      : torch::ones({1}, x.options().dtype(torch::kFloat32));
            work.emplace(kMxAmaxParts * sizeof(uint32_t));
        }
    } else {
        TORCH_CHECK(!has(g), "mx_quantize: only nvfp4 has a tensor scale");
    }
    check_cuda(launch_mx_quantize(et, f, r.data_ptr(), row_pitch(r), rows, dim, codes.data_ptr(), scales.data_ptr(),
                                  gt.defined() ? gt.data_ptr<float>() : nullptr,
                                  work ? static_cast<uint32_t*>(work->at(0)) : nullptr,
                                  cur_stream()),
               "mx_quantize");
    return {codes, scales, gt.defined() ? OptTensor(gt) : OptTensor()};
}

torch::Tensor mx_dequantize(torch::Tensor codes, torch::Tensor scales, OptTensor g, int64_t fmt, int64_t rows,
                            int64_t dim, torch::ScalarType dtype) {
    const MxFormat f = format_of(fmt);
    check_coded(f, codes, scales, rows, dim, "mx_dequantize");
    if (has(g)) check_scalar(*g, codes, "mx_dequantize");
    at::cuda::CUDAGuard guard(codes.device());
    auto out = fresh({rows, dim}, dtype, codes);
    check_cuda(launch_mx_dequantize(elt_of(out, "mx_dequantize"), f, codes.data_ptr(), scales.data_ptr(),
                                    has(g) ? g->data_ptr<float>() : nullptr, rows, dim, out.data_ptr(), cur_stream()),
               "mx_dequantize");
    return out;
}

// ---------------------------------------------------------------- RMS norm
void check_norm(const torch::Tensor& x, const torch::Tensor& w, const OptTensor& res, const char* what) {
    check_input(x, what);
    TORCH_CHECK(x.size(-1) <= kRmsMaxDim, what, ": rows of at most ", kRmsMaxDim, " elements");
    TORCH_CHECK(w.device() == x.device() && w.dim() == 1 && w.size(0) == x.size(-1) &&
                    (w.scalar_type() == x.scalar_type() || w.scalar_type() == torch::kFloat32),
                what, ": weight must be [", x.size(-1), "] of the input's dtype or fp32, on its device");
    if (has(res))
        TORCH_CHECK(res->sizes() == x.sizes() && res->scalar_type() == x.scalar_type() && res->device() == x.device(),
                    what, ": residual must match the input's shape, dtype and device");
}

torch::Tensor aligned_weight(const torch::Tensor& w) {      // vector loads
    torch::Tensor c = w.contiguous();
    return aligned16(c) ? c : c.clone();
}

struct NormOut {
    torch::Tensor y, h, rstd, codes, scales;
};
NormOut norm_forward(const torch::Tensor& x, const torch::Tensor& w_in, const OptTensor& res, double eps, bool want_rstd,
                     const MxFormat* fmt, const float* g, const char* what) {
    at::cuda::CUDAGuard guard(x.device());
    const torch::Tensor xr = as_rows(x), w = aligned_weight(w_in);
    NormOut o;
    RmsFwdArgs a{};
    a.rows = xr.size(0);
    a.dim = static_cast<int>(xr.size(1));
    a.x = xr.data_ptr();
    a.ldx = row_pitch(xr);
    torch::Tensor rr;
    if (has(res)) {
        rr = as_rows(*res);
        a.res = rr.data_ptr();
        a.ldr = row_pitch(rr);
        o.h = fresh(x.sizes(), x.scalar_type(), x);
        a.h = o.h.data_ptr();
    }
    a.w = w.data_ptr();
    a.w_f32 = w.scalar_type() == torch::kFloat32 && x.scalar_type() != torch::kFloat32;
    a.eps = static_cast<float>(eps);
    if (want_rstd) {
        o.rstd = fresh({a.rows}, torch::kFloat32, x);
        a.rstd = o.rstd.data_ptr<float>();
    }
    if (fmt) {
        o.codes = new_codes(*fmt, a.rows, a.dim, x);
        o.scales = new_scales(*fmt, a.rows, a.dim, x);
        a.codes = o.codes.data_ptr();
        a.scales = o.scales.data_ptr();
        a.g = g;
        a.fmt = *fmt;
    } else {
        o.y = fresh(x.sizes(), x.scalar_type(), x);
        a.y = o.y.data_ptr();
    }
    if (a.rows) check_cuda(launch_rms_fwd(elt_of(x, what), a, cur_stream()), what);
    return o;
}

// gx (of x and of the residual), gw
std::pair<torch::Tensor, torch::Tensor> norm_backward(const torch::Tensor& gy, const torch::Tensor& gh,
                                                      const torch::Tensor& h, const torch::Tensor& w_in,
                                                      const torch::Tensor& rstd, bool want_gw) {
    at::cuda::CUDAGuard guard(h.device());
    const torch::Tensor hr = as_rows(h), w = aligned_weight(w_in);
    RmsBwdArgs a{};
    a.rows = hr.size(0);
    a.dim = static_cast<int>(hr.size(1));
    a.h = hr.data_ptr();
    a.ldh = row_pitch(hr);
    const torch::Tensor gyr = as_rows(gy);
    torch::Tensor ghr;
    a.gy = gyr.data_ptr();
    a.ldgy = row_pitch(gyr);
    if (gh.defined()) {
        ghr = as_rows(gh);
        a.gh = ghr.data_ptr();
        a.ldgh = row_pitch(ghr);
    }
    a.w = w.data_ptr();
    a.w_f32 = w.scalar_type() == torch::kFloat32 && h.scalar_type() != torch::kFloat32;
    a.rstd = rstd.data_ptr<float>();
    a.status = mx_status_word(h.device());
    a.wait_limit = wait_limit.load(std::memory_order_relaxed);
    auto gx = fresh(h.sizes(), h.scalar_type(), h);
    a.gx = gx.data_ptr();
    torch::Tensor gw;
    c10::optional<WorkSpace> partial;
    const Elt et = elt_of(h, "rms_norm backward");
    if (want_gw) {
        gw = fresh(w.sizes(), w.scalar_type(), w);
        a.gw = gw.data_ptr();
        partial.emplace(static_cast<int64_t>(rms_bwd_partials(a.rows)) * rms_partial_pitch(a.dim) * sizeof(float));
        a.partial = static_cast<float*>(partial->at(0));
    }
    check_cuda(launch_rms_bwd(et, a, cur_stream()), "rms_norm backward");
    return {gx, gw};
}

class RmsNormFn : public torch::autograd::Function<RmsNormFn> {
public:
    static torch::autograd::variable_list forward(torch::autograd::AutogradContext* ctx, const torch::Tensor& x,
                                                  const torch::Tensor& w, const OptTensor& res, double eps) {
        NormOut o = norm_forward(x, w, res, eps, true, nullptr, nullptr, "rms_norm");
        ctx->set_materialize_grads(false);
        ctx->save_for_backward({has(res) ? o.h : x, w, o.rstd});
        ctx->saved_data["res"] = has(res);
        if (has(res)) return {o.y, o.h};
        return {o.y};
    }
    static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx,
                                                   torch::autograd::variable_list grads) {
        TORCH_CHECK(!at::GradMode::is_enabled(), "rms_norm: the backward has no gradient of its own (create_graph)");
        const bool res = ctx->saved_data["res"].toBool();
        const auto saved = ctx->get_saved_variables();
        const torch::Tensor gh = res ? grads[1] : torch::Tensor();
        if (!grads[0].defined() && !gh.defined()) return {torch::Tensor(), torch::Tensor(), torch::Tensor(), torch::Tensor()};
        if (!grads[0].defined()) return {gh, torch::Tensor(), gh, torch::Tensor()};
        auto [gx, gw] = norm_backward(grads[0], gh, saved[0], saved[1], saved[2], ctx->needs_input_grad(1));
        return {gx, gw, res ? gx : torch::Tensor(), torch::Tensor()};
    }
};

// -> y, h (undefined without a residual); differentiable
std::vector<OptTensor> rms_norm(torch::Tensor x, torch::Tensor w, OptTensor res, double eps) {
    check_norm(x, w, res, "rms_norm");
    elt_of(x, "rms_norm");
    if (at::GradMode::is_enabled() && (x.requires_grad() || w.requires_grad() || (has(res) && res->requires_grad()))) {
        auto o = RmsNormFn::apply(x, w, res, eps);
        return {o[0], has(res) ? OptTensor(o[1]) : OptTensor()};
    }
    NormOut o = norm_forward(x, w, res, eps, false, nullptr, nullptr, "rms_norm");
    return {o.y, has(res) ? OptTensor(o.h) : OptTensor()};
}

// -> codes, scales, h (undefined without a residual)
std::vector<OptTensor> rms_norm_quantized(torch::Tensor x, torch::Tensor w, OptTensor res, double eps, int64_t fmt,
                                          OptTensor g) {
    check_norm(x, w, res, "rms_norm_quantized");
    for (const torch::Tensor& t : {x, w}) no_grad_here(t, "rms_norm_quantized");
    if (has(res)) no_grad_here(*res, "rms_norm_quantized");
    const MxFormat f = format_of(fmt);
    if (has(g)) {
        TORCH_CHECK(f == MxFormat::kNvFp4, "rms_norm_quantized: only nvfp4 has a tensor scale");
        check_scalar(*g, x, "rms_norm_quantized");
    }
    NormOut o = norm_forward(x, w, res, eps, false, &f, has(g) ? g->data_ptr<float>() : nullptr, "rms_norm_quantized");
    return {o.codes, o.scales, has(res) ? OptTensor(o.h) : OptTensor()};
}

// ---------------------------------------------------------------- product
// x: [rows, k] to be quantised here, or null with x_codes / x_scales.  -> {y} or {codes, scales}
std::vector<torch::Tensor> mx_linear(OptTensor x, OptTensor x_codes, OptTensor x_scales, OptTensor x_g, int64_t rows,
                                     torch::Tensor w_codes, torch::Tensor w_scales, OptTensor w_g, int64_t fmt, int64_t n,
                                     int64_t k, OptTensor bias, int64_t act, torch::ScalarType out_dtype,
                                     bool quant_out) {
    const MxFormat f = format_of(fmt);
    check_coded(f, w_codes, w_scales, n, k, "mx_linear: weight");
    TORCH_CHECK(act >= 0 && act <= 2, "mx_linear: unknown activation");
    constexpr int64_t kMax = std::numeric_limits<int>::max() - 512;
    at::cuda::CUDAGuard guard(w_codes.device());
    torch::Tensor xr, xc, xs;
    if (has(x)) {
        check_input(*x, "mx_linear");
        no_grad_here(*x, "mx_linear");
        TORCH_CHECK(x->device() == w_codes.device() && x->size(-1) == k, "mx_linear: input [..., ", k,
                    "] on the weight's device expected, got ", x->sizes());
        elt_of(*x, "mx_linear");
        xr = as_rows(*x);
        rows = xr.size(0);
    } else {
        TORCH_CHECK(has(x_codes) && has(x_scales), "mx_linear: needs an input");
        xc = *x_codes;
        xs = *x_scales;
        check_coded(f, xc, xs, rows, k, "mx_linear: input");
        TORCH_CHECK(xc.device() == w_codes.device(), "mx_linear: input and weight on different devices");
    }
    TORCH_CHECK(rows <= kMax && n <= kMax && k <= kMax, "mx_linear: sizes below 2^31 - 512");
    if (has(x_g)) check_scalar(*x_g, w_codes, "mx_linear: input");
    if (has(w_g)) check_scalar(*w_g, w_codes, "mx_linear: weight");
    MxGemmArgs a{};
    a.m = static_cast<int>(rows);
    a.n = static_cast<int>(n);
    a.k = static_cast<int>(k);
    a.fmt = f;
    a.act = static_cast<int>(act);
    a.w_codes = w_codes.data_ptr();
    a.w_scales = w_scales.data_ptr();
    a.w_g = has(w_g) ? w_g->data_ptr<float>() : nullptr;
    a.x_g = has(x_g) ? x_g->data_ptr<float>() : nullptr;
    a.x_pitch = a.w_pitch = mx_pitch(f, k);
    torch::Tensor b, y, codes, scales;
    if (has(bias)) {
        TORCH_CHECK(bias->device() == w_codes.device() && bias->dim() == 1 && bias->size(0) == n,
                    "mx_linear: bias must be [", n, "] on the weight's device");
        no_grad_here(*bias, "mx_linear");
        b = bias->contiguous();
        a.bias = b.data_ptr();
        a.bias_elt = elt_of(b, "mx_linear: bias");
    }
    if (quant_out) {
        codes = new_codes(MxFormat::kMxFp8, rows, n, w_codes);
        scales = new_scales(MxFormat::kMxFp8, rows, n, w_codes);
        a.codes = codes.data_ptr();
        a.scales = scales.data_ptr();
        a.y_pitch = mx_pitch(MxFormat::kMxFp8, n);
    } else {
        y = fresh({rows, n}, out_dtype, w_codes);
        a.out = elt_of(y, "mx_linear: output");
        a.y = y.data_ptr();
        a.y_pitch = n * static_cast<int64_t>(y.element_size());
    }
    if (rows && n) {
        a.status = mx_status_word(w_codes.device());
        a.wait_limit = wait_limit.load(std::memory_order_relaxed);
        if (mx_few_fits(f, a.m, a.n, a.k, !xr.defined())) {
            MxFewArgs few{};
            if (xr.defined()) {
                few.x = xr.data_ptr();
                few.ldx = row_pitch(xr);
                few.x_elt = elt_of(xr, "mx_linear");
            } else {
                a.x_codes = xc.data_ptr();
                a.x_scales = xs.data_ptr();
            }
            few.g = a;
            check_cuda(launch_mx_few(few, cur_stream()), "mx_linear");
            if (quant_out) return {codes, scales};
            return {y};
        }
        c10::optional<WorkSpace> xq;
        if (xr.defined()) {
            const int64_t code_bytes = (rows * a.x_pitch + 511) / 512 * 512;
            xq.emplace(code_bytes + (rows + 127) / 128 * mx_scale_tiles(f, k) * 512);
            check_cuda(launch_mx_quantize(elt_of(xr, "mx_linear"), f, xr.data_ptr(), row_pitch(xr), rows, k, xq->at(0),
                                          xq->at(code_bytes), const_cast<float*>(a.x_g), nullptr, cur_stream()),
                       "mx_linear: quantisation");
            a.x_codes = xq->at(0);
            a.x_scales = xq->at(code_bytes);
        } else {
            a.x_codes = xc.data_ptr();
            a.x_scales = xs.data_ptr();
        }
        check_cuda(launch_mx_gemm(a, cur_stream()), "mx_linear");
    }
    if (quant_out) return {codes, scales};
    return {y};
}

}  // namespace

void register_mx_ops(pybind11::module& m) {
    namespace py = pybind11;
    m.def("mx_quantize", &mx_quantize, py::arg("x"), py::arg("fmt"), py::arg("g") = py::none());
    m.def("mx_dequantize", &mx_dequantize);
    m.def("rms_norm", &rms_norm, py::arg("x"), py::arg("w"), py::arg("res"), py::arg("eps"));
    m.def("rms_norm_quantized", &rms_norm_quantized, py::arg("x"), py::arg("w"), py::arg("res"), py::arg("eps"),
          py::arg("fmt"), py::arg("g") = py::none());
    m.def("mx_linear", &mx_linear);
    m.def("mx_status", &mx_status);
    m.def("mx_wait_limit", &mx_wait_limit);
}

}  // namespace mmltk
