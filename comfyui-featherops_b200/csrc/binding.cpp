// Python binding of the MXFP4 operators and the fused norm: argument checks, output allocation and launch in one call.
//
// These operators run in a few microseconds on the GPU, less than the same steps take in Python (linear_mxfp4 for one token: 27 us
// of host time through ctypes).  The kernels stay behind the C ABI of libfeather_b200.so: `bind` takes the addresses of its entry
// points, so this module links against torch only.  A call releases the GIL while it allocates and launches.
//
// A call does not pass torch's dispatcher.  Where somebody watches that (a tracer, a dispatch mode, a functorch transform, a tensor that is
// a subclass with its own dispatch), it returns NotImplemented once its checks are done, and the caller takes the registered operator, whose
// implementation comes back here with `direct`.
#include <Python.h>

#include <ATen/cuda/EmptyTensor.h>
#include <ATen/core/Tensor.h>
#include <ATen/core/grad_mode.h>
#include <c10/core/impl/LocalDispatchKeySet.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include "../../include/feather_b200.h"

namespace {

struct Entries {
    decltype(&feather_mxfp4_quantize) quantize;
    decltype(&feather_mxfp4_dequantize) dequantize;
    decltype(&feather_mxfp4_mm) mm;
    decltype(&feather_gated_norm) norm;
    decltype(&feather_last_error_string) error;
} g_lib;
PyObject* g_error = nullptr;          // FeatherNativeError
PyObject* g_status = nullptr;         // device index -> address of the device's status word
constexpr int kMaxDevices = 64;
int* g_status_words[kMaxDevices];

struct WithoutGil {
    PyThreadState* state = PyEval_SaveThread();
    ~WithoutGil() { PyEval_RestoreThread(state); }
};

const at::Tensor* optional_tensor(PyObject* o, const char* name) {
    if (o == Py_None) return nullptr;
    TORCH_CHECK_TYPE(THPVariable_Check(o), name, " must be a tensor or None");
    return &THPVariable_Unpack(o);
}
const at::Tensor& tensor(PyObject* o, const char* name) {
    TORCH_CHECK_TYPE(THPVariable_Check(o), name, " must be a tensor");
    return THPVariable_Unpack(o);
}
c10::optional<at::ScalarType> optional_dtype(PyObject* o, const char* name) {
    if (o == Py_None) return c10::nullopt;
    TORCH_CHECK_TYPE(THPDtype_Check(o), name, " must be a torch.dtype");
    return reinterpret_cast<THPDtype*>(o)->scalar_type;
}
double number(PyObject* o) {
    const double v = PyFloat_AsDouble(o);
    if (v == -1.0 && PyErr_Occurred()) throw python_error();
    return v;
}
bool truth(PyObject* o) {
    const int v = PyObject_IsTrue(o);
    if (v < 0) throw python_error();
    return v == 1;
}

int source_code(at::ScalarType t) {
    return t == at::kFloat ? FEATHER_SRC_FP32 : t == at::kBFloat16 ? FEATHER_SRC_BF16 : t == at::kHalf ? FEATHER_SRC_FP16 : -1;
}
bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

void refuse_grad(std::initializer_list<const at::Tensor*> tensors, const char* what) {
    for (const at::Tensor* t : tensors)                                       // undefined without a tangent, and while forward mode is off
        TORCH_CHECK(t == nullptr || !t->_fw_grad(0).defined(), what, " no forward-mode derivative: unpack the dual tensors first");
    if (!at::GradMode::is_enabled()) return;
    for (const at::Tensor* t : tensors)
        TORCH_CHECK(t == nullptr || !t->requires_grad(), what, " no backward pass: detach the inputs or call under torch.no_grad()");
}

bool has_own_dispatch(const at::Tensor& t) { return t.key_set().has(c10::DispatchKey::Python); }

// Whether the call has to go through the dispatcher.
bool watched(std::initializer_list<const at::Tensor*> tensors) {
    constexpr c10::DispatchKeySet watchers({c10::DispatchKey::Tracer, c10::DispatchKey::Python, c10::DispatchKey::PreDispatch, c10::DispatchKey::FuncTorchDynamicLayerFrontMode});
    const auto tls = c10::impl::tls_local_dispatch_key_set();
    if (((tls.included_ - tls.excluded_) & watchers) != c10::DispatchKeySet()) return true;
    for (const at::Tensor* t : tensors)
        if (t != nullptr && has_own_dispatch(*t)) return true;
    return false;
}
// Sizes that are symbols cannot be checked here.
bool symbolic(std::initializer_list<const at::Tensor*> tensors) {
    for (const at::Tensor* t : tensors)
        if (t != nullptr && t->unsafeGetTensorImpl()->has_symbolic_sizes_strides()) return true;
    return false;
}
PyObject* not_implemented() { Py_RETURN_NOTIMPLEMENTED; }

int* status_word(int device) {
    TORCH_CHECK(device >= 0 && device < kMaxDevices, "device index out of range");
    if (g_status_words[device] == nullptr) {
        PyObject* r = PyObject_CallFunction(g_status, "i", device);
        if (r == nullptr) throw python_error();
        g_status_words[device] = static_cast<int*>(PyLong_AsVoidPtr(r));
        Py_DECREF(r);
        if (PyErr_Occurred()) throw python_error();
    }
    return g_status_words[device];
}

void check(int status, const char* what) {
    if (status == FEATHER_OK) return;
    PyErr_Format(g_error, "%s failed (status %d): %s", what, status, g_lib.error());
    throw python_error();
}

// A matrix of contiguous rows over a tensor's last dimension, without a copy where its strides allow; `hold` keeps a copy alive.
struct Rows {
    at::Tensor hold;
    void* ptr;
    int64_t ld;
};
Rows rows_of(const at::Tensor& t, int64_t cols) {
    const auto sizes = t.sizes();
    const auto strides = t.strides();
    int64_t ld = cols, count = 1, next = -1;
    bool ok = (strides.back() == 1 || cols == 1) && !t.is_neg();
    for (int64_t d = t.dim() - 2; ok && d >= 0; --d) {
        if (sizes[d] == 1) continue;
        if (next < 0) ld = strides[d];
        else ok = strides[d] == next;
        next = strides[d] * sizes[d];
        count *= sizes[d];
    }
    if (ok && (count <= 1 || ld >= cols)) return {at::Tensor(), t.data_ptr(), ld};
    at::Tensor copy = t.clone(at::MemoryFormat::Contiguous).resolve_neg();
    void* const p = copy.data_ptr();
    return {std::move(copy), p, cols};
}

int64_t scale_tiles(int64_t n) { return (n + 127) / 128; }
at::Tensor empty(at::IntArrayRef sizes, at::ScalarType type, at::Device device) { return at::Tensor(at::detail::empty_cuda(sizes, type, device, c10::nullopt)); }

// ------------------------------------------------------------------------------------------------ MXFP4
struct Packed {
    const at::Tensor &data, &scales;
    int64_t rows, k;
};

Packed packed(const at::Tensor& data, const at::Tensor& scales, const char* what) {
    TORCH_CHECK(data.dim() == 2 && data.scalar_type() == at::kByte, what, " must be a uint8 [rows, K/2] tensor");
    const int64_t rows = data.size(0), k = data.size(1) * 2;
    TORCH_CHECK(k != 0 && k % 32 == 0, what, ": K must be a positive multiple of 32, got ", k);
    TORCH_CHECK(scales.scalar_type() == at::kByte && scales.dim() == 3 && scales.size(0) == scale_tiles(rows) && scales.size(1) == scale_tiles(k) && scales.size(2) == 512, what,
                "_scales must be uint8 [", scale_tiles(rows), ", ", scale_tiles(k), ", 512] (prepack_mxfp4_scales lays [rows, K/32] bytes out), got ", scales.scalar_type(), " ",
                scales.sizes());
    TORCH_CHECK(data.is_cuda() && scales.is_cuda(), what, " and its scales must be CUDA tensors");
    TORCH_CHECK(scales.device() == data.device(), what, "_scales must be on the same device as ", what);
    TORCH_CHECK(data.is_contiguous() && scales.is_contiguous(), what, " and its scales must be contiguous");
    TORCH_CHECK((has_own_dispatch(data) || aligned16(data.data_ptr())) && (has_own_dispatch(scales) || aligned16(scales.data_ptr())), what, " and its scales must be 16-byte aligned");
    return {data, scales, rows, k};
}

void check_source(const at::Tensor& x) {
    TORCH_CHECK(x.is_cuda(), "x must be a CUDA tensor");
    TORCH_CHECK(source_code(x.scalar_type()) >= 0, "cannot quantise ", x.scalar_type(), " (expected float32, bfloat16 or float16)");
}

PyObject* py_quantize(PyObject*, PyObject* const* args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    TORCH_CHECK(n == 1 || n == 2, "quantize(x[, direct])");
    const bool direct = n == 2;
    const at::Tensor& x = tensor(args[0], "x");
    refuse_grad({&x}, "MXFP4 operators have");
    if (!direct && symbolic({&x})) return not_implemented();
    check_source(x);
    TORCH_CHECK(x.dim() == 2 && x.size(1) != 0 && x.size(1) % 32 == 0, "MXFP4 needs a 2D tensor with K a positive multiple of 32, got ", x.sizes());
    if (!direct && watched({&x})) return not_implemented();
    const int64_t rows = x.size(0), k = x.size(1);
    at::Tensor data, scales;
    int status = FEATHER_OK;
    {
        WithoutGil released;
        const c10::cuda::CUDAGuard guard(x.device());
        data = empty({rows, k / 2}, at::kByte, x.device());
        scales = empty({scale_tiles(rows), scale_tiles(k), 512}, at::kByte, x.device());
        if (rows != 0) {
            const Rows src = rows_of(x, k);
            status = g_lib.quantize(src.ptr, source_code(x.scalar_type()), rows, k, src.ld, data.data_ptr<uint8_t>(), scales.data_ptr<uint8_t>(),
                                    c10::cuda::getCurrentCUDAStream(x.device().index()).stream());
        }
    }
    check(status, "feather_mxfp4_quantize");
    PyObject* const out = PyTuple_New(2);
    if (out == nullptr) throw python_error();
    PyTuple_SET_ITEM(out, 0, THPVariable_Wrap(std::move(data)));
    PyTuple_SET_ITEM(out, 1, THPVariable_Wrap(std::move(scales)));
    return out;
    END_HANDLE_TH_ERRORS
}

PyObject* py_dequantize(PyObject*, PyObject* const* args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    TORCH_CHECK(n == 3 || n == 4, "dequantize(data, scales, dtype[, direct])");
    const bool direct = n == 4;
    const auto dtype = optional_dtype(args[2], "dtype");
    TORCH_CHECK(dtype && source_code(*dtype) >= 0, "dtype must be float32, bfloat16 or float16");
    const at::Tensor &data = tensor(args[0], "data"), &scales = tensor(args[1], "scales");
    if (!direct && symbolic({&data, &scales})) return not_implemented();
    const Packed a = packed(data, scales, "data");
    if (!direct && watched({&data, &scales})) return not_implemented();
    at::Tensor out;
    int status = FEATHER_OK;
    {
        WithoutGil released;
        const c10::cuda::CUDAGuard guard(a.data.device());
        out = empty({a.rows, a.k}, *dtype, a.data.device());
        if (a.rows != 0)
            status = g_lib.dequantize(a.data.data_ptr<uint8_t>(), a.scales.data_ptr<uint8_t>(), a.rows, a.k, source_code(*dtype), out.data_ptr(),
                                      c10::cuda::getCurrentCUDAStream(a.data.device().index()).stream());
    }
    check(status, "feather_mxfp4_dequantize");
    return THPVariable_Wrap(std::move(out));
    END_HANDLE_TH_ERRORS
}

// The checks of the product beyond its operands' own; returns N.
void check_product(const at::Device& device, int64_t k, const Packed& b, const at::Tensor* bias, c10::optional<at::ScalarType> out_dtype) {
    TORCH_CHECK(k == b.k, "a and b must have the same K, got ", k, " and ", b.k);
    TORCH_CHECK(b.data.device() == device, "b must be on the same device as a");
    TORCH_CHECK(b.rows != 0, "b must have at least one row");
    if (bias != nullptr) {
        TORCH_CHECK(bias->device() == device, "bias must be on the same device as a");
        TORCH_CHECK(bias->scalar_type() == *out_dtype, "bias must have the out dtype");
        TORCH_CHECK(bias->numel() == b.rows && bias->is_contiguous(), "bias must be contiguous with N elements");
        TORCH_CHECK(!bias->is_neg(), "bias carries its sign as a flag: resolve_neg() it first");
    }
}

int launch_product(const uint8_t* a, const uint8_t* a_scales, const Packed& b, const at::Tensor* bias, const at::Tensor& out, int64_t m, int64_t ldc, int* status_dev, cudaStream_t stream) {
    return g_lib.mm(a, a_scales, b.data.data_ptr<uint8_t>(), b.scales.data_ptr<uint8_t>(), bias != nullptr ? bias->data_ptr() : nullptr, out.data_ptr(), m, b.rows, b.k, ldc,
                    out.scalar_type() == at::kBFloat16 ? FEATHER_OUT_BF16 : FEATHER_OUT_FP16, status_dev, stream);
}

PyObject* py_mm(PyObject*, PyObject* const* args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    TORCH_CHECK(n == 6 || n == 7, "mm(a, a_scales, b, b_scales, bias, out_dtype[, out or None])");
    const bool direct = n == 7;
    const at::Tensor* const bias = optional_tensor(args[4], "bias");
    const auto out_dtype = optional_dtype(args[5], "out_dtype");
    const at::Tensor* const given = n == 7 ? optional_tensor(args[6], "out") : nullptr;
    refuse_grad({bias, given}, "MXFP4 operators have");
    TORCH_CHECK(out_dtype && (*out_dtype == at::kHalf || *out_dtype == at::kBFloat16), "out_dtype must be float16 or bfloat16");
    const at::Tensor &a_data = tensor(args[0], "a"), &a_scales = tensor(args[1], "a_scales"), &b_data = tensor(args[2], "b"), &b_scales = tensor(args[3], "b_scales");
    if (!direct && symbolic({&a_data, &a_scales, &b_data, &b_scales, bias})) return not_implemented();
    const Packed a = packed(a_data, a_scales, "a"), b = packed(b_data, b_scales, "b");
    const at::Device device = a.data.device();
    check_product(device, a.k, b, bias, out_dtype);
    int64_t ldc = b.rows;
    if (given != nullptr) {
        TORCH_CHECK(given->device() == device, "out must be on the same device as a");
        TORCH_CHECK(given->scalar_type() == *out_dtype, "out must have the out dtype");
        TORCH_CHECK(given->dim() == 2 && given->size(0) == a.rows && given->size(1) == b.rows, "out must be [", a.rows, ", ", b.rows, "], got ", given->sizes());
        TORCH_CHECK(b.rows == 1 || given->stride(1) == 1, "out must have contiguous columns");
        TORCH_CHECK(!given->is_neg(), "out carries its sign as a flag: resolve_neg() it first");
        TORCH_CHECK(a.rows <= 1 || given->stride(0) >= b.rows, "rows of out overlap");
        if (a.rows > 1) ldc = given->stride(0);
    }
    if (!direct && watched({&a_data, &a_scales, &b_data, &b_scales, bias})) return not_implemented();
    int* const status_dev = status_word(device.index());
    at::Tensor out;
    int status = FEATHER_OK;
    {
        WithoutGil released;
        const c10::cuda::CUDAGuard guard(device);
        out = given != nullptr ? *given : empty({a.rows, b.rows}, *out_dtype, device);
        if (a.rows != 0)
            status = launch_product(a.data.data_ptr<uint8_t>(), a.scales.data_ptr<uint8_t>(), b, bias, out, a.rows, ldc, status_dev, c10::cuda::getCurrentCUDAStream(device.index()).stream());
    }
    check(status, "feather_mxfp4_mm");
    return THPVariable_Wrap(std::move(out));
    END_HANDLE_TH_ERRORS
}

PyObject* py_linear(PyObject*, PyObject* const* args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    TORCH_CHECK(n == 5 || n == 6, "linear(x, b, b_scales, bias, out_dtype[, direct])");
    const bool direct = n == 6;
    const at::Tensor& x = tensor(args[0], "x");
    const at::Tensor* const bias = optional_tensor(args[3], "bias");
    auto out_dtype = optional_dtype(args[4], "out_dtype");
    refuse_grad({&x, bias}, "MXFP4 operators have");
    const at::Tensor &b_data = tensor(args[1], "b"), &b_scales = tensor(args[2], "b_scales");
    if (!direct && symbolic({&x, &b_data, &b_scales, bias})) return not_implemented();
    TORCH_CHECK(x.dim() != 0, "x must have at least one dimension");
    check_source(x);
    if (!out_dtype) out_dtype = x.scalar_type() == at::kFloat ? at::kBFloat16 : x.scalar_type();
    TORCH_CHECK(*out_dtype == at::kHalf || *out_dtype == at::kBFloat16, "out_dtype must be float16 or bfloat16");
    const int64_t k = x.size(-1);
    TORCH_CHECK(k != 0 && k % 32 == 0, "x: K must be a positive multiple of 32, got ", k);
    const Packed b = packed(b_data, b_scales, "b");
    const at::Device device = x.device();
    check_product(device, k, b, bias, out_dtype);
    if (!direct && watched({&x, &b_data, &b_scales, bias})) return not_implemented();
    int* const status_dev = status_word(device.index());
    const int64_t m = x.numel() / k;
    at::Tensor out;
    int quantised = FEATHER_OK, status = FEATHER_OK;
    {
        WithoutGil released;
        const c10::cuda::CUDAGuard guard(device);
        at::DimVector sizes(x.sizes().begin(), x.sizes().end());
        sizes.back() = b.rows;
        out = empty(sizes, *out_dtype, device);
        if (m != 0) {
            // scales first: their size keeps the data behind them aligned
            const int64_t scale_bytes = scale_tiles(m) * scale_tiles(k) * 512;
            const at::Tensor operand = empty({scale_bytes + m * (k / 2)}, at::kByte, device);
            uint8_t* const scales = operand.data_ptr<uint8_t>();
            const Rows src = rows_of(x, k);
            const cudaStream_t stream = c10::cuda::getCurrentCUDAStream(device.index()).stream();
            quantised = g_lib.quantize(src.ptr, source_code(x.scalar_type()), m, k, src.ld, scales + scale_bytes, scales, stream);
            if (quantised == FEATHER_OK) status = launch_product(scales + scale_bytes, scales, b, bias, out, m, b.rows, status_dev, stream);
        }
    }
    check(quantised, "feather_mxfp4_quantize");
    check(status, "feather_mxfp4_mm");
    return THPVariable_Wrap(std::move(out));
    END_HANDLE_TH_ERRORS
}

// ------------------------------------------------------------------------------------------------ fused norm
void check_operand(const at::Tensor& t, const char* name, const at::Device& device) {
    TORCH_CHECK(source_code(t.scalar_type()) >= 0, name, " must be float32, bfloat16 or float16");
    TORCH_CHECK(t.device() == device, name, " must be on the same device as x");
}

void check_vector(const at::Tensor* t, const char* name, int64_t cols, const at::Device& device) {
    if (t == nullptr) return;
    check_operand(*t, name, device);
    TORCH_CHECK(t->numel() == cols && t->is_contiguous(), name, " must be contiguous with ", cols, " elements");
}

// [cols], or x's shape with the token dimensions after some point of size 1.  Returns how many rows of x share a row of t.
int64_t check_modulation(const at::Tensor* t, const char* name, const at::Tensor& x) {
    if (t == nullptr) return 1;
    check_operand(*t, name, x.device());
    const int64_t cols = x.size(-1), lead = x.dim() - 1, shift = x.dim() - t->dim();
    TORCH_CHECK(t->dim() != 0 && t->size(-1) == cols && shift >= 0, name, " must end in ", cols, " elements and have no more dimensions than x, got ", t->sizes());
    int64_t shared = 1;
    bool rest = false, ok = true;                       // past the last dimension that t has in full
    for (int64_t d = 0; d < lead; ++d) {
        const int64_t own = d < shift ? 1 : t->size(d - shift);
        if (!rest && own == x.size(d)) continue;
        rest = true;
        ok = ok && own == 1;
        shared *= x.size(d);
    }
    TORCH_CHECK(ok, name, " ", t->sizes(), " must have x's leading dimensions ", x.sizes().slice(0, lead), ", those after some point replaced by 1");
    return shared > 0 ? shared : 1;
}

Rows aligned_rows(const at::Tensor& t, int64_t cols, bool align) {
    Rows r = rows_of(t, cols);
    if (align && (!aligned16(r.ptr) || r.ld * t.element_size() % 16 != 0)) {
        at::Tensor copy = t.clone(at::MemoryFormat::Contiguous);
        void* const p = copy.data_ptr();
        return {std::move(copy), p, cols};
    }
    return r;
}

PyObject* py_norm(PyObject*, PyObject* const* args, Py_ssize_t n) {
    HANDLE_TH_ERRORS
    TORCH_CHECK(n == 15 || n == 16, "norm(x, y, gate, residual_scale, post_norm, post_weight, weight, bias, scale, shift, kind, eps, out_dtype, want_norm, packed[, direct])");
    const bool direct = n == 16;
    const at::Tensor& x = tensor(args[0], "x");
    const at::Tensor *const y = optional_tensor(args[1], "y"), *const gate = optional_tensor(args[2], "gate"), *const post_weight = optional_tensor(args[5], "post_weight"),
                     *const weight = optional_tensor(args[6], "weight"), *const bias = optional_tensor(args[7], "bias"), *const scale = optional_tensor(args[8], "scale"),
                     *const shift = optional_tensor(args[9], "shift");
    const double residual_scale = number(args[3]), eps = number(args[11]);
    const bool post_norm = truth(args[4]), want_norm = truth(args[13]), pack = truth(args[14]);
    auto out_dtype = optional_dtype(args[12], "out_dtype");
    refuse_grad({&x, y, gate, post_weight, weight, bias, scale, shift}, "gated_residual_norm has");
    if (!direct && symbolic({&x, y, gate, post_weight, weight, bias, scale, shift})) return not_implemented();
    TORCH_CHECK(x.is_cuda(), "x must be a CUDA tensor");
    TORCH_CHECK(source_code(x.scalar_type()) >= 0, "x must be float32, bfloat16 or float16");
    TORCH_CHECK(x.dim() != 0 && x.size(-1) != 0, "x must have at least one element in its last dimension");
    const bool rms = PyUnicode_Check(args[10]) && PyUnicode_CompareWithASCIIString(args[10], "rms") == 0;
    TORCH_CHECK(rms || (PyUnicode_Check(args[10]) && PyUnicode_CompareWithASCIIString(args[10], "layer") == 0), "kind must be 'rms' or 'layer'");
    TORCH_CHECK(eps >= 0.0, "eps must not be negative");
    const int64_t cols = x.size(-1);
    const at::Device device = x.device();
    TORCH_CHECK(cols <= 16384, "the last dimension must be at most 16384, got ", cols);
    if (y == nullptr) {
        TORCH_CHECK(gate == nullptr && !post_norm && post_weight == nullptr, "gate, post_norm and post_weight need y");
        TORCH_CHECK(want_norm, "without y there is only the norm to compute");
    } else {
        check_operand(*y, "y", device);
        TORCH_CHECK(y->sizes() == x.sizes(), "y must have x's shape ", x.sizes(), ", got ", y->sizes());
        TORCH_CHECK(post_weight == nullptr || post_norm, "post_weight needs post_norm");
    }
    TORCH_CHECK(want_norm || (weight == nullptr && bias == nullptr && scale == nullptr && shift == nullptr && !pack),
                "weight, bias, scale, shift and packed belong to the norm that want_norm=False leaves out");
    if (!out_dtype) {
        out_dtype = x.scalar_type() != at::kFloat || y == nullptr ? x.scalar_type() : y->scalar_type();
        if (pack && *out_dtype == at::kFloat) out_dtype = at::kBFloat16;
    }
    TORCH_CHECK(source_code(*out_dtype) >= 0, "out_dtype must be float32, bfloat16 or float16");
    TORCH_CHECK(!pack || cols % 32 == 0, "an MXFP4 result needs a last dimension that is a multiple of 32, got ", cols);
    TORCH_CHECK(!pack || *out_dtype != at::kFloat, "an MXFP4 result is rounded to out_dtype first: float16 or bfloat16");
    check_vector(weight, "weight", cols, device);
    check_vector(bias, "bias", cols, device);
    check_vector(post_weight, "post_weight", cols, device);
    feather_norm_args a{};
    a.gate_rows = check_modulation(gate, "gate", x);
    a.scale_rows = check_modulation(scale, "scale", x);
    a.shift_rows = check_modulation(shift, "shift", x);
    if (!direct && watched({&x, y, gate, post_weight, weight, bias, scale, shift})) return not_implemented();
    a.status_dev = status_word(device.index());

    at::Tensor r, h, h_scales;
    int status = FEATHER_OK;
    {
        WithoutGil released;
        const c10::cuda::CUDAGuard guard(device);
        const int64_t rows = x.numel() / cols;
        if (y != nullptr) r = empty(x.sizes(), x.scalar_type(), device);
        if (pack) {
            h = empty({rows, cols / 2}, at::kByte, device);
            h_scales = empty({scale_tiles(rows), scale_tiles(cols), 512}, at::kByte, device);
        } else if (want_norm) {
            h = empty(x.sizes(), *out_dtype, device);
        }
        if (rows != 0) {
            at::Tensor hold[8];
            int held = 0;
            const auto put = [&](const at::Tensor* t, const void*& ptr, int& dtype, int64_t* ld) {
                if (t == nullptr) return;
                Rows m = aligned_rows(*t, cols, pack);
                ptr = m.ptr;
                dtype = source_code(t->scalar_type());
                if (ld != nullptr) *ld = m.ld;
                hold[held++] = std::move(m.hold);
            };
            a.rows = rows;
            a.cols = cols;
            a.ldr = a.ldh = cols;
            put(&x, a.x, a.x_dtype, &a.ldx);
            put(y, a.y, a.y_dtype, &a.ldy);
            put(weight, a.weight, a.weight_dtype, nullptr);
            put(bias, a.bias, a.bias_dtype, nullptr);
            put(post_weight, a.post_weight, a.post_weight_dtype, nullptr);
            put(gate, a.gate, a.gate_dtype, &a.gate_ld);
            put(scale, a.scale, a.scale_dtype, &a.scale_ld);
            put(shift, a.shift, a.shift_dtype, &a.shift_ld);
            if (r.defined()) a.r = r.data_ptr();
            if (h.defined()) a.h = h.data_ptr();
            if (h_scales.defined()) a.h_scales = h_scales.data_ptr<uint8_t>();
            a.h_dtype = source_code(*out_dtype);
            a.residual_scale = static_cast<float>(residual_scale);
            a.eps = static_cast<float>(eps);
            a.kind = rms ? FEATHER_NORM_RMS : FEATHER_NORM_LAYER;
            a.post_norm = post_norm ? 1 : 0;
            status = g_lib.norm(&a, c10::cuda::getCurrentCUDAStream(device.index()).stream());
        }
    }
    check(status, "feather_gated_norm");
    PyObject* first;
    if (r.defined()) {
        first = THPVariable_Wrap(std::move(r));
    } else {
        Py_INCREF(args[0]);
        first = args[0];
    }
    PyObject* second;
    if (pack) {
        second = PyTuple_New(2);
        if (second == nullptr) throw python_error();
        PyTuple_SET_ITEM(second, 0, THPVariable_Wrap(std::move(h)));
        PyTuple_SET_ITEM(second, 1, THPVariable_Wrap(std::move(h_scales)));
    } else if (h.defined()) {
        second = THPVariable_Wrap(std::move(h));
    } else {
        Py_INCREF(Py_None);
        second = Py_None;
    }
    PyObject* const out = PyTuple_New(2);
    if (out == nullptr) throw python_error();
    PyTuple_SET_ITEM(out, 0, first);
    PyTuple_SET_ITEM(out, 1, second);
    return out;
    END_HANDLE_TH_ERRORS
}

// bind(addresses of quantize, dequantize, mm, norm, last_error_string; error class; status(device index) -> address)
PyObject* py_bind(PyObject*, PyObject* args) {
    unsigned long long p[5];
    PyObject *error, *status;
    if (!PyArg_ParseTuple(args, "KKKKKOO", &p[0], &p[1], &p[2], &p[3], &p[4], &error, &status)) return nullptr;
    g_lib.quantize = reinterpret_cast<decltype(g_lib.quantize)>(p[0]);
    g_lib.dequantize = reinterpret_cast<decltype(g_lib.dequantize)>(p[1]);
    g_lib.mm = reinterpret_cast<decltype(g_lib.mm)>(p[2]);
    g_lib.norm = reinterpret_cast<decltype(g_lib.norm)>(p[3]);
    g_lib.error = reinterpret_cast<decltype(g_lib.error)>(p[4]);
    Py_INCREF(error);
    Py_INCREF(status);
    g_error = error;
    g_status = status;
    Py_RETURN_NONE;
}

PyMethodDef g_methods[] = {
    {"bind", py_bind, METH_VARARGS, nullptr},
    {"quantize", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(py_quantize)), METH_FASTCALL, nullptr},
    {"dequantize", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(py_dequantize)), METH_FASTCALL, nullptr},
    {"mm", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(py_mm)), METH_FASTCALL, nullptr},
    {"linear", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(py_linear)), METH_FASTCALL, nullptr},
    {"norm", reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(py_norm)), METH_FASTCALL, nullptr},
    {nullptr, nullptr, 0, nullptr},
};

PyModuleDef g_module = {PyModuleDef_HEAD_INIT, "_feather_binding", nullptr, -1, g_methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__feather_binding() {
    return PyModule_Create(&g_module);
}
