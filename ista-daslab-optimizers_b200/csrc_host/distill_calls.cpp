// Host side of the distillation operators in native code: looks the tensors over, allocates the outputs and calls the library.
//
// What bounds a call over few rows is the host: the same checks, allocations and the autograd node in Python take 15 to 100 us, more than the kernels.
// Here a call takes a few.  A call that is not as it should be (a tensor elsewhere, another type or shape, a gradient asked for where there is none) returns None
// before anything has happened; the Python side (distillation.py) then says what is wrong.  What torch throws on the way becomes the Python exception it stands
// for, and a status of the library is returned as a number.
#define PY_SSIZE_T_CLEAN
#include <Python.h>
#include <ATen/ATen.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/core/AutogradState.h>
#include <c10/core/GradMode.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/python_variable.h>

#include <exception>
#include <optional>
#include <string>

#include "microadam_b200.h"

namespace {

// The library's entry points, handed over once (`bind`): this file is not linked against it.
struct Library {
    decltype(&mab_quantize_rows) quantize_rows = nullptr;
    decltype(&mab_int8_matmul) int8_matmul = nullptr;
    decltype(&mab_topk_logits) topk_logits = nullptr;
    decltype(&mab_distill_loss) distill_loss = nullptr;
    decltype(&mab_distill_grad) distill_grad = nullptr;
    decltype(&mab_distill_step) distill_step = nullptr;
    decltype(&mab_last_error) last_error = nullptr;
} g_library;

struct ReleasedInterpreter {
    PyThreadState* saved = PyEval_SaveThread();
    ~ReleasedInterpreter() { PyEval_RestoreThread(saved); }
};

// The device of a call, current while this lives, and its stream.
struct Target {
    std::optional<c10::cuda::CUDAGuard> guard;
    void* stream;
    explicit Target(const at::Tensor& t) {
        const auto device = t.device().index();
        if (c10::cuda::current_device() != device) guard.emplace(device);
        stream = c10::cuda::getCurrentCUDAStream(device).stream();
    }
};

PyObject* raise_python() {
    torch::translate_exception_to_python(std::current_exception());
    return nullptr;
}

bool is_float(const at::Tensor& t) { return t.scalar_type() == at::kFloat || t.scalar_type() == at::kBFloat16; }
int code(const at::Tensor& t) { return t.scalar_type() == at::kFloat ? MAB_F32 : MAB_BF16; }

// A new tensor, straight from the device's allocator.
at::Tensor fresh(at::IntArrayRef sizes, at::ScalarType type, const at::Tensor& like) { return at::detail::empty_cuda(sizes, type, like.device(), std::nullopt); }

// A matrix on a CUDA device whose rows are contiguous: its address and their distance.  (A tensor whose negation torch has put off, the imaginary part of a conjugate, holds other numbers than its memory.)
struct Rows {
    void* p = nullptr;
    int64_t pitch = 0;
    bool of(const at::Tensor& t) {
        if (t.layout() != at::kStrided || t.dim() != 2 || !t.is_cuda() || t.is_neg()) return false;
        const int64_t rows = t.size(0), cols = t.size(1);
        if (cols > 1 && t.stride(1) != 1) return false;
        pitch = rows > 1 ? t.stride(0) : std::max<int64_t>(cols, 1);
        p = t.data_ptr();
        return pitch >= cols;
    }
};

// n contiguous float32 values on the device of `like`.
bool is_vector(const at::Tensor& t, int64_t n, const at::Tensor& like) {
    return t.scalar_type() == at::kFloat && t.dim() == 1 && t.size(0) == n && t.device() == like.device() && t.is_contiguous() && !t.is_neg();
}
float* vector_at(const at::Tensor& t) { return t.defined() ? static_cast<float*>(t.data_ptr()) : nullptr; }

// An argument that is a tensor, or None where `optional`.
bool tensor(PyObject* o, at::Tensor* out, bool optional = false) {
    if (optional && o == Py_None) return true;
    if (!THPVariable_Check(o)) return false;
    *out = THPVariable_Unpack(o);
    return true;
}
// A tangent of forward-mode differentiation, which none of the operators carries on.
bool has_tangent(const at::Tensor& t) { return t.defined() && c10::AutogradState::get_tls_state().get_fw_grad_mode() && t._fw_grad(/*level=*/0).defined(); }
bool wants_gradient(const at::Tensor& t) { return t.defined() && ((t.requires_grad() && c10::GradMode::is_enabled()) || has_tangent(t)); }

// A tensor of the caller's that the library has written to: autograd has to know, where it keeps it (or what shares its memory) for a backward pass.
void written(const at::Tensor& t, PyObject* given) {
    if (given != Py_None && !t.is_inference()) torch::autograd::impl::bump_version(t);
}

PyObject* tuple(std::initializer_list<at::Tensor> tensors) {
    PyObject* r = PyTuple_New(static_cast<Py_ssize_t>(tensors.size()));
    if (r == nullptr) return nullptr;
    Py_ssize_t i = 0;
    for (const at::Tensor& t : tensors) {
        PyObject* o = THPVariable_Wrap(t);
        if (o == nullptr) { Py_DECREF(r); return nullptr; }
        PyTuple_SET_ITEM(r, i++, o);
    }
    return r;
}
PyObject* answer(int status, std::initializer_list<at::Tensor> tensors) { return status == MAB_OK ? tuple(tensors) : PyLong_FromLong(status); }

#define EXPECT(condition) do { if (!(condition)) Py_RETURN_NONE; } while (0)

// bind(addresses of the seven entry points, in the order of Library)
PyObject* bind(PyObject*, PyObject* args) {
    unsigned long long a[7];
    if (!PyArg_ParseTuple(args, "KKKKKKK", &a[0], &a[1], &a[2], &a[3], &a[4], &a[5], &a[6])) return nullptr;
    auto set = [](auto& fn, unsigned long long at) { fn = reinterpret_cast<std::remove_reference_t<decltype(fn)>>(static_cast<uintptr_t>(at)); };
    set(g_library.quantize_rows, a[0]);
    set(g_library.int8_matmul, a[1]);
    set(g_library.topk_logits, a[2]);
    set(g_library.distill_loss, a[3]);
    set(g_library.distill_grad, a[4]);
    set(g_library.distill_step, a[5]);
    set(g_library.last_error, a[6]);
    Py_RETURN_NONE;
}

// quantize_rows(x, codes or None, scales or None)
PyObject* quantize_rows(PyObject*, PyObject* const* args, Py_ssize_t n) try {
    at::Tensor x, codes, scales;
    EXPECT(n == 3 && tensor(args[0], &x) && tensor(args[1], &codes, true) && tensor(args[2], &scales, true));
    Rows xr, cr;
    EXPECT(xr.of(x) && is_float(x) && !wants_gradient(x));
    const int64_t rows = x.size(0), cols = x.size(1);
    const Target on(x);
    if (!codes.defined()) {
        codes = fresh({rows, (cols + 15) / 16 * 16}, at::kChar, x);
        if (cols % 16) codes = codes.narrow(1, 0, cols);
    }
    EXPECT(cr.of(codes) && codes.scalar_type() == at::kChar && codes.sizes() == x.sizes() && codes.device() == x.device());
    if (!scales.defined()) scales = fresh({rows}, at::kFloat, x);
    EXPECT(is_vector(scales, rows, x) && !wants_gradient(scales));
    int status;
    {
        const ReleasedInterpreter other_threads_run;
        status = g_library.quantize_rows(rows, cols, xr.p, code(x), xr.pitch, static_cast<int8_t*>(cr.p), cr.pitch, vector_at(scales), on.stream);
    }
    written(codes, args[1]);
    written(scales, args[2]);
    return answer(status, {codes, scales});
} catch (...) {
    return raise_python();
}

// int8_matmul(a, b, a_scales, b_scales, bias or None, out or None, whether a new out is bfloat16)
PyObject* int8_matmul(PyObject*, PyObject* const* args, Py_ssize_t n) try {
    at::Tensor a, b, a_scales, b_scales, bias, out;
    EXPECT(n == 7 && tensor(args[0], &a) && tensor(args[1], &b) && tensor(args[2], &a_scales) && tensor(args[3], &b_scales) && tensor(args[4], &bias, true) &&
           tensor(args[5], &out, true));
    Rows ar, br, outr;
    EXPECT(ar.of(a) && br.of(b) && a.scalar_type() == at::kChar && b.scalar_type() == at::kChar && a.device() == b.device() && a.size(1) == b.size(1));
    const int64_t m = a.size(0), channels = b.size(0), k = a.size(1);
    EXPECT(is_vector(a_scales, m, a) && is_vector(b_scales, channels, a) && (!bias.defined() || is_vector(bias, channels, a)));
    EXPECT(!wants_gradient(a_scales) && !wants_gradient(b_scales) && !wants_gradient(bias));
    const Target on(a);
    if (!out.defined()) out = fresh({m, channels}, args[6] == Py_True ? at::kBFloat16 : at::kFloat, a);
    EXPECT(outr.of(out) && is_float(out) && out.size(0) == m && out.size(1) == channels && out.device() == a.device() && !wants_gradient(out));
    if (m == 1) ar.pitch = (ar.pitch + 15) / 16 * 16;              // one row: no distance
    if (channels == 1) br.pitch = (br.pitch + 15) / 16 * 16;
    int status;
    {
        const ReleasedInterpreter other_threads_run;
        status = g_library.int8_matmul(m, channels, k, static_cast<const int8_t*>(ar.p), ar.pitch, static_cast<const int8_t*>(br.p), br.pitch, vector_at(a_scales),
                                       vector_at(b_scales), vector_at(bias), outr.p, code(out), outr.pitch, on.stream);
    }
    written(out, args[5]);
    return answer(status, {out});
} catch (...) {
    return raise_python();
}

// topk_logits(logits, k, temperature)
PyObject* topk_logits(PyObject*, PyObject* const* args, Py_ssize_t n) try {
    at::Tensor z;
    EXPECT(n == 3 && tensor(args[0], &z) && PyLong_Check(args[1]) && PyFloat_Check(args[2]));
    const int64_t k = PyLong_AsLongLong(args[1]);
    if (k == -1 && PyErr_Occurred()) { PyErr_Clear(); Py_RETURN_NONE; }
    Rows zr;
    EXPECT(zr.of(z) && is_float(z) && !wants_gradient(z) && k >= 1 && k <= z.size(1));
    const Target on(z);
    const int64_t rows = z.size(0);
    at::Tensor values = fresh({rows, k}, z.scalar_type(), z), indices = fresh({rows, k}, at::kInt, z), rest = fresh({rows}, at::kFloat, z);
    const double temperature = PyFloat_AS_DOUBLE(args[2]);
    int status;
    {
        const ReleasedInterpreter other_threads_run;
        status = g_library.topk_logits(rows, z.size(1), k, zr.p, code(z), zr.pitch, temperature, values.data_ptr(), static_cast<int32_t*>(indices.data_ptr()),
                                       vector_at(rest), on.stream);
    }
    return answer(status, {values, indices, rest});
} catch (...) {
    return raise_python();
}

// A teacher's lists beside a student's logits.
struct Lists {
    at::Tensor logits, indices, values, rest, weights;
    Rows z;
    int64_t rows, vocab, k;
    bool of(PyObject* const* args) {
        if (!tensor(args[0], &logits) || !tensor(args[1], &indices) || !tensor(args[2], &values) || !tensor(args[3], &rest, true) || !tensor(args[4], &weights, true))
            return false;
        if (!z.of(logits) || !is_float(logits)) return false;
        rows = logits.size(0);
        vocab = logits.size(1);
        if (indices.scalar_type() != at::kInt || indices.dim() != 2 || indices.size(0) != rows || indices.device() != logits.device() || !indices.is_contiguous()) return false;
        k = indices.size(1);
        if (!is_float(values) || values.sizes() != indices.sizes() || values.device() != logits.device() || !values.is_contiguous() || values.is_neg()) return false;
        if ((rest.defined() && !is_vector(rest, rows, logits)) || (weights.defined() && !is_vector(weights, rows, logits))) return false;
        return !wants_gradient(values) && !wants_gradient(rest) && !wants_gradient(weights);
    }
};

// A status of the library inside an autograd node.
void throw_if(int status, const char* what) {
    if (status != MAB_OK) throw std::runtime_error(std::string(what) + " failed with status " + std::to_string(status) + ": " + g_library.last_error());
}

at::Tensor loss_of(const Lists& l, double temperature, at::Tensor* stats, at::Tensor* list_grad) {
    const Target on(l.logits);
    at::Tensor loss = fresh({l.rows}, at::kFloat, l.logits);
    *stats = fresh({l.rows, 2}, at::kFloat, l.logits);
    *list_grad = fresh({l.rows, l.k}, at::kFloat, l.logits);
    throw_if(g_library.distill_loss(l.rows, l.vocab, l.k, l.z.p, code(l.logits), l.z.pitch, static_cast<const int32_t*>(l.indices.data_ptr()), l.values.data_ptr(), code(l.values),
                                    vector_at(l.rest), vector_at(l.weights), temperature, vector_at(loss), vector_at(*stats), vector_at(*list_grad), on.stream), "distill_loss");
    return loss;
}

struct DistillLoss : torch::autograd::Function<DistillLoss> {
    static at::Tensor forward(torch::autograd::AutogradContext* ctx, const at::Tensor& logits, const Lists* lists, double temperature) {
        at::Tensor stats, list_grad;
        at::Tensor loss = loss_of(*lists, temperature, &stats, &list_grad);
        ctx->save_for_backward({logits, lists->indices, lists->weights, stats, list_grad});
        ctx->saved_data["temperature"] = temperature;
        return loss;
    }
    static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx, torch::autograd::variable_list upstream) {
        const auto saved = ctx->get_saved_variables();
        at::Tensor up = upstream[0];
        if (!up.defined()) return {at::Tensor(), at::Tensor(), at::Tensor()};
        const bool graph = c10::GradMode::is_enabled();
        at::Tensor grad;
        {
            const c10::AutoGradMode off(false);
            const Target on(up);
            const int64_t rows = up.size(0);
            // What hooks for saved tensors give back can be anything: the library only gets what is like what was saved (its distances may be others).  (The messages are literals:
            // a compiler that links its C++ library statically has streams of its own here, which do not know torch's locale.)
            auto back = [&](size_t i, at::ScalarType type) {
                const at::Tensor& t = saved[i];
                TORCH_CHECK(t.layout() == at::kStrided && t.is_cuda() && t.device() == up.device() && t.scalar_type() == type && t.dim() >= 1 && t.size(0) == rows,
                            "distill_loss: a saved tensor came back with another device, layout, type or number of rows (hooks for saved tensors have to give back what they got)");
                return t.resolve_neg();
            };
            const at::Tensor indices = back(1, at::kInt).contiguous(), stats = back(3, at::kFloat).contiguous(), list_grad = back(4, at::kFloat).contiguous();
            const at::Tensor weights = saved[2].defined() ? back(2, at::kFloat).contiguous() : at::Tensor();
            at::Tensor logits = back(0, saved[0].scalar_type() == at::kBFloat16 ? at::kBFloat16 : at::kFloat);
            TORCH_CHECK(logits.dim() == 2 && indices.dim() == 2 && list_grad.sizes() == indices.sizes() && stats.dim() == 2 && stats.size(1) == 2 &&
                            (!weights.defined() || weights.dim() == 1),
                        "distill_loss: a saved tensor came back in another shape (hooks for saved tensors have to give back what they got)");
            Rows z;
            if (!z.of(logits)) {
                logits = logits.contiguous();
                z.of(logits);
            }
            const int64_t vocab = logits.size(1);
            if (up.scalar_type() != at::kFloat) up = up.to(at::kFloat);
            up = up.resolve_neg();
            grad = fresh({rows, vocab}, logits.scalar_type(), logits);
            throw_if(g_library.distill_grad(rows, vocab, indices.size(1), z.p, code(logits), z.pitch, static_cast<const int32_t*>(indices.data_ptr()), vector_at(weights),
                                            ctx->saved_data["temperature"].toDouble(), vector_at(stats), vector_at(list_grad), vector_at(up), up.stride(0),
                                            grad.data_ptr(), vocab, on.stream), "distill_loss backward");
        }
        if (graph) {                                     // somebody may differentiate the gradient: that is refused when it happens
            auto refuse = std::make_shared<torch::autograd::DelayedError>("distill_loss is differentiable once", 1);
            grad = (*refuse)({grad.requires_grad_()})[0];
        }
        return {grad, at::Tensor(), at::Tensor()};
    }
};

// distill_loss(logits, indices, values, rest or None, weights or None, temperature)
PyObject* distill_loss(PyObject*, PyObject* const* args, Py_ssize_t n) try {
    Lists l;
    EXPECT(n == 6 && PyFloat_Check(args[5]) && l.of(args) && !has_tangent(l.logits));
    const double temperature = PyFloat_AS_DOUBLE(args[5]);
    // (what the library refuses is found out here, without an exception)
    EXPECT(l.k >= 1 && l.k <= MAB_MAX_LIST && l.vocab >= 1 && l.vocab <= MAB_MAX_VOCAB && temperature > 1e-6 && temperature < 1e6);
    at::Tensor loss, stats, list_grad;
    {
        const ReleasedInterpreter other_threads_run;
        loss = wants_gradient(l.logits) ? DistillLoss::apply(l.logits, &l, temperature) : loss_of(l, temperature, &stats, &list_grad);
    }
    return THPVariable_Wrap(loss);
} catch (...) {
    return raise_python();
}

// distill_step(logits, indices, values, rest or None, weights or None, temperature, grad or None)
PyObject* distill_step(PyObject*, PyObject* const* args, Py_ssize_t n) try {
    Lists l;
    at::Tensor grad;
    EXPECT(n == 7 && PyFloat_Check(args[5]) && l.of(args) && tensor(args[6], &grad, true) && !has_tangent(l.logits) && !has_tangent(grad));
    const Target on(l.logits);
    if (!grad.defined()) grad = fresh({l.rows, l.vocab}, l.logits.scalar_type(), l.logits);
    Rows g;
    EXPECT(g.of(grad) && grad.sizes() == l.logits.sizes() && grad.scalar_type() == l.logits.scalar_type() && grad.device() == l.logits.device() && !grad.requires_grad());
    at::Tensor loss = fresh({l.rows}, at::kFloat, l.logits);
    const double temperature = PyFloat_AS_DOUBLE(args[5]);
    int status;
    {
        const ReleasedInterpreter other_threads_run;
        status = g_library.distill_step(l.rows, l.vocab, l.k, l.z.p, code(l.logits), l.z.pitch, static_cast<const int32_t*>(l.indices.data_ptr()), l.values.data_ptr(),
                                        code(l.values), vector_at(l.rest), vector_at(l.weights), temperature, vector_at(loss), g.p, g.pitch, on.stream);
    }
    written(grad, args[6]);
    return answer(status, {loss, grad});
} catch (...) {
    return raise_python();
}

PyCFunction fast(PyObject* (*f)(PyObject*, PyObject* const*, Py_ssize_t)) { return reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(f)); }

PyMethodDef methods[] = {{"bind", bind, METH_VARARGS, "Hands over the library's entry points."},
                         {"quantize_rows", fast(quantize_rows), METH_FASTCALL, nullptr},
                         {"int8_matmul", fast(int8_matmul), METH_FASTCALL, nullptr},
                         {"topk_logits", fast(topk_logits), METH_FASTCALL, nullptr},
                         {"distill_loss", fast(distill_loss), METH_FASTCALL, nullptr},
                         {"distill_step", fast(distill_step), METH_FASTCALL, nullptr},
                         {nullptr, nullptr, 0, nullptr}};

PyModuleDef module = {PyModuleDef_HEAD_INIT, "_distill_calls", "Native host side of the distillation operators.", -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__distill_calls(void) { return PyModule_Create(&module); }
