// Calls of the operators on feature rows from torch tensors: checks, outputs,
// workspaces and the current stream, then the C ABI (include/mdx_hip.h).
//
// A small norm or product is a few microseconds on the device; the same steps
// in Python with ctypes took 11 to 14 (31 for an AdamW step over 12 tensors), most
// of them in allocating and slicing outputs.  operators.py documents the
// functions and gives the exceptions: `init(refuse, fail)` takes
// refuse(message, path) and fail(status, message, name), which make them.
#include <Python.h>

#include <ATen/core/Tensor.h>
#include <ATen/hip/EmptyTensor.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/python_variable.h>

#include <algorithm>
#include <cmath>
#include <memory>
#include <string>
#include <utility>
#include <vector>

#include "../../include/mdx_hip.h"

namespace {

constexpr int64_t kBlock = 128; // elements per scale along a row
constexpr auto kCodes = at::kFloat8_e4m3fn;
constexpr auto kScales = at::kFloat8_e8m0fnu;

PyObject* g_refuse = nullptr;
PyObject* g_fail = nullptr;

struct Refused {
    std::string message, path;
};
struct Failed {
    int status;
    std::string message;
    const char* name;
};
struct Raised {}; // a Python exception is set

int64_t ceil_div(int64_t v, int64_t by) { return (v + by - 1) / by; }

int kind_of(at::ScalarType t) {
    switch (t) {
        case at::kFloat: return MDX_FLOAT32;
        case at::kBFloat16: return MDX_BFLOAT16;
        case at::kHalf: return MDX_FLOAT16;
        default: return -1;
    }
}

std::string type_name(at::ScalarType t) {
    PyObject* s = PyObject_Str(reinterpret_cast<PyObject*>(torch::getTHPDtype(t)));
    if (s == nullptr) throw Raised{};
    std::string name = PyUnicode_AsUTF8(s);
    Py_DECREF(s);
    return name;
}

std::string shape_of(at::IntArrayRef shape) {
    std::string s = "(";
    for (size_t i = 0; i < shape.size(); ++i) s += (i ? ", " : "") + std::to_string(shape[i]);
    return s + (shape.size() == 1 ? ",)" : ")");
}

const at::Tensor& tensor(PyObject* o, const char* name) {
    if (!THPVariable_Check(o)) throw Refused{std::string(name) + " must be a torch tensor", name};
    return THPVariable_Unpack(o);
}

const at::Tensor& on_device(PyObject* o, const char* name) {
    const at::Tensor& t = tensor(o, name);
    if (!t.is_cuda()) throw Refused{std::string(name) + " must live on a HIP device", name};
    return t;
}

void same_device(const at::Tensor& t, const char* name, at::Device device) {
    if (t.device() != device)
        throw Refused{std::string(name) + " lives on " + t.device().str() + ", not on " + device.str(), name};
}

// Elements from row to row of a matrix on `device`; checks its layout.
int64_t pitch_of(const at::Tensor& t, const char* name, at::Device device) {
    same_device(t, name, device);
    if (t.dim() != 2) throw Refused{std::string(name) + " must be two-dimensional", name};
    const int64_t rows = t.size(0), width = t.size(1);
    if (width > 1 && t.stride(1) != 1) throw Refused{std::string(name) + " must have contiguous rows", name};
    if (rows <= 1) return ceil_div(std::max<int64_t>(width, 1), kBlock) * kBlock;
    if (t.stride(0) < width) throw Refused{"the rows of " + std::string(name) + " overlap", name};
    return t.stride(0);
}

void same_matrix(const at::Tensor& t, const char* name, const at::Tensor& like, const char* of) {
    if (t.sizes() != like.sizes() || t.scalar_type() != like.scalar_type())
        throw Refused{std::string(name) + " must have the shape and type of " + of + ": " + shape_of(like.sizes()) + ", "
                          + type_name(like.scalar_type()),
                      name};
}

float* vector_of(PyObject* o, const char* name, int64_t size, at::Device device) {
    if (!THPVariable_Check(o) || THPVariable_Unpack(o).device() != device)
        throw Refused{std::string(name) + " must be a torch tensor on " + device.str(), name};
    const at::Tensor& t = THPVariable_Unpack(o);
    if (t.scalar_type() != at::kFloat || t.dim() != 1 || t.size(0) != size || !t.is_contiguous())
        throw Refused{std::string(name) + " must be a contiguous float32 tensor of shape (" + std::to_string(size) + ",)",
                      name};
    return static_cast<float*>(t.data_ptr());
}

// Whether a number is one that the device reads: other tensors of one element are numbers as Python takes them.
bool moves(PyObject* o) {
    return THPVariable_Check(o) && THPVariable_Unpack(o).is_cuda() && THPVariable_Unpack(o).scalar_type() == at::kLong;
}

const int64_t* number_at(PyObject* o, const char* name, at::Device device) {
    const at::Tensor& t = THPVariable_Unpack(o);
    if (t.device() != device || t.numel() != 1)
        throw Refused{std::string(name) + " must be a whole number or an int64 tensor of one element on " + device.str(), name};
    return static_cast<const int64_t*>(t.data_ptr());
}

at::Tensor empty(at::IntArrayRef shape, at::ScalarType type, at::Device device) {
    return at::detail::empty_cuda(shape, type, device, std::nullopt); // past the dispatcher: 0.3 us less each
}

// A matrix whose rows start at multiples of `unit` bytes.
at::Tensor empty_pitched(int64_t rows, int64_t width, int64_t unit, at::ScalarType type, at::Device device) {
    const int64_t pitch = ceil_div(width, unit) * unit;
    const at::Tensor t = empty({rows, pitch}, type, device);
    if (pitch != width) { // its storage stays whole
        const int64_t sizes[2] = {rows, width}, strides[2] = {pitch, 1};
        t.unsafeGetTensorImpl()->set_sizes_and_strides(at::IntArrayRef(sizes), at::IntArrayRef(strides));
    }
    return t;
}

at::Tensor empty_codes(int64_t rows, int64_t width, at::Device d) { return empty_pitched(rows, width, kBlock, kCodes, d); }
at::Tensor empty_scales(int64_t rows, int64_t width, at::Device d) {
    return empty_pitched(rows, ceil_div(width, kBlock), 4, kScales, d);
}

// Tells autograd that a tensor which the caller gave was written: graphs that saved it refuse to go on.
void written_to(const at::Tensor& t) {
    if (!t.is_inference()) t.unsafeGetTensorImpl()->bump_version(); // tensors made in inference mode have no version
}

// The calls record no gradients.  Where one would have to go back through a call's results (grad mode is on and an input
// requires gradients), the results lead to an error in place of nothing: a gradient that is left out of a sum shows nowhere.
class History {
public:
    History(const char* name, std::initializer_list<std::pair<const at::Tensor*, const char*>> inputs) : name_(name) {
        for (const auto& [t, what] : inputs) {
            if (!t->defined() || t->unsafeGetTensorImpl()->autograd_meta() == nullptr) continue; // nothing to do with gradients
            if (t->_fw_grad(0).defined())
                throw Refused{std::string(what) + " has a forward gradient, and " + name + " gives none", what};
            if (t->requires_grad() && at::GradMode::is_enabled()) from_.emplace_back(t, what);
        }
    }
    // of an `out` that the caller gave, as for torch's own
    void refuse_out(const at::Tensor& out) const {
        if (!from_.empty()) throw Refused{std::string("out records no gradients, but ") + from_[0].second + " requires them", "out"};
        if (out.requires_grad() && at::GradMode::is_enabled())
            throw Refused{"out requires gradients: write into it under torch.no_grad()", "out"};
    }
    void goes_to(std::initializer_list<at::Tensor> results) const {
        if (from_.empty()) return;
        torch::autograd::edge_list edges;
        for (const auto& [t, what] : from_) edges.push_back(torch::autograd::impl::gradient_edge(*t));
        const std::shared_ptr<torch::autograd::Node> node(
            new torch::autograd::NotImplemented(std::string(name_) + " (it records no gradients: call it under torch.no_grad() "
                                                                     "or in a torch.autograd.Function)",
                                                std::move(edges)),
            torch::autograd::deleteNode);
        for (const at::Tensor& t : results)
            if (t.defined() && at::isFloatingType(t.scalar_type())) torch::autograd::set_history(t, node);
    }

private:
    const char* name_;
    std::vector<std::pair<const at::Tensor*, const char*>> from_;
};

void* stream_of(at::Device device) { return c10::hip::getCurrentHIPStream(device.index()).stream(); }

template <typename Call> void run(const char* name, Call&& call) {
    int status;
    std::string message;
    Py_BEGIN_ALLOW_THREADS
    status = call();
    if (status != MDX_OK) message = mdx_hip_last_error(nullptr);
    Py_END_ALLOW_THREADS
    if (status != MDX_OK) throw Failed{status, message, name};
}

template <typename Body> PyObject* guarded(Body&& body) {
    try {
        return body();
    } catch (const Refused& e) {
        PyObject* made = PyObject_CallFunction(g_refuse, "ss", e.message.c_str(), e.path.c_str());
        if (made != nullptr) {
            PyErr_SetObject(reinterpret_cast<PyObject*>(Py_TYPE(made)), made);
            Py_DECREF(made);
        }
    } catch (const Failed& e) {
        PyObject* made = PyObject_CallFunction(g_fail, "iss", e.status, e.message.c_str(), e.name);
        if (made != nullptr) {
            PyErr_SetObject(reinterpret_cast<PyObject*>(Py_TYPE(made)), made);
            Py_DECREF(made);
        }
    } catch (const Raised&) {
    } catch (const c10::OutOfMemoryError& e) {
        PyObject* made = PyObject_CallFunction(g_fail, "iss", int(MDX_OUT_OF_MEMORY), e.what_without_backtrace(), "torch");
        if (made != nullptr) {
            PyErr_SetObject(reinterpret_cast<PyObject*>(Py_TYPE(made)), made);
            Py_DECREF(made);
        }
    } catch (const std::exception& e) {
        PyErr_SetString(PyExc_RuntimeError, e.what());
    }
    return nullptr;
}

void expect(Py_ssize_t given, Py_ssize_t wanted) {
    if (given == wanted) return;
    PyErr_Format(PyExc_TypeError, "%zd arguments, not %zd", wanted, given);
    throw Raised{};
}

double number(PyObject* o) {
    const double v = PyFloat_AsDouble(o);
    if (v == -1.0 && PyErr_Occurred()) throw Raised{};
    return v;
}

int64_t whole(PyObject* o) {
    const long long v = PyLong_AsLongLong(o);
    if (v == -1 && PyErr_Occurred()) throw Raised{};
    return v;
}

PyObject* none() {
    Py_INCREF(Py_None);
    return Py_None;
}

PyObject* tuple_of(std::initializer_list<at::Tensor> tensors) {
    PyObject* t = PyTuple_New(Py_ssize_t(tensors.size()));
    if (t == nullptr) throw Raised{};
    Py_ssize_t i = 0;
    for (const at::Tensor& x : tensors) PyTuple_SET_ITEM(t, i++, x.defined() ? THPVariable_Wrap(x) : none());
    return t;
}

at::ScalarType type_of(PyObject* o, const char* message) {
    if (!THPDtype_Check(o)) throw Refused{message, "dtype"};
    return reinterpret_cast<THPDtype*>(o)->scalar_type;
}

// rms_norm(rows, gain, residual, eps, dtype) -> (values, scales, total, rstd)
PyObject* rms_norm(PyObject*, PyObject* const* o, Py_ssize_t n) {
    return guarded([&] {
        expect(n, 5);
        const at::Tensor& rows = on_device(o[0], "rows");
        const at::Device device = rows.device();
        const at::ScalarType type = rows.scalar_type();
        const int kind = kind_of(type);
        if (kind < 0)
            throw Refused{"rows must be float32, bfloat16 or float16, not " + type_name(type), "rows"};
        mdx_norm_args a{};
        a.x_pitch = pitch_of(rows, "rows", device);
        a.rows = rows.size(0);
        a.width = rows.size(1);
        a.dtype = a.out_dtype = kind;
        if (o[4] != Py_None) {
            const at::ScalarType to = type_of(o[4], "dtype must be a torch dtype");
            if (to == kCodes) a.out_dtype = MDX_FLOAT8;
            else if (to != type)
                throw Refused{"dtype must be " + type_name(type) + " or " + type_name(kCodes) + ", not " + type_name(to),
                              "dtype"};
        }
        a.eps = number(o[3]);
        if (!(a.eps > 0.0) || !std::isfinite(a.eps)) throw Refused{"eps must be positive and finite", "eps"};
        at::Tensor residual, values, scales, total;
        if (o[2] != Py_None) {
            residual = tensor(o[2], "residual");
            a.residual_pitch = pitch_of(residual, "residual", device);
            same_matrix(residual, "residual", rows, "rows");
            a.residual = residual.data_ptr();
        }
        a.gain = vector_of(o[1], "gain", a.width, device);
        const History history("rms_norm", {{&rows, "rows"}, {&THPVariable_Unpack(o[1]), "gain"}, {&residual, "residual"}});
        if (a.out_dtype == MDX_FLOAT8) {
            values = empty_codes(a.rows, a.width, device);
            scales = empty_scales(a.rows, a.width, device);
            a.scales = static_cast<uint8_t*>(scales.data_ptr());
            a.scales_pitch = scales.stride(0);
        } else {
            values = empty({a.rows, a.width}, type, device);
        }
        if (residual.defined()) {
            total = empty({a.rows, a.width}, type, device);
            a.total = total.data_ptr();
            a.total_pitch = a.width;
        }
        at::Tensor rstd = empty({a.rows}, at::kFloat, device);
        if (a.rows > 0 && a.width > 0) {
            a.x = rows.data_ptr();
            a.values = values.data_ptr();
            a.values_pitch = values.stride(0);
            a.rstd = static_cast<float*>(rstd.data_ptr());
            void* stream = stream_of(device);
            run("rms_norm", [&] { return mdx_hip_rms_norm(device.index(), &a, stream); });
        } else if (a.rows > 0) {
            rstd.fill_(1.0 / std::sqrt(a.eps));
        }
        history.goes_to({values, scales, total, rstd});
        return tuple_of({values, scales, total, rstd});
    });
}

// rms_norm_backward(grad, total, gain, rstd, grad_total) -> (grad_rows, grad_gain)
PyObject* rms_norm_backward(PyObject*, PyObject* const* o, Py_ssize_t n) {
    return guarded([&] {
        expect(n, 5);
        const at::Tensor& total = on_device(o[1], "total");
        const at::Device device = total.device();
        const at::ScalarType type = total.scalar_type();
        if (kind_of(type) < 0)
            throw Refused{"total must be float32, bfloat16 or float16, not " + type_name(type), "total"};
        mdx_norm_backward_args a{};
        a.dtype = kind_of(type);
        a.t_pitch = pitch_of(total, "total", device);
        a.rows = total.size(0);
        a.width = total.size(1);
        const at::Tensor& grad = tensor(o[0], "grad");
        a.grad_pitch = pitch_of(grad, "grad", device);
        same_matrix(grad, "grad", total, "total");
        at::Tensor other;
        if (o[4] != Py_None) {
            other = tensor(o[4], "grad_total");
            a.grad_total_pitch = pitch_of(other, "grad_total", device);
            same_matrix(other, "grad_total", total, "total");
            a.grad_total = other.data_ptr();
        }
        a.gain = vector_of(o[2], "gain", a.width, device);
        a.rstd = vector_of(o[3], "rstd", a.rows, device);
        const History history("rms_norm_backward", {{&grad, "grad"}, {&total, "total"}, {&THPVariable_Unpack(o[2]), "gain"},
                                                    {&THPVariable_Unpack(o[3]), "rstd"}, {&other, "grad_total"}});
        at::Tensor grad_rows = empty({a.rows, a.width}, type, device), grad_gain = empty({a.width}, at::kFloat, device);
        if (a.width > 0) {
            a.workspace_bytes = mdx_hip_rms_norm_backward_workspace(a.rows, a.width);
            at::Tensor workspace;
            if (a.workspace_bytes > 0) {
                workspace = empty({a.workspace_bytes}, at::kByte, device);
                a.workspace = workspace.data_ptr();
            }
            a.grad = grad.data_ptr();
            a.t = total.data_ptr();
            a.grad_x = grad_rows.data_ptr();
            a.grad_x_pitch = a.width;
            a.grad_gain = static_cast<float*>(grad_gain.data_ptr());
            void* stream = stream_of(device);
            run("rms_norm_backward", [&] { return mdx_hip_rms_norm_backward(device.index(), &a, stream); });
        }
        history.goes_to({grad_rows, grad_gain});
        return tuple_of({grad_rows, grad_gain});
    });
}

// quantize_fp8(matrix, tile, transpose) -> (codes, scales)
PyObject* quantize_fp8(PyObject*, PyObject* const* o, Py_ssize_t n) {
    return guarded([&] {
        expect(n, 3);
        const at::Tensor& matrix = on_device(o[0], "matrix");
        const at::Device device = matrix.device();
        if (kind_of(matrix.scalar_type()) < 0)
            throw Refused{"matrix must be float32, bfloat16 or float16, not " + type_name(matrix.scalar_type()), "matrix"};
        mdx_quantize_args a{};
        a.dtype = kind_of(matrix.scalar_type());
        a.x_pitch = pitch_of(matrix, "matrix", device);
        a.rows = matrix.size(0);
        a.width = matrix.size(1);
        a.tile = int32_t(whole(o[1]));
        a.transpose = PyObject_IsTrue(o[2]);
        if (a.transpose < 0) throw Raised{};
        const History history("quantize_fp8", {{&matrix, "matrix"}});
        const int64_t down = a.transpose ? a.width : a.rows, across = a.transpose ? a.rows : a.width;
        at::Tensor codes = empty_codes(down, across, device);
        at::Tensor scales = empty_scales(ceil_div(down, a.tile), across, device);
        if (a.rows > 0 && a.width > 0) {
            a.x = matrix.data_ptr();
            a.codes = static_cast<uint8_t*>(codes.data_ptr());
            a.codes_pitch = codes.stride(0);
            a.scales = static_cast<uint8_t*>(scales.data_ptr());
            a.scales_pitch = scales.stride(0);
            void* stream = stream_of(device);
            run("quantize_fp8", [&] { return mdx_hip_quantize_fp8(device.index(), &a, stream); });
        }
        history.goes_to({codes, scales});
        return tuple_of({codes, scales});
    });
}

// Whether each row starts at a multiple of `unit` bytes and its bytes up to the next such multiple are there.
bool readable(const at::Tensor& t, int64_t pitch, int64_t unit) {
    const int64_t rows = t.size(0), width = t.size(1);
    if (reinterpret_cast<uintptr_t>(t.data_ptr()) % size_t(unit) != 0 || (rows > 1 && pitch % unit != 0)) return false;
    if (width % unit == 0) return true;
    const int64_t end = t.storage_offset() + (rows > 1 ? (rows - 1) * pitch : 0) + ceil_div(width, unit) * unit;
    return end <= int64_t(t.storage().nbytes());
}

struct Operand {
    const at::Tensor &codes, &scales;
    int64_t pitch, scales_pitch;
    bool packed;
    Operand(PyObject* c, PyObject* s, const char* name, const char* scales_name, at::Device device)
        : codes(tensor(c, name)), scales(tensor(s, scales_name)), pitch(pitch_of(codes, name, device)),
          scales_pitch(pitch_of(scales, scales_name, device)) {
        if (codes.scalar_type() != kCodes)
            throw Refused{std::string(name) + " must be " + type_name(kCodes) + ", not " + type_name(codes.scalar_type()),
                          name};
        if (scales.scalar_type() != kScales)
            throw Refused{std::string(scales_name) + " must be " + type_name(kScales) + ", not "
                              + type_name(scales.scalar_type()),
                          scales_name};
        packed = readable(codes, pitch, 16) && readable(scales, scales_pitch, 4);
    }
};

// matmul_fp8(a, a_scales, b, b_scales, dtype, out) -> out
PyObject* matmul_fp8(PyObject*, PyObject* const* o, Py_ssize_t n) {
    return guarded([&] {
        expect(n, 6);
        const at::Device device = on_device(o[0], "a").device();
        const Operand a(o[0], o[1], "a", "a_scales", device), b(o[2], o[3], "b", "b_scales", device);
        mdx_matmul_args g{};
        g.m = a.codes.size(0);
        g.k = a.codes.size(1);
        g.n = b.codes.size(0);
        if (b.codes.size(1) != g.k)
            throw Refused{"a has " + std::to_string(g.k) + " columns and b " + std::to_string(b.codes.size(1)), "b"};
        const int64_t blocks = ceil_div(g.k, kBlock);
        if (a.scales.size(0) != g.m || a.scales.size(1) != blocks)
            throw Refused{"a_scales must have shape " + shape_of({g.m, blocks}) + ", not " + shape_of(a.scales.sizes()),
                          "a_scales"};
        const int64_t tall = ceil_div(g.n, kBlock);
        if (b.scales.size(1) == blocks && b.scales.size(0) == g.n) g.b_tile = 1;
        else if (b.scales.size(1) == blocks && b.scales.size(0) == tall) g.b_tile = int32_t(kBlock);
        else
            throw Refused{"b_scales must have shape " + shape_of({g.n, blocks}) + " or " + shape_of({tall, blocks})
                              + ", not " + shape_of(b.scales.sizes()),
                          "b_scales"};
        const History history("matmul_fp8", {{&a.codes, "a"}, {&a.scales, "a_scales"}, {&b.codes, "b"}, {&b.scales, "b_scales"}});
        at::Tensor out;
        if (o[5] == Py_None) {
            const at::ScalarType type = type_of(o[4], "dtype must be a torch dtype");
            if (kind_of(type) < 0)
                throw Refused{"dtype must be float32, bfloat16 or float16, not " + type_name(type), "dtype"};
            out = empty({g.m, g.n}, type, device);
            g.out_pitch = g.n;
        } else {
            out = tensor(o[5], "out");
            g.out_pitch = pitch_of(out, "out", device);
            if (out.size(0) != g.m || out.size(1) != g.n || kind_of(out.scalar_type()) < 0)
                throw Refused{"out must be a float32, bfloat16 or float16 matrix of shape " + shape_of({g.m, g.n}), "out"};
            history.refuse_out(out);
        }
        if (g.m > 0 && g.n > 0) {
            g.a = static_cast<const uint8_t*>(a.codes.data_ptr());
            g.a_pitch = a.pitch;
            g.a_scales = static_cast<const uint8_t*>(a.scales.data_ptr());
            g.a_scales_pitch = a.scales_pitch;
            g.b = static_cast<const uint8_t*>(b.codes.data_ptr());
            g.b_pitch = b.pitch;
            g.b_scales = static_cast<const uint8_t*>(b.scales.data_ptr());
            g.b_scales_pitch = b.scales_pitch;
            g.out = out.data_ptr();
            g.out_dtype = kind_of(out.scalar_type());
            g.a_packed = a.packed;
            g.b_packed = b.packed;
            g.workspace_bytes = mdx_hip_matmul_fp8_workspace(&g);
            at::Tensor workspace;
            if (g.workspace_bytes > 0) {
                workspace = empty({g.workspace_bytes}, at::kByte, device);
                g.workspace = workspace.data_ptr();
            }
            void* stream = stream_of(device);
            run("matmul_fp8", [&] { return mdx_hip_matmul_fp8(device.index(), &g, stream); });
            if (o[5] != Py_None) written_to(out);
        }
        history.goes_to({out});
        return THPVariable_Wrap(out);
    });
}

// A list or tuple of tensors, held: the caller's list may change while a call lets go of Python.
struct Tensors {
    PyObject* held = nullptr;
    const char* name;
    Tensors(PyObject* o, const char* n) : held(PySequence_Tuple(o)), name(n) {
        if (held == nullptr) throw Raised{};
    }
    ~Tensors() { Py_XDECREF(held); }
    Tensors(const Tensors&) = delete;
    Tensors& operator=(const Tensors&) = delete;
    Py_ssize_t size() const { return PyTuple_GET_SIZE(held); }
    const at::Tensor& at(Py_ssize_t i) const { return tensor(PyTuple_GET_ITEM(held, i), name); }
};

// adamw_step(params, grads, first, second, first_scales, second_scales, step, lr, beta1, beta2, eps, decay, seed)
PyObject* adamw_step(PyObject*, PyObject* const* o, Py_ssize_t n) {
    return guarded([&] {
        expect(n, 13);
        const bool eight = o[4] != Py_None || o[5] != Py_None;
        if (eight && (o[4] == Py_None || o[5] == Py_None))
            throw Refused{"states in 8 bits need first_scales and second_scales", "first_scales"};
        static const char* const names[6] = {"params", "grads", "first", "second", "first_scales", "second_scales"};
        const int lists = eight ? 6 : 4;
        std::vector<std::unique_ptr<Tensors>> given;
        for (int i = 0; i < lists; ++i) given.push_back(std::make_unique<Tensors>(o[i], names[i]));
        const Py_ssize_t count = given[0]->size();
        for (int i = 1; i < lists; ++i)
            if (given[i]->size() != count)
                throw Refused{std::string(names[i]) + " must hold one tensor for each of the " + std::to_string(count)
                                  + " params",
                              names[i]};
        mdx_adamw_args a{};
        const bool moving_step = moves(o[6]), moving_seed = moves(o[12]);
        a.step = moving_step ? 1 : whole(o[6]);
        a.lr = number(o[7]);
        a.beta1 = number(o[8]);
        a.beta2 = number(o[9]);
        a.eps = number(o[10]);
        a.weight_decay = number(o[11]);
        if (!moving_seed) a.seed = uint32_t(PyLong_AsUnsignedLongLongMask(o[12]));
        if (PyErr_Occurred()) throw Raised{};
        a.bits = eight ? 8 : 32;
        if (a.step < 1) throw Refused{"step must be a whole number from 1 on", "step"};
        if (!(a.lr >= 0.0 && std::isfinite(a.lr) && a.weight_decay >= 0.0 && std::isfinite(a.weight_decay)))
            throw Refused{"lr and weight_decay must be finite and not negative", "lr"};
        if (!(a.beta1 >= 0.0 && a.beta1 < 1.0 && a.beta2 >= 0.0 && a.beta2 < 1.0))
            throw Refused{"betas must lie in [0, 1)", "betas"};
        if (!(a.eps > 0.0 && std::isfinite(a.eps))) throw Refused{"eps must be positive and finite", "eps"};
        if (count == 0) return none();
        const at::Tensor& lead = given[0]->at(0);
        if (!lead.is_cuda()) throw Refused{"params must live on a HIP device", "params"};
        const at::Device device = lead.device();
        const int64_t* step_at = moving_step ? number_at(o[6], "step", device) : nullptr;
        const int64_t* seed_at = moving_seed ? number_at(o[12], "seed", device) : nullptr;
        const at::ScalarType grad_type = given[1]->at(0).scalar_type();
        if (kind_of(grad_type) < 0) throw Refused{"grads must be float32, bfloat16 or float16 tensors", "grads"};
        a.grad_dtype = kind_of(grad_type);
        const at::ScalarType state = eight ? kCodes : at::kFloat;
        const at::ScalarType types[6] = {at::kFloat, grad_type, state, state, kScales, kScales};
        std::vector<mdx_adamw_tensor> table(static_cast<size_t>(count));
        for (Py_ssize_t k = 0; k < count; ++k) {
            void* at_[6] = {};
            const at::Tensor& param = given[0]->at(k);
            const int64_t size = param.numel();
            for (int i = 0; i < lists; ++i) {
                const at::Tensor& t = given[i]->at(k);
                if (t.scalar_type() != types[i] || t.device() != device || !t.is_contiguous())
                    throw Refused{std::string(names[i]) + " must be contiguous " + type_name(types[i]) + " tensors on "
                                      + device.str(),
                                  names[i]};
                if (i >= 4) {
                    if (t.numel() != ceil_div(size, kBlock))
                        throw Refused{std::string(names[i]) + " must hold one scale per 128 elements of its parameter",
                                      names[i]};
                } else if (t.sizes() != param.sizes()) {
                    throw Refused{std::string(names[i]) + " must have the shapes of params", names[i]};
                }
                at_[i] = t.data_ptr();
            }
            table[size_t(k)] = {size, static_cast<float*>(at_[0]), at_[1], at_[2], at_[3],
                                static_cast<uint8_t*>(at_[4]), static_cast<uint8_t*>(at_[5])};
        }
        a.tensors = table.data();
        a.count = count;
        void* stream = stream_of(device);
        run("adamw_step", [&] { return mdx_hip_adamw_step_at(device.index(), &a, step_at, seed_at, stream); });
        for (int i = 0; i < lists; ++i)
            for (Py_ssize_t k = 0; i != 1 && k < count; ++k) written_to(given[i]->at(k));
        return none();
    });
}

PyObject* init(PyObject*, PyObject* const* o, Py_ssize_t n) {
    return guarded([&] {
        expect(n, 2);
        Py_INCREF(o[0]);
        Py_INCREF(o[1]);
        Py_XDECREF(g_refuse);
        Py_XDECREF(g_fail);
        g_refuse = o[0];
        g_fail = o[1];
        return none();
    });
}

#define MDX_METHOD(name) {#name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(name)), METH_FASTCALL, nullptr}
PyMethodDef methods[] = {MDX_METHOD(init),         MDX_METHOD(rms_norm),   MDX_METHOD(rms_norm_backward),
                         MDX_METHOD(quantize_fp8), MDX_METHOD(matmul_fp8), MDX_METHOD(adamw_step),
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef definition = {PyModuleDef_HEAD_INIT, "mdx_torch", "Operators on feature rows, called with torch tensors.", -1,
                          methods, nullptr, nullptr, nullptr, nullptr};

} // namespace

PyMODINIT_FUNC PyInit_mdx_torch() { return PyModule_Create(&definition); }
