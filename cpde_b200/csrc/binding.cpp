// The Python side of the device-tensor operators (cpde_b200.operators): checks of
// tensors, new outputs and workspaces from torch's allocator, and the call of the
// C entry point on torch's current stream. A small call's time is its way through
// here: from Python with ctypes it took 10 to 22 us, most of it conversions.
//
// The entry points' addresses come from Python (bind), so that this module uses
// the library that cpde_b200.native has loaded.
#include <ATen/ATen.h>
#include <ATen/core/grad_mode.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cstdint>
#include <stdexcept>
#include <string>

#include "../../include/cpde_b200.h"

namespace {

struct Entries {
    decltype(&cpde_last_error) last_error;
    decltype(&cpde_embedding) embedding;
    decltype(&cpde_embedding_gradient_workspace) embedding_gradient_workspace;
    decltype(&cpde_embedding_gradient) embedding_gradient;
    decltype(&cpde_dropout) dropout;
    decltype(&cpde_group_norm_forward_workspace) group_norm_forward_workspace;
    decltype(&cpde_group_norm_workspace) group_norm_workspace;
    decltype(&cpde_group_norm) group_norm;
    decltype(&cpde_group_norm_gradient) group_norm_gradient;
} entries = {};
PyObject* engine_error = nullptr;  // cpde_b200.native.EngineError

// A Python exception is set.
struct Raised {};

void check(bool ok, const char* message) {
    if (ok) return;
    PyErr_SetString(PyExc_ValueError, message);
    throw Raised();
}

struct Engine {
    cpde_engine* handle;
    int device;
    void* stream() const {
        // The default stream's own handle: a null one selects the engine's stream.
        cudaStream_t s = c10::cuda::getCurrentCUDAStream(c10::DeviceIndex(device)).stream();
        return s ? s : reinterpret_cast<void*>(1);
    }
    void done(int status) const {
        if (status == CPDE_OK) return;
        PyObject* error = PyObject_CallFunction(engine_error, "is", status, entries.last_error(handle));
        if (error) {
            PyErr_SetObject(engine_error, error);
            Py_DECREF(error);
        }
        throw Raised();
    }
};

// Positional arguments of a call.
struct Arguments {
    PyObject* const* items;
    Py_ssize_t count, next = 0;
    PyObject* take() {
        check(next < count, "too few arguments");
        return items[next++];
    }
    int64_t integer() {
        const long long v = PyLong_AsLongLong(take());
        if (v == -1 && PyErr_Occurred()) throw Raised();
        return v;
    }
    uint64_t word() {  // modulo 2^64
        const unsigned long long v = PyLong_AsUnsignedLongLongMask(take());
        if (v == ~0ull && PyErr_Occurred()) throw Raised();
        return v;
    }
    double number() {
        const double v = PyFloat_AsDouble(take());
        if (v == -1.0 && PyErr_Occurred()) throw Raised();
        return v;
    }
    Engine engine() {
        auto* handle = reinterpret_cast<cpde_engine*>(uintptr_t(word()));
        return {handle, int(integer())};
    }
    at::Tensor tensor(const Engine& e, const char* name) {
        at::Tensor t = optional(e, name);
        check(t.defined(), (std::string(name) + " must be a tensor").c_str());
        return t;
    }
    at::Tensor optional(const Engine& e, const char* name) {
        PyObject* o = take();
        if (o == Py_None) return {};
        check(THPVariable_Check(o), (std::string(name) + " must be a tensor").c_str());
        at::Tensor t = THPVariable_Unpack(o);
        check(t.is_cuda() && t.get_device() == e.device, "every tensor must be on the engine's device");
        // The result would be detached in silence.
        check(!t.requires_grad() || !at::GradMode::is_enabled(),
              "a tensor requires gradients: use operators.Embedding, Dropout or GroupNorm, or torch.no_grad()");
        return t;
    }
    // An element type, or `none` for None.
    at::ScalarType type(at::ScalarType none) {
        PyObject* o = take();
        if (o == Py_None) return none;
        check(THPDtype_Check(o), "dtype must be a torch.dtype");
        return reinterpret_cast<THPDtype*>(o)->scalar_type;
    }
};

int32_t type_code(at::ScalarType type, const char* message) {
    check(type == at::kFloat || type == at::kBFloat16 || type == at::kHalf, message);
    return type == at::kFloat ? CPDE_F32 : type == at::kBFloat16 ? CPDE_BF16 : CPDE_F16;
}

int32_t id_code(const at::Tensor& ids) {
    check(ids.scalar_type() == at::kInt || ids.scalar_type() == at::kLong, "ids must be int32 or int64");
    return ids.scalar_type() == at::kLong ? CPDE_I64 : CPDE_I32;
}

const void* pointer(const at::Tensor& t) { return t.defined() ? t.const_data_ptr() : nullptr; }

at::Tensor made(at::IntArrayRef sizes, const at::Tensor& like, at::ScalarType type) {
    return at::empty(sizes, like.options().dtype(type).requires_grad(false));
}

// A matrix of rows with adjacent channels and their stride; other layouts
// (transposed, broadcast) are copied first.
struct Rows {
    at::Tensor t;
    int64_t rows, columns, stride;
    explicit Rows(at::Tensor from) : t(std::move(from)) {
        if (t.dim() != 2) t = t.reshape({-1, t.size(-1)});
        rows = t.size(0), columns = t.size(1);
        if ((columns > 1 && t.stride(1) != 1) || (rows > 1 && t.stride(0) < columns)) t = t.contiguous();
        stride = rows > 1 ? t.stride(0) : columns;
    }
};

// The same for (instance, point, channel) arrays.
struct Points {
    at::Tensor t;
    int64_t point, instance;
    Points(at::Tensor from, const char* message) : t(std::move(from)) {
        check(t.dim() == 3, message);
        if ((t.size(2) > 1 && t.stride(2) != 1) || (t.size(1) > 1 && t.stride(1) < t.size(2))) t = t.contiguous();
        point = std::max(t.stride(1), t.size(2));
        instance = t.stride(0);
    }
};

PyObject* embedding(Arguments& a) {
    const Engine e = a.engine();
    at::Tensor table = a.tensor(e, "table"), ids = a.tensor(e, "ids");
    const float scale = float(a.number());
    check(table.dim() == 2, "table must have shape (rows, channels)");
    const int32_t kind = type_code(table.scalar_type(), "table must be float32, bfloat16 or float16"), id_kind = id_code(ids);
    const at::ScalarType type = a.type(table.scalar_type());
    const int32_t out_kind = type_code(type, "dtype must be float32, bfloat16 or float16");
    at::DimVector sizes(ids.sizes());
    sizes.push_back(table.size(1));
    const at::Tensor out = made(sizes, table, type);
    ids = ids.contiguous();
    const Rows rows(std::move(table));
    e.done(entries.embedding(e.handle, kind, pointer(rows.t), rows.stride, rows.rows, rows.columns, id_kind, pointer(ids),
                             ids.numel(), scale, out_kind, out.mutable_data_ptr(), e.stream()));
    return THPVariable_Wrap(out);
}

PyObject* embedding_gradient(Arguments& a) {
    const Engine e = a.engine();
    at::Tensor grad = a.tensor(e, "grad"), ids = a.tensor(e, "ids");
    const int64_t rows = a.integer();
    const float scale = float(a.number());
    check(grad.dim() == ids.dim() + 1 && grad.sizes().slice(0, ids.dim()) == ids.sizes(),
          "grad must have the shape of ids and the channels");
    const int32_t kind = type_code(grad.scalar_type(), "grad must be float32, bfloat16 or float16"), id_kind = id_code(ids);
    const at::ScalarType type = a.type(grad.scalar_type());
    const int32_t out_kind = type_code(type, "dtype must be float32, bfloat16 or float16");
    const int64_t tokens = ids.numel(), channels = grad.size(-1);
    size_t bytes = 0;
    check(entries.embedding_gradient_workspace(tokens, rows, channels, &bytes) == CPDE_OK, "invalid tokens, rows or channels");
    const at::Tensor out = made({rows, channels}, grad, type);
    const at::Tensor workspace = made({int64_t(bytes)}, grad, at::kByte);
    const Rows g(std::move(grad));
    ids = ids.contiguous();
    e.done(entries.embedding_gradient(e.handle, kind, pointer(g.t), g.stride, id_kind, pointer(ids), tokens, rows, channels,
                                      scale, out_kind, out.mutable_data_ptr(), workspace.mutable_data_ptr(), bytes,
                                      e.stream()));
    return THPVariable_Wrap(out);
}

PyObject* dropout(Arguments& a) {
    const Engine e = a.engine();
    at::Tensor x = a.tensor(e, "x"), residual = a.optional(e, "residual");
    const double rate = a.number();
    const uint64_t seed = a.word(), offset = a.word();
    const int32_t kind = type_code(x.scalar_type(), "x must be float32, bfloat16 or float16");
    check(!residual.defined() || (residual.sizes() == x.sizes() && residual.scalar_type() == x.scalar_type()),
          "residual must have x's shape and type");
    const at::Tensor y = made(x.sizes(), x, x.scalar_type());
    int64_t rows = 1, columns = x.numel(), stride = columns, residual_stride = columns;
    if (!(x.is_contiguous() && (!residual.defined() || residual.is_contiguous()))) {
        const Rows r(std::move(x));
        x = r.t, rows = r.rows, columns = r.columns, stride = r.stride, residual_stride = columns;
        if (residual.defined()) {
            const Rows s(std::move(residual));
            residual = s.t, residual_stride = s.stride;
        }
    }
    e.done(entries.dropout(e.handle, kind, pointer(x), stride, pointer(residual), residual_stride, rows, columns, rate, seed,
                           offset, y.mutable_data_ptr(), e.stream()));
    return THPVariable_Wrap(y);
}

// What group norm and its gradient share, in the order of the Python arguments.
struct Norm {
    at::Tensor weight, bias, lengths;
    int32_t kind, parameter, activation;
    double rate;
    uint64_t seed, offset;
    size_t bytes = 0;
    Norm(Arguments& a, const Engine& e, const at::Tensor& x, int64_t groups,
         decltype(entries.group_norm_workspace) workspace) {
        weight = a.optional(e, "weight"), bias = a.optional(e, "bias");
        activation = int32_t(a.integer());
        lengths = a.optional(e, "lengths");
        rate = a.number(), seed = a.word(), offset = a.word();
        kind = type_code(x.scalar_type(), "x must be float32, bfloat16 or float16");
        at::ScalarType type = at::kFloat;
        for (const at::Tensor* p : {&weight, &bias})
            if (p->defined()) {
                check(p->dim() == 1 && p->size(0) == x.size(2) && p->is_contiguous(),
                      "weight and bias must be contiguous tensors with a value per channel");
                type = p->scalar_type();
            }
        check(!weight.defined() || !bias.defined() || weight.scalar_type() == bias.scalar_type(),
              "weight and bias must have one type");
        check(type == at::kFloat || type == x.scalar_type(), "weight and bias must be float32 or of x's type");
        parameter = type_code(type, "weight and bias must be float32 or of x's type");
        check(!lengths.defined() || (lengths.scalar_type() == at::kInt && lengths.dim() == 1 &&
                                     lengths.size(0) == x.size(0) && lengths.is_contiguous()),
              "lengths must be a contiguous int32 tensor with a value per instance");
        check(workspace(x.size(0), x.size(1), x.size(2), groups, &bytes) == CPDE_OK,
              "invalid sizes, or a group count that does not divide the channels");
    }
    const int32_t* counts() const { return static_cast<const int32_t*>(pointer(lengths)); }
};

PyObject* group_norm(Arguments& a) {
    const Engine e = a.engine();
    const Points x(a.tensor(e, "x"), "x must have shape (instances, points, channels)");
    const int64_t groups = a.integer();
    const double eps = a.number();
    const Norm n(a, e, x.t, groups, entries.group_norm_forward_workspace);
    const at::Tensor y = made(x.t.sizes(), x.t, x.t.scalar_type());
    const at::Tensor mean = made({x.t.size(0), groups}, x.t, at::kFloat), rstd = made({x.t.size(0), groups}, x.t, at::kFloat);
    const at::Tensor workspace = made({int64_t(n.bytes)}, x.t, at::kByte);
    e.done(entries.group_norm(e.handle, n.kind, pointer(x.t), x.point, x.instance, x.t.size(0), x.t.size(1), x.t.size(2),
                              groups, n.parameter, pointer(n.weight), pointer(n.bias), eps, n.activation, n.counts(), n.rate,
                              n.seed, n.offset, y.mutable_data_ptr(), static_cast<float*>(mean.mutable_data_ptr()),
                              static_cast<float*>(rstd.mutable_data_ptr()), workspace.mutable_data_ptr(), n.bytes,
                              e.stream()));
    return Py_BuildValue("NNN", THPVariable_Wrap(y), THPVariable_Wrap(mean), THPVariable_Wrap(rstd));
}

PyObject* group_norm_gradient(Arguments& a) {
    const Engine e = a.engine();
    at::Tensor grad_in = a.tensor(e, "grad"), x_in = a.tensor(e, "x");
    check(grad_in.sizes() == x_in.sizes() && grad_in.scalar_type() == x_in.scalar_type(), "grad must have x's shape and type");
    const Points grad(std::move(grad_in), "grad must have shape (instances, points, channels)");
    const Points x(std::move(x_in), "x must have shape (instances, points, channels)");
    const at::Tensor mean = a.tensor(e, "mean"), rstd = a.tensor(e, "rstd");
    const int64_t groups = a.integer();
    const Norm n(a, e, x.t, groups, entries.group_norm_workspace);
    for (const at::Tensor* t : {&mean, &rstd})
        check(t->scalar_type() == at::kFloat && t->dim() == 2 && t->size(0) == x.t.size(0) && t->size(1) == groups &&
                  t->is_contiguous(),
              "mean and rstd must be contiguous float32 tensors of shape (instances, groups)");
    const at::Tensor dx = made(x.t.sizes(), x.t, x.t.scalar_type());
    at::Tensor dweight, dbias;
    if (n.weight.defined()) dweight = made(n.weight.sizes(), x.t, n.weight.scalar_type());
    if (n.bias.defined()) dbias = made(n.bias.sizes(), x.t, n.bias.scalar_type());
    const at::Tensor workspace = made({int64_t(n.bytes)}, x.t, at::kByte);
    e.done(entries.group_norm_gradient(
        e.handle, n.kind, pointer(grad.t), grad.point, grad.instance, pointer(x.t), x.point, x.instance,
        static_cast<const float*>(pointer(mean)), static_cast<const float*>(pointer(rstd)), x.t.size(0), x.t.size(1),
        x.t.size(2), groups, n.parameter, pointer(n.weight), pointer(n.bias), n.activation, n.counts(), n.rate, n.seed,
        n.offset, dx.mutable_data_ptr(), const_cast<void*>(pointer(dweight)), const_cast<void*>(pointer(dbias)),
        workspace.mutable_data_ptr(), n.bytes, e.stream()));
    auto wrap = [](const at::Tensor& t) {
        if (t.defined()) return THPVariable_Wrap(t);
        Py_INCREF(Py_None);
        return Py_None;
    };
    return Py_BuildValue("NNN", wrap(dx), wrap(dweight), wrap(dbias));
}

// bind(EngineError, {name: address}).
PyObject* bind(Arguments& a) {
    PyObject* error = a.take();
    PyObject* addresses = a.take();
    auto address = [&](const char* name) -> void* {
        PyObject* v = PyDict_GetItemString(addresses, name);
        check(v, "an entry point is missing");
        return reinterpret_cast<void*>(uintptr_t(PyLong_AsUnsignedLongLongMask(v)));
    };
    Entries e;
    e.last_error = reinterpret_cast<decltype(e.last_error)>(address("cpde_last_error"));
    e.embedding = reinterpret_cast<decltype(e.embedding)>(address("cpde_embedding"));
    e.embedding_gradient_workspace =
        reinterpret_cast<decltype(e.embedding_gradient_workspace)>(address("cpde_embedding_gradient_workspace"));
    e.embedding_gradient = reinterpret_cast<decltype(e.embedding_gradient)>(address("cpde_embedding_gradient"));
    e.dropout = reinterpret_cast<decltype(e.dropout)>(address("cpde_dropout"));
    e.group_norm_forward_workspace =
        reinterpret_cast<decltype(e.group_norm_forward_workspace)>(address("cpde_group_norm_forward_workspace"));
    e.group_norm_workspace = reinterpret_cast<decltype(e.group_norm_workspace)>(address("cpde_group_norm_workspace"));
    e.group_norm = reinterpret_cast<decltype(e.group_norm)>(address("cpde_group_norm"));
    e.group_norm_gradient = reinterpret_cast<decltype(e.group_norm_gradient)>(address("cpde_group_norm_gradient"));
    entries = e;
    Py_XDECREF(engine_error);
    Py_INCREF(error);
    engine_error = error;
    Py_RETURN_NONE;
}

template <PyObject* (*F)(Arguments&)>
PyObject* guarded(PyObject*, PyObject* const* items, Py_ssize_t count) {
    try {
        Arguments a{items, count};
        return F(a);
    } catch (const Raised&) {
    } catch (const std::exception& e) {
        PyErr_SetString(PyExc_RuntimeError, e.what());
    }
    return nullptr;
}

template <PyObject* (*F)(Arguments&)>
PyMethodDef method(const char* name) {
    return {name, reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(&guarded<F>)), METH_FASTCALL, nullptr};
}

PyMethodDef methods[] = {method<bind>("bind"), method<embedding>("embedding"),
                         method<embedding_gradient>("embedding_gradient"), method<dropout>("dropout"),
                         method<group_norm>("group_norm"), method<group_norm_gradient>("group_norm_gradient"),
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_operators", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__operators() { return PyModule_Create(&module); }
