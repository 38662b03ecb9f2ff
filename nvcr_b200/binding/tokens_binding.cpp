// The token operators for Python: takes torch tensors, checks what the C ABI
// cannot see (types, shapes, strides, devices), allocates the outputs and calls
// include/nvcr_sm100.h on torch's current stream or a given one. A step of a
// token model is a row of short calls, whose cost on the host is the user's
// waiting time: through ctypes, with the checks in Python, a norm of one token
// took 13.6 us of host time, of which the launch is 3.6.
//
// nvcr_b200/tokens.py wraps these functions and documents them. Arguments are
// positional; an optional tensor or stream is None.

#include <Python.h>

#include <ATen/ATen.h>
#include <c10/cuda/CUDAFunctions.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cmath>
#include <cstdint>
#include <exception>
#include <initializer_list>
#include <string>

#include "../../include/nvcr_sm100.h"

namespace {

PyObject* refuse_function = nullptr;  // refuse(message) raises ExecutorError(invalid_argument)
PyObject* check_function = nullptr;   // check(status) raises ExecutorError of the library's last error

struct Refusal {
    std::string message;
};
struct Failure {
    int status;
};
struct Raised {};  // a Python exception is set

std::string name_of(const at::Tensor& t) {
    std::string text = std::string("a ") + c10::toString(t.scalar_type()) + " tensor of shape (";
    for (std::int64_t i = 0; i < t.dim(); ++i) text += (i > 0 ? ", " : "") + std::to_string(t.size(i));
    return text + ") on " + t.device().str();
}

void check(int status) {
    if (status != 0) throw Failure{status};
}

void require(bool condition, const char* message) {
    if (!condition) throw Refusal{message};
}

const at::Tensor& tensor(PyObject* object, const char* what) {
    if (!THPVariable_Check(object)) throw Refusal{std::string(what) + " must be a torch tensor"};
    return THPVariable_Unpack(object);
}

// Arguments that are no tensors.
std::int64_t whole(PyObject* object) {
    const std::int64_t value = PyLong_AsLongLong(object);
    if (value == -1 && PyErr_Occurred() != nullptr) throw Raised{};
    return value;
}
int small(PyObject* object, const char* what) {
    const std::int64_t value = whole(object);
    if (value < INT32_MIN || value > INT32_MAX) throw Refusal{std::string(what) + " is out of range"};
    return static_cast<int>(value);
}
bool truth(PyObject* object) {
    const int value = PyObject_IsTrue(object);
    if (value < 0) throw Raised{};
    return value != 0;
}
double real(PyObject* object) {
    const double value = PyFloat_AsDouble(object);
    if (value == -1.0 && PyErr_Occurred() != nullptr) throw Raised{};
    return value;
}
void* address(PyObject* object) {
    void* value = PyLong_AsVoidPtr(object);
    if (value == nullptr && PyErr_Occurred() != nullptr) throw Raised{};
    return value;
}

int type_of(const at::Tensor& t) {
    switch (t.scalar_type()) {
    case at::kHalf: return NVCR_SM100_TOKEN_F16;
    case at::kBFloat16: return NVCR_SM100_TOKEN_BF16;
    case at::kFloat: return NVCR_SM100_TOKEN_F32;
    default: return -1;
    }
}

// The library launches on the current device, and the default stream's handle is the same for all of them. (Asking
// which one is current takes 0.15 us: not where there is only one.)
void require_current(int device) {
    static const int devices = c10::cuda::device_count();
    if (devices == 1 && device == 0) return;
    c10::DeviceIndex current = -1;
    if (c10::cuda::GetDevice(&current) != cudaSuccess || current != device) {
        throw Refusal{"the tensors are on cuda:" + std::to_string(device) + ", which is not the current CUDA device"};
    }
}

void* stream_of(PyObject* object, int device) {
    if (object != Py_None) return address(object);
    return c10::cuda::getCurrentCUDAStream(static_cast<c10::DeviceIndex>(device)).stream();
}

// The address of a contiguous tensor of a type and shape on a device.
void* plain(const at::Tensor& t, const char* what, at::ScalarType type, std::initializer_list<std::int64_t> shape,
            int device) {
    if (t.scalar_type() != type || t.sizes() != at::IntArrayRef(shape) || !t.is_cuda() || t.get_device() != device ||
        !t.is_contiguous()) {
        std::string wanted = std::string(what) + " must be a contiguous " + c10::toString(type) + " tensor of shape (";
        bool first = true;
        for (std::int64_t n : shape) wanted += (first ? "" : ", ") + std::to_string(n), first = false;
        throw Refusal{wanted + ") on cuda:" + std::to_string(device) + ", and is " + name_of(t)};
    }
    return t.data_ptr();
}

void* plain_or_null(PyObject* object, const char* what, at::ScalarType type, std::initializer_list<std::int64_t> shape,
                    int device) {
    return object == Py_None ? nullptr : plain(tensor(object, what), what, type, shape, device);
}

// The address of a tensor of a type and shape whose last dimension is contiguous.
void* strided(const at::Tensor& t, const char* what, at::ScalarType type, at::IntArrayRef shape, int device) {
    if (t.scalar_type() != type || t.sizes() != shape || !t.is_cuda() || t.get_device() != device ||
        (t.stride(-1) != 1 && t.size(-1) > 1 && t.numel() > 0)) {
        std::string wanted = std::string(what) + " must be a " + c10::toString(type) + " tensor of shape (";
        for (std::size_t i = 0; i < shape.size(); ++i) wanted += (i > 0 ? ", " : "") + std::to_string(shape[i]);
        throw Refusal{wanted + ") on cuda:" + std::to_string(device) + " whose last dimension is contiguous, and is " +
                      name_of(t)};
    }
    return t.data_ptr();
}

PyObject* wrapped(const at::Tensor& t) {
    if (!t.defined()) Py_RETURN_NONE;
    return THPVariable_Wrap(t);
}

PyObject* pair(const at::Tensor& a, const at::Tensor& b) {
    PyObject* result = PyTuple_New(2);
    if (result == nullptr) return nullptr;
    PyObject* first = wrapped(a);
    PyObject* second = wrapped(b);
    if (first == nullptr || second == nullptr) {
        Py_XDECREF(first);
        Py_XDECREF(second);
        Py_DECREF(result);
        return nullptr;
    }
    PyTuple_SET_ITEM(result, 0, first);
    PyTuple_SET_ITEM(result, 1, second);
    return result;
}

// Runs `body`; what it throws becomes a Python exception.
template <typename F>
PyObject* guarded(Py_ssize_t given, Py_ssize_t wanted, F&& body) {
    if (given != wanted) {
        PyErr_Format(PyExc_TypeError, "%zd arguments wanted, %zd given", wanted, given);
        return nullptr;
    }
    PyObject* raised = nullptr;
    try {
        return body();
    } catch (const Refusal& refusal) {
        raised = PyObject_CallFunction(refuse_function, "s", refusal.message.c_str());
    } catch (const Failure& failure) {
        raised = PyObject_CallFunction(check_function, "i", failure.status);
    } catch (const Raised&) {
        return nullptr;
    } catch (...) {  // torch's own exceptions as torch raises them
        torch::translate_exception_to_python(std::current_exception());
        return nullptr;
    }
    if (raised != nullptr) {  // neither returns without raising
        Py_DECREF(raised);
        PyErr_SetString(PyExc_RuntimeError, "a refused call did not raise");
    }
    return nullptr;
}

// norm(block, residual, gate, post, post_weight, post_bias, pre_weight, pre_bias, layer, residual_scale,
//      weight_offset, epsilon, hidden, normed, stream) -> (hidden, normed)
PyObject* norm(PyObject*, PyObject* const* args, Py_ssize_t count) {
    return guarded(count, 15, [&] {
        const at::Tensor& block = tensor(args[0], "block");
        const int type = type_of(block);
        require(type >= 0 && block.dim() == 2, "block must be a [rows, width] tensor of a float type");
        const bool hidden = truth(args[12]), normed = truth(args[13]);
        require(hidden || normed, "neither hidden nor normed is wanted");
        require(block.is_cuda(), "tensors must be on a CUDA device");
        const at::ScalarType kind = block.scalar_type();
        const int device = block.get_device();
        require_current(device);
        const at::IntArrayRef shape = block.sizes();
        const std::int64_t rows = shape[0], width = shape[1];
        const void* const from = strided(block, "block", kind, shape, device);
        const void *residual = nullptr, *gate = nullptr;
        std::int64_t residual_stride = 0, gate_stride = 0;
        if (args[1] != Py_None) {
            const at::Tensor& t = tensor(args[1], "residual");
            residual = strided(t, "residual", kind, shape, device), residual_stride = t.stride(0);
        }
        if (args[2] != Py_None) {
            const at::Tensor& t = tensor(args[2], "gate");
            if (t.dim() == 1) {
                gate = plain(t, "gate", kind, {width}, device);
            } else {
                gate = strided(t, "gate", kind, shape, device), gate_stride = t.stride(0);
            }
        }
        const void* const post_weight = plain_or_null(args[4], "post_weight", kind, {width}, device);
        const void* const post_bias = plain_or_null(args[5], "post_bias", kind, {width}, device);
        const void* const pre_weight = plain_or_null(args[6], "pre_weight", kind, {width}, device);
        const void* const pre_bias = plain_or_null(args[7], "pre_bias", kind, {width}, device);
        require(width <= INT32_MAX, "width is out of range");
        at::Tensor sum, out;
        if (hidden) sum = at::empty(shape, block.options());
        if (normed) out = at::empty(shape, block.options());
        check(nvcr_sm100_token_norm(type, small(args[8], "layer"), truth(args[3]), from, block.stride(0), residual,
                                    residual_stride, gate, gate_stride, post_weight, post_bias, pre_weight, pre_bias,
                                    hidden ? sum.data_ptr() : nullptr, normed ? out.data_ptr() : nullptr, rows,
                                    static_cast<std::int32_t>(width), static_cast<float>(real(args[9])),
                                    static_cast<float>(real(args[10])), static_cast<float>(real(args[11])),
                                    stream_of(args[14], device)));
        return pair(sum, out);
    });
}

bool is_half(const at::Tensor& t) { return t.scalar_type() == at::kHalf || t.scalar_type() == at::kBFloat16; }

// append(cache, device, keys, values, slots, queries, positions, cosines, sines, interleaved, stream) -> rotated queries
PyObject* append(PyObject*, PyObject* const* args, Py_ssize_t count) {
    return guarded(count, 11, [&] {
        const auto* cache = static_cast<const nvcr_sm100_token_cache*>(address(args[0]));
        const int device = small(args[1], "device");
        require_current(device);
        const at::Tensor& keys = tensor(args[2], "keys");
        const at::Tensor& values = tensor(args[3], "values");
        require(keys.dim() == 3 && is_half(keys), "keys must be a float16 or bfloat16 tensor of three dimensions");
        const at::ScalarType kind = keys.scalar_type();
        const std::int64_t tokens = keys.size(0);
        const std::int64_t shape[3] = {tokens, cache->kv_heads, cache->head_dim};
        const void* const key = strided(keys, "keys", kind, shape, device);
        const void* const value = strided(values, "values", kind, shape, device);
        const void* const slots = plain(tensor(args[4], "slots"), "slots", at::kLong, {tokens}, device);
        at::Tensor rotated;
        const void* query = nullptr;
        std::int64_t query_stride = 0, query_head_stride = 0, query_heads = 0;
        if (args[5] != Py_None) {
            const at::Tensor& queries = tensor(args[5], "queries");
            require(queries.dim() == 3, "queries have three dimensions");
            query_heads = queries.size(1);
            require(query_heads <= INT32_MAX, "queries have too many heads");
            const std::int64_t query_shape[3] = {tokens, query_heads, cache->head_dim};
            query = strided(queries, "queries", kind, query_shape, device);
            query_stride = queries.stride(0), query_head_stride = queries.stride(1);
            rotated = at::empty(query_shape, queries.options());
        }
        const void *positions = nullptr, *cosines = nullptr, *sines = nullptr;
        std::int64_t table_rows = 0, half = 0;
        if (args[6] != Py_None) {
            require(args[7] != Py_None && args[8] != Py_None, "positions need rotation tables");
            const at::Tensor& table = tensor(args[7], "cosines");
            require(table.dim() == 2, "cosines have two dimensions");
            table_rows = table.size(0), half = table.size(1);
            require(half <= cache->head_dim, "the rotation tables are wider than half a head");
            positions = plain(tensor(args[6], "positions"), "positions", at::kInt, {tokens}, device);
            cosines = plain(table, "cosines", at::kFloat, {table_rows, half}, device);
            sines = plain(tensor(args[8], "sines"), "sines", at::kFloat, {table_rows, half}, device);
        }
        check(nvcr_sm100_token_append(
            cache, type_of(keys), key, keys.stride(0), keys.stride(1), value, values.stride(0), values.stride(1),
            static_cast<const std::int64_t*>(slots), tokens, query, query_stride, query_head_stride,
            static_cast<std::int32_t>(query_heads), query != nullptr ? rotated.data_ptr() : nullptr,
            static_cast<const std::int32_t*>(positions), static_cast<const float*>(cosines),
            static_cast<const float*>(sines), table_rows, static_cast<std::int32_t>(2 * half), truth(args[9]),
            stream_of(args[10], device)));
        return wrapped(rotated);
    });
}

// read(cache, device, slots, type, stream) -> (keys, values)
PyObject* read(PyObject*, PyObject* const* args, Py_ssize_t count) {
    return guarded(count, 5, [&] {
        const auto* cache = static_cast<const nvcr_sm100_token_cache*>(address(args[0]));
        const int device = small(args[1], "device"), type = small(args[3], "dtype");
        require_current(device);
        const at::Tensor& slots = tensor(args[2], "slots");
        require(slots.dim() == 1, "slots have one dimension");
        const std::int64_t tokens = slots.size(0);
        const void* const at_slots = plain(slots, "slots", at::kLong, {tokens}, device);
        const at::ScalarType kind = type == NVCR_SM100_TOKEN_F16 ? at::kHalf
            : type == NVCR_SM100_TOKEN_BF16                       ? at::kBFloat16
                                                                  : at::kFloat;
        const std::int64_t shape[3] = {tokens, cache->kv_heads, cache->head_dim};
        const at::TensorOptions options = slots.options().dtype(kind);
        const at::Tensor keys = at::empty(shape, options), values = at::empty(shape, options);
        check(nvcr_sm100_token_read(cache, type, static_cast<const std::int64_t*>(at_slots), tokens, keys.data_ptr(),
                                    values.data_ptr(), stream_of(args[4], device)));
        return pair(keys, values);
    });
}

// attend(context, cache, device, queries, page_table, lengths, query_offsets, max_queries, max_length, scale, stream)
PyObject* attend(PyObject*, PyObject* const* args, Py_ssize_t count) {
    return guarded(count, 11, [&] {
        auto* context = static_cast<nvcr_sm100_token_context*>(address(args[0]));
        const auto* cache = static_cast<const nvcr_sm100_token_cache*>(address(args[1]));
        const int device = small(args[2], "device");
        require_current(device);
        const at::Tensor& queries = tensor(args[3], "queries");
        const at::Tensor& table = tensor(args[4], "page_table");
        const at::Tensor& lengths = tensor(args[5], "lengths");
        require(queries.dim() == 3 && is_half(queries), "queries must be a float16 or bfloat16 tensor of three dimensions");
        const std::int64_t tokens = queries.size(0), heads = queries.size(1);
        require(heads <= INT32_MAX, "queries have too many heads");
        const std::int64_t shape[3] = {tokens, heads, cache->head_dim};
        const void* const query = strided(queries, "queries", queries.scalar_type(), shape, device);
        require(lengths.dim() == 1 && table.dim() == 2, "lengths have one dimension and page_table two");
        const std::int64_t batch = lengths.size(0), columns = table.size(1);
        require(batch <= INT32_MAX && columns <= INT32_MAX, "page_table is too large");
        const std::int64_t table_shape[2] = {batch, columns};
        const void* const pages = strided(table, "page_table", at::kInt, table_shape, device);
        const void* const length = plain(lengths, "lengths", at::kInt, {batch}, device);
        const void* const offsets = plain_or_null(args[6], "query_offsets", at::kInt, {batch + 1}, device);
        const double scale = args[9] == Py_None ? 1.0 / std::sqrt(static_cast<double>(cache->head_dim)) : real(args[9]);
        const at::Tensor out = at::empty(shape, queries.options());
        check(nvcr_sm100_token_attend(
            context, cache, type_of(queries), query, queries.stride(0), queries.stride(1), tokens,
            static_cast<std::int32_t>(heads), static_cast<const std::int32_t*>(pages), table.stride(0),
            static_cast<std::int32_t>(columns), static_cast<const std::int32_t*>(length), static_cast<std::int32_t>(batch),
            static_cast<const std::int32_t*>(offsets), small(args[7], "max_queries"), small(args[8], "max_length"),
            static_cast<float>(scale), out.data_ptr(), stream_of(args[10], device)));
        return wrapped(out);
    });
}

// multiply(codes, scales, outputs, inputs, group, device, x, bias, stream) -> y
PyObject* multiply(PyObject*, PyObject* const* args, Py_ssize_t count) {
    return guarded(count, 9, [&] {
        const int outputs = small(args[2], "outputs"), inputs = small(args[3], "inputs"), group = small(args[4], "group");
        const int device = small(args[5], "device");
        require_current(device);
        const at::Tensor& x = tensor(args[6], "x");
        require(x.dim() == 2 && is_half(x), "x must be a float16 or bfloat16 tensor of two dimensions");
        const std::int64_t rows = x.size(0);
        const std::int64_t shape[2] = {rows, inputs};
        const void* const from = strided(x, "x", x.scalar_type(), shape, device);
        const void* const bias = plain_or_null(args[7], "bias", x.scalar_type(), {outputs}, device);
        const at::Tensor y = at::empty({rows, outputs}, x.options());
        check(nvcr_sm100_token_multiply(type_of(x), from, x.stride(0), rows, address(args[0]), address(args[1]), outputs,
                                        inputs, group, bias, y.data_ptr(), stream_of(args[8], device)));
        return wrapped(y);
    });
}

// on_current(device): refuses another device than the current one.
PyObject* on_current(PyObject*, PyObject* const* args, Py_ssize_t count) {
    return guarded(count, 1, [&]() -> PyObject* {
        require_current(small(args[0], "device"));
        Py_RETURN_NONE;
    });
}

// bind(refuse, check): the functions that raise.
PyObject* bind(PyObject*, PyObject* const* args, Py_ssize_t count) {
    return guarded(count, 2, [&]() -> PyObject* {
        Py_INCREF(args[0]);
        Py_INCREF(args[1]);
        Py_XSETREF(refuse_function, args[0]);
        Py_XSETREF(check_function, args[1]);
        Py_RETURN_NONE;
    });
}

#define TOKEN_METHOD(name) {#name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(name)), METH_FASTCALL, nullptr}
PyMethodDef methods[] = {TOKEN_METHOD(norm),     TOKEN_METHOD(append), TOKEN_METHOD(read), TOKEN_METHOD(attend),
                         TOKEN_METHOD(multiply), TOKEN_METHOD(on_current), TOKEN_METHOD(bind), {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "nvcr_tokens", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit_nvcr_tokens() { return PyModule_Create(&module); }
