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
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/Exceptions.h>
#include <torch/csrc/autograd/python_variable.h>

#include <cmath>
#include <cstdint>
#include <exception>
#include <initializer_list>
#include <optional>
#include <string>
#include <type_traits>

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

// Working memory of one call, of the call's own stream: its allocator hands it on to that stream's later work only.
at::Tensor workspace(std::size_t bytes, int device, PyObject* stream) {
    std::optional<c10::cuda::CUDAStreamGuard> guard;
    if (stream != Py_None) {
        const auto index = static_cast<c10::DeviceIndex>(device);
        auto handle = static_cast<cudaStream_t>(address(stream));
        guard.emplace(handle == nullptr ? c10::cuda::getDefaultCUDAStream(index)
                                        : c10::cuda::getStreamFromExternal(handle, index));
    }
    return at::empty({static_cast<std::int64_t>(bytes)},
                     at::TensorOptions().dtype(at::kByte).device(at::kCUDA, static_cast<c10::DeviceIndex>(device)));
}

// bytes_multiply(packed, scales, outputs, inputs, status, device, x, bias, stream) -> y
PyObject* bytes_multiply(PyObject*, PyObject* const* args, Py_ssize_t count) {
    return guarded(count, 9, [&] {
        const int outputs = small(args[2], "outputs"), inputs = small(args[3], "inputs");
        const int device = small(args[5], "device");
        require_current(device);
        const at::Tensor& x = tensor(args[6], "x");
        const int type = type_of(x);
        require(x.dim() == 2 && type >= 0, "x must be a tensor of a float type of two dimensions");
        const std::int64_t rows = x.size(0);
        const std::int64_t shape[2] = {rows, inputs};
        const void* const from = strided(x, "x", x.scalar_type(), shape, device);
        const void* const bias = plain_or_null(args[7], "bias", x.scalar_type(), {outputs}, device);
        std::size_t bytes = 0;
        check(nvcr_sm100_token_bytes_workspace(rows, outputs, inputs, &bytes));
        const at::Tensor y = at::empty({rows, outputs}, x.options());
        const at::Tensor room = workspace(bytes, device, args[8]);
        check(nvcr_sm100_token_bytes_multiply(type, from, x.stride(0), rows, address(args[0]),
                                              static_cast<const float*>(address(args[1])), outputs, inputs, bias,
                                              y.data_ptr(), room.data_ptr(), bytes,
                                              static_cast<std::uint32_t*>(address(args[4])), stream_of(args[8], device)));
        return wrapped(y);
    });
}

// experts_multiply(packed, scales, experts, outputs, inputs, status, device, x, choices, weights, stream) -> y
PyObject* experts_multiply(PyObject*, PyObject* const* args, Py_ssize_t count) {
    return guarded(count, 11, [&] {
        const int experts = small(args[2], "experts"), outputs = small(args[3], "outputs"), inputs = small(args[4], "inputs");
        const int device = small(args[6], "device");
        require_current(device);
        const at::Tensor& x = tensor(args[7], "x");
        const at::Tensor& choices = tensor(args[8], "choices");
        const int type = type_of(x);
        require((x.dim() == 2 || x.dim() == 3) && type >= 0, "x must be a tensor of a float type of two or three dimensions");
        require(choices.dim() == 2, "choices have two dimensions");
        const std::int64_t tokens = choices.size(0), chosen = choices.size(1);
        require(chosen <= INT32_MAX, "choices are out of range");
        const bool rows_each = x.dim() == 3;
        const std::int64_t flat[2] = {tokens, inputs}, deep[3] = {tokens, chosen, inputs};
        const void* const from =
            strided(x, "x", x.scalar_type(), rows_each ? at::IntArrayRef(deep) : at::IntArrayRef(flat), device);
        const void* const which = plain(choices, "choices", at::kInt, {tokens, chosen}, device);
        const void* const weights = plain_or_null(args[9], "weights", at::kFloat, {tokens, chosen}, device);
        std::size_t bytes = 0;
        check(nvcr_sm100_token_experts_workspace(tokens, static_cast<std::int32_t>(chosen), weights != nullptr, experts,
                                                 outputs, inputs, &bytes));
        const at::Tensor y = weights != nullptr ? at::empty({tokens, outputs}, x.options())
                                                : at::empty({tokens, chosen, outputs}, x.options());
        const at::Tensor room = workspace(bytes, device, args[10]);
        check(nvcr_sm100_token_experts_multiply(
            type, from, x.stride(0), rows_each ? x.stride(1) : 0, rows_each, tokens,
            static_cast<const std::int32_t*>(which), static_cast<std::int32_t>(chosen),
            static_cast<const float*>(weights), address(args[0]), static_cast<const float*>(address(args[1])), experts,
            outputs, inputs, y.data_ptr(), room.data_ptr(), bytes, static_cast<std::uint32_t*>(address(args[5])),
            stream_of(args[10], device)));
        return wrapped(y);
    });
}

// route(scores, count, sigmoid, bias, groups, kept_groups, renormalise, scale, stream) -> (choices, weights)
PyObject* route(PyObject*, PyObject* const* args, Py_ssize_t count) {
    return guarded(count, 9, [&] {
        const at::Tensor& scores = tensor(args[0], "scores");
        const int type = type_of(scores);
        require(type >= 0 && scores.dim() == 2, "scores must be a [tokens, experts] tensor of a float type");
        require(scores.is_cuda(), "tensors must be on a CUDA device");
        const int device = scores.get_device();
        require_current(device);
        const std::int64_t tokens = scores.size(0), experts = scores.size(1);
        require(experts <= INT32_MAX, "scores have too many experts");
        const int chosen = small(args[1], "count");
        require(chosen > 0 && chosen <= experts, "count must be 1 to the number of experts");
        const void* const from = strided(scores, "scores", scores.scalar_type(), scores.sizes(), device);
        const void* const bias = plain_or_null(args[3], "bias", at::kFloat, {experts}, device);
        const at::Tensor choices = at::empty({tokens, chosen}, scores.options().dtype(at::kInt));
        const at::Tensor weights = at::empty({tokens, chosen}, scores.options().dtype(at::kFloat));
        check(nvcr_sm100_token_route(type, from, scores.stride(0), tokens, static_cast<std::int32_t>(experts), chosen,
                                     truth(args[2]), static_cast<const float*>(bias), small(args[4], "groups"),
                                     small(args[5], "kept_groups"), truth(args[6]), static_cast<float>(real(args[7])),
                                     choices.data_ptr<std::int32_t>(), weights.data_ptr<float>(),
                                     stream_of(args[8], device)));
        return pair(choices, weights);
    });
}

// A number for every row, or a tensor with one for each.
template <typename T>
struct EachRow {
    const T* values = nullptr;
    T value{};
    EachRow(PyObject* object, const char* what, at::ScalarType type, std::int64_t rows, int device) {
        if (THPVariable_Check(object)) {
            values = static_cast<const T*>(plain(tensor(object, what), what, type, {rows}, device));
        } else if constexpr (std::is_same_v<T, float>) {
            value = static_cast<float>(real(object));
        } else {
            value = small(object, what);
        }
    }
};

// sample(logits, uniforms, temperature, top_k, top_p, min_p, stream) -> (symbols, probabilities)
PyObject* sample(PyObject*, PyObject* const* args, Py_ssize_t count) {
    return guarded(count, 7, [&] {
        const at::Tensor& logits = tensor(args[0], "logits");
        const int type = type_of(logits);
        require(type >= 0 && logits.dim() == 2, "logits must be a [rows, symbols] tensor of a float type");
        require(logits.is_cuda(), "tensors must be on a CUDA device");
        const int device = logits.get_device();
        require_current(device);
        const std::int64_t rows = logits.size(0), symbols = logits.size(1);
        require(symbols <= INT32_MAX, "logits have too many symbols");
        const void* const from = strided(logits, "logits", logits.scalar_type(), logits.sizes(), device);
        const void* const uniforms = plain(tensor(args[1], "uniforms"), "uniforms", at::kFloat, {rows}, device);
        const EachRow<float> temperature(args[2], "temperature", at::kFloat, rows, device);
        const EachRow<std::int32_t> top_k(args[3], "top_k", at::kInt, rows, device);
        const EachRow<float> top_p(args[4], "top_p", at::kFloat, rows, device);
        const EachRow<float> min_p(args[5], "min_p", at::kFloat, rows, device);
        const at::Tensor chosen = at::empty({rows}, logits.options().dtype(at::kLong));
        const at::Tensor probabilities = at::empty({rows}, logits.options().dtype(at::kFloat));
        std::size_t bytes = 0;
        check(nvcr_sm100_token_sample_workspace(type, rows, static_cast<std::int32_t>(symbols), &bytes));
        at::Tensor room;
        if (bytes > 0) room = workspace(bytes, device, args[6]);
        check(nvcr_sm100_token_sample(type, from, logits.stride(0), rows, static_cast<std::int32_t>(symbols),
                                      static_cast<const float*>(uniforms), temperature.values, temperature.value,
                                      top_k.values, top_k.value, top_p.values, top_p.value, min_p.values, min_p.value,
                                      chosen.data_ptr<std::int64_t>(), probabilities.data_ptr<float>(),
                                      bytes > 0 ? room.data_ptr() : nullptr, bytes, stream_of(args[6], device)));
        return pair(chosen, probabilities);
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
                         TOKEN_METHOD(multiply), TOKEN_METHOD(bytes_multiply), TOKEN_METHOD(experts_multiply),
                         TOKEN_METHOD(route),    TOKEN_METHOD(sample), TOKEN_METHOD(on_current), TOKEN_METHOD(bind),
                         {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "nvcr_tokens", nullptr, -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit_nvcr_tokens() { return PyModule_Create(&module); }
