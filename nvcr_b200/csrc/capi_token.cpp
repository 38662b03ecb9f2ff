// The token operators of include/nvcr_sm100.h: argument checks and launches.

#include "../../include/nvcr_sm100.h"

#include "capi_internal.hpp"
#include "token_kernels.hpp"

#include <algorithm>
#include <cmath>
#include <cstdint>
#include <exception>
#include <limits>
#include <memory>
#include <mutex>
#include <new>
#include <string>
#include <vector>

struct nvcr_sm100_token_context {
    int device = 0;
    nvcr_sm100::token::AttendWorkspace workspace{};
    bool captured = false;  // a graph holds the workspace's address
};

int nvcr_sm100::token::sm_count() {
    static const int count = [] {
        int device = 0, found = 0;
        if (cudaGetDevice(&device) != cudaSuccess ||
            cudaDeviceGetAttribute(&found, cudaDevAttrMultiProcessorCount, device) != cudaSuccess || found <= 0) {
            cudaGetLastError();
            return 148;
        }
        return found;
    }();
    return count;
}

namespace {

using nvcr_sm100::Code;
using nvcr_sm100::Error;
using nvcr_sm100::report_error;
using nvcr_sm100::report_ok;
namespace token = nvcr_sm100::token;

// Workspaces of destroyed contexts for the next ones, which wait for the calls
// that may still use them; a captured one is nobody's again, as its graph may be
// replayed. `contexts` counts those made, so `spares` never grows past its
// reservation.
std::mutex spare_lock;
std::vector<std::unique_ptr<nvcr_sm100_token_context>> spares;
std::size_t contexts = 0;

int refuse(const char* reason) { return report_error(Error{Code::invalid_argument, reason}); }

int launched(cudaError_t status) {
    if (status == cudaSuccess) return report_ok();
    if (status == cudaErrorInvalidValue) return refuse("a size is past what a launch can hold");
    return report_error(Error{Code::backend_error, cudaGetErrorString(status)});
}

template <typename F>
int guarded(F&& body) {
    try {
        return body();
    } catch (const std::bad_alloc&) {
        return report_error(Error{Code::resource_exhausted, "host allocation failed"});
    } catch (const std::exception& exception) {
        return report_error(Error{Code::internal_error, exception.what()});
    } catch (...) {
        return report_error(Error{Code::internal_error, "unknown exception"});
    }
}

bool half_type(int type) { return type == NVCR_SM100_TOKEN_F16 || type == NVCR_SM100_TOKEN_BF16; }
bool any_type(int type) { return half_type(type) || type == NVCR_SM100_TOKEN_F32; }

constexpr std::int64_t most_rows = std::numeric_limits<std::int32_t>::max();
// Kernels walk a row, or look ahead in a sequence, in steps that pass its end: 32-bit places stay clear of 2^31.
constexpr std::int32_t most_places = 1 << 30;

// Null when the cache's shape and buffers can be used, else why not.
const char* cache_refusal(const nvcr_sm100_token_cache* cache) {
    if (cache == nullptr || cache->key_codes == nullptr || cache->key_scales == nullptr ||
        cache->value_codes == nullptr || cache->value_scales == nullptr) {
        return "null cache buffer";
    }
    if (cache->pages <= 0 || cache->kv_heads <= 0 || cache->kv_heads > 65535) return "cache pages or heads out of range";
    if (cache->page_size <= 0 || cache->page_size % 16 != 0) return "cache page_size must be a positive multiple of 16";
    if (cache->head_dim != 64 && cache->head_dim != 128 && cache->head_dim != 256) {
        return "cache head_dim must be 64, 128 or 256";
    }
    if ((cache->group != 32 && cache->group != 64 && cache->group != 128) || cache->group > cache->head_dim ||
        cache->head_dim > 4 * cache->group) {
        return "cache group must be 32, 64 or 128, with 1, 2 or 4 groups a head";
    }
    if (static_cast<std::int64_t>(cache->pages) * cache->kv_heads > most_rows / (cache->page_size / 16)) {
        return "cache has 2^31 runs of 16 places or more";
    }
    for (const void* buffer : {static_cast<const void*>(cache->key_codes), static_cast<const void*>(cache->key_scales),
                               static_cast<const void*>(cache->value_codes),
                               static_cast<const void*>(cache->value_scales)}) {
        if (reinterpret_cast<std::uintptr_t>(buffer) % 16 != 0) return "cache buffers must be 16-byte aligned";
    }
    return nullptr;
}

token::Cache cache_of(const nvcr_sm100_token_cache& cache) {
    return {cache.key_codes, cache.key_scales, cache.value_codes, cache.value_scales, cache.status,
            cache.pages,     cache.kv_heads,   cache.page_size,   cache.head_dim,     cache.group};
}

// 8 rows of 98304 inputs fit the shared memory of a cluster of eight blocks.
bool matrix_shape(std::int32_t outputs, std::int32_t inputs, std::int32_t group) {
    return outputs > 0 && outputs <= most_rows - 15 && inputs > 0 && inputs <= 98304 && (group == 32 || group == 64 || group == 128) && inputs % group == 0;
}

// 131072 products of -128 and 127 stay below 2^31.
bool byte_matrix_shape(std::int64_t matrices, std::int32_t outputs, std::int32_t inputs) {
    return matrices > 0 && matrices <= most_rows && outputs > 0 && outputs <= 1 << 24 && inputs > 0 && inputs <= 131072;
}
constexpr const char* byte_matrix_reason = "a matrix has 1 to 2^24 outputs and 1 to 131072 inputs";

// Of this thread's next call of a product in 8 bits, which takes it.
struct WaitTest {
    unsigned long long limit_ns = 0;
    std::int32_t block = -1;
};
thread_local WaitTest wait_test;

void take_wait_test(token::BytesArgs& args) {
    args.wait_ns = wait_test.limit_ns, args.withheld = wait_test.block;
    wait_test = {};
}

bool aligned(const void* buffer) { return reinterpret_cast<std::uintptr_t>(buffer) % 16 == 0; }

// Null when the experts' call can be made, else why not. Rows of experts are padded by up to 15, and counted in 32 bits.
const char* experts_refusal(std::int64_t tokens, std::int32_t chosen, std::int32_t experts, std::int32_t outputs,
                            std::int32_t inputs) {
    if (experts <= 0 || experts > token::most_experts) return "experts must be 1 to 1024";
    if (!byte_matrix_shape(experts, outputs, inputs)) return byte_matrix_reason;
    if (chosen <= 0 || tokens < 0 || tokens > most_places / chosen) return "tokens or chosen out of range";
    return nullptr;
}

token::BytesArgs experts_args(std::int64_t tokens, std::int32_t chosen, const std::int32_t* choices, const float* weights,
                              std::int32_t experts, std::int32_t outputs, std::int32_t inputs) {
    token::BytesArgs args{};
    args.tokens = tokens, args.chosen = chosen, args.inner = 1;
    args.choices = choices, args.weights = weights;
    args.experts = experts, args.outputs = outputs, args.inputs = inputs;
    return args;
}

token::BytesArgs matrix_args(std::int64_t rows, std::int32_t outputs, std::int32_t inputs) {
    token::BytesArgs args{};
    args.tokens = rows, args.inner = args.chosen = args.experts = 1;
    args.outputs = outputs, args.inputs = inputs;
    return args;
}

}  // namespace

extern "C" {

int nvcr_sm100_token_norm(int type, int layer, int post, const void* block, int64_t block_stride, const void* residual,
                          int64_t residual_stride, const void* gate, int64_t gate_stride, const void* post_weight,
                          const void* post_bias, const void* pre_weight, const void* pre_bias, void* hidden,
                          void* normed, int64_t rows, int32_t width, float residual_scale, float weight_offset,
                          float epsilon, void* stream) {
    return guarded([&] {
        if (!any_type(type)) return refuse("unknown type");
        if (rows < 0 || rows > most_rows || width <= 0 || width > most_places) return refuse("rows or width out of range");
        if (rows > 0 && hidden == nullptr && normed == nullptr) return refuse("neither hidden nor normed is wanted");
        if (rows > 0 && block == nullptr) return refuse("null block");
        if (!(epsilon >= 0.0f)) return refuse("epsilon must not be negative");
        return launched(token::block_norm({static_cast<token::Type>(type), layer != 0, post != 0, block, block_stride,
                                           residual, residual_stride, gate, gate_stride, post_weight, post_bias,
                                           pre_weight, pre_bias, hidden, normed, rows, width, residual_scale,
                                           weight_offset, epsilon},
                                          static_cast<cudaStream_t>(stream)));
    });
}

int nvcr_sm100_token_append(const nvcr_sm100_token_cache* cache, int type, const void* keys, int64_t key_stride,
                            int64_t key_head_stride, const void* values, int64_t value_stride,
                            int64_t value_head_stride, const int64_t* slots, int64_t tokens, const void* queries,
                            int64_t query_stride, int64_t query_head_stride, int32_t query_heads, void* rotated,
                            const int32_t* positions, const float* cosines, const float* sines, int64_t table_rows,
                            int32_t rotary, int interleaved, void* stream) {
    return guarded([&] {
        if (const char* reason = cache_refusal(cache)) return refuse(reason);
        if (!half_type(type)) return refuse("type must be F16 or BF16");
        if (tokens < 0 || tokens > most_rows) return refuse("tokens out of range");
        if (tokens > 0 && (keys == nullptr || values == nullptr || slots == nullptr)) {
            return refuse("null keys, values or slots");
        }
        if (queries != nullptr && (rotated == nullptr || query_heads <= 0 || query_heads > 65535)) {
            return refuse("queries need an output and 1 to 65535 heads");
        }
        if (positions != nullptr) {
            if (cosines == nullptr || sines == nullptr || table_rows <= 0) return refuse("null or empty rotation table");
            if (rotary <= 0 || rotary % 2 != 0 || rotary > cache->head_dim) {
                return refuse("rotary must be even, positive and at most head_dim");
            }
        }
        return launched(token::append(cache_of(*cache),
                                      {static_cast<token::Type>(type), keys, key_stride, key_head_stride, values,
                                       value_stride, value_head_stride, slots, tokens, queries, query_stride,
                                       query_head_stride, query_heads, rotated, positions, cosines, sines, table_rows,
                                       rotary, interleaved != 0},
                                      static_cast<cudaStream_t>(stream)));
    });
}

int nvcr_sm100_token_read(const nvcr_sm100_token_cache* cache, int type, const int64_t* slots, int64_t count,
                          void* keys, void* values, void* stream) {
    return guarded([&] {
        if (const char* reason = cache_refusal(cache)) return refuse(reason);
        if (!any_type(type)) return refuse("unknown type");
        if (count < 0 || count > most_rows) return refuse("count out of range");
        if (count > 0 && (slots == nullptr || keys == nullptr || values == nullptr)) {
            return refuse("null slots, keys or values");
        }
        return launched(token::read(cache_of(*cache), static_cast<token::Type>(type), slots, count, keys, values,
                                    static_cast<cudaStream_t>(stream)));
    });
}

int nvcr_sm100_token_context_create(nvcr_sm100_token_context** context) {
    return guarded([&] {
        if (context == nullptr) return refuse("null argument");
        *context = nullptr;
        int device = 0;
        cudaError_t status = cudaGetDevice(&device);
        if (status != cudaSuccess) return launched(status);
        const std::size_t ticket_bytes = (token::attend_ticket_bytes() + 255) / 256 * 256;
        {
            std::unique_lock<std::mutex> guard(spare_lock);
            auto spare = std::find_if(spares.begin(), spares.end(),
                                      [&](const auto& c) { return c->device == device && !c->captured; });
            if (spare != spares.end()) {
                std::unique_ptr<nvcr_sm100_token_context> found = std::move(*spare);
                spares.erase(spare);
                guard.unlock();
                status = cudaDeviceSynchronize();  // the destroyed context's calls
                if (status == cudaSuccess) status = cudaMemset(found->workspace.tickets, 0, ticket_bytes);
                if (status == cudaSuccess) status = cudaStreamSynchronize(nullptr);
                if (status != cudaSuccess) {
                    guard.lock();
                    spares.push_back(std::move(found));
                    return launched(status);
                }
                *context = found.release();
                return report_ok();
            }
            spares.reserve(++contexts);  // so that destroying one needs no memory
        }
        auto made = std::make_unique<nvcr_sm100_token_context>();
        made->device = device;
        unsigned char* memory = nullptr;
        status = cudaMalloc(&memory, ticket_bytes + token::attend_partial_bytes());
        if (status == cudaErrorMemoryAllocation) {
            cudaGetLastError();
            return report_error(Error{Code::resource_exhausted, "no device memory for the context's workspace"});
        }
        if (status == cudaSuccess) status = cudaMemset(memory, 0, ticket_bytes);
        // the memset is on the default stream, which other streams need not wait for
        if (status == cudaSuccess) status = cudaStreamSynchronize(nullptr);
        if (status != cudaSuccess) {
            cudaFree(memory);
            return launched(status);
        }
        made->workspace = {reinterpret_cast<float*>(memory + ticket_bytes), reinterpret_cast<unsigned*>(memory)};
        *context = made.release();
        return report_ok();
    });
}

void nvcr_sm100_token_context_destroy(nvcr_sm100_token_context* context) {
    if (context == nullptr) return;
    // No CUDA call: this may come at any time, in the middle of a capture or of the calls that use the workspace.
    std::lock_guard<std::mutex> guard(spare_lock);
    spares.emplace_back(context);
}

int nvcr_sm100_token_attend(nvcr_sm100_token_context* context, const nvcr_sm100_token_cache* cache, int type,
                            const void* queries, int64_t query_stride, int64_t query_head_stride, int64_t tokens,
                            int32_t heads, const int32_t* page_table, int64_t table_stride, int32_t table_pages,
                            const int32_t* lengths, int32_t batch, const int32_t* query_offsets, int32_t max_queries,
                            int32_t max_length, float scale, void* output, void* stream) {
    return guarded([&] {
        if (context == nullptr) return refuse("null context");
        if (const char* reason = cache_refusal(cache)) return refuse(reason);
        if (!half_type(type)) return refuse("type must be F16 or BF16");
        if (tokens < 0 || tokens > most_rows || batch < 0 || batch > 65535) return refuse("tokens or batch out of range");
        if (heads <= 0 || heads > 65535 || heads % cache->kv_heads != 0) {
            return refuse("heads must be a positive multiple of the cache's heads");
        }
        if (max_queries <= 0 || max_queries > 65535) return refuse("max_queries out of range");
        if (query_offsets == nullptr && tokens != batch) return refuse("without query_offsets there is one token a sequence");
        if (max_length > most_places) return refuse("max_length is at most 2^30");
        if (max_length < 0 || table_pages < 0 ||
            max_length > static_cast<std::int64_t>(table_pages) * cache->page_size) {
            return refuse("max_length needs more pages than page_table has");
        }
        if (!std::isfinite(scale)) return refuse("scale must be finite");
        if (tokens > 0 &&
            (output == nullptr || (batch > 0 && (queries == nullptr || page_table == nullptr || lengths == nullptr)))) {
            return refuse("null queries, page_table, lengths or output");
        }
        if (reinterpret_cast<std::uintptr_t>(output) % 16 != 0) return refuse("output must be 16-byte aligned");
        int device = 0;
        const cudaError_t status = cudaGetDevice(&device);
        if (status != cudaSuccess) return launched(status);
        if (device != context->device) {
            return report_error(Error{Code::invalid_state, "the context belongs to device " +
                                                               std::to_string(context->device)});
        }
        if (!context->captured) {
            cudaStreamCaptureStatus capture = cudaStreamCaptureStatusNone;
            const cudaError_t asked = cudaStreamIsCapturing(static_cast<cudaStream_t>(stream), &capture);
            if (asked != cudaSuccess) return launched(asked);
            context->captured = capture != cudaStreamCaptureStatusNone;
        }
        return launched(token::attend(cache_of(*cache),
                                      {static_cast<token::Type>(type), queries, query_stride, query_head_stride, tokens,
                                       heads, page_table, table_stride, lengths, batch, query_offsets, max_queries,
                                       max_length, scale, output},
                                      context->workspace, static_cast<cudaStream_t>(stream)));
    });
}

int nvcr_sm100_token_packed_bytes(int32_t outputs, int32_t inputs, int32_t group, size_t* code_bytes,
                                  size_t* scale_bytes) {
    return guarded([&] {
        if (code_bytes == nullptr || scale_bytes == nullptr) return refuse("null argument");
        if (!matrix_shape(outputs, inputs, group)) return refuse("inputs must be a multiple of a group of 32, 64 or 128, and at most 98304");
        *code_bytes = token::packed_code_bytes(outputs, inputs);
        *scale_bytes = token::packed_scale_bytes(outputs, inputs, group);
        return report_ok();
    });
}

int nvcr_sm100_token_pack(const uint8_t* codes, const uint16_t* scales, const uint16_t* minimums, int32_t outputs,
                          int32_t inputs, int32_t group, void* packed_codes, void* packed_scales, void* stream) {
    return guarded([&] {
        if (!matrix_shape(outputs, inputs, group)) return refuse("inputs must be a multiple of a group of 32, 64 or 128, and at most 98304");
        if (codes == nullptr || scales == nullptr || minimums == nullptr || packed_codes == nullptr ||
            packed_scales == nullptr) {
            return refuse("null argument");
        }
        if (reinterpret_cast<std::uintptr_t>(packed_codes) % 16 != 0 ||
            reinterpret_cast<std::uintptr_t>(packed_scales) % 16 != 0) {
            return refuse("packed buffers must be 16-byte aligned");
        }
        return launched(token::pack(codes, scales, minimums, outputs, inputs, group,
                                    static_cast<std::uint8_t*>(packed_codes), static_cast<std::uint16_t*>(packed_scales),
                                    static_cast<cudaStream_t>(stream)));
    });
}

int nvcr_sm100_token_multiply(int type, const void* x, int64_t x_stride, int64_t rows, const void* packed_codes,
                              const void* packed_scales, int32_t outputs, int32_t inputs, int32_t group,
                              const void* bias, void* y, void* stream) {
    return guarded([&] {
        if (!half_type(type)) return refuse("type must be F16 or BF16");
        if (!matrix_shape(outputs, inputs, group)) return refuse("inputs must be a multiple of a group of 32, 64 or 128, and at most 98304");
        if (rows < 0 || rows > 65535) return refuse("rows out of range");
        if (packed_codes == nullptr || packed_scales == nullptr || (rows > 0 && (x == nullptr || y == nullptr))) {
            return refuse("null argument");
        }
        if (reinterpret_cast<std::uintptr_t>(packed_codes) % 16 != 0 ||
            reinterpret_cast<std::uintptr_t>(packed_scales) % 16 != 0) {
            return refuse("packed buffers must be 16-byte aligned");
        }
        return launched(token::multiply({static_cast<token::Type>(type), x, x_stride, rows,
                                         static_cast<const std::uint8_t*>(packed_codes),
                                         static_cast<const std::uint16_t*>(packed_scales), outputs, inputs, group, bias,
                                         y},
                                        static_cast<cudaStream_t>(stream)));
    });
}

int nvcr_sm100_token_bytes_packed(int64_t matrices, int32_t outputs, int32_t inputs, size_t* bytes) {
    return guarded([&] {
        if (bytes == nullptr) return refuse("null argument");
        if (!byte_matrix_shape(matrices, outputs, inputs)) return refuse(byte_matrix_reason);
        *bytes = token::byte_matrix_bytes(matrices, outputs, inputs);
        return report_ok();
    });
}

int nvcr_sm100_token_bytes_pack(const int8_t* codes, int64_t matrices, int32_t outputs, int32_t inputs, void* packed,
                                void* stream) {
    return guarded([&] {
        if (!byte_matrix_shape(matrices, outputs, inputs)) return refuse(byte_matrix_reason);
        if (codes == nullptr || packed == nullptr) return refuse("null argument");
        if (!aligned(packed)) return refuse("packed buffers must be 16-byte aligned");
        return launched(token::pack_bytes(codes, matrices, outputs, inputs, packed, static_cast<cudaStream_t>(stream)));
    });
}

int nvcr_sm100_token_bytes_workspace(int64_t rows, int32_t outputs, int32_t inputs, size_t* bytes) {
    return guarded([&] {
        if (bytes == nullptr) return refuse("null argument");
        if (!byte_matrix_shape(1, outputs, inputs)) return refuse(byte_matrix_reason);
        if (rows < 0 || rows > most_places) return refuse("rows out of range");
        *bytes = token::bytes_workspace(matrix_args(rows, outputs, inputs));
        return report_ok();
    });
}

int nvcr_sm100_token_bytes_multiply(int type, const void* x, int64_t x_stride, int64_t rows, const void* packed,
                                    const float* scales, int32_t outputs, int32_t inputs, const void* bias, void* y,
                                    void* workspace, size_t workspace_bytes, uint32_t* status, void* stream) {
    return guarded([&] {
        if (!any_type(type)) return refuse("unknown type");
        if (!byte_matrix_shape(1, outputs, inputs)) return refuse(byte_matrix_reason);
        if (rows < 0 || rows > most_places) return refuse("rows out of range");
        if (packed == nullptr || scales == nullptr ||
            (rows > 0 && (x == nullptr || y == nullptr || workspace == nullptr))) {
            return refuse("null argument");
        }
        if (!aligned(packed) || !aligned(workspace)) return refuse("packed and workspace buffers must be 16-byte aligned");
        token::BytesArgs args = matrix_args(rows, outputs, inputs);
        if (workspace_bytes < token::bytes_workspace(args)) return refuse("the workspace is too small");
        args.type = static_cast<token::Type>(type);
        args.x = x, args.x_stride = x_stride;
        args.packed = packed, args.scales = scales, args.bias = bias, args.y = y;
        args.workspace = workspace, args.status = status;
        take_wait_test(args);
        return launched(token::multiply_bytes(args, static_cast<cudaStream_t>(stream)));
    });
}

int nvcr_sm100_token_experts_workspace(int64_t tokens, int32_t chosen, int weighted, int32_t experts, int32_t outputs,
                                       int32_t inputs, size_t* bytes) {
    return guarded([&] {
        if (bytes == nullptr) return refuse("null argument");
        if (const char* reason = experts_refusal(tokens, chosen, experts, outputs, inputs)) return refuse(reason);
        // the size goes by whether there are choices and weights, not by what they are
        const std::int32_t choices = 0;
        const float weights = 0.0f;
        *bytes = token::bytes_workspace(
            experts_args(tokens, chosen, &choices, weighted != 0 ? &weights : nullptr, experts, outputs, inputs));
        return report_ok();
    });
}

int nvcr_sm100_token_experts_multiply(int type, const void* x, int64_t x_stride, int64_t x_row_stride, int rows_each,
                                      int64_t tokens, const int32_t* choices, int32_t chosen, const float* weights,
                                      const void* packed, const float* scales, int32_t experts, int32_t outputs,
                                      int32_t inputs, void* y, void* workspace, size_t workspace_bytes,
                                      uint32_t* status, void* stream) {
    return guarded([&] {
        if (!any_type(type)) return refuse("unknown type");
        if (const char* reason = experts_refusal(tokens, chosen, experts, outputs, inputs)) return refuse(reason);
        if (packed == nullptr || scales == nullptr ||
            (tokens > 0 && (x == nullptr || choices == nullptr || y == nullptr || workspace == nullptr))) {
            return refuse("null argument");
        }
        if (!aligned(packed) || !aligned(workspace)) return refuse("packed and workspace buffers must be 16-byte aligned");
        if (tokens == 0) return report_ok();
        token::BytesArgs args = experts_args(tokens, chosen, choices, weights, experts, outputs, inputs);
        if (workspace_bytes < token::bytes_workspace(args)) return refuse("the workspace is too small");
        args.type = static_cast<token::Type>(type);
        args.x = x, args.x_stride = x_stride;
        if (rows_each != 0) args.inner = chosen, args.x_inner_stride = x_row_stride;
        args.packed = packed, args.scales = scales, args.y = y;
        args.workspace = workspace, args.status = status;
        take_wait_test(args);
        return launched(token::multiply_bytes(args, static_cast<cudaStream_t>(stream)));
    });
}

int nvcr_sm100_token_test_wait_timeout(unsigned int limit_ms, int32_t block) {
    return guarded([&] {
        if (limit_ms == 0 || limit_ms > 4000) return refuse("the limit must be 1 to 4000 ms");
        if (block < 0) return refuse("block out of range");
        wait_test = {limit_ms * 1000000ull, block};
        return report_ok();
    });
}

int nvcr_sm100_token_route(int type, const void* scores, int64_t stride, int64_t tokens, int32_t experts,
                           int32_t count, int sigmoid, const float* bias, int32_t groups, int32_t kept_groups,
                           int renormalise, float scale, int32_t* choices, float* weights, void* stream) {
    return guarded([&] {
        if (!any_type(type)) return refuse("unknown type");
        if (tokens < 0 || tokens > most_rows) return refuse("tokens out of range");
        if (experts <= 0 || experts > token::most_experts) return refuse("experts must be 1 to 1024");
        if (count <= 0 || count > experts) return refuse("count must be 1 to the number of experts");
        if (groups <= 0 || experts % groups != 0) return refuse("experts must be a multiple of groups");
        if (kept_groups <= 0 || kept_groups > groups) return refuse("kept_groups must be 1 to groups");
        if (!std::isfinite(scale)) return refuse("scale must be finite");
        if (tokens > 0 && (scores == nullptr || choices == nullptr || weights == nullptr)) {
            return refuse("null scores, choices or weights");
        }
        return launched(token::route({static_cast<token::Type>(type), scores, stride, tokens, experts, count, sigmoid != 0,
                                      bias, groups, kept_groups, renormalise != 0, scale, choices, weights},
                                     static_cast<cudaStream_t>(stream)));
    });
}

int nvcr_sm100_token_sample_workspace(int type, int64_t rows, int32_t symbols, size_t* bytes) {
    return guarded([&] {
        if (bytes == nullptr) return refuse("null argument");
        if (!any_type(type)) return refuse("unknown type");
        if (rows < 0 || rows > most_rows) return refuse("rows out of range");
        if (symbols <= 0 || symbols > token::most_symbols) return refuse("symbols must be 1 to 2^20");
        *bytes = token::sample_workspace(static_cast<token::Type>(type), rows, symbols);
        return report_ok();
    });
}

int nvcr_sm100_token_sample(int type, const void* logits, int64_t stride, int64_t rows, int32_t symbols,
                            const float* uniforms, const float* temperatures, float temperature,
                            const int32_t* top_ks, int32_t top_k, const float* top_ps, float top_p, const float* min_ps,
                            float min_p, int64_t* chosen, float* probabilities, void* workspace, size_t workspace_bytes,
                            void* stream) {
    return guarded([&] {
        if (!any_type(type)) return refuse("unknown type");
        if (rows < 0 || rows > most_rows) return refuse("rows out of range");
        if (symbols <= 0 || symbols > token::most_symbols) return refuse("symbols must be 1 to 2^20");
        if (!aligned(workspace)) return refuse("the workspace must be 16-byte aligned");
        const std::size_t needed = token::sample_workspace(static_cast<token::Type>(type), rows, symbols);
        if (workspace_bytes < needed || (needed > 0 && workspace == nullptr)) return refuse("the workspace is too small");
        if (rows > 0 && (logits == nullptr || uniforms == nullptr || chosen == nullptr || probabilities == nullptr)) {
            return refuse("null logits, uniforms, chosen or probabilities");
        }
        return launched(token::sample({static_cast<token::Type>(type), logits, stride, rows, symbols, uniforms, temperatures,
                                       top_ks, top_ps, min_ps, temperature, top_k, top_p, min_p, chosen, probabilities,
                                       workspace},
                                      static_cast<cudaStream_t>(stream)));
    });
}

}  // extern "C"
