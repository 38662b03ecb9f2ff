#pragma once

// Launchers of the token operators (k_token_*.cu): the steps of a token model
// in low-bit form. Every launcher enqueues on `stream` and returns the launch
// status; the entry points in capi_token.cpp have checked the arguments.
//
// The 4-bit group form, of cached keys and values and of weights: `group`
// consecutive values are held as codes c in 0..15 (two a byte, the even index
// in the low half), an FP16 scale s and an FP16 minimum m, and stand for
// c * s + m.

#include <cstddef>
#include <cstdint>

#include <cuda_runtime.h>

namespace nvcr_sm100::token {

// Streaming multiprocessors of the current device (looked up once; a process
// drives GPUs of one kind).
int sm_count();

enum class Type : int { f16 = 0, bf16 = 1, f32 = 2 };

// Bits of a cache's status word: what a kernel found wrong in device data.
constexpr unsigned status_slot = 1;      // a slot past the cache's end
constexpr unsigned status_position = 2;  // a position outside the rotation table
constexpr unsigned status_page = 4;      // a page number outside the cache
constexpr unsigned status_length = 8;    // a sequence's length or offsets outside what the call said

// Rows of one batch of vectors whose last dimension is contiguous; strides in elements.
struct NormArgs {
    Type type;
    bool layer;      // subtract the mean (layer norm), else root mean square
    bool post;       // norm of the block's output
    const void* block;
    std::int64_t block_stride;
    const void* residual;  // null: none
    std::int64_t residual_stride;
    const void* gate;  // null: one
    std::int64_t gate_stride;  // 0: the same for every row
    const void* post_weight;   // null weights are one, null biases zero
    const void* post_bias;
    const void* pre_weight;
    const void* pre_bias;
    void* hidden;  // null: not wanted
    void* normed;  // null: not wanted, and no norm of the sum
    std::int64_t rows;
    int width;
    float residual_scale;
    float weight_offset;
    float epsilon;
};
cudaError_t block_norm(const NormArgs& args, cudaStream_t stream);

// Pages of codes [pages][kv_heads][page_size][head_dim / 2] and of (scale,
// minimum) pairs [pages][kv_heads][page_size][head_dim / group][2].
struct Cache {
    std::uint8_t* key_codes;
    std::uint16_t* key_scales;
    std::uint8_t* value_codes;
    std::uint16_t* value_scales;
    unsigned* status;  // null: not wanted
    int pages;
    int kv_heads;
    int page_size;
    int head_dim;
    int group;
};

struct AppendArgs {
    Type type;
    const void* keys;
    std::int64_t key_stride, key_head_stride;
    const void* values;
    std::int64_t value_stride, value_head_stride;
    const std::int64_t* slots;
    std::int64_t tokens;
    const void* queries;  // null: none
    std::int64_t query_stride, query_head_stride;
    int query_heads;
    void* rotated;  // [tokens][query_heads][head_dim]
    const std::int32_t* positions;  // null: no rotation
    const float* cosines;           // [table_rows][rotary / 2]
    const float* sines;
    std::int64_t table_rows;
    int rotary;
    bool interleaved;
};
cudaError_t append(const Cache& cache, const AppendArgs& args, cudaStream_t stream);
cudaError_t read(const Cache& cache, Type type, const std::int64_t* slots, std::int64_t count, void* keys, void* values,
                 cudaStream_t stream);

struct AttendArgs {
    Type type;
    const void* queries;
    std::int64_t query_stride, query_head_stride;
    std::int64_t tokens;
    int heads;
    const std::int32_t* page_table;
    std::int64_t table_stride;
    const std::int32_t* lengths;
    int batch;
    const std::int32_t* query_offsets;  // null: one token of each sequence
    int max_queries;
    int max_length;
    float scale;
    void* output;  // [tokens][heads][head_dim]
};
// Where ranges of one sequence's length are joined; tickets are zero between calls.
struct AttendWorkspace {
    float* partials;
    unsigned* tickets;
};
std::size_t attend_partial_bytes();
std::size_t attend_ticket_bytes();
cudaError_t attend(const Cache& cache, const AttendArgs& args, const AttendWorkspace& workspace, cudaStream_t stream);

struct MultiplyArgs {
    Type type;
    const void* x;
    std::int64_t x_stride;
    std::int64_t rows;
    const std::uint8_t* codes;
    const std::uint16_t* scales;
    int outputs;
    int inputs;
    int group;
    const void* bias;  // null: none
    void* y;           // [rows][outputs]
};
// The packed form of codes [outputs][inputs / 2] with scales and minimums
// [outputs][inputs / group], and its sizes in bytes.
std::size_t packed_code_bytes(int outputs, int inputs);
std::size_t packed_scale_bytes(int outputs, int inputs, int group);
cudaError_t pack(const std::uint8_t* codes, const std::uint16_t* scales, const std::uint16_t* minimums, int outputs,
                 int inputs, int group, std::uint8_t* packed_codes, std::uint16_t* packed_scales, cudaStream_t stream);
cudaError_t multiply(const MultiplyArgs& args, cudaStream_t stream);

// Products in 8 bits: one matrix for all rows, or (choices not null) for each row of a token's `chosen` ones that of
// an expert.
struct BytesArgs {
    Type type;
    const void* x;  // [tokens][inner][inputs]
    std::int64_t x_stride, x_inner_stride;
    std::int64_t tokens;
    int inner;   // rows of x a token: 1, or chosen
    int chosen;  // rows of products a token
    const std::int32_t* choices;  // [tokens][chosen]; null: one matrix, and chosen is 1
    const float* weights;         // [tokens][chosen], or null: products are not summed
    const void* packed;
    const float* scales;  // [experts][outputs]
    int experts;
    int outputs;
    int inputs;
    const void* bias;  // [outputs], or null; null with choices
    void* y;           // [tokens][chosen][outputs], or with weights [tokens][outputs]
    void* workspace;
    unsigned* status;  // null: not wanted
    // self-test: after how long a wait gives up (0: the kernels' limit), and the block that copies nothing (-1: none)
    unsigned long long wait_ns = 0;
    int withheld = -1;
};
std::size_t byte_matrix_bytes(std::int64_t matrices, int outputs, int inputs);
cudaError_t pack_bytes(const std::int8_t* codes, std::int64_t matrices, int outputs, int inputs, void* packed,
                       cudaStream_t stream);
std::size_t bytes_workspace(const BytesArgs& args);
cudaError_t multiply_bytes(const BytesArgs& args, cudaStream_t stream);

struct RouteArgs {
    Type type;
    const void* scores;
    std::int64_t stride;
    std::int64_t tokens;
    int experts;
    int count;
    bool sigmoid;
    const float* bias;  // null: none
    int groups;
    int kept_groups;
    bool renormalise;
    float scale;
    std::int32_t* choices;  // [tokens][count]
    float* weights;
};
constexpr int most_experts = 1024;
cudaError_t route(const RouteArgs& args, cudaStream_t stream);

struct SampleArgs {
    Type type;
    const void* logits;
    std::int64_t stride;
    std::int64_t rows;
    int symbols;
    const float* uniforms;
    const float* temperatures;  // null: `temperature` for every row; the same of the others
    const std::int32_t* top_ks;
    const float* top_ps;
    const float* min_ps;
    float temperature;
    int top_k;
    float top_p;
    float min_p;
    std::int64_t* chosen;
    float* probabilities;
    void* workspace;
};
constexpr int most_symbols = 1 << 20;
std::size_t sample_workspace(Type type, std::int64_t rows, int symbols);
cudaError_t sample(const SampleArgs& args, cudaStream_t stream);

}  // namespace nvcr_sm100::token
