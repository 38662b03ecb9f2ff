#pragma once

// What the kernels of products in 8 bits share: the layout of the weights and how a row of x becomes codes.
//
// Weights lie as blocks of 128 outputs by 128 inputs, [matrix][tile of outputs][block of inputs][128][128], zeros past the
// edges; within a block as the tensor cores read it from shared memory: the 16-byte piece c of row r lies at piece c ^ (r % 8).

#include "token_elements.cuh"

namespace nvcr_sm100::token {

constexpr int block_rows = 128;   // outputs of a weight block: the MMA's M
constexpr int block_bytes = 128;  // inputs of a block: a swizzled row
constexpr int weight_block = block_rows * block_bytes;

inline int blocks_of(int inputs) { return (inputs + block_bytes - 1) / block_bytes; }
inline int tiles_of(int outputs) { return (outputs + block_rows - 1) / block_rows; }

// A few rows, by kernels that read the weights without the tensor cores (k_token_bytes_few.cu).
bool few_rows(const BytesArgs& args);
cudaError_t multiply_few(const BytesArgs& args, cudaStream_t stream);

// Values at .. at + 15 of a row, zeros past its end; `vector`: the row begins on a 16-byte boundary.
template <typename T>
__device__ __forceinline__ void load_sixteen(const T* row, int at, int inputs, bool vector, float (&v)[16]) {
    if (vector && at + 16 <= inputs) {
        constexpr int each = 16 / sizeof(T);
#pragma unroll
        for (int part = 0; part < 16 / each; ++part) {
            const uint4 words = *reinterpret_cast<const uint4*>(row + at + part * each);
            const unsigned word[4] = {words.x, words.y, words.z, words.w};
#pragma unroll
            for (int i = 0; i < each; ++i) {
                if constexpr (sizeof(T) == 4) {
                    v[part * each + i] = __uint_as_float(word[i]);
                } else {
                    const std::uint16_t bits = static_cast<std::uint16_t>(word[i / 2] >> (i % 2 * 16));
                    v[part * each + i] = widen(reinterpret_cast<const T&>(bits));
                }
            }
        }
    } else {
#pragma unroll
        for (int i = 0; i < 16; ++i) v[i] = at + i < inputs ? widen(row[at + i]) : 0.0f;
    }
}

// The scale of a row whose largest magnitude is `most`, and codes by it.
struct RowScale {
    float scale, inverse;
    bool finite;
    __device__ __forceinline__ explicit RowScale(float most) {
        scale = fmaxf(__fmul_rn(most, 1.0f / 127.0f), 1.17549435e-38f);  // 2^-126: the inverse of a smaller one would overflow
        inverse = __frcp_rn(scale);
        finite = most <= 3.40282347e38f;
    }
    // A row that holds a NaN or an infinity gives no numbers.
    __device__ __forceinline__ float told() const { return finite ? scale : __int_as_float(0x7fffffff); }
    __device__ __forceinline__ uint4 codes(const float (&v)[16]) const {
        unsigned words[4];
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            unsigned byte[4];
#pragma unroll
            for (int b = 0; b < 4; ++b) {
                // within 127.5 of zero: adding 1.5 * 2^23 rounds to a whole number, whose low byte is the code
                byte[b] = __float_as_uint(__fadd_rn(__fmul_rn(v[4 * w + b], inverse), 12582912.0f));
            }
            words[w] = __byte_perm(__byte_perm(byte[0], byte[1], 0x0040), __byte_perm(byte[2], byte[3], 0x0040), 0x5410);
        }
        return {words[0], words[1], words[2], words[3]};
    }
};

}  // namespace nvcr_sm100::token
