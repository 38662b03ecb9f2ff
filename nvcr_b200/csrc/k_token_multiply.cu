// Products of a few rows with a matrix of 4-bit weights in groups:
//   y[r][n] = sum_k x[r][k] * (c[n][k] * s[n][k / group] + m[n][k / group]) + bias[n],
// summed in FP32. HBM-bound: the codes are read once.
#include "token_elements.cuh"

namespace nvcr_sm100::token {
namespace {

constexpr int threads = 128;

// One warp an (output, row); a lane takes every 32nd byte of codes.
template <typename T>
__global__ void __launch_bounds__(threads) multiply_kernel(MultiplyArgs a) {
    const int lane = threadIdx.x % 32;
    const int output = blockIdx.x * (threads / 32) + threadIdx.x / 32;
    const std::int64_t row = blockIdx.y;
    if (output >= a.outputs) return;
    const T* x = static_cast<const T*>(a.x) + row * a.x_stride;
    const std::uint8_t* codes = a.codes + static_cast<std::int64_t>(output) * (a.inputs / 2);
    const std::uint16_t* scales = a.scales + static_cast<std::int64_t>(output) * (a.inputs / a.group) * 2;
    float sum = 0.0f;
    for (int byte = lane; byte < a.inputs / 2; byte += 32) {
        const unsigned code = codes[byte];
        const float s = half_bits(scales[2 * byte / a.group * 2]), m = half_bits(scales[2 * byte / a.group * 2 + 1]);
        sum = fmaf(widen(x[2 * byte]), fmaf(static_cast<float>(code & 15u), s, m), sum);
        sum = fmaf(widen(x[2 * byte + 1]), fmaf(static_cast<float>(code >> 4), s, m), sum);
    }
    sum = warp_sum(sum);
    if (lane == 0) {
        if (a.bias != nullptr) sum += widen(static_cast<const T*>(a.bias)[output]);
        static_cast<T*>(a.y)[row * a.outputs + output] = narrow<T>(sum);
    }
}

__global__ void interleave_kernel(const std::uint16_t* scales, const std::uint16_t* minimums, std::size_t count,
                                  std::uint16_t* packed) {
    const std::size_t i = static_cast<std::size_t>(blockIdx.x) * blockDim.x + threadIdx.x;
    if (i >= count) return;
    packed[2 * i] = scales[i];
    packed[2 * i + 1] = minimums[i];
}

}  // namespace

std::size_t packed_code_bytes(int outputs, int inputs) { return static_cast<std::size_t>(outputs) * (inputs / 2); }

std::size_t packed_scale_bytes(int outputs, int inputs, int group) {
    return static_cast<std::size_t>(outputs) * (inputs / group) * 4;
}

cudaError_t pack(const std::uint8_t* codes, const std::uint16_t* scales, const std::uint16_t* minimums, int outputs,
                 int inputs, int group, std::uint8_t* packed_codes, std::uint16_t* packed_scales, cudaStream_t stream) {
    const cudaError_t copied = cudaMemcpyAsync(packed_codes, codes, packed_code_bytes(outputs, inputs),
                                               cudaMemcpyDeviceToDevice, stream);
    if (copied != cudaSuccess) return copied;
    const std::size_t count = packed_scale_bytes(outputs, inputs, group) / 4;
    interleave_kernel<<<static_cast<unsigned>((count + 255) / 256), 256, 0, stream>>>(scales, minimums, count,
                                                                                       packed_scales);
    return cudaGetLastError();
}

cudaError_t multiply(const MultiplyArgs& args, cudaStream_t stream) {
    if (args.rows == 0) return cudaSuccess;
    const dim3 grid(static_cast<unsigned>((args.outputs + threads / 32 - 1) / (threads / 32)),
                    static_cast<unsigned>(args.rows));
    if (args.type == Type::f16) {
        multiply_kernel<__half><<<grid, threads, 0, stream>>>(args);
    } else {
        multiply_kernel<__nv_bfloat16><<<grid, threads, 0, stream>>>(args);
    }
    return cudaGetLastError();
}

}  // namespace nvcr_sm100::token
