// Norms after and before a block, fused with the block's gate and the residual:
//   p = post ? N(block) : block,  hidden = residual_scale * residual + gate * p,
//   normed = N(hidden), with N(v) = v / sqrt(mean(v^2) + epsilon) * (weight +
//   weight_offset) + bias, of v - mean(v) for a layer norm.
// Sums, the residual sum and everything between the inputs and the two outputs
// are FP32; `normed` comes from the unrounded sum. Each input is read once and
// each output written once.
//
// Measured on a B200: 4096 x 4096 BF16, five tensors of rows (168 MB): 32 us, 5.3
// TB/s, bound by HBM; FP32 (336 MB) 56.5 us, 5.9 TB/s. One row of 2048 FP16: 2.1 to 2.2
// us, bound by the launch and two sums across a block. Element by element: 77 x 1111
// FP32 2.7 us, 2048 x 4097 BF16 69 us (1.2 TB/s). Rows past the registers, 512 x 20000
// FP32: 138 us (1.5 TB/s). Rows held in
// registers, with every load issued before the first sum, took the first from 82
// us (the row re-read for each pass) to 47, and 64 registers a thread, which lets
// twice as many rows be in flight, to 32.
#include "token_elements.cuh"

#include <type_traits>

namespace nvcr_sm100::token {
namespace {

constexpr int threads = 256;

__device__ __forceinline__ float block_sum(float v, float* scratch) {
    v = warp_sum(v);
    __syncthreads();
    if (threadIdx.x % 32 == 0) scratch[threadIdx.x / 32] = v;
    __syncthreads();
    float total = 0.0f;
    for (int w = 0; w < threads / 32; ++w) total += scratch[w];
    return total;
}

template <typename T>
__device__ __forceinline__ float weight_at(const void* weight, int i, float offset) {
    return weight == nullptr ? 1.0f : widen(static_cast<const T*>(weight)[i]) + offset;
}

template <typename T>
__device__ __forceinline__ float bias_at(const void* bias, int i) {
    return bias == nullptr ? 0.0f : widen(static_cast<const T*>(bias)[i]);
}

// One row a block, re-reading the row for each pass: rows too long for the registers.
template <typename T>
__global__ void __launch_bounds__(threads) long_norm_kernel(NormArgs a) {
    __shared__ float scratch[threads / 32];
    join_chain();
    const std::int64_t row = blockIdx.x;
    const T* block = static_cast<const T*>(a.block) + row * a.block_stride;
    const T* residual = a.residual == nullptr ? nullptr : static_cast<const T*>(a.residual) + row * a.residual_stride;
    const T* gate = a.gate == nullptr ? nullptr : static_cast<const T*>(a.gate) + row * a.gate_stride;
    const float inverse = 1.0f / static_cast<float>(a.width);
    float mean = 0.0f, factor = 1.0f;
    if (a.post) {
        if (a.layer) {
            float sum = 0.0f;
            for (int i = threadIdx.x; i < a.width; i += threads) sum += widen(block[i]);
            mean = block_sum(sum, scratch) * inverse;
        }
        float squares = 0.0f;
        for (int i = threadIdx.x; i < a.width; i += threads) {
            const float v = widen(block[i]) - mean;
            squares = fmaf(v, v, squares);
        }
        factor = rsqrtf(block_sum(squares, scratch) * inverse + a.epsilon);
    }
    auto hidden_at = [&](int i) {
        float p = widen(block[i]);
        if (a.post) p = fmaf((p - mean) * factor, weight_at<T>(a.post_weight, i, a.weight_offset), bias_at<T>(a.post_bias, i));
        if (gate != nullptr) p *= widen(gate[i]);
        return residual == nullptr ? p : fmaf(widen(residual[i]), a.residual_scale, p);
    };
    float hidden_mean = 0.0f, hidden_factor = 1.0f;
    if (a.normed != nullptr) {
        if (a.layer) {
            float sum = 0.0f;
            for (int i = threadIdx.x; i < a.width; i += threads) sum += hidden_at(i);
            hidden_mean = block_sum(sum, scratch) * inverse;
        }
        float squares = 0.0f;
        for (int i = threadIdx.x; i < a.width; i += threads) {
            const float v = hidden_at(i) - hidden_mean;
            squares = fmaf(v, v, squares);
        }
        hidden_factor = rsqrtf(block_sum(squares, scratch) * inverse + a.epsilon);
    }
    for (int i = threadIdx.x; i < a.width; i += threads) {
        const float h = hidden_at(i);
        if (a.hidden != nullptr) static_cast<T*>(a.hidden)[row * a.width + i] = narrow<T>(h);
        if (a.normed != nullptr) {
            static_cast<T*>(a.normed)[row * a.width + i] = narrow<T>(fmaf(
                (h - hidden_mean) * hidden_factor, weight_at<T>(a.pre_weight, i, a.weight_offset), bias_at<T>(a.pre_bias, i)));
        }
    }
}

// VEC consecutive elements in one access: 16 bytes as words, or a single element.
template <typename T, int VEC>
struct Pack {
    uint4 words;
    __device__ __forceinline__ unsigned word(int i) const {
        return i == 0 ? words.x : i == 1 ? words.y : i == 2 ? words.z : words.w;
    }
    __device__ __forceinline__ float get(int i) const {
        if constexpr (sizeof(T) == 4) {
            return __uint_as_float(word(i));
        } else if constexpr (std::is_same_v<T, __nv_bfloat16>) {
            return __uint_as_float(i % 2 == 0 ? word(i / 2) << 16 : word(i / 2) & 0xffff0000u);
        } else {
            const unsigned pair = word(i / 2);
            const float2 both = __half22float2(reinterpret_cast<const __half2&>(pair));
            return i % 2 == 0 ? both.x : both.y;
        }
    }
    __device__ __forceinline__ void set(const float (&v)[VEC]) {
        unsigned made[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if constexpr (sizeof(T) == 4) {
                made[i] = __float_as_uint(v[i]);
            } else if constexpr (std::is_same_v<T, __nv_bfloat16>) {
                const __nv_bfloat162 pair = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
                made[i] = reinterpret_cast<const unsigned&>(pair);
            } else {
                const __half2 pair = __floats2half2_rn(v[2 * i], v[2 * i + 1]);
                made[i] = reinterpret_cast<const unsigned&>(pair);
            }
        }
        words = {made[0], made[1], made[2], made[3]};
    }
};
template <typename T>
struct Pack<T, 1> {
    T value;
    __device__ __forceinline__ float get(int) const { return widen(value); }
    __device__ __forceinline__ void set(const float (&v)[1]) { value = narrow<T>(v[0]); }
};

// One row a block (or a warp, rows threadIdx.y, when blockDim.x is 32), held in registers: a thread has C times VEC
// elements, and everything the row needs is loaded before the first sum.
template <typename T, int VEC, int C>
__global__ void __launch_bounds__(C == 1 ? 1024 : 512, VEC > 1 && C == 2 ? 2 : 1) norm_kernel(NormArgs a) {
    using P = Pack<T, VEC>;
    __shared__ float scratch[4][32];
    join_chain();
    const std::int64_t row = static_cast<std::int64_t>(blockIdx.x) * blockDim.y + threadIdx.y;
    if (row >= a.rows) return;  // whole warps of a block without barriers
    const int warps = blockDim.x / 32, lane = threadIdx.x % 32, warp = threadIdx.x / 32;
    int sums = 0;
    auto row_sum = [&](float v) {  // one barrier: each sum of the row has its own scratch
        v = warp_sum(v);
        if (warps == 1) return v;
        if (lane == 0) scratch[sums][warp] = v;
        __syncthreads();
        v = warp_sum(lane < warps ? scratch[sums][lane] : 0.0f);
        ++sums;
        return v;
    };
    int at[C];
    bool in[C];
#pragma unroll
    for (int c = 0; c < C; ++c) {
        at[c] = (c * static_cast<int>(blockDim.x) + static_cast<int>(threadIdx.x)) * VEC;
        in[c] = at[c] < a.width;
    }
    auto load = [&](const void* base, std::int64_t offset, P (&to)[C]) {
        if (base == nullptr) return;
#pragma unroll
        for (int c = 0; c < C; ++c) {
            if (in[c]) to[c] = *reinterpret_cast<const P*>(static_cast<const T*>(base) + offset + at[c]);
        }
    };
    P block[C], residual[C], gate[C], weight[C], bias[C];
    load(a.block, row * a.block_stride, block);
    load(a.residual, row * a.residual_stride, residual);
    load(a.gate, row * a.gate_stride, gate);
    constexpr bool early = C == 1;  // the weights too; else there are not the registers, and many rows find them in L1
    if (early) load(a.post_weight, 0, weight), load(a.post_bias, 0, bias);
    float v[C][VEC];
#pragma unroll
    for (int c = 0; c < C; ++c) {
#pragma unroll
        for (int i = 0; i < VEC; ++i) v[c][i] = in[c] ? block[c].get(i) : 0.0f;
    }
    const float inverse = 1.0f / static_cast<float>(a.width);
    // v becomes its norm; elements past the width stay out of the sums and keep any value
    auto normalise = [&](const void* has_weight, const void* has_bias) {
        float mean = 0.0f;
        if (a.layer) {
            float sum = 0.0f;
#pragma unroll
            for (int c = 0; c < C; ++c) {
#pragma unroll
                for (int i = 0; i < VEC; ++i) sum += in[c] ? v[c][i] : 0.0f;
            }
            mean = row_sum(sum) * inverse;
        }
        float squares = 0.0f;
#pragma unroll
        for (int c = 0; c < C; ++c) {
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
                v[c][i] -= mean;
                squares = in[c] ? fmaf(v[c][i], v[c][i], squares) : squares;
            }
        }
        const float factor = rsqrtf(row_sum(squares) * inverse + a.epsilon);
        if (!early) load(has_weight, 0, weight), load(has_bias, 0, bias);
#pragma unroll
        for (int c = 0; c < C; ++c) {
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
                const float w = has_weight == nullptr ? 1.0f : weight[c].get(i) + a.weight_offset;
                const float b = has_bias == nullptr ? 0.0f : bias[c].get(i);
                v[c][i] = fmaf(v[c][i] * factor, w, b);
            }
        }
    };
    if (a.post) normalise(a.post_weight, a.post_bias);
    if (early && a.normed != nullptr) load(a.pre_weight, 0, weight), load(a.pre_bias, 0, bias);
#pragma unroll
    for (int c = 0; c < C; ++c) {
#pragma unroll
        for (int i = 0; i < VEC; ++i) {
            if (a.gate != nullptr) v[c][i] *= gate[c].get(i);
            if (a.residual != nullptr) v[c][i] = fmaf(residual[c].get(i), a.residual_scale, v[c][i]);
        }
    }
    auto store = [&](void* base) {
#pragma unroll
        for (int c = 0; c < C; ++c) {
            P out;
            out.set(v[c]);
            if (in[c]) *reinterpret_cast<P*>(static_cast<T*>(base) + row * a.width + at[c]) = out;
        }
    };
    if (a.hidden != nullptr) store(a.hidden);
    if (a.normed != nullptr) {
        normalise(a.pre_weight, a.pre_bias);
        store(a.normed);
    }
}

template <typename T, int VEC, int C>
cudaError_t launch_rows(const NormArgs& a, cudaStream_t stream) {
    const int vectors = (a.width + VEC - 1) / VEC, lanes = (vectors + C - 1) / C;
    const unsigned threads = static_cast<unsigned>((lanes + 31) / 32 * 32);
    const unsigned together = threads == 32 ? 8 : 1;  // rows of a block
    const unsigned grid = static_cast<unsigned>((a.rows + together - 1) / together);
    return kernels::launch_overlapped(norm_kernel<T, VEC, C>, dim3(grid), dim3(threads, together), 0, stream, a);
}

template <typename T>
cudaError_t launch_type(const NormArgs& a, cudaStream_t stream) {
    constexpr int vec = 16 / sizeof(T);
    const auto aligned = [](const void* p, std::int64_t stride) {
        return reinterpret_cast<std::uintptr_t>(p) % 16 == 0 && stride % (16 / static_cast<std::int64_t>(sizeof(T))) == 0;
    };
    const bool vectors = a.width % vec == 0 && aligned(a.block, a.block_stride) && aligned(a.residual, a.residual_stride) &&
        aligned(a.gate, a.gate_stride) && aligned(a.post_weight, 0) && aligned(a.post_bias, 0) &&
        aligned(a.pre_weight, 0) && aligned(a.pre_bias, 0) && aligned(a.hidden, 0) && aligned(a.normed, 0);
    if (vectors) {
        // A thread with one vector is done soonest; with two, more of many rows are in flight. FP16, us with one and with
        // two: 1 x 2048 2.1, 2.6; 64 x 4096 2.6, 3.0; 296 x 4096 3.6, 3.6; 592 x 4096 6.3, 4.8; 4096 x 4096 42, 31.
        const int count = a.width / vec;
        const bool many = a.rows >= 4 * static_cast<std::int64_t>(sm_count());
        if (count <= 1024 && !(many && count > 64)) return launch_rows<T, vec, 1>(a, stream);
        if (count <= 1024) return launch_rows<T, vec, 2>(a, stream);
        if (count <= 2048) return launch_rows<T, vec, 4>(a, stream);
    } else {
        if (a.width <= 8 * 512) return launch_rows<T, 1, 8>(a, stream);
        if (a.width <= 16 * 512) return launch_rows<T, 1, 16>(a, stream);
    }
    return kernels::launch_overlapped(long_norm_kernel<T>, dim3(static_cast<unsigned>(a.rows)), dim3(threads), 0, stream, a);
}

}  // namespace

cudaError_t block_norm(const NormArgs& args, cudaStream_t stream) {
    if (args.rows == 0) return cudaSuccess;
    switch (args.type) {
    case Type::f16: return launch_type<__half>(args, stream);
    case Type::bf16: return launch_type<__nv_bfloat16>(args, stream);
    case Type::f32: return launch_type<float>(args, stream);
    }
    return cudaErrorInvalidValue;
}

}  // namespace nvcr_sm100::token
