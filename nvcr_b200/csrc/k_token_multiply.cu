// Products of a few rows with a matrix of 4-bit weights in groups:
//   y[r][n] = sum_k x[r][k] (c[n][k] s[n][g] + m[n][g]) + bias[n]
//           = sum_g s[n][g] (x . c)_g + m[n][g] sum(x)_g + bias[n].
// Both inner sums are tensor-core products (mma.m16n8k16: 16 outputs, 8 rows of
// x): the codes themselves, and ones for sum(x). With x in FP16 a nibble masked
// out of its place is the FP16 number c 2^-24 or, four bits up, c 2^-20
// (subnormal, exact), in two sums whose powers of two join the scale. bfloat16
// has no room for that in FP32's range, and there a nibble under the exponent of
// 128 is 128 + c (exact), whose 128 leaves through the minimum: m - 128 s. Sums
// are FP32, a group at a time.
//
// A few rows make this a stream of the weights: HBM-bound, or launch- and
// latency-bound where they are small. So they are laid out once in the order in
// which lanes want them: 16 outputs x 64 inputs are 512 consecutive bytes, 16 a
// lane; a lane loads whole fragments with one 16-byte load, straight to
// registers, several steps of 128 inputs ahead. A block's eight warps share the
// inputs of 16, 32 or 64 outputs and are summed in shared memory; where that
// leaves SMs idle, up to eight blocks of a cluster share the inputs and are
// summed over distributed shared memory, in order: no workspace, one launch.
#include "token_elements.cuh"

#include <algorithm>
#include <type_traits>

#include <cooperative_groups.h>

namespace nvcr_sm100::token {
namespace {

namespace cg = cooperative_groups;

constexpr int warps = 8;
constexpr int step_inputs = 128;

template <typename T>
__device__ __forceinline__ void mma(float (&d)[4], const unsigned (&a)[4], unsigned b0, unsigned b1) {
    if constexpr (std::is_same_v<T, __half>) {
        asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
            "{%0, %1, %2, %3};"
            : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    } else {
        asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
            "{%0, %1, %2, %3};"
            : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    }
}

// The packed form, from 16 x 128 steps: codes [tile of 16 outputs][step][2][lane][4 words], where lane (r, j) =
// (lane / 4, lane % 4) holds, of 64 inputs, word 0 = output r, inputs 8 j .. 8 j + 7 of the first 32; word 1 = output
// r + 8, the same; words 2 and 3 = the second 32. In a word, inputs 0 .. 7 are nibbles 0, 4, 1, 5, 2, 6, 3, 7: pairs of
// inputs are 16 bits apart. Pairs (scale, minimum) [tile][step][group][r][2 outputs]. What lies past the matrix is zero.
__host__ __device__ constexpr int tiles_of(int outputs) { return (outputs + 15) / 16; }
__host__ __device__ constexpr int steps_of(int inputs) { return (inputs + step_inputs - 1) / step_inputs; }

struct Shape {
    int steps;
    int tiles;
    bool aligned;  // x can be read 16 bytes at a time
};

// R tiles of 16 outputs, NT times 8 rows.
template <typename T, int G, int NT, int R>
__global__ void __launch_bounds__(32 * warps) multiply_kernel(const MultiplyArgs a, const Shape shape) {
    constexpr bool half = std::is_same_v<T, __half>;
    constexpr int groups = step_inputs / G, quarters = G / 32;  // 32 inputs each
    constexpr int depth = R == 1 ? 4 : R == 2 ? 2 : 1;          // steps of weights in flight
    constexpr unsigned one = half ? 0x3c003c00u : 0x3f803f80u;
    __shared__ float sums[warps][R][16][8 * NT];
    const int lane = threadIdx.x % 32, warp = threadIdx.x / 32, r = lane / 4, j = lane % 4;
    const cg::cluster_group cluster = cg::this_cluster();
    const int parts = static_cast<int>(cluster.num_blocks()), part = static_cast<int>(cluster.block_rank());
    const int first_tile = blockIdx.x / parts * R;
    const std::int64_t first_row = static_cast<std::int64_t>(blockIdx.y) * (8 * NT);
    const int stride = warps * parts, start = part * warps + warp;
    const int count = start < shape.steps ? (shape.steps - start + stride - 1) / stride : 0;

    const uint4* codes[R];
    const uint2* scales[R];
#pragma unroll
    for (int t = 0; t < R; ++t) {  // a tile past the last reads the last and is not stored
        const std::int64_t at = static_cast<std::int64_t>(min(first_tile + t, shape.tiles - 1)) * shape.steps + start;
        codes[t] = reinterpret_cast<const uint4*>(a.codes) + at * 64 + lane;
        scales[t] = reinterpret_cast<const uint2*>(a.scales) + at * (8 * groups) + r;
    }
    uint4 code[depth][R][2];
    uint2 pair[depth][R][groups];
    auto load_weights = [&](int i, int slot) {
        if (i >= count) return;
#pragma unroll
        for (int t = 0; t < R; ++t) {
            code[slot][t][0] = __ldcs(codes[t] + static_cast<std::int64_t>(i) * stride * 64);
            code[slot][t][1] = __ldcs(codes[t] + static_cast<std::int64_t>(i) * stride * 64 + 32);
#pragma unroll
            for (int g = 0; g < groups; ++g) {
                pair[slot][t][g] = __ldg(scales[t] + static_cast<std::int64_t>(i) * stride * (8 * groups) + 8 * g);
            }
        }
    };
    const T* x[NT];
#pragma unroll
    for (int n = 0; n < NT; ++n) x[n] = static_cast<const T*>(a.x) + (first_row + 8 * n + r) * a.x_stride + 8 * j;
    uint4 value[NT][4], value_next[NT][4];
    auto load_x = [&](int i, uint4 (&to)[NT][4]) {
#pragma unroll
        for (int n = 0; n < NT; ++n) {
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const int k = (start + i * stride) * step_inputs + 32 * q;
                uint4 v = {0u, 0u, 0u, 0u};
                if (i < count && k < a.inputs && first_row + 8 * n + r < a.rows) {
                    if (shape.aligned) {
                        v = __ldg(reinterpret_cast<const uint4*>(x[n] + k));
                    } else {
                        alignas(16) T values[8];
#pragma unroll
                        for (int e = 0; e < 8; ++e) values[e] = x[n][k + e];
                        v = *reinterpret_cast<const uint4*>(values);
                    }
                }
                to[n][q] = v;
            }
        }
    };
#pragma unroll
    for (int s = 0; s < depth; ++s) load_weights(s, s);
    load_x(0, value);

    float y[R][NT][4];
#pragma unroll
    for (int t = 0; t < R; ++t) {
#pragma unroll
        for (int n = 0; n < NT; ++n) y[t][n][0] = y[t][n][1] = y[t][n][2] = y[t][n][3] = 0.0f;
    }
    for (int base = 0; base < count; base += depth) {
#pragma unroll
        for (int s = 0; s < depth; ++s) {
            if (base + s >= count) break;
            load_x(base + s + 1, value_next);
#pragma unroll
            for (int g = 0; g < groups; ++g) {
                float x_sum[NT][4];
                const unsigned ones[4] = {one, one, one, one};
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    x_sum[n][0] = x_sum[n][1] = x_sum[n][2] = x_sum[n][3] = 0.0f;
#pragma unroll
                    for (int q = g * quarters; q < (g + 1) * quarters; ++q) {
                        mma<T>(x_sum[n], ones, value[n][q].x, value[n][q].z);
                        mma<T>(x_sum[n], ones, value[n][q].y, value[n][q].w);
                    }
                }
#pragma unroll
                for (int t = 0; t < R; ++t) {
                    float even[NT][4], odd[NT][4];  // for bfloat16 all of them in `even`
#pragma unroll
                    for (int n = 0; n < NT; ++n) {
#pragma unroll
                        for (int i = 0; i < 4; ++i) even[n][i] = odd[n][i] = 0.0f;
                    }
#pragma unroll
                    for (int q = g * quarters; q < (g + 1) * quarters; ++q) {
                        const uint4 raw = code[s][t][q / 2];
                        const unsigned near = q % 2 == 0 ? raw.x : raw.z, far = q % 2 == 0 ? raw.y : raw.w;
                        unsigned front[4], back[4];
                        if constexpr (half) {
                            const unsigned near8 = near >> 8, far8 = far >> 8;
                            front[0] = near & 0x000f000fu, front[1] = far & 0x000f000fu;
                            front[2] = near8 & 0x000f000fu, front[3] = far8 & 0x000f000fu;
                            back[0] = near & 0x00f000f0u, back[1] = far & 0x00f000f0u;
                            back[2] = near8 & 0x00f000f0u, back[3] = far8 & 0x00f000f0u;
                        } else {
                            front[0] = (near & 0x000f000fu) | 0x43004300u, front[1] = (far & 0x000f000fu) | 0x43004300u;
                            front[2] = (near >> 8 & 0x000f000fu) | 0x43004300u;
                            front[3] = (far >> 8 & 0x000f000fu) | 0x43004300u;
                            back[0] = (near >> 4 & 0x000f000fu) | 0x43004300u;
                            back[1] = (far >> 4 & 0x000f000fu) | 0x43004300u;
                            back[2] = (near >> 12 & 0x000f000fu) | 0x43004300u;
                            back[3] = (far >> 12 & 0x000f000fu) | 0x43004300u;
                        }
#pragma unroll
                        for (int n = 0; n < NT; ++n) {
                            mma<T>(even[n], front, value[n][q].x, value[n][q].z);
                            mma<T>(half ? odd[n] : even[n], back, value[n][q].y, value[n][q].w);
                        }
                    }
                    const float2 near_pair = __half22float2(reinterpret_cast<const __half2&>(pair[s][t][g].x));
                    const float2 far_pair = __half22float2(reinterpret_cast<const __half2&>(pair[s][t][g].y));
                    const float near_scale = half ? near_pair.x * 0x1p24f : near_pair.x;
                    const float far_scale = half ? far_pair.x * 0x1p24f : far_pair.x;
                    const float near_low = half ? near_pair.y : fmaf(-128.0f, near_pair.x, near_pair.y);
                    const float far_low = half ? far_pair.y : fmaf(-128.0f, far_pair.x, far_pair.y);
#pragma unroll
                    for (int n = 0; n < NT; ++n) {
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const float dot = half ? fmaf(odd[n][i], 0.0625f, even[n][i]) : even[n][i];
                            const float with_low = fmaf(i < 2 ? near_low : far_low, x_sum[n][i], y[t][n][i]);
                            y[t][n][i] = fmaf(i < 2 ? near_scale : far_scale, dot, with_low);
                        }
                    }
                }
            }
            load_weights(base + s + depth, s);
#pragma unroll
            for (int n = 0; n < NT; ++n) {
#pragma unroll
                for (int q = 0; q < 4; ++q) value[n][q] = value_next[n][q];
            }
        }
    }

#pragma unroll
    for (int t = 0; t < R; ++t) {
#pragma unroll
        for (int n = 0; n < NT; ++n) {
#pragma unroll
            for (int i = 0; i < 4; ++i) sums[warp][t][r + (i & 2) * 4][8 * n + 2 * j + (i & 1)] = y[t][n][i];
        }
    }
    __syncthreads();
    constexpr int outs = R * 16 * 8 * NT;
    for (int e = threadIdx.x; e < outs; e += 32 * warps) {
        float* const at = &sums[0][0][0][0] + e;
        float total = 0.0f;
#pragma unroll
        for (int w = 0; w < warps; ++w) total += at[w * outs];
        *at = total;  // this thread alone reads and writes element e of every warp
    }
    if (parts > 1) {
        cluster.sync();
    } else {
        __syncthreads();
    }
    if (part == 0) {
        for (int e = threadIdx.x; e < outs; e += 32 * warps) {
            const int output = e % (16 * R), row = e / (16 * R);  // neighbouring threads store neighbouring outputs
            float* const at = &sums[0][output / 16][output % 16][row];
            float total = *at;
            for (int p = 1; p < parts; ++p) total += *cluster.map_shared_rank(at, p);
            const int n = first_tile * 16 + output;
            if (n < a.outputs && first_row + row < a.rows) {
                if (a.bias != nullptr) total += widen(static_cast<const T*>(a.bias)[n]);
                static_cast<T*>(a.y)[(first_row + row) * a.outputs + n] = narrow<T>(total);
            }
        }
    }
    if (parts > 1) cluster.sync();  // the other blocks' sums stay until they are read
}

template <typename T, int G, int NT, int R>
cudaError_t launch(const MultiplyArgs& a, const Shape& shape, cudaStream_t stream) {
    const int blocks = (shape.tiles + R - 1) / R;
    const unsigned row_blocks = static_cast<unsigned>((a.rows + 8 * NT - 1) / (8 * NT));
    // Blocks of a cluster share the inputs while the SMs are not all taken and every warp keeps two steps.
    int parts = 1;
    while (parts < 8 && static_cast<std::int64_t>(blocks) * row_blocks * parts * 2 <= sm_count() &&
           shape.steps >= 2 * warps * parts * 2) {
        parts *= 2;
    }
    cudaLaunchConfig_t config{};
    config.gridDim = dim3(static_cast<unsigned>(blocks * parts), row_blocks);
    config.blockDim = dim3(32 * warps);
    config.stream = stream;
    cudaLaunchAttribute attribute[1];
    attribute[0].id = cudaLaunchAttributeClusterDimension;
    attribute[0].val.clusterDim = {static_cast<unsigned>(parts), 1, 1};
    config.attrs = attribute;
    config.numAttrs = 1;
    return cudaLaunchKernelEx(&config, multiply_kernel<T, G, NT, R>, a, shape);
}

template <typename T, int G, int NT>
cudaError_t launch_tiles(const MultiplyArgs& a, const Shape& shape, cudaStream_t stream) {
    // More outputs a block read x fewer times; fewer spread a small matrix over the SMs.
    if (shape.tiles >= 4 * sm_count()) return launch<T, G, NT, 4>(a, shape, stream);
    if (shape.tiles >= 2 * sm_count()) return launch<T, G, NT, 2>(a, shape, stream);
    return launch<T, G, NT, 1>(a, shape, stream);
}

template <typename T, int G>
cudaError_t launch_rows(const MultiplyArgs& a, const Shape& shape, cudaStream_t stream) {
    return a.rows <= 8 ? launch_tiles<T, G, 1>(a, shape, stream) : launch_tiles<T, G, 2>(a, shape, stream);
}

template <typename T>
cudaError_t launch_group(const MultiplyArgs& a, const Shape& shape, cudaStream_t stream) {
    return a.group == 32 ? launch_rows<T, 32>(a, shape, stream)
        : a.group == 64  ? launch_rows<T, 64>(a, shape, stream)
                         : launch_rows<T, 128>(a, shape, stream);
}

// One thread a packed word of codes.
__global__ void pack_codes_kernel(const std::uint8_t* __restrict__ codes, int outputs, int inputs, int steps,
                                  std::int64_t count, unsigned* __restrict__ packed) {
    const std::int64_t i = static_cast<std::int64_t>(blockIdx.x) * blockDim.x + threadIdx.x;
    if (i >= count) return;
    const int word = static_cast<int>(i % 4), lane = static_cast<int>(i / 4 % 32), part = static_cast<int>(i / 128 % 2);
    const std::int64_t block = i / 256;
    const std::int64_t output = block / steps * 16 + lane / 4 + word % 2 * 8;
    const std::int64_t input = block % steps * step_inputs + part * 64 + word / 2 * 32 + lane % 4 * 8;
    unsigned bits = 0;
    if (output < outputs && input < inputs) {  // inputs are a multiple of 32, so all eight are inside
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const unsigned byte = codes[output * (inputs / 2) + (input + e) / 2];
            bits |= (byte >> (e % 2 * 4) & 15u) << (4 * (e / 2 + e % 2 * 4));
        }
    }
    packed[i] = bits;
}

// One thread a pair (scale, minimum).
__global__ void pack_scales_kernel(const std::uint16_t* __restrict__ scales, const std::uint16_t* __restrict__ minimums,
                                   int outputs, int inputs, int group, int steps, std::int64_t count,
                                   unsigned* __restrict__ packed) {
    const std::int64_t i = static_cast<std::int64_t>(blockIdx.x) * blockDim.x + threadIdx.x;
    if (i >= count) return;
    const int groups = step_inputs / group, of_tile = static_cast<int>(i % 16);
    const std::int64_t output = i / 16 / groups / steps * 16 + of_tile / 2 + of_tile % 2 * 8;
    const std::int64_t at = i / 16 / groups % steps * groups + i / 16 % groups;
    const bool inside = output < outputs && at < inputs / group;
    const std::int64_t from = output * (inputs / group) + at;
    packed[i] = inside ? scales[from] | static_cast<unsigned>(minimums[from]) << 16 : 0u;
}

}  // namespace

std::size_t packed_code_bytes(int outputs, int inputs) {
    return static_cast<std::size_t>(tiles_of(outputs)) * steps_of(inputs) * 1024;
}

std::size_t packed_scale_bytes(int outputs, int inputs, int group) {
    return static_cast<std::size_t>(tiles_of(outputs)) * steps_of(inputs) * (step_inputs / group) * 64;
}

cudaError_t pack(const std::uint8_t* codes, const std::uint16_t* scales, const std::uint16_t* minimums, int outputs,
                 int inputs, int group, std::uint8_t* packed_codes, std::uint16_t* packed_scales, cudaStream_t stream) {
    const std::int64_t words = static_cast<std::int64_t>(packed_code_bytes(outputs, inputs) / 4);
    const std::int64_t pairs = static_cast<std::int64_t>(packed_scale_bytes(outputs, inputs, group) / 4);
    if ((words + 255) / 256 > 0x7fffffff) return cudaErrorInvalidValue;
    pack_codes_kernel<<<static_cast<unsigned>((words + 255) / 256), 256, 0, stream>>>(
        codes, outputs, inputs, steps_of(inputs), words, reinterpret_cast<unsigned*>(packed_codes));
    pack_scales_kernel<<<static_cast<unsigned>((pairs + 255) / 256), 256, 0, stream>>>(
        scales, minimums, outputs, inputs, group, steps_of(inputs), pairs, reinterpret_cast<unsigned*>(packed_scales));
    return cudaGetLastError();
}

cudaError_t multiply(const MultiplyArgs& args, cudaStream_t stream) {
    if (args.rows == 0) return cudaSuccess;
    const Shape shape{steps_of(args.inputs), tiles_of(args.outputs),
                      reinterpret_cast<std::uintptr_t>(args.x) % 16 == 0 && args.x_stride % 8 == 0};
    return args.type == Type::f16 ? launch_group<__half>(args, shape, stream)
                                  : launch_group<__nv_bfloat16>(args, shape, stream);
}

}  // namespace nvcr_sm100::token
