// Products in 8 bits for a few rows, where the weights' bytes are the work and a launch's latency most of the time: one
// launch, in which every block loads its first weights, takes its rows of x as codes into shared memory and multiplies
// them by dp4a (one row of 4096 -> 4096: 7.0 to 7.3 us, of which 2.6 are the weights at HBM's rate). Sums are exact in
// int32, so their splits and orders change no bit.
//
// The first weights are meant to be on their way while the codes are made, but two blocks an SM leave 64 registers a
// thread, of which the weights are 32 and a piece of x in FP32 another 16: all variants spill 156 to 252 bytes a thread
// then, and a register whose load is under way is stored only once it has come. So how much of the two runs side by side is
// not known.
//
// A warp has eight outputs at a time: rows 16 g + 4 h + {0..3} and those 8 below, whose pieces of a swizzled block lie
// alike, so that a lane's piece of x serves two loads of weights.
#include "token_bytes.cuh"

#include <algorithm>

namespace nvcr_sm100::token {
namespace {

constexpr int threads = 512;
constexpr int warps = threads / 32;
constexpr int unit = 8;       // outputs of a warp
constexpr int most_room = 64 * 1024;  // of codes: two blocks an SM
constexpr int depth = 4;      // blocks of inputs under way

struct FewArgs {
    const void* x;
    std::int64_t stride, inner_stride;
    bool vector;
    int inputs, k_blocks;
    const std::uint8_t* weights;
    const float* scales;
    int outputs, tiles, units;  // units of a matrix
    int splits;                 // warps that share a unit's inputs
    const void* bias;
    void* y;
    int rows;                       // of x: of the call, or (experts) of a token
    const std::int32_t* choices;    // experts: [tokens][chosen]
    const float* choice_weights;
    int chosen, experts;
};

__device__ __forceinline__ int dot(const uint4& w, const uint4& x, int sum) {
    sum = __dp4a(static_cast<int>(w.x), static_cast<int>(x.x), sum);
    sum = __dp4a(static_cast<int>(w.y), static_cast<int>(x.y), sum);
    sum = __dp4a(static_cast<int>(w.z), static_cast<int>(x.z), sum);
    return __dp4a(static_cast<int>(w.w), static_cast<int>(x.w), sum);
}

// Weights are read once: past the caches that other data could use.
__device__ __forceinline__ uint4 stream_load(const std::uint8_t* at) {
    uint4 v;
    asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(at));
    return v;
}

// Rows of x as codes [row][k_blocks * 128] in shared memory, each by warps / Rows warps (Rows a power of two).
template <typename T, int Rows>
__device__ __forceinline__ void quantise(const FewArgs& a, const T* x, std::int64_t stride, int rows, uint4* codes, float* scales,
                                         float* scratch) {
    constexpr int group = threads / Rows;
    const int row = static_cast<int>(threadIdx.x) / group, part = static_cast<int>(threadIdx.x) % group;
    const int pieces = a.k_blocks * (block_bytes / 16);
    const T* from = x + row * stride;
    float kept[16], most = 0.0f;  // a thread's first piece stays in registers, the others are read again
    const bool there = row < rows;
    if (there && part < pieces) {
        load_sixteen(from, part * 16, a.inputs, a.vector, kept);
#pragma unroll
        for (int i = 0; i < 16; ++i) most = max_nan(most, fabsf(kept[i]));
    }
#pragma unroll 1
    for (int piece = part + group; there && piece < pieces; piece += group) {
        float v[16];
        load_sixteen(from, piece * 16, a.inputs, a.vector, v);
#pragma unroll
        for (int i = 0; i < 16; ++i) most = max_nan(most, fabsf(v[i]));
    }
#pragma unroll
    for (int offset = 16; offset > 0; offset /= 2) most = max_nan(most, __shfl_xor_sync(0xffffffffu, most, offset));
    if constexpr (Rows < warps) {
        if (threadIdx.x % 32 == 0) scratch[threadIdx.x / 32] = most;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < warps / Rows; ++w) most = max_nan(most, scratch[row * (warps / Rows) + w]);
    }
    if (!there) return;
    const RowScale scale(most);
    if (part == 0) scales[row] = scale.told();
    if (part < pieces) codes[row * pieces + part] = scale.codes(kept);
#pragma unroll 1
    for (int piece = part + group; piece < pieces; piece += group) {
        float v[16];
        load_sixteen(from, piece * 16, a.inputs, a.vector, v);
        codes[row * pieces + piece] = scale.codes(v);
    }
}

// Where a lane's weights of a unit begin, and which piece of x they are multiplied with.
__device__ __forceinline__ const std::uint8_t* lane_weights(const FewArgs& a, std::int64_t matrix, int u, int lane, int& piece) {
    const int row = u / 2 * 16 + u % 2 * 4 + lane / 8;  // and row + 8
    piece = (lane % 8) ^ (row & 7);
    return a.weights + (matrix * a.tiles + row / block_rows) * a.k_blocks * weight_block + row % block_rows * block_bytes + lane % 8 * 16;
}
__device__ __forceinline__ int output_of(int u, int nth) { return u / 2 * 16 + u % 2 * 4 + nth / 4 * 8 + nth % 4; }

// One matrix, up to Rows rows. A warp has a unit and a part of its inputs: blocks part, part + splits, ...
template <typename T, int Rows>
__global__ void __launch_bounds__(threads, 2) few_kernel(FewArgs a) {
    extern __shared__ uint4 codes[];
    __shared__ float row_scales[Rows], scratch[warps];
    __shared__ int sums[warps][unit][Rows];
    kernels::launch_dependents();
    const int warp = static_cast<int>(threadIdx.x) / 32, lane = static_cast<int>(threadIdx.x) % 32;
    const int here = warps / a.splits;  // units of the block
    const int u = static_cast<int>(blockIdx.x) * here + warp / a.splits;
    const int part = warp % a.splits;
    const bool there = u < a.units;
    int piece = 0;
    const std::uint8_t* from = lane_weights(a, 0, there ? u : 0, lane, piece);
    // The kernel before this one may still be writing: until it has ended the weights only come as far as L2.
    const std::uint8_t* unit_rows = from - lane / 8 * block_bytes - lane % 8 * 16;
    for (int i = lane; there && part + i / 8 * a.splits < a.k_blocks; i += 32) {  // lines of 128 bytes: four rows, and the four 8 below
        const std::uint8_t* line = unit_rows + static_cast<std::int64_t>(part + i / 8 * a.splits) * weight_block +
            (i % 8 < 4 ? i % 8 : 4 + i % 8) * block_bytes;
        asm volatile("prefetch.global.L2 [%0];" ::"l"(line));
    }
    kernels::grid_dependency_wait();
    uint4 w[depth][2];
#pragma unroll
    for (int d = 0; d < depth; ++d) {
        const int k = part + d * a.splits;
        if (there && k < a.k_blocks) {
            w[d][0] = stream_load(from + static_cast<std::int64_t>(k) * weight_block);
            w[d][1] = stream_load(from + static_cast<std::int64_t>(k) * weight_block + 8 * block_bytes);
        } else {
            w[d][0] = w[d][1] = uint4{0, 0, 0, 0};
        }
    }
    quantise<T, Rows>(a, static_cast<const T*>(a.x), a.stride, a.rows, codes, row_scales, scratch);
    __syncthreads();
    const int pieces = a.k_blocks * (block_bytes / 16);
    int sum[2][Rows] = {};
    if (there) {
        for (int k0 = part; k0 < a.k_blocks; k0 += depth * a.splits) {
#pragma unroll
            for (int d = 0; d < depth; ++d) {
                const int k = k0 + d * a.splits, next = k + depth * a.splits;
                const uint4 one = w[d][0], two = w[d][1];
                if (next < a.k_blocks) {
                    w[d][0] = stream_load(from + static_cast<std::int64_t>(next) * weight_block);
                    w[d][1] = stream_load(from + static_cast<std::int64_t>(next) * weight_block + 8 * block_bytes);
                }
                if (k < a.k_blocks) {
#pragma unroll
                    for (int r = 0; r < Rows; ++r) {  // rows past the call's are summed and not stored
                        const uint4 x = codes[r * pieces + k * (block_bytes / 16) + piece];
                        sum[0][r] = dot(one, x, sum[0][r]), sum[1][r] = dot(two, x, sum[1][r]);
                    }
                }
            }
        }
    }
#pragma unroll
    for (int r = 0; r < Rows; ++r) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
#pragma unroll
            for (int o = 4; o > 0; o /= 2) sum[h][r] += __shfl_xor_sync(0xffffffffu, sum[h][r], o);
            if (lane % 8 == 0) sums[warp][h * 4 + lane / 8][r] = sum[h][r];
        }
    }
    __syncthreads();
    for (int i = static_cast<int>(threadIdx.x); i < here * unit * a.rows; i += threads) {
        const int r = i / (here * unit), nth = i % unit, local = i / unit % here;
        const int output = output_of(static_cast<int>(blockIdx.x) * here + local, nth);
        if (output >= a.outputs) continue;
        int total = 0;
        for (int s = 0; s < a.splits; ++s) total += sums[local * a.splits + s][nth][r];
        float v = __fmul_rn(__fmul_rn(__int2float_rn(total), a.scales[output]), row_scales[r]);
        if (a.bias != nullptr) v = __fadd_rn(v, widen(static_cast<const T*>(a.bias)[output]));
        static_cast<T*>(a.y)[static_cast<std::int64_t>(r) * a.outputs + output] = narrow<T>(v);
    }
}

constexpr int most_chosen = 16;

// A token's products with the matrices of its experts: a block has one unit at least, and each of its warps a choice and a
// part of the inputs.
template <typename T, int Rows>
__global__ void __launch_bounds__(threads, 2) few_experts_kernel(FewArgs a) {
    extern __shared__ uint4 codes[];
    __shared__ float row_scales[Rows], scratch[warps];
    __shared__ int sums[warps][unit];
    kernels::launch_dependents();
    kernels::grid_dependency_wait();
    const int warp = static_cast<int>(threadIdx.x) / 32, lane = static_cast<int>(threadIdx.x) % 32;
    const std::int64_t token = blockIdx.y;
    const int each = a.chosen * a.splits;  // warps of a unit
    const int here = warps / each;
    const int local = warp / each, nth_choice = warp % each / a.splits, part = warp % a.splits;
    const int u = static_cast<int>(blockIdx.x) * here + local;
    const std::int32_t* choices = a.choices + token * a.chosen;
    const int expert = local < here ? choices[nth_choice] : -1;
    const bool there = u < a.units && expert >= 0 && expert < a.experts;
    int piece = 0;
    const std::uint8_t* from = lane_weights(a, there ? expert : 0, there ? u : 0, lane, piece);
    uint4 w[depth][2];
#pragma unroll
    for (int d = 0; d < depth; ++d) {
        const int k = part + d * a.splits;
        if (there && k < a.k_blocks) {
            w[d][0] = stream_load(from + static_cast<std::int64_t>(k) * weight_block);
            w[d][1] = stream_load(from + static_cast<std::int64_t>(k) * weight_block + 8 * block_bytes);
        } else {
            w[d][0] = w[d][1] = uint4{0, 0, 0, 0};
        }
    }
    quantise<T, Rows>(a, static_cast<const T*>(a.x) + token * a.stride, a.inner_stride, a.rows, codes, row_scales, scratch);
    __syncthreads();
    const int pieces = a.k_blocks * (block_bytes / 16);
    const int row = a.rows == 1 ? 0 : nth_choice;
    int sum[2] = {};
    if (there) {
        for (int k0 = part; k0 < a.k_blocks; k0 += depth * a.splits) {
#pragma unroll
            for (int d = 0; d < depth; ++d) {
                const int k = k0 + d * a.splits, next = k + depth * a.splits;
                const uint4 one = w[d][0], two = w[d][1];
                if (next < a.k_blocks) {
                    w[d][0] = stream_load(from + static_cast<std::int64_t>(next) * weight_block);
                    w[d][1] = stream_load(from + static_cast<std::int64_t>(next) * weight_block + 8 * block_bytes);
                }
                if (k < a.k_blocks) {
                    const uint4 x = codes[row * pieces + k * (block_bytes / 16) + piece];
                    sum[0] = dot(one, x, sum[0]), sum[1] = dot(two, x, sum[1]);
                }
            }
        }
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
#pragma unroll
        for (int o = 4; o > 0; o /= 2) sum[h] += __shfl_xor_sync(0xffffffffu, sum[h], o);
        if (lane % 8 == 0) sums[warp][h * 4 + lane / 8] = sum[h];
    }
    __syncthreads();
    auto product = [&](int of_unit, int j, int nth, int output) {
        const int e = choices[j];
        int total = 0;
        for (int s = 0; s < a.splits; ++s) total += sums[of_unit * each + j * a.splits + s][nth];
        return __fmul_rn(__fmul_rn(__int2float_rn(total), a.scales[static_cast<std::int64_t>(e) * a.outputs + output]),
                         row_scales[a.rows == 1 ? 0 : j]);
    };
    const bool summed = a.choice_weights != nullptr;
    for (int i = static_cast<int>(threadIdx.x); i < here * unit * (summed ? 1 : a.chosen); i += threads) {
        const int nth = i % unit, of_unit = i / unit % here, j = i / unit / here;
        const int output = output_of(static_cast<int>(blockIdx.x) * here + of_unit, nth);
        if (output >= a.outputs) continue;
        if (summed) {
            float v = 0.0f;
            for (int n = 0; n < a.chosen; ++n) {
                if (choices[n] >= 0 && choices[n] < a.experts) {
                    v = fmaf(a.choice_weights[token * a.chosen + n], product(of_unit, n, nth, output), v);
                }
            }
            static_cast<T*>(a.y)[token * a.outputs + output] = narrow<T>(v);
        } else {
            const bool some = choices[j] >= 0 && choices[j] < a.experts;
            static_cast<T*>(a.y)[(token * a.chosen + j) * a.outputs + output] = narrow<T>(some ? product(of_unit, j, nth, output) : 0.0f);
        }
    }
}

template <typename T, int Rows, bool Experts>
cudaError_t launch(const FewArgs& a, dim3 grid, cudaStream_t stream) {
    static SharedAllowance allowance;
    void (*kernel)(FewArgs);
    if constexpr (Experts) {
        kernel = few_experts_kernel<T, Rows>;
    } else {
        kernel = few_kernel<T, Rows>;
    }
    const cudaError_t status = allowance.allow(kernel, most_room);
    if (status != cudaSuccess) return status;
    return kernels::launch_overlapped(kernel, grid, dim3(threads), static_cast<std::size_t>(Rows) * a.k_blocks * block_bytes, stream, a);
}

template <typename T, bool Experts>
cudaError_t by_rows(const FewArgs& a, dim3 grid, cudaStream_t stream) {
    if (a.rows == 1) return launch<T, 1, Experts>(a, grid, stream);
    if (a.rows == 2) return launch<T, 2, Experts>(a, grid, stream);
    if (a.rows <= 4) return launch<T, 4, Experts>(a, grid, stream);
    if (a.rows <= 8) return launch<T, 8, Experts>(a, grid, stream);
    if constexpr (Experts) return launch<T, 16, Experts>(a, grid, stream);
    return cudaErrorInvalidValue;
}

template <bool Experts>
cudaError_t by_type(Type type, const FewArgs& a, dim3 grid, cudaStream_t stream) {
    switch (type) {
    case Type::f16: return by_rows<__half, Experts>(a, grid, stream);
    case Type::bf16: return by_rows<__nv_bfloat16, Experts>(a, grid, stream);
    default: return by_rows<float, Experts>(a, grid, stream);
    }
}

int power_of_two(int n) {
    int p = 1;
    while (p < n) p *= 2;
    return p;
}

}  // namespace

// One or two rows always. Every block takes all rows as codes for itself and multiplies without the tensor cores, so with
// more rows only where there is little to multiply: 3 rows of 4096 -> 4096 (50 M products) 8.7 us here and 9.1 by the tensor
// cores, 4 rows 9.4 and 9.1, 8 rows of 1024 -> 1024 5.5 and 8.0, of 4096 -> 16384 26.6 and 17.9. By experts, whose other
// way takes three launches: 4 tokens by 8 of 128, 2048 -> 1024 (67 M), 13 us and 23; 32 tokens by 2 of 8 (134 M) 20 and 15.
bool few_rows(const BytesArgs& a) {
    const std::int64_t rows = a.choices == nullptr ? a.tokens : a.inner, pairs = a.choices == nullptr ? a.tokens : a.tokens * a.chosen;
    if (rows > 16 || power_of_two(static_cast<int>(rows)) * blocks_of(a.inputs) > most_room / block_bytes) return false;
    const std::int64_t products = static_cast<std::int64_t>(a.inputs) * a.outputs;
    if (a.choices == nullptr) return rows <= 2 || (rows <= 8 && rows * products <= 3 << 24);
    return a.chosen <= most_chosen && pairs <= 64 && pairs * products <= 1 << 26;
}

cudaError_t multiply_few(const BytesArgs& a, cudaStream_t stream) {
    const int elements = a.type == Type::f32 ? 4 : 2;
    FewArgs f{};
    f.x = a.x, f.stride = a.x_stride, f.inner_stride = a.x_inner_stride;
    f.vector = reinterpret_cast<std::uintptr_t>(a.x) % 16 == 0 && a.x_stride * elements % 16 == 0 && a.x_inner_stride * elements % 16 == 0;
    f.inputs = a.inputs, f.k_blocks = blocks_of(a.inputs);
    f.weights = static_cast<const std::uint8_t*>(a.packed), f.scales = a.scales;
    f.outputs = a.outputs, f.tiles = tiles_of(a.outputs), f.units = (a.outputs + 15) / 16 * 2;
    f.bias = a.bias, f.y = a.y;
    f.rows = a.choices == nullptr ? static_cast<int>(a.tokens) : a.inner;
    f.choices = a.choices, f.choice_weights = a.weights, f.chosen = a.chosen, f.experts = a.experts;
    // warps that share a unit's inputs: while all blocks run at once, and a warp has two blocks of inputs at least
    const std::int64_t pairs = a.choices == nullptr ? 1 : a.tokens * a.chosen;
    const int most = a.choices == nullptr ? warps : warps / a.chosen;
    f.splits = 1;
    while (f.splits * 2 <= most && f.splits * 4 <= f.k_blocks && f.units * pairs * f.splits * 2 <= 2ll * warps * sm_count()) f.splits *= 2;
    const int here = warps / (f.splits * (a.choices == nullptr ? 1 : a.chosen));
    const dim3 grid(static_cast<unsigned>((f.units + here - 1) / here), static_cast<unsigned>(a.choices == nullptr ? 1 : a.tokens));
    return a.choices == nullptr ? by_type<false>(a.type, f, grid, stream) : by_type<true>(a.type, f, grid, stream);
}

}  // namespace nvcr_sm100::token
