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
// registers, a few steps of 128 inputs ahead. x goes to shared memory once, as
// fragments, with its groups' sums. A block of 16 warps, one an SM, takes up to 16
// consecutive tiles of 16 outputs; their steps in a row are divided evenly among
// the warps, so a warp streams without a barrier to its end, whatever the sizes,
// and leaves a sum in shared memory wherever its part of a tile ends. Where tiles
// are fewer than SMs, or x is larger than shared memory, up to eight blocks of a
// cluster divide the inputs and are summed over distributed shared memory. All
// sums are in a fixed order: no atomics, no workspace, one launch.
//
// Measured on a B200, weights from HBM: one FP16 row, 4096 -> 4096 (8.9 MB): 6.2 us,
// 1.4 TB/s, bound by latency (5.0 us with the arithmetic left out; 5.4 with weights
// that are in L2); 16 BF16 rows, 4096 -> 16384 (38 MB): 20.1 us, 1.9 TB/s, bound by
// the conversion and the sums (13.2 us without arithmetic); 5 rows, 1088 -> 1001 with
// a bias: 3.9 us.
#include "token_elements.cuh"

#include <algorithm>
#include <type_traits>

#include <cooperative_groups.h>

namespace nvcr_sm100::token {
namespace {

namespace cg = cooperative_groups;

constexpr int warps = 16;
constexpr int step_inputs = 128;
constexpr int most_tiles = 16;  // of a block

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
    int steps;       // of 128 inputs
    int tiles;       // of 16 outputs
    int part_steps;  // of each block of a cluster
    bool aligned;    // x can be read 16 bytes at a time
};

// Shared memory: x as fragments [step][quarter of 32 inputs][row][j] of 16 bytes (a lane whose row is past the last
// reads the last: its column of the product is not stored), the groups' sums of x [step][group][8 NT], and the warps'
// sums of (16 outputs, 8 NT rows): warp w's of the block's tile t is number w + t, which grows along the warps' row of
// steps.
template <int G, int NT>
__host__ __device__ constexpr int x_step_bytes(int rows) { return rows * 256 + (step_inputs / G) * 8 * NT * 4; }
template <int NT>
constexpr int sum_floats = 16 * 8 * NT;
template <int NT>
constexpr int sums_bytes = (warps + most_tiles - 1) * sum_floats<NT> * 4;
// x's part of it, which holds the block's own sums when a cluster joins them.
template <int G, int NT>
__host__ __device__ constexpr int x_bytes(int steps, int rows) {
    const int x = steps * x_step_bytes<G, NT>(rows), own = most_tiles * sum_floats<NT> * 4;
    return x > own ? x : own;
}

// One output of one row, value by value in the order of the inputs: an output that is no finite number is taken again
// here, as an infinite x times codes and minimums apart is no number where x times their values is an infinity (and 128
// times a bfloat16 sum may overflow). A row of 4096 inputs with an infinity takes 120 us to 4096 outputs; a NaN ends the
// loop.
template <typename T, int G>
__device__ __noinline__ float product_of_values(const T* x, const unsigned* codes, const unsigned* pairs, int inputs,
                                                int steps, int output) {
    constexpr int groups = step_inputs / G;
    const int row = output % 16, r = row % 8, far = row / 8;
    const std::int64_t first = static_cast<std::int64_t>(output / 16) * steps;
    float sum = 0.0f;
    for (int octet = 0; octet < inputs / 8 && sum == sum; ++octet) {
        const std::int64_t step = first + octet / 16;
        const int part = octet / 8 % 2, word = octet / 4 % 2 * 2 + far;
        const unsigned code = codes[step * 256 + part * 128 + (r * 4 + octet % 4) * 4 + word];
        const unsigned pair = pairs[(step * groups + octet % 16 * 8 / G) * 16 + r * 2 + far];
        const float scale = half_bits(static_cast<std::uint16_t>(pair));
        const float minimum = half_bits(static_cast<std::uint16_t>(pair >> 16));
        for (int i = 0; i < 8; ++i) {
            const float c = static_cast<float>(code >> (4 * (i / 2 + i % 2 * 4)) & 15u);
            sum = fmaf(widen(x[octet * 8 + i]), fmaf(c, scale, minimum), sum);
        }
    }
    return sum;
}

template <typename T, int G, int NT>
__global__ void __launch_bounds__(32 * warps) multiply_kernel(const MultiplyArgs a, const Shape shape) {
    constexpr bool half = std::is_same_v<T, __half>;
    constexpr int groups = step_inputs / G, quarters = G / 32;
    // steps of weights in flight, as the registers allow
    constexpr int depth = (G == 128 ? 5 : G == 64 ? 4 : 3) + (NT == 1 ? 1 : 0);
    constexpr unsigned one = half ? 0x3c003c00u : 0x3f803f80u;
    extern __shared__ __align__(128) std::uint8_t shared[];
    join_chain();
    const int lane = threadIdx.x % 32, warp = threadIdx.x / 32, r = lane / 4, j = lane % 4;
    const cg::cluster_group cluster = cg::this_cluster();
    const int parts = static_cast<int>(cluster.num_blocks()), part = static_cast<int>(cluster.block_rank());
    const int blocks = static_cast<int>(gridDim.x) / parts, block = static_cast<int>(blockIdx.x) / parts;
    const int first_tile = static_cast<int>(static_cast<std::int64_t>(shape.tiles) * block / blocks);
    const int tiles = static_cast<int>(static_cast<std::int64_t>(shape.tiles) * (block + 1) / blocks) - first_tile;
    const int first_step = part * shape.part_steps;
    const int steps = max(0, min(shape.part_steps, shape.steps - first_step));
    const std::int64_t first_row = static_cast<std::int64_t>(blockIdx.y) * (8 * NT);
    const int rows = static_cast<int>(min(static_cast<std::int64_t>(8 * NT), a.rows - first_row));
    uint4* const x_parts = reinterpret_cast<uint4*>(shared);
    float* const x_sums = reinterpret_cast<float*>(shared + shape.part_steps * (rows * 256));
    float* const sums = reinterpret_cast<float*>(shared + x_bytes<G, NT>(shape.part_steps, rows));

    // ---- this warp's part of the steps of the block's tiles in a row, and its first weights ----
    const int total = tiles * steps;
    const int begin = total * warp / warps, end = total * (warp + 1) / warps;
    uint4 code[depth][2];
    uint2 pair[depth][groups];
    const int begin_tile = steps > 0 ? begin / steps : 0;
    const std::int64_t begin_at =
        static_cast<std::int64_t>(first_tile + begin_tile) * shape.steps + first_step + (begin - begin_tile * steps);
    const uint4* codes = reinterpret_cast<const uint4*>(a.codes) + begin_at * 64 + lane;
    const uint2* scales = reinterpret_cast<const uint2*>(a.scales) + begin_at * (8 * groups) + r;
    int to_load = end - begin, to_tile_end = steps - (begin - begin_tile * steps);
    auto load_weights = [&](int slot) {
        if (to_load <= 0) return;
        code[slot][0] = __ldcs(codes);
        code[slot][1] = __ldcs(codes + 32);
#pragma unroll
        for (int g = 0; g < groups; ++g) pair[slot][g] = __ldcs(scales + 8 * g);
        codes += 64, scales += 8 * groups, --to_load;
        if (--to_tile_end == 0) {  // over the other blocks' steps
            to_tile_end = steps;
            codes += (shape.steps - steps) * 64, scales += (shape.steps - steps) * (8 * groups);
        }
    };
#pragma unroll
    for (int s = 0; s < depth; ++s) load_weights(s);

    // ---- x to shared memory, and its groups' sums as products with ones ----
    // the fragments in a row, an octet of inputs a thread; 32 * warps / 4 (quarter, row) pairs on at a time
    int x_row = static_cast<int>(threadIdx.x) / 4 % rows, x_quarter = static_cast<int>(threadIdx.x) / 4 / rows;
    const int more_rows = 32 * warps / 4 % rows, more_quarters = 32 * warps / 4 / rows;
    for (int e = threadIdx.x; e < steps * 16 * rows; e += 32 * warps) {
        const int k = first_step * step_inputs + 32 * x_quarter + 8 * j;
        const bool inside = k < a.inputs;  // zeros past the inputs, which are a multiple of 32
        const T* const from = static_cast<const T*>(a.x) + (first_row + x_row) * a.x_stride + (inside ? k : 0);
        if (shape.aligned) {
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(
                             static_cast<unsigned>(__cvta_generic_to_shared(x_parts + e))),
                         "l"(from), "r"(inside ? 16 : 0)
                         : "memory");
        } else {
            alignas(16) T values[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) values[i] = inside ? from[i] : narrow<T>(0.0f);
            x_parts[e] = *reinterpret_cast<const uint4*>(values);
        }
        x_row += more_rows, x_quarter += more_quarters;
        if (x_row >= rows) x_row -= rows, ++x_quarter;
    }
    int x_lane[NT];  // of this lane's row in a quarter
#pragma unroll
    for (int n = 0; n < NT; ++n) x_lane[n] = min(8 * n + r, rows - 1) * 4 + j;
    asm volatile("cp.async.wait_all;" ::: "memory");
    __syncthreads();
    for (int e = warp; e < steps * groups; e += warps) {
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
            const unsigned ones[4] = {one, one, one, one};
#pragma unroll
            for (int q = 0; q < quarters; ++q) {
                const uint4 v = x_parts[(e * quarters + q) * (rows * 4) + x_lane[n]];
                mma<T>(sum, ones, v.x, v.z);
                mma<T>(sum, ones, v.y, v.w);
            }
            if (r == 0) *reinterpret_cast<float2*>(x_sums + e * (8 * NT) + 8 * n + 2 * j) = {sum[0], sum[1]};
        }
    }
    __syncthreads();

    // ---- the stream of weights ----
    float y[NT][4];
#pragma unroll
    for (int n = 0; n < NT; ++n) y[n][0] = y[n][1] = y[n][2] = y[n][3] = 0.0f;
    int tile = begin_tile, step = begin - tile * steps;
    for (int base = begin; base < end; base += depth) {
#pragma unroll
        for (int s = 0; s < depth; ++s) {
            if (base + s >= end) break;
            const uint4* const x_step = x_parts + step * (rows * 16);
            const float* const x_sum_step = x_sums + step * (groups * 8 * NT) + 2 * j;
#pragma unroll
            for (int g = 0; g < groups; ++g) {
                float even[NT][4], odd[NT][4];  // for bfloat16 all of them in `even`
#pragma unroll
                for (int n = 0; n < NT; ++n) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) even[n][i] = odd[n][i] = 0.0f;
                }
#pragma unroll
                for (int q = g * quarters; q < (g + 1) * quarters; ++q) {
                    const uint4 raw = code[s][q / 2];
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
                        const uint4 v = x_step[q * (rows * 4) + x_lane[n]];
                        mma<T>(even[n], front, v.x, v.z);
                        mma<T>(half ? odd[n] : even[n], back, v.y, v.w);
                    }
                }
                const float2 near_pair = __half22float2(reinterpret_cast<const __half2&>(pair[s][g].x));
                const float2 far_pair = __half22float2(reinterpret_cast<const __half2&>(pair[s][g].y));
                const float near_scale = half ? near_pair.x * 0x1p24f : near_pair.x;
                const float far_scale = half ? far_pair.x * 0x1p24f : far_pair.x;
                const float near_low = half ? near_pair.y : fmaf(-128.0f, near_pair.x, near_pair.y);
                const float far_low = half ? far_pair.y : fmaf(-128.0f, far_pair.x, far_pair.y);
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    const float2 x_sum = *reinterpret_cast<const float2*>(x_sum_step + g * (8 * NT) + 8 * n);
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const float dot = half ? fmaf(odd[n][i], 0.0625f, even[n][i]) : even[n][i];
                        const float with_low = fmaf(i < 2 ? near_low : far_low, i % 2 == 0 ? x_sum.x : x_sum.y, y[n][i]);
                        y[n][i] = fmaf(i < 2 ? near_scale : far_scale, dot, with_low);
                    }
                }
            }
            load_weights(s);
            ++step;
            if (step == steps || base + s + 1 == end) {  // the tile's end, or this warp's
                float* const to = sums + (warp + tile) * sum_floats<NT> + r;
#pragma unroll
                for (int n = 0; n < NT; ++n) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) {  // [row][output]
                        to[(8 * n + 2 * j + (i & 1)) * 16 + (i & 2) * 4] = y[n][i];
                        y[n][i] = 0.0f;
                    }
                }
                step = 0, ++tile;
            }
        }
    }
    __syncthreads();

    // ---- join the warps, then the blocks of the cluster ----
    auto warp_of = [&](int at) { return ((at + 1) * warps - 1) / total; };  // whose part holds step `at` of the row
    const int outs = tiles * sum_floats<NT>;
    auto joined = [&](int e) {
        const int t = e / sum_floats<NT>, within = e % sum_floats<NT>;
        float value = 0.0f;
        if (total > 0) {
            const int last = warp_of((t + 1) * steps - 1);
            for (int w = warp_of(t * steps); w <= last; ++w) {
                if (total * w / warps == total * (w + 1) / warps) continue;  // fewer steps than warps: this one had none
                value += sums[(w + t) * sum_floats<NT> + within];
            }
        }
        return value;
    };
    auto store = [&](int e, float value) {
        const int output = (first_tile + e / sum_floats<NT>) * 16 + e % 16;
        const std::int64_t row = first_row + e % sum_floats<NT> / 16;
        if (output >= a.outputs || row >= a.rows) return;
        if (!(fabsf(value) < INFINITY)) {
            value = product_of_values<T, G>(static_cast<const T*>(a.x) + row * a.x_stride,
                                            reinterpret_cast<const unsigned*>(a.codes),
                                            reinterpret_cast<const unsigned*>(a.scales), a.inputs, shape.steps, output);
        }
        if (a.bias != nullptr) value += widen(static_cast<const T*>(a.bias)[output]);
        static_cast<T*>(a.y)[row * a.outputs + output] = narrow<T>(value);
    };
    if (parts == 1) {
        for (int e = threadIdx.x; e < outs; e += 32 * warps) store(e, joined(e));
        return;
    }
    float* const whole = reinterpret_cast<float*>(shared);  // over x, which is not read any more
    for (int e = threadIdx.x; e < outs; e += 32 * warps) whole[e] = joined(e);
    cluster.sync();
    for (int e = part * 32 * warps + threadIdx.x; e < outs; e += parts * 32 * warps) {
        float value = 0.0f;
        for (int p = 0; p < parts; ++p) value += *cluster.map_shared_rank(whole + e, p);
        store(e, value);
    }
    cluster.sync();  // the other blocks' sums stay until they are read
}

// Clusters of `parts` blocks, one block an SM, that run at once (asked once: clusters keep to groups of SMs whose
// sizes are not multiples of theirs).
template <typename T, int G, int NT>
int clusters_at_once(int parts) {
    if (parts == 1) return sm_count();
    static std::atomic<int> known[4];  // 1, 2, 4, 8 parts
    std::atomic<int>& found = known[parts == 2 ? 1 : parts == 4 ? 2 : 3];
    int clusters = found.load(std::memory_order_relaxed);
    if (clusters > 0) return clusters;
    cudaLaunchConfig_t config{};
    config.gridDim = dim3(static_cast<unsigned>(parts * sm_count()));
    config.blockDim = dim3(32 * warps);
    config.dynamicSmemBytes = 120 * 1024;  // one block an SM
    cudaLaunchAttribute attribute[1];
    attribute[0].id = cudaLaunchAttributeClusterDimension;
    attribute[0].val.clusterDim = {static_cast<unsigned>(parts), 1, 1};
    config.attrs = attribute;
    config.numAttrs = 1;
    if (cudaOccupancyMaxActiveClusters(&clusters, multiply_kernel<T, G, NT>, &config) != cudaSuccess || clusters <= 0) {
        cudaGetLastError();
        clusters = std::max(1, sm_count() / parts);
    }
    found.store(clusters, std::memory_order_relaxed);
    return clusters;
}

template <typename T, int G, int NT>
cudaError_t launch(const MultiplyArgs& a, Shape shape, cudaStream_t stream) {
    constexpr int room = 226 * 1024 - sums_bytes<NT>;
    static SharedAllowance allowance;
    const cudaError_t allowed = allowance.allow(multiply_kernel<T, G, NT>, room + sums_bytes<NT>);
    if (allowed != cudaSuccess) return allowed;
    const std::int64_t row_blocks = (a.rows + 8 * NT - 1) / (8 * NT);
    // Blocks of a cluster divide the inputs where x would not fit, and while the SMs are not all taken and every warp
    // still has a step. us divided and whole, one row of FP16: 16384 -> 1024 6.9, 9.2; 8192 -> 1024 5.5, 6.2; 4096 ->
    // 1024 4.6, 4.5 (16 rows 6.3, 7.2).
    const int step_bytes = x_step_bytes<G, NT>(static_cast<int>(std::min<std::int64_t>(a.rows, 8 * NT)));
    int parts = 1;
    while (parts < 8 && (shape.steps + parts - 1) / parts * step_bytes > room) parts *= 2;
    if ((shape.steps + parts - 1) / parts * step_bytes > room) {
        if constexpr (NT == 2) return launch<T, G, 1>(a, shape, stream);  // 8 rows at a time
        return cudaErrorInvalidValue;
    }
    while (parts < 8 && shape.tiles * row_blocks * parts * 2 <= sm_count() && shape.steps >= warps * parts * 2) parts *= 2;
    shape.part_steps = (shape.steps + parts - 1) / parts;
    const int x_rows = static_cast<int>(std::min<std::int64_t>(a.rows, 8 * NT));
    const std::size_t bytes = static_cast<std::size_t>(x_bytes<G, NT>(shape.part_steps, x_rows) + sums_bytes<NT>);
    const int at_once = std::max<int>(1, static_cast<int>(clusters_at_once<T, G, NT>(parts) / row_blocks));
    const int rounds = (shape.tiles + most_tiles * at_once - 1) / (most_tiles * at_once);
    const int blocks = std::min(shape.tiles, at_once * rounds);
    cudaLaunchConfig_t config{};
    config.gridDim = dim3(static_cast<unsigned>(blocks * parts), static_cast<unsigned>(row_blocks));
    config.blockDim = dim3(32 * warps);
    config.dynamicSmemBytes = bytes;
    config.stream = stream;
    cudaLaunchAttribute attributes[2];
    attributes[0].id = cudaLaunchAttributeClusterDimension;
    attributes[0].val.clusterDim = {static_cast<unsigned>(parts), 1, 1};
    attributes[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attributes[1].val.programmaticStreamSerializationAllowed = 1;
    config.attrs = attributes;
    config.numAttrs = 2;
    return cudaLaunchKernelEx(&config, multiply_kernel<T, G, NT>, a, static_cast<const Shape&>(shape));
}

template <typename T, int G>
cudaError_t launch_rows(const MultiplyArgs& a, const Shape& shape, cudaStream_t stream) {
    // Blocks of 16 rows read the weights once for twice the rows; of 8 rows, they are twice as many and have half the x
    // to lay out. us with 16 and with 8, 16 rows of FP16: 1088 -> 1001 4.6, 3.9; 2048 -> 2048 5.6, 4.9; 4096 -> 4096
    // 9.2, 8.7; 4096 -> 16384 18.5, 20.0. Of BF16: 2048 -> 2048 5.5, 5.1; 4096 -> 4096 9.4, 9.7; 4096 -> 16384 18.6,
    // 22.5. 32 rows, 2048 -> 2048: 6.3, 5.9 (BF16 6.3, 6.2); 4096 -> 4096 BF16: 12.1, 13.3.
    const bool small = a.rows <= 32 && static_cast<std::int64_t>(a.inputs) * a.outputs <= 1 << 22;
    return a.rows <= 8 || small ? launch<T, G, 1>(a, shape, stream) : launch<T, G, 2>(a, shape, stream);
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
    const Shape shape{steps_of(args.inputs), tiles_of(args.outputs), 0,
                      reinterpret_cast<std::uintptr_t>(args.x) % 16 == 0 && args.x_stride % 8 == 0};
    return args.type == Type::f16 ? launch_group<__half>(args, shape, stream)
                                  : launch_group<__nv_bfloat16>(args, shape, stream);
}

}  // namespace nvcr_sm100::token
