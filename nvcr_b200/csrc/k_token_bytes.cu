// Products in 8-bit integers: y[t][n] = (sum_k q[t][k] w[n][k]) * scale[n] * s[t] + bias[n], the rows of x taken as
// codes q = rint(x / s) with a scale s of their own, one matrix for all rows or the matrix of the expert that each
// row has chosen. The sums are exact in int32, so their order, and a split of them, change no bit.
//
// Four launches at most: where the rows of each expert go (`arrange`; up to 1024 pairs the next one finds that itself), the
// rows as codes (`quantise`), the product, and for weighted sums over experts their products' sums (`combine`).
// Both operands lie in memory as the tensor cores read them from shared memory, in the 128-byte swizzle: weights as
// blocks of 128 outputs by 128 inputs, rows as [128 inputs][row][128 bytes]. So every tile is one contiguous copy,
// with neither a tensor map nor an alignment that a caller has to keep.
#include "tcgen05.cuh"
#include "token_bytes.cuh"

#include <algorithm>
#include <cmath>
#include <type_traits>

namespace nvcr_sm100::token {
namespace {

using namespace kernels;

constexpr int step_rows = 16;      // rows of x are padded to the MMA's step of N
constexpr int pair_step_rows = 32; // with two blocks a tile
constexpr int most_tile = 256;     // rows of x a tile

std::int64_t padded(std::int64_t rows) { return (rows + step_rows - 1) / step_rows * step_rows; }
std::size_t aligned(std::size_t bytes) { return (bytes + 255) / 256 * 256; }

// ---- weights: [matrix][tile of outputs][block of inputs][128][128], zeros past the edges, laid out once ----

// Products read one matrix's weights before they wait for the kernel before them, so a kernel that writes weights neither
// starts early nor lets the next one: no programmatic launch here.
__global__ void __launch_bounds__(256) pack_kernel(const std::int8_t* codes, std::int64_t blocks, int outputs, int inputs,
                                                   int tiles, int k_blocks, uint4* packed) {
    // a thread a 16-byte piece: piece c of row r lies at piece c ^ (r % 8)
    for (std::int64_t i = blockIdx.x * 256ll + threadIdx.x; i < blocks * (weight_block / 16);
         i += static_cast<std::int64_t>(gridDim.x) * 256) {
        const std::int64_t block = i / (weight_block / 16);
        const int row = static_cast<int>(i / 8 % block_rows), piece = static_cast<int>(i % 8) ^ (row & 7);
        const int k = static_cast<int>(block % k_blocks) * block_bytes + piece * 16;
        const int output = static_cast<int>(block / k_blocks % tiles) * block_rows + row;
        const std::int64_t matrix = block / k_blocks / tiles;
        unsigned words[4] = {0, 0, 0, 0};
        if (output < outputs) {
            const std::int8_t* from = codes + (matrix * outputs + output) * inputs + k;
            for (int b = 0; b < 16; ++b) {
                if (k + b < inputs) words[b / 4] |= static_cast<unsigned>(static_cast<std::uint8_t>(from[b])) << (b % 4 * 8);
            }
        }
        packed[i] = {words[0], words[1], words[2], words[3]};
    }
}

// ---- clusters ----

__device__ __forceinline__ void cluster_arrive() {
    __syncwarp();
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
}
__device__ __forceinline__ void cluster_wait() {
    __syncwarp();
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}

__device__ __forceinline__ int peer_load(const int* here, int rank) {
    int v;
    asm volatile("{\n\t.reg .b32 there;\n\tmapa.shared::cluster.u32 there, %1, %2;\n\tld.shared::cluster.b32 %0, [there];\n\t}"
                 : "=r"(v)
                 : "r"(smem_address(here)), "r"(rank)
                 : "memory");
    return v;
}

// ---- where the rows of each expert go ----

constexpr int arrange_threads = 1024;

struct Arranged {
    int* place;       // [pairs]: the row of a pair, or -1
    int* pair;        // [rows]: the pair of a row
    int4* tiles;      // expert, first row, rows
    int* tile_count;
    int* given_up;    // whether a block of the product has: some products are missing
};

constexpr int arrange_blocks = 8;

// One cluster, a part of the pairs each block's; a thread an expert. Which of an expert's rows a pair gets is decided by
// atomics, and changes no output: rows are independent and their sums exact. 16384 pairs of 32 experts: 9.7 us, 11
// by one block, which more pairs would keep longer.
__global__ void __cluster_dims__(arrange_blocks, 1, 1) __launch_bounds__(arrange_threads)
    arrange_kernel(const std::int32_t* choices, std::int64_t pairs, int experts, int tile_rows, Arranged out) {
    __shared__ int counts[arrange_threads], next[arrange_threads], scratch[64];
    static_assert(most_experts <= arrange_threads);
    const int thread = threadIdx.x, lane = thread % 32, warp = thread / 32;
    const int rank = static_cast<int>(blockIdx.x);
    counts[thread] = 0;
    join_chain();
    __syncthreads();
    const std::int64_t from = pairs * rank / arrange_blocks, to = pairs * (rank + 1) / arrange_blocks;
#pragma unroll 4
    for (std::int64_t i = from + thread; i < to; i += arrange_threads) {
        const int e = choices[i];
        if (e >= 0 && e < experts) atomicAdd(&counts[e], 1);
    }
    cluster_arrive();
    cluster_wait();
    int count = 0, before = 0;  // of the expert: all, and those of earlier blocks
    int some[arrange_blocks];
#pragma unroll
    for (int b = 0; b < arrange_blocks; ++b) some[b] = peer_load(&counts[thread], b);
#pragma unroll
    for (int b = 0; b < arrange_blocks; ++b) count += some[b], before += b < rank ? some[b] : 0;
    cluster_arrive();  // the others' counts are read
    const int rows = (count + step_rows - 1) / step_rows * step_rows;
    const int tiles = (count + tile_rows - 1) / tile_rows;
    int row = rows, tile = tiles;
    for (int o = 1; o < 32; o *= 2) {
        const int r = __shfl_up_sync(0xffffffffu, row, o), t = __shfl_up_sync(0xffffffffu, tile, o);
        if (lane >= o) row += r, tile += t;
    }
    if (lane == 31) scratch[warp] = row, scratch[32 + warp] = tile;
    __syncthreads();
    int all_tiles = 0;
    for (int w = 0; w < arrange_threads / 32; ++w) {
        if (w < warp) row += scratch[w], tile += scratch[32 + w];
        all_tiles += scratch[32 + w];
    }
    row -= rows, tile -= tiles;
    if (rank == 0) {
        for (int t = 0; t < tiles; ++t) {
            out.tiles[tile + t] = {thread, row + t * tile_rows, min(tile_rows, count - t * tile_rows), 0};
        }
        if (thread == 0) *out.tile_count = all_tiles, *out.given_up = 0;
    }
    next[thread] = row + before;
    __syncthreads();
#pragma unroll 4
    for (std::int64_t i = from + thread; i < to; i += arrange_threads) {
        const int e = choices[i];
        int at = -1;
        if (e >= 0 && e < experts) {
            at = atomicAdd(&next[e], 1);
            out.pair[at] = static_cast<int>(i);
        }
        out.place[i] = at;
    }
    cluster_wait();
}

// ---- rows as codes ----

struct QuantiseArgs {
    const void* x;
    std::int64_t stride, inner_stride;  // of a token, and of a row within a token
    int inner;                          // rows a token
    std::int64_t rows;
    int inputs, k_blocks;
    bool vector;          // rows begin on 16-byte boundaries
    const int* place;     // null: row r goes to row r; else to rows place[r * fan ..]
    int fan;
    std::int64_t out_rows;
    std::uint8_t* codes;  // [k_blocks][out_rows][128], swizzled
    float* scales;        // [out_rows]
    void* zeros;          // null, or the output whose rows without a place are zeros
    int outputs;
    // for blocks that find the places themselves
    const std::int32_t* choices;
    int pairs, experts, tile_rows;
    Arranged arranged;
};

constexpr int most_own_pairs = 1024;

// The places of a few pairs, found by every block of `quantise_kernel` for itself, which saves a launch: `places` of the
// block's own pairs first .. first + count - 1. The first block writes the tiles. 256 threads.
__device__ __forceinline__ void find_places(const QuantiseArgs& a, int first, int count, int* choices, int* starts, int* places) {
    __shared__ int scratch[16];
    const int thread = threadIdx.x, lane = thread % 32, warp = thread / 32;
    for (int e = thread; e < a.experts; e += 256) starts[e] = 0;
    for (int i = thread; i < a.pairs; i += 256) {
        const int e = a.choices[i];
        choices[i] = e >= 0 && e < a.experts ? e : -1;
    }
    __syncthreads();
    for (int i = thread; i < a.pairs; i += 256) {
        if (choices[i] >= 0) atomicAdd(&starts[choices[i]], 1);
    }
    __syncthreads();
    // a thread a run of experts: their rows, padded, and tiles before its first
    const int run = (a.experts + 255) / 256, from = min(a.experts, thread * run), to = min(a.experts, from + run);
    int rows = 0, tiles = 0;
    for (int e = from; e < to; ++e) {
        rows += (starts[e] + step_rows - 1) / step_rows * step_rows;
        tiles += (starts[e] + a.tile_rows - 1) / a.tile_rows;
    }
    int row = rows, tile = tiles;
    for (int o = 1; o < 32; o *= 2) {
        const int r = __shfl_up_sync(0xffffffffu, row, o), t = __shfl_up_sync(0xffffffffu, tile, o);
        if (lane >= o) row += r, tile += t;
    }
    if (lane == 31) scratch[warp] = row, scratch[8 + warp] = tile;
    __syncthreads();
    int all_tiles = 0;
    for (int w = 0; w < 8; ++w) {
        if (w < warp) row += scratch[w], tile += scratch[8 + w];
        all_tiles += scratch[8 + w];
    }
    row -= rows, tile -= tiles;
    for (int e = from; e < to; ++e) {
        const int have = starts[e];
        starts[e] = row;
        if (blockIdx.x == 0) {
            for (int t = 0; t * a.tile_rows < have; ++t) {
                a.arranged.tiles[tile++] = {e, row + t * a.tile_rows, min(a.tile_rows, have - t * a.tile_rows), 0};
            }
        }
        row += (have + step_rows - 1) / step_rows * step_rows;
    }
    if (blockIdx.x == 0 && thread == 0) *a.arranged.tile_count = all_tiles, *a.arranged.given_up = 0;
    __syncthreads();
    for (int n = warp; n < count; n += 8) {  // a warp a pair: those with the same expert before it
        const int i = first + n, e = choices[i];
        int before = 0;
        for (int j = 0; j < i; j += 32) before += __popc(__ballot_sync(0xffffffffu, j + lane < i && choices[j + lane] == e));
        if (lane == 0) {
            places[n] = e < 0 ? -1 : starts[e] + before;
            if (e >= 0) a.arranged.pair[starts[e] + before] = i;
        }
    }
    __syncthreads();
}

// Sixteen values of a row as they are in memory.
template <typename T>
struct Sixteen {
    uint4 words[sizeof(T)];
    __device__ __forceinline__ void load(const T* row, int at, int inputs, bool vector) {
        if (vector && at + 16 <= inputs) {
#pragma unroll
            for (int i = 0; i < static_cast<int>(sizeof(T)); ++i) words[i] = reinterpret_cast<const uint4*>(row + at)[i];
        } else {
            unsigned made[4 * sizeof(T)];
#pragma unroll
            for (int i = 0; i < static_cast<int>(4 * sizeof(T)); ++i) {
                if constexpr (sizeof(T) == 4) {
                    made[i] = at + i < inputs ? __float_as_uint(row[at + i]) : 0u;
                } else {
                    const auto* bits = reinterpret_cast<const std::uint16_t*>(row);
                    const unsigned low = at + 2 * i < inputs ? bits[at + 2 * i] : 0u, high = at + 2 * i + 1 < inputs ? bits[at + 2 * i + 1] : 0u;
                    made[i] = low | high << 16;
                }
            }
#pragma unroll
            for (int i = 0; i < static_cast<int>(sizeof(T)); ++i) words[i] = {made[4 * i], made[4 * i + 1], made[4 * i + 2], made[4 * i + 3]};
        }
    }
    __device__ __forceinline__ unsigned word(int i) const {
        const uint4& w = words[i / 4];
        return i % 4 == 0 ? w.x : i % 4 == 1 ? w.y : i % 4 == 2 ? w.z : w.w;
    }
    // The largest magnitude's bits so far, by halves for 16-bit types: magnitudes are ordered as their bits are, infinities
    // and then NaNs above all.
    __device__ __forceinline__ unsigned largest(unsigned so_far) const {
#pragma unroll
        for (int i = 0; i < static_cast<int>(4 * sizeof(T)); ++i) {
            if constexpr (sizeof(T) == 4) {
                so_far = max(so_far, word(i) & 0x7fffffffu);
            } else {
                so_far = __vmaxu2(so_far, word(i) & 0x7fff7fffu);
            }
        }
        return so_far;
    }
    __device__ __forceinline__ void values(float (&v)[16]) const {
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            if constexpr (sizeof(T) == 4) {
                v[i] = __uint_as_float(word(i));
            } else if constexpr (std::is_same_v<T, __nv_bfloat16>) {
                v[i] = __uint_as_float(i % 2 == 0 ? word(i / 2) << 16 : word(i / 2) & 0xffff0000u);
            } else {
                v[i] = half_bits(static_cast<std::uint16_t>(word(i / 2) >> (i % 2 * 16)));
            }
        }
    }
};

// Warps warps a row, a thread 16 values at a time, of which the first Held stay in registers between the row's maximum and
// its codes; longer rows are read again. One warp a row, with the whole of it in registers, where there are rows for all
// warps of an SM: 8192 x 4096 BF16 30 -> 24 us.
template <typename T, int Warps, int Held, bool Arrange>
__global__ void __launch_bounds__(256) quantise_kernel(QuantiseArgs a) {
    extern __shared__ int own[];  // Arrange: places of the block's pairs, then choices and starts
    constexpr int threads = Warps * 32;
    __shared__ unsigned maxima[8];
    join_chain();
    if constexpr (Arrange) {
        const int first = static_cast<int>(blockIdx.x) * (8 / Warps) * a.fan, room = 8 / Warps * a.fan;
        find_places(a, first, min(room, a.pairs - first), own + room, own + room + a.pairs, own);
    }
    const int part = threadIdx.x % threads;
    const std::int64_t row = blockIdx.x * static_cast<std::int64_t>(8 / Warps) + threadIdx.x / threads;
    const bool there = row < a.rows;
    const T* x = static_cast<const T*>(a.x);
    if (there) x += a.inner == 1 ? row * a.stride : row / a.inner * a.stride + row % a.inner * a.inner_stride;
    const int pieces = a.k_blocks * (block_bytes / 16);
    Sixteen<T> kept[Held];
    unsigned largest = 0;
#pragma unroll
    for (int h = 0; h < Held; ++h) {
        if (there && part + h * threads < pieces) kept[h].load(x, (part + h * threads) * 16, a.inputs, a.vector);
    }
#pragma unroll
    for (int h = 0; h < Held; ++h) {
        if (there && part + h * threads < pieces) largest = kept[h].largest(largest);
    }
#pragma unroll 1
    for (int piece = part + Held * threads; there && piece < pieces; piece += threads) {
        Sixteen<T> v;
        v.load(x, piece * 16, a.inputs, a.vector);
        largest = v.largest(largest);
    }
    if constexpr (sizeof(T) == 2) largest = max(largest >> 16, largest & 0xffffu);
    largest = __reduce_max_sync(0xffffffffu, largest);
    if constexpr (Warps > 1) {
        if (threadIdx.x % 32 == 0) maxima[threadIdx.x / 32] = largest;
        __syncthreads();
        const int first = threadIdx.x / threads * Warps;
#pragma unroll
        for (int w = 0; w < Warps; ++w) largest = max(largest, maxima[first + w]);
    }
    if (!there) return;
    float most;
    if constexpr (sizeof(T) == 4) {
        most = __uint_as_float(largest);
    } else {
        const auto bits = static_cast<std::uint16_t>(largest);
        most = widen(reinterpret_cast<const T&>(bits));
    }
    const RowScale scale(most);
    auto place = [&](int f) -> std::int64_t {
        if constexpr (Arrange) return own[static_cast<int>(threadIdx.x) / threads * a.fan + f];
        return a.place == nullptr ? row : a.place[row * a.fan + f];
    };
    auto store = [&](const Sixteen<T>& sixteen, int piece) {
        float v[16];
        sixteen.values(v);
        const uint4 words = scale.codes(v);
        std::uint8_t* block = a.codes + piece / 8 * a.out_rows * block_bytes;
        for (int f = 0; f < a.fan; ++f) {
            const std::int64_t to = place(f);
            if (to >= 0) reinterpret_cast<uint4*>(block + to * block_bytes)[(piece % 8) ^ static_cast<int>(to & 7)] = words;
        }
    };
#pragma unroll
    for (int h = 0; h < Held; ++h) {
        if (part + h * threads < pieces) store(kept[h], part + h * threads);
    }
#pragma unroll 1
    for (int piece = part + Held * threads; piece < pieces; piece += threads) {
        Sixteen<T> v;
        v.load(x, piece * 16, a.inputs, a.vector);
        store(v, piece);
    }
    for (int f = part; f < a.fan; f += threads) {
        const std::int64_t to = place(f);
        if (to >= 0) a.scales[to] = scale.told();
    }
    if (a.zeros != nullptr) {
        for (int f = 0; f < a.fan; ++f) {
            if (place(f) >= 0) continue;
            T* out = static_cast<T*>(a.zeros) + (row * a.fan + f) * a.outputs;
            for (int i = part; i < a.outputs; i += threads) out[i] = narrow<T>(0.0f);
        }
    }
}

// ---- the product ----

constexpr int epilogue_warps = 8;
constexpr int copy_warp = 8, copy_warps = 4, mma_warp = 12;
constexpr int product_threads = 32 * 13;
constexpr int most_stages = 12;

struct ProductArgs {
    const std::uint8_t* weights;
    const float* scales;
    const void* bias;
    const std::uint8_t* codes;
    const float* row_scales;
    Arranged arranged;  // tiles null: rows 0 .. rows - 1 of one matrix
    std::int64_t rows, out_rows;
    int experts, outputs, tiles, k_blocks;
    int tile_rows, stages, splits;
    unsigned tmem_columns;
    void* y;
    unsigned* status;
    unsigned long long wait_ns;  // after which a wait gives up
    int withheld;                // the block that copies nothing, so that waits do (a self-test), or -1
};

struct ProductTail {
    // of the tile's columns: the rows' scales, and the rows of y; by turns, as one tile's stores overlap the next one's loads
    alignas(16) float row_scales[2][most_tile];
    alignas(16) int rows[2][most_tile];
    std::uint64_t full[most_stages], empty[most_stages], tmem_full[2], tmem_empty[2], drain;
    std::uint32_t tmem;
    unsigned status;  // of waits: told to the caller's at the end
    int abort;
    int given_up;     // by a block of the cluster, which tells all: its sums are missing
};

__device__ __forceinline__ void bulk_load(std::uint32_t to, const void* from, std::uint32_t bytes, std::uint32_t barrier) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(to),
                 "l"(__cvta_generic_to_global(from)), "r"(bytes), "r"(barrier)
                 : "memory");
}

__device__ __forceinline__ void peer_store(std::uint32_t address, int rank, int v) {
    asm volatile("{\n\t.reg .b32 there;\n\tmapa.shared::cluster.u32 there, %0, %1;\n\tst.shared::cluster.b32 [there], %2;\n\t}" ::"r"(address),
                 "r"(rank), "r"(v)
                 : "memory");
}

// A barrier of the epilogue's threads: whether any of them says so. bar.red takes whole warps.
__device__ __forceinline__ bool epilogue_any(bool mine) {
    __syncwarp();
    int any;
    asm volatile(
        "{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %1, 0;\n\tbar.red.or.pred q, 1, 256, p;\n\tselp.b32 %0, 1, 0, q;\n\t}"
        : "=r"(any)
        : "r"(static_cast<int>(mine))
        : "memory");
    return any != 0;
}

// What a block whose wait ran out leaves behind: its status, and that sums over experts are not to be made.
template <bool Experts>
__device__ __forceinline__ void give_up(const ProductArgs& a, unsigned status) {
    if (a.status != nullptr) atomicOr(a.status, status);
    if (Experts) atomicExch(a.arranged.given_up, 1);
}

struct Tile {
    int expert, output;          // output: first of the tile
    std::int64_t row;            // first row of the codes
    int rows, columns;           // columns: rows padded to the MMA's step
};

// Tiles of one group of rows after another; with Pair the outputs are those of two blocks.
template <bool Experts, bool Pair = false>
__device__ __forceinline__ Tile tile_at(const ProductArgs& a, int item) {
    const int tiles = Pair ? (a.tiles + 1) / 2 : a.tiles;
    const int nth = item / tiles;
    Tile t;
    t.output = (item - nth * tiles) * (Pair ? 2 * block_rows : block_rows);
    if constexpr (Experts) {
        const int4 found = a.arranged.tiles[nth];
        t.expert = found.x, t.row = found.y, t.rows = found.z;
    } else {
        t.expert = 0, t.row = static_cast<std::int64_t>(nth) * a.tile_rows;
        t.rows = static_cast<int>(min(static_cast<std::int64_t>(a.tile_rows), a.rows - t.row));
    }
    constexpr int step = Pair ? pair_step_rows : step_rows;
    t.columns = (t.rows + step - 1) / step * step;
    return t;
}

// What a tile's stores need of its rows, by a thread a row; the caller synchronises.
template <bool Experts>
__device__ __forceinline__ void stage_rows(const ProductArgs& a, const Tile& t, ProductTail& tail, int buffer) {
    const int column = static_cast<int>(threadIdx.x);
    if (column >= t.rows) return;
    tail.row_scales[buffer][column] = a.row_scales[t.row + column];
    if constexpr (Experts) tail.rows[buffer][column] = a.arranged.pair[t.row + column];
}

// An epilogue warp's part of a tile, scaled and stored: 32 outputs from `first` on, half of the columns.
template <typename T, bool Experts>
__device__ __forceinline__ void store_tile(const ProductArgs& a, const Tile& t, const ProductTail& tail, int buffer, int first,
                                           std::uint32_t sums, int half) {
    const int output = first + static_cast<int>(threadIdx.x) % 32;
    const bool inside = output < a.outputs;
    const std::int64_t channel = static_cast<std::int64_t>(t.expert) * a.outputs + output;
    const float scale = inside ? a.scales[channel] : 0.0f;
    const float bias = inside && a.bias != nullptr ? widen(static_cast<const T*>(a.bias)[channel]) : 0.0f;
    T* y = static_cast<T*>(a.y) + output;
    if constexpr (!Experts) y += t.row * a.outputs;
    __syncwarp();
    int ahead[16];  // the next columns, under way while the ones before are scaled
    if (half * 16 < t.columns) tmem_load16(sums + static_cast<std::uint32_t>(half * 16), ahead);
#pragma unroll 1
    for (int column = half * 16; column < t.columns; column += 32) {
        int acc[16];
        tmem_load_wait();
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            acc[i] = ahead[i];
            asm volatile("" : "+r"(acc[i]));  // not read before the wait
        }
        if (column + 32 < t.columns) tmem_load16(sums + static_cast<std::uint32_t>(column + 32), ahead);
        if (inside) {
            float row_scale[16];
            int row[16];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float4 v = reinterpret_cast<const float4*>(tail.row_scales[buffer])[column / 4 + i];
                row_scale[4 * i] = v.x, row_scale[4 * i + 1] = v.y, row_scale[4 * i + 2] = v.z, row_scale[4 * i + 3] = v.w;
                if constexpr (Experts) {
                    const int4 r = reinterpret_cast<const int4*>(tail.rows[buffer])[column / 4 + i];
                    row[4 * i] = r.x, row[4 * i + 1] = r.y, row[4 * i + 2] = r.z, row[4 * i + 3] = r.w;
                }
            }
            T* to = y + static_cast<std::int64_t>(column) * a.outputs;
            auto value = [&](int i) {
                const float v = __fmul_rn(__fmul_rn(__int2float_rn(acc[i]), scale), row_scale[i]);
                return narrow<T>(a.bias != nullptr ? __fadd_rn(v, bias) : v);
            };
            if (column + 16 <= t.rows) {
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    if constexpr (Experts) {
                        y[static_cast<std::int64_t>(row[i]) * a.outputs] = value(i);
                    } else {
                        *to = value(i);
                        to += a.outputs;
                    }
                }
            } else {
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    if (column + i < t.rows) y[static_cast<std::int64_t>(Experts ? row[i] : column + i) * a.outputs] = value(i);
                }
            }
        }
        __syncwarp();  // the TMEM instructions take whole warps: reconverge before the next columns
    }
    tmem_load_wait();
}

// A block takes tiles of 128 outputs by tile_rows rows one after another: four warps copy blocks of weights and rows into a
// ring, a thread issues the MMAs into one of two accumulators, eight warps scale and store the other. A copy holds up the
// warp that issues it for some 800 cycles, but takes as many lanes' copies as there are: one warp that copied the two
// operands of each block, for which the MMAs of 256 rows take 512 cycles, had set the pace (880 cycles a block). With
// `splits` > 1 a cluster of that many blocks has one tile, each block a part of its inputs; each sends its sums of an
// output to the block that adds up and stores that output.
template <typename T, bool Experts>
__global__ void __launch_bounds__(product_threads, 1) product_kernel(const ProductArgs a) {
    extern __shared__ std::uint8_t dynamic[];
    __shared__ ProductTail tail;
    const std::uint32_t raw = smem_address(dynamic);
    const std::uint32_t ring = (raw + 1023u) & ~1023u;
    const std::uint32_t row_bytes = static_cast<std::uint32_t>(a.tile_rows) * block_bytes;
    const std::uint32_t rows_ring = ring + static_cast<std::uint32_t>(a.stages) * weight_block;
    const std::uint32_t exchange = rows_ring + static_cast<std::uint32_t>(a.stages) * row_bytes;  // [block][column][output]
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    const int splits = a.splits;
    const int rank = static_cast<int>(blockIdx.x) % splits;
    const int first_item = static_cast<int>(blockIdx.x) / splits, item_step = static_cast<int>(gridDim.x) / splits;
    const int k_from = static_cast<int>(static_cast<std::int64_t>(a.k_blocks) * rank / splits);
    const int k_to = static_cast<int>(static_cast<std::int64_t>(a.k_blocks) * (rank + 1) / splits);

    if (warp == copy_warp && lane == 0) {
        for (int s = 0; s < a.stages; ++s) {
            barrier_init(smem_address(&tail.full[s]), 1);
            barrier_init(smem_address(&tail.empty[s]), 1);
        }
        for (int b = 0; b < 2; ++b) {
            barrier_init(smem_address(&tail.tmem_full[b]), 1);
            barrier_init(smem_address(&tail.tmem_empty[b]), epilogue_warps * 32);
        }
        barrier_init(smem_address(&tail.drain), 1);
        tail.status = 0;
        tail.abort = tail.given_up = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        fence_proxy_async_shared();
    }
    if (warp == mma_warp) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_address(&tail.tmem)),
                     "r"(a.tmem_columns)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tmem_fence_before();
    __syncthreads();
    tmem_fence_after();
    const std::uint32_t tmem = tail.tmem;
    if (splits > 1) cluster_arrive();  // the others' memory is there once all have
    volatile int* abort = &tail.abort;
    unsigned* waits = &tail.status;
    launch_dependents();
    if (Experts || warp < copy_warp || warp >= copy_warp + copy_warps) grid_dependency_wait();
    int items = 0;
    if (Experts) {
        items = *a.arranged.tile_count * a.tiles;
    } else {
        items = static_cast<int>((a.rows + a.tile_rows - 1) / a.tile_rows) * a.tiles;
    }

    if (warp >= copy_warp && warp < copy_warp + copy_warps) {
        // The block's copies are numbered q = 0, 1, ..., a block of inputs each, tile after tile; this warp has every
        // fourth one. Those that fill the ring go out a lane each, the later ones a lane an operand. (There are four stages
        // at least: a warp that ran ahead by two uses of a stage would take the parity of its barrier's phase before last for
        // the last one's.)
        const int blocks = k_to - k_from;
        const bool copying = first_item < items && static_cast<int>(blockIdx.x) != a.withheld;
        const std::int64_t mine = copying ? static_cast<std::int64_t>((items - first_item + item_step - 1) / item_step) * blocks : 0;
        auto of = [&](std::int64_t q, std::uint32_t& bytes, const std::uint8_t*& weights, const std::uint8_t*& rows) {
            const std::int64_t nth = q / blocks;
            const int k = k_from + static_cast<int>(q - nth * blocks);
            const Tile t = tile_at<Experts>(a, first_item + static_cast<int>(nth) * item_step);
            bytes = static_cast<std::uint32_t>(t.columns) * block_bytes;
            weights = a.weights + ((static_cast<std::int64_t>(t.expert) * a.tiles + t.output / block_rows) * a.k_blocks + k) * weight_block;
            rows = a.codes + (t.row + k * a.out_rows) * block_bytes;
        };
        const int own = lane * copy_warps + warp - copy_warp;
        const bool filling = own < a.stages && own < mine;
        const std::uint32_t own_full = smem_address(&tail.full[filling ? own : 0]);
        std::uint32_t bytes = 0;
        const std::uint8_t *weights = nullptr, *rows = nullptr;
        if (filling) {
            of(own, bytes, weights, rows);
            barrier_expect_bytes(own_full, weight_block + bytes);
            // The kernel before this one makes the codes; it lets this one start only after its own wait, so when all
            // before it have ended, and weights are written by kernels that let nothing start early: one matrix's need not
            // wait. Which expert's, the tiles have said.
            bulk_load(ring + own * weight_block, weights, weight_block, own_full);
        }
        __syncwarp();
        if (!Experts) grid_dependency_wait();
        if (filling) bulk_load(rows_ring + own * row_bytes, rows, bytes, own_full);
        __syncwarp();
        std::int64_t q = warp - copy_warp;
        while (q < a.stages) q += copy_warps;
        if (lane < 2) {
            std::int64_t nth = q / blocks;
            int k = static_cast<int>(q - nth * blocks), slot = static_cast<int>(q) % a.stages;
            std::uint32_t pass = static_cast<std::uint32_t>(q) / static_cast<std::uint32_t>(a.stages);
            bool moved = true;  // to another tile
            const std::uint8_t* from = nullptr;
            const std::int64_t step = lane == 0 ? weight_block : a.out_rows * block_bytes;
            for (; q < mine; q += copy_warps) {
                if (moved) {
                    of(nth * blocks, bytes, weights, rows);
                    from = lane == 0 ? weights : rows;
                    moved = false;
                }
                bool free = true;
                if (lane == 0) free = !*abort && barrier_wait_for(smem_address(&tail.empty[slot]), (pass & 1u) ^ 1u, waits, a.wait_ns);
                if (!__shfl_sync(3u, free, 0)) {
                    *abort = 1;
                    break;
                }
                const std::uint32_t full = smem_address(&tail.full[slot]);
                if (lane == 0) barrier_expect_bytes(full, weight_block + bytes);
                __syncwarp(3u);
                bulk_load(lane == 0 ? ring + slot * weight_block : rows_ring + slot * row_bytes, from + k * step,
                          lane == 0 ? weight_block : bytes, full);
                for (slot += copy_warps; slot >= a.stages; slot -= a.stages) ++pass;
                for (k += copy_warps; k >= blocks; k -= blocks) ++nth, moved = true;
            }
            if (*abort && lane == 0) {  // the copies under way: of q - 4, q - 8, ...
                for (std::int64_t last = q - copy_warps; last >= 0 && last > q - copy_warps - a.stages; last -= copy_warps) {
                    if (last < mine) barrier_wait_for(smem_address(&tail.full[last % a.stages]), last / a.stages & 1, waits, a.wait_ns);
                }
            }
        }
    } else if (warp == mma_warp) {
        if (lane == 0) {
            int slot = 0, buffer = 0;
            std::uint32_t phase = 0, pass = 0;
            const std::uint64_t first_weights = sw128_descriptor(ring), first_rows = sw128_descriptor(rows_ring);
            Tile next = first_item < items ? tile_at<Experts>(a, first_item) : Tile{};
            for (int item = first_item; item < items && !*abort; item += item_step) {
                const Tile t = next;
                if (items - item > item_step) next = tile_at<Experts>(a, item + item_step);  // its latency under this one's products
                const std::uint32_t instruction = i8_instruction(t.columns);
                bool going = barrier_wait_for(smem_address(&tail.tmem_empty[buffer]), pass ^ 1u, waits, a.wait_ns);
                tmem_fence_after();
                const std::uint32_t sums = tmem + static_cast<std::uint32_t>(buffer * a.tile_rows);
                for (int k = k_from; going && k < k_to; ++k) {
                    going = barrier_wait_for(smem_address(&tail.full[slot]), phase, waits, a.wait_ns);
                    if (!going) break;
                    tmem_fence_after();
                    const std::uint64_t w = first_weights + static_cast<std::uint64_t>(slot * (weight_block >> 4));
                    const std::uint64_t x = first_rows + static_cast<std::uint64_t>(slot * (static_cast<int>(row_bytes) >> 4));
#pragma unroll
                    for (int step = 0; step < block_bytes / 32; ++step) {
                        mma_i8(sums, w + 2 * step, x + 2 * step, instruction, k > k_from || step > 0);
                    }
                    mma_commit(smem_address(&tail.empty[slot]));
                    if (++slot == a.stages) slot = 0, phase ^= 1u;
                }
                if (going) {
                    mma_commit(smem_address(&tail.tmem_full[buffer]));
                } else {
                    *abort = 1;
                }
                if (++buffer == 2) buffer = 0, pass ^= 1u;
            }
            if (*abort) {  // the MMAs under way
                mma_commit(smem_address(&tail.drain));
                barrier_wait_for(smem_address(&tail.drain), 0, waits, a.wait_ns);
            }
        }
    } else {
        const int quarter = warp % 4, half = warp / 4;
        int buffer = 0;
        std::uint32_t pass = 0;
        if (splits > 1) cluster_wait();
        for (int item = first_item; item < items; item += item_step) {
            const Tile t = tile_at<Experts>(a, item);
            if (splits == 1) stage_rows<Experts>(a, t, tail, buffer);
            if (epilogue_any(*abort != 0)) break;  // all of them, as the next ones wait for one another here
            // the TMEM loads take whole warps, so a warp takes one decision
            if (!__all_sync(0xffffffffu, barrier_wait_for(smem_address(&tail.tmem_full[buffer]), pass, waits, a.wait_ns))) {
                *abort = 1;
                continue;
            }
            tmem_fence_after();
            const std::uint32_t sums = tmem + static_cast<std::uint32_t>(buffer * a.tile_rows) +
                (static_cast<std::uint32_t>(quarter * 32) << 16);
            if (splits == 1) {
                store_tile<T, Experts>(a, t, tail, buffer, t.output + quarter * 32, sums, half);
            } else {
                const int mine = block_rows / splits;  // outputs that a block adds up
                const int channel = quarter * 32 + lane;
                const std::uint32_t to = exchange + static_cast<std::uint32_t>(rank * a.tile_rows * mine + channel % mine) * 4;
                for (int column = half * 16; column < t.columns; column += 32) {
                    int acc[16];
                    tmem_load16(sums + static_cast<std::uint32_t>(column), acc);
                    tmem_load_wait();
#pragma unroll
                    for (int i = 0; i < 16; ++i) peer_store(to + static_cast<std::uint32_t>((column + i) * mine) * 4, channel / mine, acc[i]);
                }
            }
            tmem_fence_before();
            barrier_arrive(smem_address(&tail.tmem_empty[buffer]));
            if (++buffer == 2) buffer = 0, pass ^= 1u;
        }
    }
    __syncwarp();

    if (splits > 1) {
        if (warp >= epilogue_warps) cluster_wait();
        if (*abort && lane < splits) peer_store(smem_address(&tail.given_up), lane, 1);  // the warp that gave up is one of them
        cluster_arrive();
        cluster_wait();
        if (first_item < items && !*static_cast<volatile int*>(&tail.given_up)) {
            const Tile t = tile_at<Experts>(a, first_item);
            const int mine = block_rows / splits;
            const int* sums = reinterpret_cast<const int*>(dynamic + (exchange - raw));
            for (int i = threadIdx.x; i < mine * t.rows; i += product_threads) {
                const int column = i / mine, output = t.output + rank * mine + i % mine;
                if (output >= a.outputs) continue;
                int sum = 0;
#pragma unroll 8
                for (int r = 0; r < splits; ++r) sum += sums[r * a.tile_rows * mine + i];
                const std::int64_t channel = static_cast<std::int64_t>(t.expert) * a.outputs + output;
                const std::int64_t row = t.row + column;
                float v = __fmul_rn(__fmul_rn(__int2float_rn(sum), a.scales[channel]), a.row_scales[row]);
                if (a.bias != nullptr) v = __fadd_rn(v, widen(static_cast<const T*>(a.bias)[channel]));
                const std::int64_t to = Experts ? a.arranged.pair[row] : row;
                static_cast<T*>(a.y)[to * a.outputs + output] = narrow<T>(v);
            }
        }
    }
    tmem_fence_before();
    __syncthreads();
    if (warp == mma_warp) {
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(a.tmem_columns) : "memory");
        if (lane == 0 && tail.status != 0) give_up<Experts>(a, tail.status);
    }
}

// Large products: two blocks of a cluster have a tile of 256 outputs, each with half of its outputs' weights and half of its
// rows in its shared memory, which the tensor cores of both read. A block of 128 inputs so takes 32 KB a block in place of
// 48, where 128 x 256 tiles loaded 66 bytes a cycle and SM, which is all that L2 gave. The copies of both blocks count on
// the first one's barriers, whose thread issues the MMAs: a thread that told it of the second one's, by an arrival with
// release, took 1300 cycles a block of inputs. A stage of the ring holds two blocks of inputs, as a wait, four MMAs and a
// commit take that thread 690 cycles, and the tensor cores 512.
constexpr int pair_blocks = 2;                                // of inputs a stage
constexpr unsigned copy_lanes = (2u << pair_blocks) - 1;      // of a copying warp

template <typename T, bool Experts>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(product_threads, 1) pair_kernel(
    const __grid_constant__ CUtensorMap weights_map, const __grid_constant__ CUtensorMap codes_map, const ProductArgs a) {
    extern __shared__ std::uint8_t dynamic[];
    __shared__ ProductTail tail;
    const std::uint32_t ring = (smem_address(dynamic) + 1023u) & ~1023u;
    const std::uint32_t row_bytes = static_cast<std::uint32_t>(a.tile_rows) / 2 * block_bytes;
    const std::uint32_t rows_ring = ring + static_cast<std::uint32_t>(a.stages) * pair_blocks * weight_block;
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    const int rank = static_cast<int>(blockIdx.x) % 2;
    const int first_item = static_cast<int>(blockIdx.x) / 2, item_step = static_cast<int>(gridDim.x) / 2;
    const int blocks = a.k_blocks, groups = (blocks + pair_blocks - 1) / pair_blocks;

    if (warp == copy_warp && lane == 0) {
        for (int s = 0; s < a.stages; ++s) {
            barrier_init(smem_address(&tail.full[s]), 1);
            barrier_init(smem_address(&tail.empty[s]), 1);
        }
        for (int b = 0; b < 2; ++b) {
            barrier_init(smem_address(&tail.tmem_full[b]), 1);
            barrier_init(smem_address(&tail.tmem_empty[b]), 2 * epilogue_warps);
        }
        barrier_init(smem_address(&tail.drain), 1);
        tail.status = 0;
        tail.abort = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        fence_proxy_async_shared();
    }
    if (warp == mma_warp) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_address(&tail.tmem)),
                     "r"(a.tmem_columns)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    }
    tmem_fence_before();
    __syncthreads();
    cluster_arrive();
    cluster_wait();
    tmem_fence_after();
    const std::uint32_t tmem = tail.tmem;
    volatile int* abort = &tail.abort;
    unsigned* waits = &tail.status;
    launch_dependents();
    grid_dependency_wait();
    const int row_tiles = Experts ? *a.arranged.tile_count : static_cast<int>((a.rows + a.tile_rows - 1) / a.tile_rows);
    const int items = row_tiles * ((a.tiles + 1) / 2);

    if (warp >= copy_warp && warp < copy_warp + copy_warps) {
        const bool copying = first_item < items && static_cast<int>(blockIdx.x) != a.withheld;
        const std::int64_t mine = copying ? static_cast<std::int64_t>((items - first_item + item_step - 1) / item_step) * groups : 0;
        // No more warps take turns than there are stages: one that ran ahead by two uses of a stage would take the parity of
        // its barrier's phase before last for the last one's.
        const int turns = min(copy_warps, a.stages);
        if (lane <= pair_blocks && warp - copy_warp < turns) {  // the first lane copies weights, the others a block of codes each
            std::int64_t nth = (warp - copy_warp) / groups;
            int group = (warp - copy_warp) % groups, slot = (warp - copy_warp) % a.stages;
            std::uint32_t pass = static_cast<std::uint32_t>((warp - copy_warp) / a.stages);
            bool moved = true;  // to another tile
            int from = 0;       // row of 128 bytes
            const CUtensorMap* map = lane == 0 ? &weights_map : &codes_map;
            const int step = lane == 0 ? block_rows : static_cast<int>(a.out_rows);
            const std::uint32_t to = lane == 0 ? ring : rows_ring + (lane - 1) * row_bytes;
            const std::uint32_t to_step = pair_blocks * (lane == 0 ? weight_block : row_bytes);
            // of both blocks: boxes are whole, past the last row and the last block of inputs too (zeros past the codes' end)
            const std::uint32_t stage = 2 * pair_blocks * (weight_block + row_bytes);
            std::int64_t q = warp - copy_warp;
            for (; q < mine; q += turns) {
                if (moved) {
                    const Tile t = tile_at<Experts, true>(a, first_item + static_cast<int>(nth) * item_step);
                    // past an odd last tile the second block's products are of no output
                    const std::int64_t tile = static_cast<std::int64_t>(t.expert) * a.tiles + min(t.output / block_rows + rank, a.tiles - 1);
                    from = static_cast<int>(lane == 0 ? tile * blocks * block_rows
                                                      : t.row + rank * (t.columns / 2) + static_cast<std::int64_t>(lane - 1) * a.out_rows);
                    moved = false;
                }
                bool free = true;
                if (lane == 0) free = !*abort && barrier_wait_for(smem_address(&tail.empty[slot]), (pass & 1u) ^ 1u, waits, a.wait_ns);
                if (!__shfl_sync(copy_lanes, free, 0)) {
                    *abort = 1;
                    break;
                }
                const std::uint32_t full = smem_address(&tail.full[slot]);
                if (lane == 0 && rank == 0) barrier_expect_bytes(full, stage);
                __syncwarp(copy_lanes);
                tma_load_2d_pair(to + slot * to_step, map, full, 0, from + group * pair_blocks * step);
                for (slot += turns; slot >= a.stages; slot -= a.stages) ++pass;
                for (group += turns; group >= groups; group -= groups) ++nth, moved = true;
            }
            if (*abort && lane == 0 && rank == 0) {  // the copies under way, the other block's too
                for (std::int64_t last = q - turns; last >= 0 && last > q - turns - a.stages; last -= turns) {
                    barrier_wait_for(smem_address(&tail.full[last % a.stages]), last / a.stages & 1, waits, a.wait_ns);
                }
            }
        }
    } else if (warp == mma_warp && rank == 1) {  // the first block's thread issues for both
    } else if (warp == mma_warp) {
        if (lane == 0) {
            int slot = 0, buffer = 0;
            std::uint32_t phase = 0, pass = 0;
            const std::uint64_t first_weights = sw128_descriptor(ring), first_rows = sw128_descriptor(rows_ring);
            Tile next = first_item < items ? tile_at<Experts, true>(a, first_item) : Tile{};
            for (int item = first_item; item < items && !*abort; item += item_step) {
                const Tile t = next;
                if (items - item > item_step) next = tile_at<Experts, true>(a, item + item_step);  // its latency under this one's products
                const std::uint32_t instruction = i8_pair_instruction(t.columns);
                bool going = barrier_wait_for(smem_address(&tail.tmem_empty[buffer]), pass ^ 1u, waits, a.wait_ns);
                tmem_fence_after();
                const std::uint32_t sums = tmem + static_cast<std::uint32_t>(buffer * a.tile_rows);
                for (int k = 0; going && k < blocks; k += pair_blocks) {
                    going = barrier_wait_for(smem_address(&tail.full[slot]), phase, waits, a.wait_ns);
                    if (!going) break;
                    tmem_fence_after();
                    const std::uint64_t w = first_weights + static_cast<std::uint64_t>(slot * (pair_blocks * weight_block >> 4));
                    const std::uint64_t x = first_rows + static_cast<std::uint64_t>(slot * (pair_blocks * static_cast<int>(row_bytes) >> 4));
#pragma unroll
                    for (int block = 0; block < pair_blocks; ++block) {
                        if (k + block >= blocks) break;
#pragma unroll
                        for (int step = 0; step < block_bytes / 32; ++step) {
                            mma_i8_pair(sums, w + static_cast<std::uint64_t>(block * (weight_block >> 4) + 2 * step),
                                        x + static_cast<std::uint64_t>(block * (static_cast<int>(row_bytes) >> 4) + 2 * step), instruction,
                                        k > 0 || block > 0 || step > 0);
                        }
                    }
                    mma_commit_pair(smem_address(&tail.empty[slot]));
                    if (++slot == a.stages) slot = 0, phase ^= 1u;
                }
                if (going) {
                    mma_commit_pair(smem_address(&tail.tmem_full[buffer]));
                } else {
                    *abort = 1;
                }
                if (++buffer == 2) buffer = 0, pass ^= 1u;
            }
            if (*abort) {  // the MMAs under way
                mma_commit_pair(smem_address(&tail.drain));
                barrier_wait_for(smem_address(&tail.drain), 0, waits, a.wait_ns);
            }
        }
    } else {
        const int quarter = warp % 4, half = warp / 4;
        int buffer = 0;
        std::uint32_t pass = 0;
        for (int item = first_item; item < items; item += item_step) {
            const Tile t = tile_at<Experts, true>(a, item);
            stage_rows<Experts>(a, t, tail, buffer);
            if (epilogue_any(*abort != 0)) break;  // all of them, as the next ones wait for one another here
            // the TMEM loads take whole warps, so a warp takes one decision
            if (!__all_sync(0xffffffffu, barrier_wait_for(smem_address(&tail.tmem_full[buffer]), pass, waits, a.wait_ns))) {
                *abort = 1;
                continue;
            }
            tmem_fence_after();
            const std::uint32_t sums = tmem + static_cast<std::uint32_t>(buffer * a.tile_rows) +
                (static_cast<std::uint32_t>(quarter * 32) << 16);
            store_tile<T, Experts>(a, t, tail, buffer, t.output + rank * block_rows + quarter * 32, sums, half);
            tmem_fence_before();
            __syncwarp();
            if (lane == 0) barrier_arrive_at(smem_address(&tail.tmem_empty[buffer]), 0);
            if (++buffer == 2) buffer = 0, pass ^= 1u;
        }
    }
    tmem_fence_before();
    __syncthreads();
    cluster_arrive();  // the other block's memory is read, and this one's barriers are arrived on, no more
    cluster_wait();
    if (warp == mma_warp) {
        asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(a.tmem_columns) : "memory");
        if (lane == 0 && tail.status != 0) give_up<Experts>(a, tail.status);
    }
}

// ---- y[t] = sum_j weights[t][j] * products[t][j], in the order of j ----

// A thread Each outputs: four where rows of outputs are whole vectors.
template <typename T, int Each>
__global__ void __launch_bounds__(128) combine_kernel(const float* products, const std::int32_t* choices, const float* weights,
                                                      int chosen, int experts, int outputs, const int* given_up, T* y) {
    join_chain();
    const bool whole = *given_up == 0;  // else products are missing, and nothing is written
    const std::int64_t token = blockIdx.x;
    for (int output = static_cast<int>(blockIdx.y * 128 + threadIdx.x) * Each; output < outputs; output += static_cast<int>(gridDim.y) * 128 * Each) {
        float sum[Each] = {};
#pragma unroll 4
        for (int j = 0; j < chosen; ++j) {
            const std::int64_t pair = token * chosen + j;
            const int e = choices[pair];
            if (e < 0 || e >= experts) continue;
            const float weight = weights[pair];
            const float* from = products + pair * outputs + output;
            if constexpr (Each == 4) {
                const float4 v = *reinterpret_cast<const float4*>(from);
                sum[0] = fmaf(weight, v.x, sum[0]), sum[1] = fmaf(weight, v.y, sum[1]);
                sum[2] = fmaf(weight, v.z, sum[2]), sum[3] = fmaf(weight, v.w, sum[3]);
            } else {
                sum[0] = fmaf(weight, *from, sum[0]);
            }
        }
#pragma unroll
        for (int i = 0; i < Each; ++i) {
            if (whole) y[token * outputs + output + i] = narrow<T>(sum[i]);
        }
    }
}

// ---- launches ----

template <typename T, int Warps, int Held>
cudaError_t quantise_rows(const QuantiseArgs& a, cudaStream_t stream) {
    const auto blocks = static_cast<unsigned>((a.rows + 8 / Warps - 1) / (8 / Warps));
    if (a.choices == nullptr) return launch_overlapped(quantise_kernel<T, Warps, Held, false>, dim3(blocks), dim3(256), 0, stream, a);
    const std::size_t shared = sizeof(int) * (static_cast<std::size_t>(8 / Warps) * a.fan + a.pairs + a.experts);
    return launch_overlapped(quantise_kernel<T, Warps, Held, true>, dim3(blocks), dim3(256), shared, stream, a);
}

template <typename T>
cudaError_t quantise(const QuantiseArgs& a, cudaStream_t stream) {
    constexpr int held = 16 / sizeof(T);  // 64 registers
    const bool many = a.rows >= 8 * sm_count();
    if (a.inputs <= 1024) return quantise_rows<T, 1, 2>(a, stream);
    if (many && a.inputs <= 512 * held) return quantise_rows<T, 1, held>(a, stream);
    if (a.inputs <= 2048) return quantise_rows<T, 2, 2>(a, stream);
    return quantise_rows<T, 8, 2>(a, stream);
}

cudaError_t quantise(Type type, const QuantiseArgs& a, cudaStream_t stream) {
    switch (type) {
    case Type::f16: return quantise<__half>(a, stream);
    case Type::bf16: return quantise<__nv_bfloat16>(a, stream);
    default: return quantise<float>(a, stream);
    }
}

template <typename T, bool Experts>
cudaError_t product(ProductArgs a, std::int64_t most_items, cudaStream_t stream) {
    static SharedAllowance allowance;
    const int exchange = a.splits > 1 ? block_rows * a.tile_rows * 4 : 0;
    const int room = 208 * 1024 - exchange;
    const int stage = weight_block + a.tile_rows * block_bytes;
    a.stages = std::min(most_stages, room / stage);
    if (a.stages < copy_warps) return cudaErrorInvalidValue;  // as the copying warps' turns need (at 256 rows there are four)
    a.tmem_columns = 32;
    while (a.tmem_columns < 2u * static_cast<unsigned>(a.tile_rows)) a.tmem_columns *= 2;
    const int bytes = a.stages * stage + exchange + 1024;
    cudaError_t status = allowance.allow(product_kernel<T, Experts>, 210 * 1024);
    if (status != cudaSuccess) return status;
    cudaLaunchConfig_t config{};
    config.gridDim = dim3(static_cast<unsigned>(a.splits > 1 ? most_items * a.splits
                                                             : std::min<std::int64_t>(most_items, sm_count())));
    config.blockDim = dim3(product_threads);
    config.dynamicSmemBytes = static_cast<std::size_t>(bytes);
    config.stream = stream;
    cudaLaunchAttribute attributes[2];
    attributes[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attributes[0].val.programmaticStreamSerializationAllowed = 1;
    attributes[1].id = cudaLaunchAttributeClusterDimension;
    attributes[1].val.clusterDim.x = static_cast<unsigned>(a.splits);
    attributes[1].val.clusterDim.y = attributes[1].val.clusterDim.z = 1;
    config.attrs = attributes;
    config.numAttrs = a.splits > 1 ? 2 : 1;
    return cudaLaunchKernelEx(&config, product_kernel<T, Experts>, a);
}

using EncodeTiled = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                                 const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                 CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

// `rows` rows of 128 bytes, copied `box` at a time (their swizzle is in memory already).
bool encode(CUtensorMap& map, const void* memory, std::uint64_t rows, int box) {
    static const EncodeTiled function = [] {
        void* pointer = nullptr;
        cudaDriverEntryPointQueryResult found{};
        if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &pointer, 12000, cudaEnableDefault, &found) != cudaSuccess ||
            found != cudaDriverEntryPointSuccess) {
            return static_cast<EncodeTiled>(nullptr);
        }
        return reinterpret_cast<EncodeTiled>(pointer);
    }();
    if (function == nullptr) return false;
    const cuuint64_t sizes[2] = {block_bytes, rows}, strides[1] = {block_bytes};
    const cuuint32_t boxes[2] = {block_bytes, static_cast<cuuint32_t>(box)}, steps[2] = {1, 1};
    return function(&map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(memory), sizes, strides, boxes, steps,
                    CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                    CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <typename T, bool Experts>
cudaError_t pair_product(ProductArgs a, std::int64_t most_items, cudaStream_t stream) {
    static SharedAllowance allowance;
    const int stage = pair_blocks * (weight_block + a.tile_rows / 2 * block_bytes);
    a.stages = std::min(most_stages, 208 * 1024 / stage);
    a.tmem_columns = 32;
    while (a.tmem_columns < 2u * static_cast<unsigned>(a.tile_rows)) a.tmem_columns *= 2;
    const cudaError_t status = allowance.allow(pair_kernel<T, Experts>, 210 * 1024);
    if (status != cudaSuccess) return status;
    CUtensorMap weights, codes;
    const std::uint64_t blocks = static_cast<std::uint64_t>(a.arranged.tiles == nullptr ? 1 : a.experts) * a.tiles * a.k_blocks;
    if (!encode(weights, a.weights, blocks * block_rows, pair_blocks * block_rows) ||
        !encode(codes, a.codes, static_cast<std::uint64_t>(a.k_blocks) * a.out_rows, a.tile_rows / 2)) {
        return cudaErrorUnknown;
    }
    const auto pairs = static_cast<unsigned>(std::min<std::int64_t>(most_items, sm_count() / 2));
    return launch_overlapped(pair_kernel<T, Experts>, dim3(2 * pairs), dim3(product_threads),
                             static_cast<std::size_t>(a.stages * stage + 1024), stream, weights, codes, a);
}

template <bool Experts>
cudaError_t product(Type type, const ProductArgs& a, std::int64_t most_items, bool pair, cudaStream_t stream) {
    if (pair) {
        switch (type) {
        case Type::f16: return pair_product<__half, Experts>(a, most_items, stream);
        case Type::bf16: return pair_product<__nv_bfloat16, Experts>(a, most_items, stream);
        default: return pair_product<float, Experts>(a, most_items, stream);
        }
    }
    switch (type) {
    case Type::f16: return product<__half, Experts>(a, most_items, stream);
    case Type::bf16: return product<__nv_bfloat16, Experts>(a, most_items, stream);
    default: return product<float, Experts>(a, most_items, stream);
    }
}

constexpr int most_split_tile = 64;  // rows of a tile that a cluster shares: its sums have a place of their own

// Blocks that share a tile's inputs: while they all run at once and each has two blocks of them. No more than four: of
// clusters of eight blocks with an SM each, 16 do not run at once (16 rows of 2048 -> 2048 11.4 us, 7.6 by four).
int splits_of(std::int64_t items, int tile_rows, int k_blocks) {
    int splits = 1;
    while (tile_rows <= most_split_tile && splits < 4 && items * splits * 2 <= sm_count() && k_blocks >= splits * 4) splits *= 2;
    return splits;
}

struct Shape {
    int tile_rows;
    bool pair;  // two blocks a tile
};

// Rows a tile, and the kernel: what takes the fewest cycles by a model. A block of inputs is loaded at 60 bytes a cycle or
// multiplied at two cycles a row (at least 240); a tile's stores, which overlap the next tile's products, take 24 cycles a
// row.
Shape shape_of(bool experts, double groups, double rows, int tiles, int k_blocks) {
    Shape best{step_rows, false};
    double least = -1.0;
    for (const bool pair : {false, true}) {
        const int step = pair ? pair_step_rows : step_rows, sets = sm_count() / (pair ? 2 : 1);
        for (int n = step; n <= most_tile; n += step) {
            // rows of a group are spread around their mean, so beyond one tile the last is half full
            const double items = groups * (pair ? (tiles + 1) / 2 : tiles) * (!experts ? std::ceil(rows / n) : std::max(1.0, rows / n + 0.5));
            const int splits = pair ? 1 : splits_of(static_cast<std::int64_t>(items), n, k_blocks);
            const double block = std::max({(weight_block + (pair ? n / 2 : n) * block_bytes) / 60.0, 2.0 * n, 240.0});
            const double product = std::ceil(static_cast<double>(k_blocks) / splits) * block, stores = 600.0 + 24.0 * n;
            const double cost = std::ceil(items * splits / sets) * std::max(product, stores) + stores + (splits > 1 ? 1500.0 : 0.0) + (pair ? 1500.0 : 0.0);
            if (least < 0.0 || cost < least) least = cost, best = {n, pair};
            if (n >= rows && !experts) break;
        }
    }
    return best;
}

// Where the parts of a call's working memory are: for any shape of its tiles, which takes a microsecond to choose.
struct Plan {
    std::int64_t out_rows, groups;
    std::size_t codes, scales, place, pair, table, count, products, bytes;
};

Plan plan_of(const BytesArgs& a) {
    Plan p{};
    const std::int64_t pairs = a.tokens * a.chosen;
    std::size_t at = 0;
    auto take = [&](std::size_t bytes) {
        const std::size_t here = at;
        at += aligned(bytes);
        return here;
    };
    p.groups = a.choices == nullptr ? 1 : std::max<std::int64_t>(std::min<std::int64_t>(a.experts, pairs), 1);
    p.out_rows = a.choices == nullptr ? padded(a.tokens) : padded(pairs + p.groups * (step_rows - 1));
    p.codes = take(static_cast<std::size_t>(blocks_of(a.inputs)) * p.out_rows * block_bytes);
    p.scales = take(p.out_rows * sizeof(float));
    if (a.choices != nullptr) {
        p.place = take(pairs * sizeof(int));
        p.pair = take(p.out_rows * sizeof(int));
        p.table = take((pairs / step_rows + p.groups) * sizeof(int4));
        p.count = take(2 * sizeof(int));
        if (a.weights != nullptr) p.products = take(static_cast<std::size_t>(pairs) * a.outputs * sizeof(float));
    }
    p.bytes = at;
    return p;
}

template <typename T>
cudaError_t combine(const BytesArgs& a, const float* products, const int* given_up, cudaStream_t stream) {
    const int each = a.outputs % 4 == 0 ? 4 : 1;
    const dim3 grid(static_cast<unsigned>(a.tokens), static_cast<unsigned>(std::min((a.outputs + 128 * each - 1) / (128 * each), 65535)));
    auto kernel = each == 4 ? combine_kernel<T, 4> : combine_kernel<T, 1>;
    return launch_overlapped(kernel, grid, dim3(128), 0, stream, products, a.choices, a.weights, a.chosen, a.experts, a.outputs,
                             given_up, static_cast<T*>(a.y));
}

}  // namespace

std::size_t byte_matrix_bytes(std::int64_t matrices, int outputs, int inputs) {
    return static_cast<std::size_t>(matrices) * tiles_of(outputs) * blocks_of(inputs) * weight_block;
}

cudaError_t pack_bytes(const std::int8_t* codes, std::int64_t matrices, int outputs, int inputs, void* packed,
                       cudaStream_t stream) {
    const std::int64_t blocks = matrices * tiles_of(outputs) * blocks_of(inputs);
    const std::int64_t grid = std::min<std::int64_t>((blocks * (weight_block / 16) + 255) / 256, 16ll * sm_count());
    pack_kernel<<<static_cast<unsigned>(grid), 256, 0, stream>>>(codes, blocks, outputs, inputs, tiles_of(outputs),
                                                                  blocks_of(inputs), static_cast<uint4*>(packed));
    return cudaGetLastError();
}

std::size_t bytes_workspace(const BytesArgs& a) { return plan_of(a).bytes; }

cudaError_t multiply_bytes(const BytesArgs& a, cudaStream_t stream) {
    if (a.tokens == 0) return cudaSuccess;
    if (few_rows(a)) return multiply_few(a, stream);
    const Plan p = plan_of(a);
    auto* memory = static_cast<std::uint8_t*>(a.workspace);
    const std::int64_t pairs = a.tokens * a.chosen;
    const Shape shape = shape_of(a.choices != nullptr, static_cast<double>(p.groups), static_cast<double>(pairs) / static_cast<double>(p.groups),
                                 tiles_of(a.outputs), blocks_of(a.inputs));
    const std::int64_t row_tiles = a.choices == nullptr ? (pairs + shape.tile_rows - 1) / shape.tile_rows : pairs / shape.tile_rows + p.groups;
    const int elements = a.type == Type::f32 ? 4 : 2;
    if (row_tiles * tiles_of(a.outputs) > INT32_MAX - 1024) return cudaErrorInvalidValue;  // tiles are counted in 32 bits
    Arranged arranged{};
    if (a.choices != nullptr) {
        arranged = {reinterpret_cast<int*>(memory + p.place), reinterpret_cast<int*>(memory + p.pair),
                    reinterpret_cast<int4*>(memory + p.table), reinterpret_cast<int*>(memory + p.count),
                    reinterpret_cast<int*>(memory + p.count) + 1};
    }
    QuantiseArgs q{};
    if (a.choices != nullptr && pairs <= most_own_pairs) {
        q.choices = a.choices, q.pairs = static_cast<int>(pairs), q.experts = a.experts, q.tile_rows = shape.tile_rows;
        q.arranged = arranged;
    } else if (a.choices != nullptr) {
        const cudaError_t status = launch_overlapped(arrange_kernel, dim3(arrange_blocks), dim3(arrange_threads), 0, stream, a.choices,
                                                     pairs, a.experts, shape.tile_rows, arranged);
        if (status != cudaSuccess) return status;
    }
    q.x = a.x, q.stride = a.x_stride, q.inner_stride = a.x_inner_stride;
    q.inner = a.inner;
    q.rows = a.tokens * q.inner;
    q.inputs = a.inputs, q.k_blocks = blocks_of(a.inputs);
    q.vector = reinterpret_cast<std::uintptr_t>(a.x) % 16 == 0 && a.x_stride * elements % 16 == 0 &&
        a.x_inner_stride * elements % 16 == 0;
    q.place = arranged.place, q.fan = a.chosen / q.inner;
    q.out_rows = p.out_rows;
    q.codes = memory + p.codes, q.scales = reinterpret_cast<float*>(memory + p.scales);
    q.zeros = a.choices != nullptr && a.weights == nullptr ? a.y : nullptr, q.outputs = a.outputs;
    cudaError_t status = quantise(a.type, q, stream);
    if (status != cudaSuccess) return status;

    ProductArgs r{};
    r.weights = static_cast<const std::uint8_t*>(a.packed), r.scales = a.scales, r.bias = a.bias;
    r.codes = q.codes, r.row_scales = q.scales, r.arranged = arranged;
    r.rows = a.tokens, r.out_rows = p.out_rows;
    r.experts = a.experts, r.outputs = a.outputs, r.tiles = tiles_of(a.outputs), r.k_blocks = q.k_blocks;
    r.tile_rows = shape.tile_rows;
    const std::int64_t items = row_tiles * (shape.pair ? (r.tiles + 1) / 2 : r.tiles);
    r.splits = shape.pair ? 1 : splits_of(items, r.tile_rows, r.k_blocks);
    r.status = a.status, r.wait_ns = a.wait_ns != 0 ? a.wait_ns : wait_limit_ns, r.withheld = a.withheld;
    if (a.choices == nullptr) {
        r.y = a.y;
        return product<false>(a.type, r, items, shape.pair, stream);
    }
    if (a.weights == nullptr) {
        r.y = a.y;
        return product<true>(a.type, r, items, shape.pair, stream);
    }
    auto* products = reinterpret_cast<float*>(memory + p.products);
    r.y = products;
    // FP32 products, so that a token's sum is rounded once
    status = product<true>(Type::f32, r, items, shape.pair, stream);
    if (status != cudaSuccess) return status;
    switch (a.type) {
    case Type::f16: return combine<__half>(a, products, arranged.given_up, stream);
    case Type::bf16: return combine<__nv_bfloat16>(a, products, arranged.given_up, stream);
    default: return combine<float>(a, products, arranged.given_up, stream);
    }
}

}  // namespace nvcr_sm100::token
