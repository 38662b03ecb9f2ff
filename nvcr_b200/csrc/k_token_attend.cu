// Attention of new tokens over the paged 4-bit cache. Token i of a sequence's
// count new ones is at position length - count + i and sees the keys up to its
// own position; one that sees none gives zeros, as does a token that belongs to
// no sequence, or to one whose offsets or length are out of range. Grouped heads:
// query head h reads cache head h / (heads / kv_heads).
//
// The codes are never expanded to values. With s, m a group's scale and minimum,
//   score = sum_g s_g (q_g . c_g) + m_g sum(q_g),
//   out_d = sum_t (p_t s_tg) (c_td - 8) + sum_t p_t (m_tg + 8 s_tg),
// so both products run on the codes themselves. For keys, a nibble masked out of
// its place in a 16-bit half is the FP16 number c 2^-24 or, four bits up, c 2^-20
// (subnormal, exact in the tensor cores), and the powers of two are taken out
// with the scales: five integer instructions give eight codes of an operand.
// For values, the same nibbles under the exponent of 1024 give c - 8 with one
// FP16 operation a pair (exact): the weights' rounding and the tensor cores'
// truncated sums then weigh on c - 8, not on c, which a long mean of values
// around zero needs (131072 keys: error 6.0e-4 with c, see the tests' bound).
// Keys and transposed values are the 16-row operand of mma.m16n8k16, the query
// rows that share a cache head (grouped heads times new tokens) its 8 columns:
// a step's work is a cache read of 4.5 bits a value against one or two such
// columns, so what bounds it is HBM and the conversion, not the tensor pipe,
// and the warp-level instruction leaves codes, scores and weights in registers.
// Queries are scaled by a power of two per row into FP16's range (exact but for
// channels 2^-35 of the row's largest); weights p s are rounded to FP16
// after scaling to the group's largest scale so far, as a 16-bit operand must.
// Scores, softmax statistics and sums are FP32.
//
// Work is cut evenly over the blocks, one an SM, whatever the lengths: a segment is
// one cache head, 8 or 16 query rows and a sequence's whole length, in units of 256
// or 128 keys (two runs of 16, or one, for each of eight warps); all segments' units
// in a row are divided among the blocks (segments of one length alike, each among
// as many), or taken whole where a cut saves less than its join costs. A warp
// streams its runs through a ring of its own in shared memory (cp.async; 16-byte
// chunks XOR-swizzled so that the fragment reads touch every bank once) and keeps
// its own running maximum and sum; the next piece's copies and queries are on
// their way while a piece is joined. A block joins its warps in shared memory; a
// segment that several blocks share is joined in the context's workspace by the
// last of them, in order: the same bits every time.
//
// Measured on a B200: 131072 keys, 32 heads over 8 of 128 channels, one token
// (142.6 MB): 47.4 us, 3.0 TB/s; 32 sequences of 1 to 4096 keys (76 MB): 35.5 us; 200
// keys: 5.5 us. What bounds a long stream is the integer pipe that takes the
// codes apart (174 of a launch's 348 instructions for each run of 16 keys, at half
// rate) and the warps' latency: 171 cycles a run while an SM is active. Two blocks an
// SM with 128 registers a thread streamed as fast (47.2 us), but had twice the fixed
// work: 6.3 us for 200 keys. Short calls are bound by the chain lengths -> page
// table -> cache -> join, about 1 us a link.
#include "token_elements.cuh"

#include <algorithm>
#include <cfloat>

namespace nvcr_sm100::token {
namespace {

constexpr int warps = 8;
// In keys: the least a block takes on average where segments are cut, what joining a cut segment costs, and what
// starting on one costs.
constexpr int least_keys = 512, join_keys = 768, lead_keys = 512;
constexpr int most_blocks = 160;
constexpr float log2_e = 1.4426950408889634f;
// A running maximum is raised only when a score passes it by this much (in
// powers of two): weights stay below 2^8, and few tiles rescale their sums.
constexpr float top_slack = 8.0f;

__device__ __forceinline__ void note(const Cache& cache, unsigned bit) {
    if (cache.status != nullptr) atomicOr(cache.status, bit);
}

__device__ __forceinline__ void copy_async(unsigned shared, const void* global) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(shared), "l"(global) : "memory");
}

__device__ __forceinline__ void mma(float (&d)[4], const unsigned (&a)[4], unsigned b0, unsigned b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
        "{%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ void mma_from_zero(float (&d)[4], const unsigned (&a)[4], unsigned b0, unsigned b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
        "{%10, %10, %10, %10};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.0f));
}

__device__ __forceinline__ unsigned transpose8x8(unsigned v) {
    unsigned r;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
    return r;
}

// Nibbles 0 and 4 (even) or 1 and 5 (odd) of a word as the FP16 pair c - 8: under the exponent of 1024 they read
// 1024 + c and 1024 + 16 c. (Published for 4-bit weights by Kim, Henry, Fahim and Awadalla, 2022, arXiv 2211.10017.)
__device__ __forceinline__ unsigned even_codes(unsigned v) {
    unsigned codes;
    asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(codes) : "r"((v & 0x000f000fu) | 0x64006400u), "r"(0x64086408u));
    return codes;
}
__device__ __forceinline__ unsigned odd_codes(unsigned v) {  // times 1 / 16, less 72
    unsigned codes;
    asm("fma.rn.f16x2 %0, %1, %2, %3;"
        : "=r"(codes)
        : "r"((v & 0x00f000f0u) | 0x64006400u), "r"(0x2c002c00u), "r"(0xd480d480u));
    return codes;
}

__device__ __forceinline__ unsigned pack_half(float low, float high) {
    const __half2 v = __floats2half2_rn(low, high);
    return reinterpret_cast<const unsigned&>(v);
}

__device__ __forceinline__ float2 pair_at(const std::uint8_t* scales, int byte) {
    return __half22float2(*reinterpret_cast<const __half2*>(scales + byte));
}

struct Work {
    Cache cache;
    AttendArgs a;
    Divisor runs_per_page;  // runs of 16 places
    Divisor by_ratio;
    int ratio;              // query heads of a cache head
    float* partials;        // [block][2][rows (D + 2)]: a segment begun before the block, one that goes on after it
    unsigned* tickets;      // [block], zero between calls
    bool aligned;           // queries can be read 16 bytes at a time
};

// Fragment row r of a run of 8 keys holds key row_key(r): with it the four keys
// that a value fragment reads at once lie in different rows of banks.
__device__ __forceinline__ int row_key(int r) { return (r & 4) | (r & 1) << 1 | (r & 2) >> 1; }

// XOR of the 16-byte chunk index of key t's row of D / 2 bytes.
template <int D>
__device__ __forceinline__ int swizzle(int t) {
    if (D == 64) return t >> 2 & 1;
    if (D == 128) return ((t >> 1 ^ t >> 2) & 1) << 1 | (t >> 2 & 1);
    return (t & 1) << 1 | ((t >> 1 ^ t >> 2) & 1) << 2;
}

// A run of 16 keys in the ring: [key][chunk ^ swizzle] codes of keys, of values, then [key][group] scales of each.
template <int D, int G>
constexpr int run_bytes = 16 * (D + 8 * (D / G));

// Runs of 16 keys a warp takes at once: two share a warp's control, copies and vote, where the registers allow.
template <int D, int NT>
constexpr int together = NT == 1 && D < 256 ? 2 : 1;

// Slots of that many runs in a warp's ring.
template <int D, int G, int NT>
constexpr int ring_slots = together<D, NT> == 2 ? (D == 128 && G == 32 ? 2 : 3) : D == 256 ? 3 : 4;

template <int D, int G, int NT>
constexpr int shared_bytes = warps * (ring_slots<D, G, NT> * together<D, NT> * run_bytes<D, G> + 8 * NT * (D + 4) * 4);

// What a block takes of one segment.
struct Piece {
    int segment_start, segment_end;  // in the row of all segments
    int first_unit, last_unit;
    int kv_head, first, before;      // `first` of the sequence's new tokens, which are at positions `before` and on
    int first_row, total_rows, used_rows;
    int visible_first, visible_last; // keys that the first and the last row see
    int begin, end, steps;           // this warp's places
    const std::int32_t* table;
    bool complete;
};

// The units of one sequence: `blocks` blocks of rows times `units` of each segment.
struct Share {
    int count, length, blocks, units;
    int first;  // of its new tokens; -1: out of range, and left out
};

// A sequence's tokens and length; false where they are out of range, and the sequence is left out.
__device__ __forceinline__ bool extent_of(const std::int32_t* offsets, const std::int32_t* lengths, int max_queries,
                                          int max_length, std::int64_t tokens, int sequence, int& first, int& last,
                                          int& length) {
    first = sequence, last = sequence + 1;
    if (offsets != nullptr) first = offsets[sequence], last = offsets[sequence + 1];
    length = lengths[sequence];
    return first >= 0 && last <= tokens && last >= first && last - first <= max_queries && length >= 0 && length <= max_length;
}

// Zeros for the tokens of no sequence, a warp each. Not inlined: the kernel's registers are for its stream of keys.
__device__ __noinline__ void clear_left_out(const std::int32_t* offsets, const std::int32_t* lengths, int batch,
                                            int max_queries, int max_length, std::int64_t tokens, uint4* output,
                                            int row_chunks) {
    const int lane = threadIdx.x % 32;
    int first, last, length;
    bool all_good = true;  // then the sequences' tokens lie in a row
    for (int b = lane; b < batch; b += 32) {
        all_good = all_good && extent_of(offsets, lengths, max_queries, max_length, tokens, b, first, last, length);
    }
    all_good = __all_sync(0xffffffffu, all_good);
    for (std::int64_t token = static_cast<std::int64_t>(blockIdx.x) * warps + threadIdx.x / 32; token < tokens;
         token += static_cast<std::int64_t>(gridDim.x) * warps) {
        bool inside = false;
        if (all_good) {
            inside = offsets == nullptr || (token >= offsets[0] && token < offsets[batch]);
        } else {
            for (int b = lane; b < batch; b += 32) {
                const bool good = extent_of(offsets, lengths, max_queries, max_length, tokens, b, first, last, length);
                inside = inside || (good && token >= first && token < last);
            }
            inside = __any_sync(0xffffffffu, inside);
        }
        if (inside) continue;
        for (int i = lane; i < row_chunks; i += 32) output[token * row_chunks + i] = {0u, 0u, 0u, 0u};
    }
}

// One block an SM, said to the compiler: it then takes 222 registers for FP16 heads of 128 in groups of 128, and 168
// without (131072 keys: 47.3 us, 51.7 us).
template <typename T, int D, int G, int NT>
__global__ void __launch_bounds__(32 * warps, 1) attend_kernel(const Work work) {
    constexpr int groups = D / G, rows = 8 * NT, H = together<D, NT>, ring = ring_slots<D, G, NT>;
    constexpr int unit = 16 * H * warps, slot_bytes = H * run_bytes<D, G>;  // unit: keys
    constexpr int least_units = (least_keys + unit - 1) / unit, join_units = (join_keys + unit - 1) / unit;
    constexpr int lead_units = (lead_keys + unit - 1) / unit;
    constexpr int row_bytes = D / 2, chunks = row_bytes / 16;
    constexpr int words = G / 32;  // 32-bit words of codes a lane holds of a group of one key
    constexpr int tiles = G / 16;  // 16-channel tiles of a group
    constexpr int partial_floats = rows * (D + 2);
    extern __shared__ __align__(128) std::uint8_t shared[];
    __shared__ float joint_top[warps][rows], joint_sum[warps][rows];
    __shared__ int joint_units[warps], joint_segments[warps], joint_longest[warps], joint_sequence, joint_before;
    __shared__ bool joint_last;
    __shared__ __align__(16) __half joint_query[NT][D * 8];  // [word][lane][fragment registers]
    __shared__ float joint_query_sum[rows][groups], joint_factor[rows];
    join_chain();
    const Cache& cache = work.cache;
    const AttendArgs& a = work.a;
    const int lane = threadIdx.x % 32, warp = threadIdx.x / 32, r = lane / 4, j = lane % 4;

    // ---- this block's part of all the segments' units ----
    auto share_of = [&](int sequence, bool tell) {
        int first, last, length;
        if (!extent_of(a.query_offsets, a.lengths, a.max_queries, a.max_length, a.tokens, sequence, first, last, length)) {
            if (tell) note(cache, status_length);
            return Share{0, 0, 0, 0, -1};
        }
        Share s{last - first, length, 0, 0, first};
        s.blocks = (s.count * work.ratio + rows - 1) / rows;
        s.units = max(1, (s.length + unit - 1) / unit);
        return s;
    };
    // Up to 32 sequences are one to a lane in every warp; more are divided among the block's threads.
    const bool few = a.batch <= 32;
    const int each = few ? 1 : (a.batch + 32 * warps - 1) / (32 * warps), counter = few ? lane : static_cast<int>(threadIdx.x);
    const int from = min(a.batch, counter * each), to = min(a.batch, from + each);
    Share own{0, 0, 0, 0, 0};  // of the last of them
    int units = 0, segments = 0, longest = 0;
    // Every token is some sequence's: each sequence's begin where the last one's end.
    bool covered = true;
    for (int b = from; b < to; ++b) {
        own = share_of(b, blockIdx.x == 0);
        covered = covered && own.first >= 0 && (b > 0 || own.first == 0) && (b < a.batch - 1 || own.first + own.count == a.tokens);
        units += own.blocks * own.units * cache.kv_heads;
        segments += own.blocks * cache.kv_heads;
        if (own.blocks > 0) longest = max(longest, own.units);
    }
    int units_to = units, segments_to = segments;  // become those of the threads up to this one
#pragma unroll
    for (int offset = 1; offset < 32; offset *= 2) {
        const int other = __shfl_up_sync(0xffffffffu, units_to, offset);
        const int others = __shfl_up_sync(0xffffffffu, segments_to, offset);
        if (lane >= offset) units_to += other, segments_to += others;
    }
    longest = __reduce_max_sync(0xffffffffu, longest);
    int all_units = __shfl_sync(0xffffffffu, units_to, 31), all_segments = __shfl_sync(0xffffffffu, segments_to, 31);
    if (!few) {
        if (lane == 31) joint_units[warp] = units_to, joint_segments[warp] = segments_to, joint_longest[warp] = longest;
        covered = __syncthreads_and(covered);
        all_units = all_segments = 0;
#pragma unroll
        for (int w = 0; w < warps; ++w) {
            if (w < warp) units_to += joint_units[w], segments_to += joint_segments[w];
            all_units += joint_units[w], all_segments += joint_segments[w];
            longest = max(longest, joint_longest[w]);
        }
    }
    if (__any_sync(0xffffffffu, !covered)) {
        clear_left_out(a.query_offsets, a.lengths, a.batch, a.max_queries, a.max_length, a.tokens,
                       static_cast<uint4*>(a.output), a.heads * (D / 8));
    }
    // Segments are cut only where that saves more units than joining costs.
    const int grid = static_cast<int>(gridDim.x);
    const bool whole = (all_segments + grid - 1) / grid * longest <= max(all_units / grid, least_units) + join_units;
    int blocks = max(1, min(grid, whole ? all_segments : all_units / least_units));
    // Segments of one length are cut alike, `per` blocks each, so that none has a second piece to start on; others at
    // any unit, the first `more` blocks having one more than `fewer`, where starting on a segment counts as `lead` units
    // before its first. A segment that is not cut counts as one.
    const int per = !whole && longest * all_segments == all_units && all_segments > 0 ? blocks / all_segments : 0;
    const int lead = whole || per > 0 ? 0 : lead_units;
    const int total = whole ? all_segments : all_units + lead * all_segments;
    const int mine = whole ? segments : units + lead * segments;
    const int before = (whole ? segments_to : units_to + lead * segments_to) - mine;
    auto span_of = [&](const Share& s) { return whole ? 1 : s.units + lead; };
    if (per > 0) blocks = per * all_segments;
    if (static_cast<int>(blockIdx.x) >= blocks) return;
    const int fewer = total / blocks, more = total - fewer * blocks;
    auto start_of = [&](int block) {
        if (per > 0) return block / per * longest + block % per * longest / per;
        return block * fewer + min(block, more);
    };
    auto block_of = [&](int at) {
        if (per > 0) return at / longest * per + ((at % longest + 1) * per - 1) / longest;
        const int wide = more * (fewer + 1);
        return at < wide ? at / (fewer + 1) : more + (at - wide) / fewer;
    };
    int at = start_of(blockIdx.x);
    const int stop = start_of(blockIdx.x + 1);
    if (at >= stop) return;  // no work at all
    auto share_at = [&](int sequence) {
        if (!few) return share_of(sequence, false);
        return Share{__shfl_sync(0xffffffffu, own.count, sequence), __shfl_sync(0xffffffffu, own.length, sequence),
                     __shfl_sync(0xffffffffu, own.blocks, sequence), __shfl_sync(0xffffffffu, own.units, sequence),
                     __shfl_sync(0xffffffffu, own.first, sequence)};
    };
    int sequence, sequence_start;
    const bool here = at >= before && at < before + mine;
    if (few) {
        sequence = __ffs(__ballot_sync(0xffffffffu, here)) - 1;
        sequence_start = __shfl_sync(0xffffffffu, before, sequence);
    } else {
        if (here) {
            int start = before, b = from;
            for (;; ++b) {
                const Share s = share_of(b, false);
                const int next = start + s.blocks * span_of(s) * cache.kv_heads;
                if (at < next) break;
                start = next;
            }
            joint_sequence = b;
            joint_before = start;
        }
        __syncthreads();
        sequence = joint_sequence, sequence_start = joint_before;
    }
    Share share = share_at(sequence);

    // ---- what does not change from piece to piece ----
    const unsigned ring_base = static_cast<unsigned>(__cvta_generic_to_shared(shared)) + warp * ring * slot_bytes;
    const std::uint8_t* const ring_bytes = shared + warp * ring * slot_bytes;
    const int my_key = row_key(r);                // score rows my_key and my_key + 8 of a run
    const int pair_key = (j & 1) | (j & 2) << 1;  // value keys pair_key and pair_key + 2, and 8 on
    int key_offset[groups], value_offset[groups][2];
#pragma unroll
    for (int g = 0; g < groups; ++g) {
        const int kb = g * (G / 2) + j * (G / 8), vb = g * (G / 2) + r * (G / 16);
        key_offset[g] = my_key * row_bytes + (((kb / 16) ^ swizzle<D>(my_key)) * 16 + kb % 16);
        value_offset[g][0] = pair_key * row_bytes + (((vb / 16) ^ swizzle<D>(pair_key)) * 16 + vb % 16);
        value_offset[g][1] = (pair_key + 2) * row_bytes + (((vb / 16) ^ swizzle<D>(pair_key + 2)) * 16 + vb % 16);
    }
    // Chunk lane + 32 i of a run's codes lies on key lane / chunks + i * 32 / chunks; the swizzle repeats every 8 keys.
    constexpr int copies = 16 * chunks / 32, copy_keys = 32 / chunks;
    unsigned copy_to[D == 256 ? 2 : 1];  // in a slot, of copy i modulo their number; others lie 8 keys on
#pragma unroll
    for (int i = 0; i < static_cast<int>(sizeof(copy_to) / 4); ++i) {
        const int k = lane / chunks + i * copy_keys;
        copy_to[i] = ring_base + k * row_bytes + ((lane % chunks) ^ swizzle<D>(k & 7)) * 16;
    }
    const std::uint8_t* const key_source = cache.key_codes + lane * 16;
    const std::uint8_t* const value_source = cache.value_codes + lane * 16;
    const std::uint8_t* const scale_source = lane < 4 * groups
        ? reinterpret_cast<const std::uint8_t*>(cache.key_scales) + lane * 16
        : reinterpret_cast<const std::uint8_t*>(cache.value_scales) + (lane - 4 * groups) * 16;
    const unsigned scale_to = ring_base + 16 * D + lane * 16;
    const unsigned page_runs = static_cast<unsigned>(cache.page_size) / 16;

    // ---- pieces of segments: the copies and queries of the next one are on their way while one is joined ----
    Piece feed;  // the piece whose copies go on
    auto advance = [&] {
        while (at < stop) {
            while (at >= sequence_start + share.blocks * span_of(share) * cache.kv_heads) {
                sequence_start += share.blocks * span_of(share) * cache.kv_heads;
                share = share_at(++sequence);
            }
            const int span = span_of(share), segment = (at - sequence_start) / span;
            feed.segment_start = sequence_start + segment * span;
            feed.segment_end = feed.segment_start + span;
            feed.kv_head = segment / share.blocks;
            feed.first_unit = whole ? 0 : max(0, at - feed.segment_start - lead);
            feed.last_unit = whole ? share.units : min(stop - feed.segment_start, span) - lead;
            feed.complete = feed.first_unit == 0 && feed.last_unit == share.units;
            at = feed.segment_start + min(stop - feed.segment_start, span);
            if (feed.last_unit <= feed.first_unit) continue;  // the lead alone: the next block has the first unit
            feed.first = share.first, feed.before = share.length - share.count;
            feed.first_row = (segment - feed.kv_head * share.blocks) * rows;
            feed.total_rows = share.count * work.ratio;
            feed.used_rows = min(rows, feed.total_rows - feed.first_row);
            // keys that the block's first and last row see
            feed.visible_first = max(0, feed.before + static_cast<int>(divide(feed.first_row, work.by_ratio)) + 1);
            feed.visible_last =
                max(0, feed.before + static_cast<int>(divide(feed.first_row + feed.used_rows - 1, work.by_ratio)) + 1);
            feed.end = min(feed.visible_last, feed.last_unit * unit);
            feed.begin = feed.first_unit * unit + 16 * H * warp;
            feed.steps = feed.end > feed.begin ? (feed.end - feed.begin + unit - 1) / unit : 0;
            feed.table = a.page_table + sequence * a.table_stride;
            return true;
        }
        return false;
    };
    // The ring: step k of this warp takes places begin + k * unit .. + 16 H - 1, H runs of 16.
    int ahead = 0;     // lane l: where run l of the next 32 to copy lies, in runs of 16 places; -1 without a page
    unsigned bad = 0;  // bits: runs of the ring without a page, or past the end
    auto look_ahead = [&](int step) {
        const int place = feed.begin + (step + lane / H) * unit + lane % H * 16;
        ahead = -1;
        if (place >= feed.end) return;
        const unsigned index = static_cast<unsigned>(place) / 16;
        const unsigned column = divide(index, work.runs_per_page);
        const int page = feed.table[column];
        const bool good = page >= 0 && page < cache.pages;
        if (!good) note(cache, status_page);
        if (good) ahead = static_cast<int>((page * cache.kv_heads + feed.kv_head) * page_runs + (index - column * page_runs));
    };
    auto issue = [&](int step, int slot) {
        if (step < feed.steps) {
            if (step % (32 / H) == 0) look_ahead(step);
#pragma unroll
            for (int h = 0; h < H; ++h) {
                const int place = __shfl_sync(0xffffffffu, ahead, step % (32 / H) * H + h);
                const unsigned bit = 1u << (slot * H + h);
                bad = place < 0 ? bad | bit : bad & ~bit;
                if (place >= 0) {
                    const unsigned slot_at = slot * slot_bytes + h * run_bytes<D, G>;
                    const std::uint8_t* keys = key_source + static_cast<std::int64_t>(place) * (16 * row_bytes);
                    const std::uint8_t* values = value_source + static_cast<std::int64_t>(place) * (16 * row_bytes);
#pragma unroll
                    for (int i = 0; i < copies; ++i) {
                        constexpr int kinds = sizeof(copy_to) / 4;
                        const unsigned in_slot = copy_to[i % kinds] + slot_at + i / kinds * kinds * copy_keys * row_bytes;
                        copy_async(in_slot, keys + i * 512);
                        copy_async(in_slot + 16 * row_bytes, values + i * 512);
                    }
                    if (lane < 8 * groups) {
                        copy_async(scale_to + slot_at, scale_source + static_cast<std::int64_t>(place) * (64 * groups));
                    }
                }
            }
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    constexpr int per_lane = D / 32;  // channels lane * per_lane .. of a row of the queries
    constexpr int own_rows = (rows + warps - 1) / warps;
    alignas(16) T query_raw[own_rows][per_lane];  // this warp's rows, w and w + warps
    auto start = [&] {
#pragma unroll
        for (int n = 0; n < own_rows; ++n) {
            const int row = min(feed.first_row + warps * n + warp, feed.total_rows - 1);
            const int token = static_cast<int>(divide(row, work.by_ratio));
            const T* source = static_cast<const T*>(a.queries) + static_cast<std::int64_t>(feed.first + token) * a.query_stride +
                static_cast<std::int64_t>(feed.kv_head * work.ratio + row - token * work.ratio) * a.query_head_stride +
                lane * per_lane;
            if (!work.aligned) {
#pragma unroll
                for (int i = 0; i < per_lane; ++i) query_raw[n][i] = source[i];
            } else if constexpr (per_lane == 8) {
                *reinterpret_cast<uint4*>(query_raw[n]) = *reinterpret_cast<const uint4*>(source);
            } else if constexpr (per_lane == 4) {
                *reinterpret_cast<uint2*>(query_raw[n]) = *reinterpret_cast<const uint2*>(source);
            } else {
                *reinterpret_cast<unsigned*>(query_raw[n]) = *reinterpret_cast<const unsigned*>(source);
            }
        }
#pragma unroll
        for (int s = 0; s < ring - 1; ++s) issue(s, s);
    };
    if (!advance()) return;
    start();
    for (;;) {
        const Piece now = feed;
        // ---- the queries: each warp prepares its rows, every warp then reads all of them as fragments ----
#pragma unroll
        for (int n = 0; n < own_rows; ++n) {
            const int in_block = warps * n + warp;
            if (in_block >= rows) break;
            const bool used = now.first_row + in_block < now.total_rows;
            float q[per_lane];
#pragma unroll
            for (int i = 0; i < per_lane; ++i) q[i] = used ? widen(query_raw[n][i]) : 0.0f;
            float largest = 0.0f;
#pragma unroll
            for (int i = 0; i < per_lane; ++i) largest = max_nan(largest, fabsf(q[i]));
            // as bits: a NaN's are above every number's
            const unsigned bits = __reduce_max_sync(0xffffffffu, __float_as_uint(largest) & 0x7fffffffu);
            // below 2^13 after the scaling; a row below 2^-114 keeps the factor of that size
            const int exponent = max(13, static_cast<int>(bits >> 23));
            const float up = __uint_as_float(static_cast<unsigned>(266 - exponent) << 23);
            float sum = 0.0f;
#pragma unroll
            for (int i = 0; i < per_lane; ++i) {
                const float v = q[i] * up;
                sum += v;
                // channel 8 w + i of the G / 4 that lane j takes of a group: the even places of a word hold c 2^-24, the
                // odd ones c 2^-20; places i and i + 4 are one fragment register
                const int channel = lane * per_lane + i, g = channel / G, in_group = channel % G;
                const int to_j = in_group / (G / 4), w = in_group % (G / 4) / 8, at_place = in_group % 8;
                const int odd = at_place & 1, reg = at_place >> 1 & 1, high = at_place >> 2;
                joint_query[in_block / 8][((g * words + w) * 32 + in_block % 8 * 4 + to_j) * 8 + odd * 4 + reg * 2 + high] =
                    __float2half_rn(odd ? v * 0.0625f : v);
            }
#pragma unroll
            for (int offset = 1; offset < G / per_lane; offset *= 2) sum += __shfl_xor_sync(0xffffffffu, sum, offset);
            // the codes' 2^-24 goes into the group's sum as well
            if (lane % (G / per_lane) == 0) joint_query_sum[in_block][lane / (G / per_lane)] = sum * 0x1p-24f;
            if (lane == 0) {
                joint_factor[in_block] =
                    __uint_as_float(static_cast<unsigned>(exponent - 12) << 23) * 0x1p24f * (a.scale * log2_e);
            }
        }
        __syncthreads();
        unsigned query[groups][words][2][2][NT];
        float query_sum[groups][NT][2], factor[NT][2];
        int visible[NT][2];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
#pragma unroll
            for (int g = 0; g < groups; ++g) {
#pragma unroll
                for (int w = 0; w < words; ++w) {
                    const uint4 raw = *reinterpret_cast<const uint4*>(&joint_query[n][((g * words + w) * 32 + lane) * 8]);
                    query[g][w][0][0][n] = raw.x, query[g][w][0][1][n] = raw.y;
                    query[g][w][1][0][n] = raw.z, query[g][w][1][1][n] = raw.w;
                }
                query_sum[g][n][0] = joint_query_sum[8 * n + 2 * j][g];
                query_sum[g][n][1] = joint_query_sum[8 * n + 2 * j + 1][g];
            }
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                factor[n][i] = joint_factor[8 * n + 2 * j + i];
                const int column = now.first_row + 8 * n + 2 * j + i;
                visible[n][i] = column < now.total_rows
                    ? now.before + static_cast<int>(divide(column, work.by_ratio)) + 1
                    : now.visible_last;
            }
        }

        // ---- one pass over the keys ----
        float top[NT][2], limit[NT][2], sum[NT][2], low[groups][NT][2], acc[groups][tiles][NT][4];
        float value_top[groups], value_factor[groups];
#pragma unroll
        for (int n = 0; n < NT; ++n) {
#pragma unroll
            for (int i = 0; i < 2; ++i) top[n][i] = limit[n][i] = -FLT_MAX, sum[n][i] = 0.0f;
        }
#pragma unroll
        for (int g = 0; g < groups; ++g) {
            value_top[g] = 0.0f, value_factor[g] = 1.0f;
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                low[g][n][0] = low[g][n][1] = 0.0f;
#pragma unroll
                for (int t = 0; t < tiles; ++t) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) acc[g][t][n][i] = 0.0f;
                }
            }
        }

        // A step's H runs of 16 keys. `edge`: some keys are hidden from some rows, or hold nothing (a bit of `absent`: a
        // whole run).
        auto process = [&](const std::uint8_t* slot_codes, int place, bool edge, unsigned absent) {
            float x[H][NT][4];
            auto scores = [&](int h) {
                const std::uint8_t* const codes = slot_codes + h * run_bytes<D, G>;
                const std::uint8_t* const key_scales = codes + 16 * D;
#pragma unroll
                for (int n = 0; n < NT; ++n) x[h][n][0] = x[h][n][1] = x[h][n][2] = x[h][n][3] = 0.0f;
#pragma unroll
                for (int g = 0; g < groups; ++g) {
                    unsigned near[words], far[words];
                    const std::uint8_t* from_key = codes + key_offset[g];
                    if constexpr (words == 4) {
                        *reinterpret_cast<uint4*>(near) = *reinterpret_cast<const uint4*>(from_key);
                        *reinterpret_cast<uint4*>(far) = *reinterpret_cast<const uint4*>(from_key + 8 * row_bytes);
                    } else if constexpr (words == 2) {
                        *reinterpret_cast<uint2*>(near) = *reinterpret_cast<const uint2*>(from_key);
                        *reinterpret_cast<uint2*>(far) = *reinterpret_cast<const uint2*>(from_key + 8 * row_bytes);
                    } else {
                        near[0] = *reinterpret_cast<const unsigned*>(from_key);
                        far[0] = *reinterpret_cast<const unsigned*>(from_key + 8 * row_bytes);
                    }
                    float dot[2][NT][4];  // of the even and of the odd places, two chains
#pragma unroll
                    for (int w = 0; w < words; ++w) {
                        const unsigned near8 = near[w] >> 8, far8 = far[w] >> 8;
                        const unsigned even[4] = {near[w] & 0x000f000fu, far[w] & 0x000f000fu, near8 & 0x000f000fu,
                                                  far8 & 0x000f000fu};
                        const unsigned odd[4] = {near[w] & 0x00f000f0u, far[w] & 0x00f000f0u, near8 & 0x00f000f0u,
                                                 far8 & 0x00f000f0u};
#pragma unroll
                        for (int n = 0; n < NT; ++n) {
                            if (w == 0) {
                                mma_from_zero(dot[0][n], even, query[g][w][0][0][n], query[g][w][0][1][n]);
                                mma_from_zero(dot[1][n], odd, query[g][w][1][0][n], query[g][w][1][1][n]);
                            } else {
                                mma(dot[0][n], even, query[g][w][0][0][n], query[g][w][0][1][n]);
                                mma(dot[1][n], odd, query[g][w][1][0][n], query[g][w][1][1][n]);
                            }
                        }
                    }
                    const float2 pair_near = pair_at(key_scales, (my_key * groups + g) * 4);
                    const float2 pair_far = pair_at(key_scales, ((my_key + 8) * groups + g) * 4);
#pragma unroll
                    for (int n = 0; n < NT; ++n) {
#pragma unroll
                        for (int i = 0; i < 2; ++i) {
                            x[h][n][i] = fmaf(pair_near.x, dot[0][n][i] + dot[1][n][i],
                                              fmaf(pair_near.y, query_sum[g][n][i], x[h][n][i]));
                            x[h][n][i + 2] = fmaf(pair_far.x, dot[0][n][i + 2] + dot[1][n][i + 2],
                                                  fmaf(pair_far.y, query_sum[g][n][i], x[h][n][i + 2]));
                        }
                    }
                }
#pragma unroll
                for (int n = 0; n < NT; ++n) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) x[h][n][i] *= factor[n][i & 1];
                }
            };
#pragma unroll
            for (int h = 0; h < H; ++h) scores(h);
            // Values' pairs (scale, minimum) of keys my_key and my_key + 8; places past the block's last visible key are no
            // one's, whatever they hold.
            auto value_pair = [&](int h, int far, int g) {
                const int key = my_key + 8 * far;
                float2 pair = pair_at(slot_codes + h * run_bytes<D, G> + 16 * D + 64 * groups, (key * groups + g) * 4);
                if (edge && ((absent >> h & 1u) != 0 || place + 16 * h + key >= now.end)) pair = {0.0f, 0.0f};
                return pair;
            };
            bool raise = false;
            float largest[groups];
#pragma unroll
            for (int g = 0; g < groups; ++g) {
                largest[g] = 0.0f;  // an infinite scale raises nothing
#pragma unroll
                for (int h = 0; h < H; ++h) {
#pragma unroll
                    for (int far = 0; far < 2; ++far) largest[g] = fmaxf(largest[g], fabsf(value_pair(h, far, g).x));
                }
                raise |= largest[g] > value_top[g];
            }
            if (edge) {
#pragma unroll
                for (int h = 0; h < H; ++h) {
                    const int last = (absent >> h & 1u) != 0 ? 0 : now.end - place - 16 * h;
#pragma unroll
                    for (int n = 0; n < NT; ++n) {
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const int key = my_key + (i & 2) * 4;
                            if (key >= last || place + 16 * h + key >= visible[n][i & 1]) x[h][n][i] = -INFINITY;
                        }
                    }
                }
            }
            float most_of[NT][2];
#pragma unroll
            for (int n = 0; n < NT; ++n) {
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    most_of[n][i] = fmaxf(x[0][n][i], x[0][n][i + 2]);
#pragma unroll
                    for (int h = 1; h < H; ++h) most_of[n][i] = fmaxf(most_of[n][i], fmaxf(x[h][n][i], x[h][n][i + 2]));
                    raise |= most_of[n][i] > limit[n][i];
                }
            }
            if (__any_sync(0xffffffffu, raise)) {
#pragma unroll
                for (int n = 0; n < NT; ++n) {
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        float most = most_of[n][i];
                        most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 4));
                        most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 8));
                        most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 16));
                        most = fmaxf(most, top[n][i]);
                        const float shrink = exp2_fast(top[n][i] - most);
                        top[n][i] = most;
                        limit[n][i] = most + top_slack;
                        sum[n][i] *= shrink;
#pragma unroll
                        for (int g = 0; g < groups; ++g) {
                            low[g][n][i] *= shrink;
#pragma unroll
                            for (int t = 0; t < tiles; ++t) acc[g][t][n][i] *= shrink, acc[g][t][n][i + 2] *= shrink;
                        }
                    }
                }
#pragma unroll
                for (int g = 0; g < groups; ++g) {
                    const float finite = largest[g] < INFINITY ? largest[g] : 0.0f;
                    const float most = __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(finite)));
                    if (most > value_top[g]) {  // the power of two above it becomes 2^6
                        const unsigned exponent = (__float_as_uint(most) >> 23) + 1;
                        value_top[g] = __uint_as_float(exponent << 23);
                        const float scaled = __uint_as_float((260u - exponent) << 23);
                        const float change = scaled / value_factor[g];
                        value_factor[g] = scaled;
#pragma unroll
                        for (int n = 0; n < NT; ++n) {
#pragma unroll
                            for (int t = 0; t < tiles; ++t) {
#pragma unroll
                                for (int i = 0; i < 4; ++i) acc[g][t][n][i] *= change;
                            }
                        }
                    }
                }
            }
            auto accumulate = [&](int h) {
                const std::uint8_t* const values = slot_codes + h * run_bytes<D, G> + 16 * row_bytes;
                float p[NT][4];
#pragma unroll
                for (int n = 0; n < NT; ++n) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) p[n][i] = exp2_fast(x[h][n][i] - top[n][i & 1]);
                    sum[n][0] += p[n][0] + p[n][2];
                    sum[n][1] += p[n][1] + p[n][3];
                }
#pragma unroll
                for (int g = 0; g < groups; ++g) {
                    unsigned b[NT][2];
                    const float2 near_pair = value_pair(h, 0, g), far_pair = value_pair(h, 1, g);
                    const float near_scale = near_pair.x * value_factor[g], far_scale = far_pair.x * value_factor[g];
                    const float near_middle = fmaf(8.0f, near_pair.x, near_pair.y);
                    const float far_middle = fmaf(8.0f, far_pair.x, far_pair.y);
#pragma unroll
                    for (int n = 0; n < NT; ++n) {
                        float w[4], m[4];
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            w[i] = p[n][i] * (i < 2 ? near_scale : far_scale);
                            m[i] = i < 2 ? near_middle : far_middle;
                        }
                        if (edge) {  // a hidden key's weight is 0 even against a scale that is no number
#pragma unroll
                            for (int i = 0; i < 4; ++i) {
                                if (x[h][n][i] == -INFINITY) w[i] = m[i] = 0.0f;
                            }
                        }
                        low[g][n][0] = fmaf(p[n][0], m[0], fmaf(p[n][2], m[2], low[g][n][0]));
                        low[g][n][1] = fmaf(p[n][1], m[1], fmaf(p[n][3], m[3], low[g][n][1]));
                        b[n][0] = transpose8x8(pack_half(w[0], w[1]));
                        b[n][1] = transpose8x8(pack_half(w[2], w[3]));
                    }
                    // the lane's channels of four keys: 4 codes of each (halves), 8 (a word) or 16 (two words)
                    constexpr int value_words = G == 128 ? 2 : 1;
                    unsigned code[4][value_words];
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        const std::uint8_t* from_value = values + value_offset[g][k & 1] + (k & 2) * 4 * row_bytes;
                        if constexpr (G == 128) {
                            *reinterpret_cast<uint2*>(code[k]) = *reinterpret_cast<const uint2*>(from_value);
                        } else if constexpr (G == 64) {
                            code[k][0] = *reinterpret_cast<const unsigned*>(from_value);
                        } else {
                            code[k][0] = *reinterpret_cast<const std::uint16_t*>(from_value);
                        }
                    }
#pragma unroll
                    for (int t = 0; t < tiles; t += 2) {
                        const int w = t / 4;
                        const unsigned select = t % 4 == 0 ? 0x5410u : 0x7632u;
                        const unsigned one = __byte_perm(code[0][w], code[1][w], select);
                        const unsigned two = __byte_perm(code[2][w], code[3][w], select);
                        const unsigned front[4] = {even_codes(one), odd_codes(one), even_codes(two), odd_codes(two)};
                        const unsigned back[4] = {even_codes(one >> 8), odd_codes(one >> 8), even_codes(two >> 8),
                                                  odd_codes(two >> 8)};
#pragma unroll
                        for (int n = 0; n < NT; ++n) {
                            mma(acc[g][t][n], front, b[n][0], b[n][1]);
                            mma(acc[g][t + 1][n], back, b[n][0], b[n][1]);
                        }
                    }
                }
            };
#pragma unroll
            for (int h = 0; h < H; ++h) accumulate(h);
        };

        const int edge_from = min(now.visible_first, now.end) - 16 * H;  // steps that start after it have an edge
        for (int step = 0, slot = 0; step < now.steps; ++step) {
            asm volatile("cp.async.wait_group %0;" ::"n"(ring - 2) : "memory");
            __syncwarp();  // every lane's copies are here, and every lane is done with the slot before this one
            issue(step + ring - 1, slot == 0 ? ring - 1 : slot - 1);
            const int place = now.begin + step * unit;
            const unsigned absent = bad >> (slot * H) & ((1u << H) - 1u);
            process(ring_bytes + slot * slot_bytes, place, absent != 0 || place > edge_from, absent);
            slot = slot + 1 == ring ? 0 : slot + 1;
        }
        asm volatile("cp.async.wait_group 0;" ::: "memory");
        __syncwarp();  // every lane is done with the ring
        const bool another = advance();
        if (another) start();

        // ---- join the warps ----
        constexpr int pitch = D + 4;
        float* const outs = reinterpret_cast<float*>(shared + warps * ring * slot_bytes);  // [warp][row][pitch]
#pragma unroll
        for (int n = 0; n < NT; ++n) {
#pragma unroll
            for (int i = 0; i < 2; ++i) {
#pragma unroll
                for (int offset = 4; offset < 32; offset *= 2) {
                    sum[n][i] += __shfl_xor_sync(0xffffffffu, sum[n][i], offset);
                }
                if (r == 0) {
                    joint_top[warp][8 * n + 2 * j + i] = top[n][i];
                    joint_sum[warp][8 * n + 2 * j + i] = sum[n][i];
                }
            }
        }
#pragma unroll
        for (int g = 0; g < groups; ++g) {
            const float unscale = 1.0f / value_factor[g];
#pragma unroll
            for (int n = 0; n < NT; ++n) {
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    float m = low[g][n][i];
#pragma unroll
                    for (int offset = 4; offset < 32; offset *= 2) m += __shfl_xor_sync(0xffffffffu, m, offset);
                    float* row = outs + (warp * rows + 8 * n + 2 * j + i) * pitch + g * G + r * (G / 8);
#pragma unroll
                    for (int t = 0; t < tiles; ++t) {
                        const float2 o = {fmaf(acc[g][t][n][i], unscale, m), fmaf(acc[g][t][n][i + 2], unscale, m)};
                        *reinterpret_cast<float2*>(row + 2 * t) = o;
                    }
                }
            }
        }
        __syncthreads();
        auto store = [&](int row, int d, float4 value, float whole) {
            const int at_row = now.first_row + row, token = static_cast<int>(divide(at_row, work.by_ratio));
            const float inverse = whole == 0.0f ? 0.0f : 1.0f / whole;
            T* to = static_cast<T*>(a.output) +
                (static_cast<std::int64_t>(now.first + token) * a.heads + now.kv_head * work.ratio + at_row - token * work.ratio) * D + d;
            alignas(8) T out[4] = {narrow<T>(value.x * inverse), narrow<T>(value.y * inverse), narrow<T>(value.z * inverse),
                                   narrow<T>(value.w * inverse)};
            *reinterpret_cast<uint2*>(to) = *reinterpret_cast<const uint2*>(out);
        };
        const int begin_block = now.complete ? 0 : block_of(now.segment_start + lead);
        float* const part = work.partials +
            (2 * static_cast<std::int64_t>(blockIdx.x) + (static_cast<int>(blockIdx.x) == begin_block)) * partial_floats;
        const int quads = now.used_rows * (D / 4);
        for (int e = threadIdx.x; e < quads; e += 32 * warps) {
            const int row = e / (D / 4), d = e % (D / 4) * 4;
            float most = -FLT_MAX, whole = 0.0f;
            float4 value = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int w = 0; w < warps; ++w) most = fmaxf(most, joint_top[w][row]);
#pragma unroll
            for (int w = 0; w < warps; ++w) {
                const float weight = exp2_fast(joint_top[w][row] - most);
                const float4 o = *reinterpret_cast<const float4*>(outs + (w * rows + row) * pitch + d);
                whole = fmaf(joint_sum[w][row], weight, whole);
                value.x = fmaf(o.x, weight, value.x), value.y = fmaf(o.y, weight, value.y);
                value.z = fmaf(o.z, weight, value.z), value.w = fmaf(o.w, weight, value.w);
            }
            if (now.complete) {
                store(row, d, value, whole);
            } else {
                *reinterpret_cast<float4*>(part + row * D + d) = value;
                if (d == 0) part[rows * D + row] = most, part[rows * D + rows + row] = whole;
            }
        }

        // ---- join the blocks of a segment: the last of them to get here ----
        if (!now.complete) {
            const int pieces = block_of(now.segment_end - 1) - begin_block + 1;
            __syncthreads();
            if (threadIdx.x == 0) {  // releases the block's sums, and acquires the others'
                unsigned before_me;
                asm volatile("atom.acq_rel.gpu.global.add.u32 %0, [%1], 1;"
                             : "=r"(before_me)
                             : "l"(work.tickets + begin_block)
                             : "memory");
                joint_last = before_me + 1 == static_cast<unsigned>(pieces);
                if (joint_last) work.tickets[begin_block] = 0;
            }
            __syncthreads();
            if (joint_last) {
                auto part_of = [&](int piece) {
                    return work.partials +
                        (2 * static_cast<std::int64_t>(begin_block + piece) + (piece == 0)) * partial_floats;
                };
                float* const weights = outs;                         // [piece][row]
                float* const totals = weights + most_blocks * rows;       // [piece][row]
                float4* const sums = reinterpret_cast<float4*>(totals + most_blocks * rows);
                const int shares = max(1, 32 * warps / quads);  // threads that divide one quad's pieces
                const int quad = shares > 1 ? static_cast<int>(threadIdx.x) % quads : static_cast<int>(threadIdx.x);
                const int mine_of = shares > 1 ? static_cast<int>(threadIdx.x) / quads : 0;
                constexpr int early = 4;  // pieces on their way before the weights are known
                float4 first_sums[early];
#pragma unroll
                for (int k = 0; k < early; ++k) {
                    const int piece = mine_of + k * shares;
                    if (quad < quads && mine_of < shares && piece < pieces) {
                        first_sums[k] = __ldcg(reinterpret_cast<const float4*>(part_of(piece) + quad * 4));
                    }
                }
                for (int e = threadIdx.x; e < pieces * rows; e += 32 * warps) {
                    if (e % rows < now.used_rows) {
                        const float* const one = part_of(e / rows) + rows * D + e % rows;
                        weights[e] = __ldcg(one), totals[e] = __ldcg(one + rows);
                    }
                }
                __syncthreads();
                for (int row = warp; row < now.used_rows; row += warps) {
                    float most = -FLT_MAX, whole_sum = 0.0f;
                    for (int piece = lane; piece < pieces; piece += 32) most = fmaxf(most, weights[piece * rows + row]);
#pragma unroll
                    for (int offset = 16; offset > 0; offset /= 2) {
                        most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, offset));
                    }
                    for (int piece = lane; piece < pieces; piece += 32) {
                        const float weight = exp2_fast(weights[piece * rows + row] - most);
                        weights[piece * rows + row] = weight;
                        whole_sum = fmaf(totals[piece * rows + row], weight, whole_sum);
                    }
                    whole_sum = warp_sum(whole_sum);
                    if (lane == 0) joint_sum[0][row] = whole_sum;
                }
                __syncthreads();
                for (int base = 0; base < quads; base += 32 * warps) {
                    const int e = base + quad, row = e / (D / 4), d = e % (D / 4) * 4;
                    float4 value = {0.0f, 0.0f, 0.0f, 0.0f};
                    auto add = [&](const float4& o, int piece) {
                        const float weight = weights[piece * rows + row];
                        value.x = fmaf(o.x, weight, value.x), value.y = fmaf(o.y, weight, value.y);
                        value.z = fmaf(o.z, weight, value.z), value.w = fmaf(o.w, weight, value.w);
                    };
                    if (e < quads && mine_of < shares) {
                        int piece = mine_of;
                        if (base == 0) {
#pragma unroll
                            for (int k = 0; k < early; ++k) {
                                if (piece < pieces) add(first_sums[k], piece);
                                piece += shares;
                            }
                        }
#pragma unroll 8
                        for (; piece < pieces; piece += shares) {
                            add(__ldcg(reinterpret_cast<const float4*>(part_of(piece) + row * D + d)), piece);
                        }
                    }
                    if (shares > 1) {
                        sums[threadIdx.x] = value;
                        __syncthreads();
                        for (int s = 1; s < shares && mine_of == 0; ++s) {
                            const float4 o = sums[threadIdx.x + s * quads];
                            value.x += o.x, value.y += o.y, value.z += o.z, value.w += o.w;
                        }
                    }
                    if (e < quads && mine_of == 0) store(row, d, value, joint_sum[0][row]);
                }
            }
        }
        if (!another) return;
    }
}

template <typename T, int D, int G, int NT>
cudaError_t launch(Work& work, cudaStream_t stream) {
    constexpr int bytes = shared_bytes<D, G, NT>;
    static_assert(warps * 8 * NT * (D + 4) * 4 >= 2 * most_blocks * 8 * NT * 4 + 32 * warps * 16, "the blocks' join fits");
    static SharedAllowance allowance;
    const cudaError_t allowed = allowance.allow(attend_kernel<T, D, G, NT>, bytes);
    if (allowed != cudaSuccess) return allowed;
    // the blocks that run at once, and no more than there can be units
    constexpr int unit = 16 * together<D, NT> * warps;
    const std::int64_t rows = static_cast<std::int64_t>(work.a.max_queries) * work.ratio;
    const std::int64_t segments = static_cast<std::int64_t>(work.a.batch) * work.cache.kv_heads * ((rows + 8 * NT - 1) / (8 * NT));
    const std::int64_t most = 0x7fffffff, each = std::max(1, (work.a.max_length + unit - 1) / unit);  // the kernel's are 32 bits
    constexpr int lead_units = (lead_keys + unit - 1) / unit;
    if (segments > most || segments * (each + lead_units) > most) return cudaErrorInvalidValue;
    const std::int64_t units = segments * each;
    const std::int64_t grid = std::min<std::int64_t>(std::min(sm_count(), most_blocks), units);
    return kernels::launch_overlapped(attend_kernel<T, D, G, NT>, dim3(static_cast<unsigned>(grid)), dim3(32 * warps), bytes,
                                      stream, static_cast<const Work&>(work));
}

template <typename T, int D, int G>
cudaError_t launch_rows(Work& work, cudaStream_t stream) {
    // Segments of 16 rows read the cache once for twice the rows, of 8 rows take two runs at a time and have a shorter
    // chain: 8 while each such segment has an SM of its own. Heads of 128, 8 cache heads, 16 rows each, 1024 keys, us
    // with 16 rows and with 8: one sequence (16 segments of 8) 14.7, 10.1; 8 sequences (128) 15.1, 10.3; 12 (192) 15.2,
    // 18.1; 32 (512) 28.2, 33.9. 4096 keys: 15.4, 11.9; 28.5, 27.7; 44.2, 41.9; 84.2, 97.9. The rule's worst: 2 cache
    // heads, 12 sequences of 4096 keys (48) 23.0, 28.0. With heads of 256 channels 16 rows' sums do not fit the registers.
    if constexpr (D < 256) {
        const std::int64_t rows = static_cast<std::int64_t>(work.a.max_queries) * work.ratio;
        const std::int64_t eights = static_cast<std::int64_t>(work.a.batch) * work.cache.kv_heads * ((rows + 7) / 8);
        if (rows > 8 && eights > sm_count()) return launch<T, D, G, 2>(work, stream);
    }
    return launch<T, D, G, 1>(work, stream);
}

template <typename T>
cudaError_t launch_shape(Work& work, cudaStream_t stream) {
    const int d = work.cache.head_dim, g = work.cache.group;
    if (d == 64) return g == 32 ? launch_rows<T, 64, 32>(work, stream) : launch_rows<T, 64, 64>(work, stream);
    if (d == 128) {
        return g == 32 ? launch_rows<T, 128, 32>(work, stream)
            : g == 64  ? launch_rows<T, 128, 64>(work, stream)
                       : launch_rows<T, 128, 128>(work, stream);
    }
    return g == 64 ? launch_rows<T, 256, 64>(work, stream) : launch_rows<T, 256, 128>(work, stream);
}

}  // namespace

std::size_t attend_partial_bytes() {
    return static_cast<std::size_t>(most_blocks) * 2 * std::max(16 * (128 + 2), 8 * (256 + 2)) * sizeof(float);
}

std::size_t attend_ticket_bytes() { return most_blocks * sizeof(unsigned); }

cudaError_t attend(const Cache& cache, const AttendArgs& args, const AttendWorkspace& workspace, cudaStream_t stream) {
    if (args.tokens == 0) return cudaSuccess;
    if (args.batch == 0) {
        const std::size_t values = static_cast<std::size_t>(args.tokens) * static_cast<std::size_t>(args.heads) *
            static_cast<std::size_t>(cache.head_dim);
        return cudaMemsetAsync(args.output, 0, values * 2, stream);
    }
    Work work{};
    work.cache = cache;
    work.a = args;
    work.ratio = args.heads / cache.kv_heads;
    work.runs_per_page = divisor(static_cast<unsigned>(cache.page_size / 16));
    work.by_ratio = divisor(static_cast<unsigned>(work.ratio));
    work.partials = workspace.partials;
    work.tickets = workspace.tickets;
    work.aligned = reinterpret_cast<std::uintptr_t>(args.queries) % 16 == 0 && args.query_stride % 8 == 0 &&
        args.query_head_stride % 8 == 0;
    return args.type == Type::f16 ? launch_shape<__half>(work, stream) : launch_shape<__nv_bfloat16>(work, stream);
}

}  // namespace nvcr_sm100::token
