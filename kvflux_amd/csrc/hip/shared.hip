// Decode attention of a batch whose rows share long prefixes, each prefix
// computed once for all of its rows.
//
// Row r of group g attends to the group's P_g first tokens and to its own
// tokens [P_g, len_r): with scores s = q . k / sqrt(D) over both,
//   o_r = sum_t exp(s_t - m) v_t / sum_t exp(s_t - m),
// and a softmax over a union is the merge of (m, sum, weighted sum) over its
// parts. So the work is a list of streams, one or more for each segment: a
// segment is a group's prefix (its columns are the query heads of all its
// rows) or a row's own tokens (its columns are that row's heads), a stream is
// one kv head and up to kCols columns of a segment, walked over the segment's
// tokens in tiles. Every tile has a cost, and workgroup w of N takes the tiles
// whose place in the sum of all costs T lies in [wT/N, (w+1)T/N): whole streams
// and parts of them, so any mix of long and short segments is spread evenly
// and compute-bound prefix tiles run beside memory-bound own ones. Each part
// leaves partials (m, sum, weighted sum) that a second kernel merges.
//
// A tile is 32 KiB of K and 32 KiB of V, loaded straight into LDS (two
// buffers; the next tile's loads are in flight while this one is computed). A
// wavefront owns 16 columns and a share of the tile's tokens: all of them with
// 8 blocks of columns, fewer where there are fewer blocks, merged through LDS
// at a part's end.
//   S^T = K Q^T, O^T += V^T P^T  on v_mfma_f32_16x16x32 with Q (scale folded
// in) and the weights as three 16-bit parts each: products exact in FP32, sums
// FP32. FP32 caches: v_mfma_f32_16x16x4_f32 on the values as they are.
#include "mfma_parts.h"

#include <cmath>
#include <type_traits>

namespace kvflux_hip {
namespace {

struct ShF32 {};

constexpr int kThreads = 512;  // 8 wavefronts, two per SIMD
constexpr int kWaves = kThreads / 64;
constexpr std::uint32_t kCols = 128;        // columns of a stream: 16 a wavefront
constexpr std::uint32_t kWorkgroups = 256;  // one per CU (two tiles fill its LDS)
constexpr std::uint32_t kMaxRows = 4096;    // rows and groups whose costs are summed in LDS
constexpr std::uint32_t kMaxGroups = 512;
constexpr int kBufferBytes = 65536;         // K and V of a tile

template <typename E, int kD>
struct Shape {
    static constexpr bool kF32 = std::is_same<E, ShF32>::value;
    static constexpr int kRowBytes = kD * (kF32 ? 4 : 2);
    static constexpr int kCpr = kRowBytes / 16;                  // 16-byte chunks of a token's row
    static constexpr std::uint32_t kTile = kBufferBytes / 2 / kRowBytes;  // tokens
    static constexpr std::uint32_t kStep = kF32 ? 16 : 32;       // tokens of a wavefront's step
    static constexpr std::uint32_t kSteps = kTile / kStep;
    // The fewest blocks of columns a tile's wavefronts are laid out for: with
    // fewer, they would not have a step each.
    static constexpr std::uint32_t kLeastBlocks = kSteps >= kWaves ? 1 : kWaves / kSteps;
    static constexpr int kLoads = kBufferBytes / 2 / (kThreads * 16);  // loads of a thread, K and V each
};

// Blocks of 16 columns that the wavefronts are laid out for (a power of two);
// kWaves / it groups of wavefronts share a tile's tokens.
__host__ __device__ inline std::uint32_t layout_blocks(std::uint32_t blocks, std::uint32_t least) {
    std::uint32_t n = least;
    while (n < blocks) n *= 2;
    return n < kWaves ? n : kWaves;
}

struct SharedParams {
    const void* key_cache;
    const void* value_cache;
    std::uint64_t num_blocks;
    std::uint32_t heads;   // kv heads
    FastDiv block_size;
    const std::uint64_t* table;  // [rows][width]
    std::uint64_t width;
    const std::uint64_t* lens;   // [rows]
    std::uint32_t kv_len;        // bound of every length, at most width * block_size
    std::uint32_t rows;
    std::uint32_t query_heads;
    FastDiv group;               // query heads per kv head
    const std::uint64_t* starts; // [groups + 1]
    const std::uint64_t* prefixes;  // [groups]
    std::uint32_t groups;
    std::uint32_t max_prefix;    // bound of every prefix
    const float* query;
    float* output;
    float scale_log2;            // log2(e) / sqrt(D)
    // Workspace: total cost and the rows' plans for the merge, partials.
    std::uint64_t* total;
    struct RowPlan* plans;
    float* prefix_acc;  // [slot][kCols][D]
    float* prefix_ml;   // [slot][kCols][2]
    float* row_acc;     // [slot][row_cols][D]
    float* row_ml;      // [slot][row_cols][2]
    std::uint32_t row_cols;   // min(group, kCols)
    std::uint32_t row_tiles;  // ceil(group / kCols): streams of a row for each kv head
};

// What the merge needs of a row.
struct RowPlan {
    std::uint64_t prefix_cost, own_cost;  // costs before the segments
    std::uint32_t prefix_tiles, prefix_weight, prefix_col_tiles, prefix_stream;
    std::uint32_t first_row, own_tiles, own_weight, len;
};

// A segment: the columns (of row first_row on), the tokens [begin, end) of
// table row first_row, its tiles and the cost of one.
struct Segment {
    std::uint32_t first_row, cols, col_tiles, begin, end, tiles, weight;
    __device__ std::uint64_t stream_cost() const { return static_cast<std::uint64_t>(tiles) * weight; }
    __device__ std::uint64_t cost(std::uint32_t heads) const { return stream_cost() * (heads * col_tiles); }
};

// Cost of a tile by its layout's blocks of columns.
template <typename E, int kD>
__device__ inline std::uint32_t tile_weight(std::uint32_t cols) {
    const std::uint32_t blocks = layout_blocks((cols + 15) / 16, Shape<E, kD>::kLeastBlocks);
    return blocks < kWaves ? 1u : 2u;
}

template <typename E, int kD>
__device__ inline Segment make_segment(std::uint32_t first_row, std::uint32_t cols, std::uint32_t begin, std::uint32_t end) {
    constexpr std::uint32_t kTile = Shape<E, kD>::kTile;
    Segment s{first_row, cols, (cols + kCols - 1) / kCols, begin, end, 0, 1};
    s.tiles = end > begin ? (end - begin - 1) / kTile + 1 : 0;
    s.weight = tile_weight<E, kD>(cols < kCols ? cols : kCols);
    return s;
}

// Group of a row: the last whose first row is not behind it (rows past the
// last group's end, or before the first group's start: none).
__device__ inline std::uint32_t group_of(const std::uint32_t* first, std::uint32_t groups, std::uint32_t row) {
    std::uint32_t lo = 0, hi = groups;
    while (hi - lo > 1) {
        const std::uint32_t mid = (lo + hi) / 2;
        if (first[mid] <= row) lo = mid;
        else hi = mid;
    }
    return first[lo] <= row && row < first[lo + 1] ? lo : groups;
}

// Stream numbers before a group's: every group may end in a started tile of
// columns, so group + floor(columns of the rows before it / kCols).
__device__ inline std::uint32_t group_stream(const SharedParams& p, std::uint32_t g, std::uint32_t first_row) {
    return (g + first_row * p.group.divisor / kCols) * p.heads;
}

__device__ inline std::uint64_t share_begin(std::uint64_t total, std::uint32_t w) {
    return (total * w + kWorkgroups - 1) / kWorkgroups;
}

// exp2(m - top) for merging partials: 0 for a part that saw no key.
__device__ inline float merge_weight(float m, float top) {
    return m == -INFINITY ? 0.0f : m == top ? 1.0f : __builtin_amdgcn_exp2f(m - top);
}

__device__ __attribute__((aligned(16))) unsigned char sh_zero_row[512];

template <typename E, int kD>
__global__ __launch_bounds__(kThreads) void shared_attention_kernel(SharedParams p) {
    using S = Shape<E, kD>;
    constexpr bool kF32 = S::kF32;
    using M = typename std::conditional<kF32, PfBf16Exact, E>::type;
    using Vec = typename M::Vec;
    constexpr std::uint32_t kTile = S::kTile, kStep = S::kStep;
    constexpr int kRowBytes = S::kRowBytes, kCpr = S::kCpr, kLoads = S::kLoads;
    constexpr int kKk = kD / 32;   // 16-bit: K steps of S^T
    constexpr int kDt = kD / 16;   // accumulator tiles of O^T
    constexpr float kWeightScale = kF32 ? 1.0f : M::kWeightScale;
    constexpr float kLazy = kF32 ? 8.0f : M::kLazyLog2;

    __shared__ __attribute__((aligned(16))) unsigned char buffers[2][kBufferBytes];
    __shared__ std::uint32_t first_of[kMaxGroups + 1];  // first row of a group, and the end
    __shared__ std::uint32_t prefix_of[kMaxGroups];     // its shared tokens (0: fewer than two rows, or past the bound)
    __shared__ float2 part_ml[kWaves][16];
    __shared__ std::uint32_t bad_tile[2];               // the serial number of a tile with a missing page
    __shared__ std::uint32_t found;

    const int tid = threadIdx.x, wave = tid / 64, lane = tid % 64;
    const int col = lane % 16, quad = lane / 16;
    const auto uniform = [](std::uint32_t x) {
        return static_cast<std::uint32_t>(__builtin_amdgcn_readfirstlane(static_cast<int>(x)));
    };
    const auto uniform64 = [&](std::uint64_t x) {
        return static_cast<std::uint64_t>(uniform(static_cast<std::uint32_t>(x >> 32))) << 32 |
               uniform(static_cast<std::uint32_t>(x));
    };

    // ---- plan: the groups (starts made monotone, whatever the caller gave),
    // then the sum of costs over all segments: groups first, then rows.
    if (wave == 0) {
        std::uint32_t carry = 0;
        for (std::uint32_t base = 0; base <= p.groups; base += 64) {
            const std::uint32_t g = base + lane;
            std::uint32_t v = 0;
            if (g <= p.groups) {
                const std::uint64_t s = p.starts[g];
                v = s < p.rows ? static_cast<std::uint32_t>(s) : p.rows;
            }
#pragma unroll
            for (int off = 1; off < 64; off <<= 1) {
                const auto o = static_cast<std::uint32_t>(__shfl_up(static_cast<int>(v), off));
                if (lane >= off && o > v) v = o;
            }
            v = v > carry ? v : carry;
            if (g <= p.groups) first_of[g] = v;
            carry = static_cast<std::uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(v), 63));
        }
    }
    if (tid < 2) bad_tile[tid] = 0;
    __syncthreads();
    for (std::uint32_t g = tid; g < p.groups; g += kThreads) {
        const std::uint64_t n = p.prefixes[g];
        prefix_of[g] = first_of[g + 1] - first_of[g] >= 2 && n <= p.max_prefix ? static_cast<std::uint32_t>(n) : 0u;
    }
    __syncthreads();
    const auto group_segment = [&](std::uint32_t g) {
        return make_segment<E, kD>(first_of[g], (first_of[g + 1] - first_of[g]) * p.group.divisor, 0, prefix_of[g]);
    };
    // A row shorter than its group's prefix takes no part in it.
    const auto row_segment = [&](std::uint32_t r, std::uint32_t* group) {
        const std::uint64_t full = p.lens[r];
        const std::uint32_t len = full < p.kv_len ? static_cast<std::uint32_t>(full) : p.kv_len;
        const std::uint32_t g = group_of(first_of, p.groups, r);
        const std::uint32_t shared = g < p.groups && prefix_of[g] <= len ? prefix_of[g] : 0u;
        if (group) *group = shared ? g : p.groups;
        return make_segment<E, kD>(r, p.group.divisor, shared, len);
    };
    const auto segment = [&](std::uint32_t s) {
        return s < p.groups ? group_segment(s) : row_segment(s - p.groups, nullptr);
    };
    const std::uint32_t segments = p.groups + p.rows;
    // The buffers hold no tile yet: costs before every segment, and wave totals.
    auto* const cost_before = reinterpret_cast<std::uint64_t*>(buffers[0]);
    auto* const wave_cost = reinterpret_cast<std::uint64_t*>(buffers[1]);
    static_assert((kMaxRows + kMaxGroups) * 8 <= kBufferBytes, "costs fit a buffer");
    const std::uint32_t per = (segments + kThreads - 1) / kThreads;
    std::uint64_t mine = 0;
    for (std::uint32_t i = 0; i < per; ++i) {
        const std::uint32_t s = tid * per + i;
        if (s < segments) mine += segment(s).cost(p.heads);
    }
    std::uint64_t upto = mine;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
        const std::uint64_t add = __shfl_up(static_cast<unsigned long long>(upto), off);
        if (lane >= off) upto += add;
    }
    if (lane == 63) wave_cost[wave] = upto;
    if (tid == 0) found = ~0u;
    __syncthreads();
    std::uint64_t before = upto - mine, total = 0;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
        before += w < wave ? wave_cost[w] : 0;
        total += wave_cost[w];
    }
    total = uniform64(total);
    // Neighbouring shares on one XCD (workgroups go round the 8 XCDs), so the
    // streams of a kv head meet in its L2.
    const std::uint32_t w = (blockIdx.x % 8) * (kWorkgroups / 8) + blockIdx.x / 8;
    const std::uint64_t share = share_begin(total, w), share_end = share_begin(total, w + 1);
    for (std::uint32_t i = 0; i < per; ++i) {
        const std::uint32_t s = tid * per + i;
        if (s < segments) {
            const std::uint64_t cost = segment(s).cost(p.heads);
            cost_before[s] = before;
            if (before <= share && share < before + cost) found = s;  // one segment at most
            before += cost;
        }
    }
    __syncthreads();
    if (w == 0) {  // uniform: the rows' plans for the merge
        if (tid == 0) *p.total = total;
        for (std::uint32_t r = tid; r < p.rows; r += kThreads) {
            std::uint32_t g;
            const Segment own = row_segment(r, &g);
            RowPlan plan{0, cost_before[p.groups + r], 0, 1, 1, 0, 0, own.tiles, own.weight, own.end};
            if (g < p.groups) {
                const Segment prefix = group_segment(g);
                plan.prefix_cost = cost_before[g];
                plan.prefix_tiles = prefix.tiles;
                plan.prefix_weight = prefix.weight;
                plan.prefix_col_tiles = prefix.col_tiles;
                plan.prefix_stream = group_stream(p, g, prefix.first_row);
                plan.first_row = prefix.first_row;
            }
            p.plans[r] = plan;
        }
    }
    std::uint32_t seg = uniform(found);
    if (share >= share_end || seg == ~0u) return;  // uniform: no tile starts in this share
    const auto uniform_segment = [&](std::uint32_t s) {
        const Segment x = segment(s);
        return Segment{uniform(x.first_row), uniform(x.cols), uniform(x.col_tiles), uniform(x.begin), uniform(x.end),
                       uniform(x.tiles), uniform(x.weight)};
    };
    Segment cur = uniform_segment(seg);
    std::uint64_t cost = uniform64(cost_before[seg]);  // costs before the current stream
    std::uint32_t stream = uniform(static_cast<std::uint32_t>((share - cost) / cur.stream_cost()));
    cost += stream * cur.stream_cost();
    std::uint32_t tile = uniform(static_cast<std::uint32_t>((share - cost + cur.weight - 1) / cur.weight));
    __syncthreads();  // cost_before is read: the buffers are free

    // The part at hand: tiles [tile, tile_end) of stream `stream` of segment
    // `seg`. settle() moves to the next part that has tiles; false at the end
    // of the share.
    std::uint32_t tile_end = 0;
    const auto settle = [&]() -> bool {
        while (true) {
            if (tile < cur.tiles) {
                const std::uint64_t at = cost + static_cast<std::uint64_t>(tile) * cur.weight;
                if (at >= share_end) return false;
                const std::uint64_t left = (share_end - cost + cur.weight - 1) / cur.weight;
                tile_end = left < cur.tiles ? static_cast<std::uint32_t>(left) : cur.tiles;
                return true;
            }
            cost += cur.stream_cost();
            tile = 0;
            if (cost >= share_end) return false;
            if (cur.tiles != 0 && ++stream < p.heads * cur.col_tiles) continue;
            stream = 0;
            do {
                if (++seg >= segments) return false;
                cur = uniform_segment(seg);
            } while (cur.tiles == 0);
        }
    };
    if (!settle()) return;  // uniform

    // ---- tile loads. Load i of a wavefront fills 1 KiB of the buffer in lane
    // order: chunk e = (i * 8 + wave) * 64 + lane is slot e % kCpr of row
    // e / kCpr. Which chunk of the row a lane fetches sets the swizzle that
    // keeps the reads below free of bank conflicts.
    const auto kswz = [](int row) { return kCpr >= 16 ? (row & 15) : ((row >> 1) & 7); };
    const auto vswz = [](int row) { return kF32 ? 0 : kCpr / 8 * (row & 7); };
    const std::uint32_t bs = p.block_size.divisor;
    const std::uint64_t head_bytes = static_cast<std::uint64_t>(bs) * kRowBytes;
    const std::uint64_t page_bytes = head_bytes * p.heads;
    std::uint32_t row_of[kLoads];
#pragma unroll
    for (int i = 0; i < kLoads; ++i) row_of[i] = ((i * kWaves + wave) * 64 + lane) / kCpr;
    const int slot = lane % kCpr;
    struct Where {  // a tile to load
        const std::uint64_t* table;
        std::uint32_t first, end, kvh;
    };
    const auto where = [&](std::uint32_t t) {
        return Where{p.table + static_cast<std::uint64_t>(cur.first_row) * p.width, cur.begin + t * kTile, cur.end,
                     stream / cur.col_tiles};
    };
    std::uint64_t ids[kLoads];
    const auto fetch_ids = [&](const Where& at) {
#pragma unroll
        for (int i = 0; i < kLoads; ++i) {
            const std::uint32_t token = at.first + row_of[i] < at.end ? at.first + row_of[i] : at.end - 1;
            ids[i] = at.table[p.block_size.div(token)];
        }
    };
    const auto issue = [&](const Where& at, std::uint32_t buffer, std::uint32_t serial) {
        const char* kc = static_cast<const char*>(p.key_cache) + at.kvh * head_bytes;
        const char* vc = static_cast<const char*>(p.value_cache) + at.kvh * head_bytes;
        const std::uint32_t base = lds_address(buffers[0]) + buffer * kBufferBytes + wave * 1024;
#pragma unroll
        for (int i = 0; i < kLoads; ++i) {
            const std::uint32_t token = at.first + row_of[i];
            const bool inside = token < at.end, present = ids[i] < p.num_blocks;
            if (inside && !present) bad_tile[buffer] = serial;
            const int kchunk = (slot ^ kswz(row_of[i])) * 16, vchunk = (slot ^ vswz(row_of[i])) * 16;
            const char *k, *v;
            if (inside && present) {
                const std::uint32_t off = token - p.block_size.div(token) * bs;
                const std::uint64_t row = ids[i] * page_bytes + off * static_cast<std::uint64_t>(kRowBytes);
                k = kc + row + kchunk;
                v = vc + row + vchunk;
            } else {  // a token past the end, or of a missing page: zeros, under a weight of zero
                k = reinterpret_cast<const char*>(sh_zero_row) + kchunk;
                v = reinterpret_cast<const char*>(sh_zero_row) + vchunk;
            }
            load_to_lds(k, uniform(base + i * (kWaves * 1024)));
            load_to_lds(v, uniform(base + kBufferBytes / 2 + i * (kWaves * 1024)));
        }
    };

    const std::uint32_t k_read = col * kRowBytes + (quad ^ kswz(col)) * 16;
    std::uint32_t v_read;
    if constexpr (kF32) {
        v_read = 4 * quad * kRowBytes + col * 16;
    } else {
        const int s = lane % 16, r = 4 * quad + s / 4, c = (4 * (s % 4)) / 8;
        v_read = r * kRowBytes + ((c ^ vswz(r)) * 16) + (s % 2) * 8;
    }

    std::uint32_t buffer = 0, serial = 1;
    {
        const Where at = where(tile);
        fetch_ids(at);
        issue(at, buffer, serial);
    }
    bool more = true;
    while (more) {
        // ---- a part: its columns and this wavefront's place.
        const std::uint32_t first_row = cur.first_row, kvh = stream / cur.col_tiles;
        const std::uint32_t col0 = (stream - kvh * cur.col_tiles) * kCols;
        const std::uint32_t cols = cur.cols - col0 < kCols ? cur.cols - col0 : kCols;
        const std::uint32_t layout = uniform(layout_blocks((cols + 15) / 16, S::kLeastBlocks));
        const std::uint32_t shares = kWaves / layout;  // groups of wavefronts over a tile's tokens
        const std::uint32_t block = uniform(wave / shares), token_share = uniform(wave % shares);
        const bool active = block * 16 < cols;  // uniform in a wavefront
        const bool is_prefix = seg < p.groups;
        const std::uint32_t slot_of_part =
            is_prefix ? group_stream(p, seg, first_row) + stream + w
                      : (seg - p.groups) * p.heads * p.row_tiles + stream + w;
        const std::uint32_t my_col = block * 16 + col;
        const std::uint32_t c = col0 + (my_col < cols ? my_col : 0);
        const std::uint32_t row_in = p.group.div(c);
        const float* q = p.query + (static_cast<std::uint64_t>(first_row + row_in) * p.query_heads +
                                    kvh * p.group.divisor + (c - row_in * p.group.divisor)) * kD;
        Vec qb[kF32 ? 1 : 3][kKk];
        float qf[kF32 ? kD / 4 : 1];
        if constexpr (kF32) {
#pragma unroll
            for (int m = 0; m < kD / 16; ++m) {
                const float4 x = *reinterpret_cast<const float4*>(q + 16 * m + 4 * quad);
                qf[4 * m] = x.x * p.scale_log2;
                qf[4 * m + 1] = x.y * p.scale_log2;
                qf[4 * m + 2] = x.z * p.scale_log2;
                qf[4 * m + 3] = x.w * p.scale_log2;
            }
        } else {
#pragma unroll
            for (int kk = 0; kk < kKk; ++kk) {
                const float4 lo = *reinterpret_cast<const float4*>(q + 32 * kk + 8 * quad);
                const float4 hi = *reinterpret_cast<const float4*>(q + 32 * kk + 8 * quad + 4);
                const float v[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
                std::uint32_t parts[3][4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    std::uint32_t x[3];
                    M::split3(v[2 * e] * p.scale_log2, v[2 * e + 1] * p.scale_log2, x);
#pragma unroll
                    for (int k = 0; k < 3; ++k) parts[k][e] = x[k];
                }
#pragma unroll
                for (int k = 0; k < 3; ++k)
                    qb[k][kk] = __builtin_bit_cast(Vec, make_uint4(parts[k][0], parts[k][1], parts[k][2], parts[k][3]));
            }
        }
        pf_f32x4_t acc[kDt];
#pragma unroll
        for (int dt = 0; dt < kDt; ++dt) acc[dt] = pf_f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
        // Minus the column's reference (in all accumulator lanes: the seed of
        // the score chains), and what a score may pass it by; -inf until the
        // column has seen a key.
        float nref = 0.0f, lazy = -INFINITY, sum_hi = 0.0f, sum_lo = 0.0f;

        const std::uint32_t seg_begin = cur.begin, seg_end = cur.end;
        const std::uint64_t* const table_row = p.table + static_cast<std::uint64_t>(first_row) * p.width;
        for (std::uint32_t left = tile_end - tile; left != 0; --left) {
            // The tile has landed, for every wavefront, and the other buffer is
            // no longer read.
            wait_vm<0>();
            wait_lgkm0();
            lds_barrier();
            const std::uint32_t here = buffer, here_serial = serial, here_first = seg_begin + tile * kTile;
            buffer ^= 1;
            ++serial;
            ++tile;
            if (left > 1 || (more = settle())) {  // settle() moves on to the next part
                const Where at = where(tile);
                fetch_ids(at);
                issue(at, buffer, serial);
            }
            if (active) {
                const unsigned char* kt = buffers[here];
                const unsigned char* vt = buffers[here] + kBufferBytes / 2;
                const bool bad = bad_tile[here] == here_serial;
                const std::uint32_t per_wave = S::kSteps / shares;
                for (std::uint32_t st = 0; st < per_wave; ++st) {
                    const std::uint32_t row0 = (token_share * per_wave + st) * kStep;
                    const std::uint32_t token0 = here_first + row0;
                    if (token0 >= seg_end) break;  // uniform in a wavefront
                    constexpr int kSubs = kF32 ? 1 : 2;  // 16-token score tiles of a step
                    pf_f32x4_t s[kSubs];
#pragma unroll
                    for (int b = 0; b < kSubs; ++b) s[b] = pf_f32x4_t{nref, nref, nref, nref};
                    if constexpr (kF32) {
#pragma unroll
                        for (int m = 0; m < kD / 16; ++m) {
                            const float4 x = *reinterpret_cast<const float4*>(kt + row0 * kRowBytes + (k_read ^ (m << 6)));
                            s[0] = __builtin_amdgcn_mfma_f32_16x16x4f32(x.x, qf[4 * m], s[0], 0, 0, 0);
                            s[0] = __builtin_amdgcn_mfma_f32_16x16x4f32(x.y, qf[4 * m + 1], s[0], 0, 0, 0);
                            s[0] = __builtin_amdgcn_mfma_f32_16x16x4f32(x.z, qf[4 * m + 2], s[0], 0, 0, 0);
                            s[0] = __builtin_amdgcn_mfma_f32_16x16x4f32(x.w, qf[4 * m + 3], s[0], 0, 0, 0);
                        }
                    } else {
#pragma unroll
                        for (int kk = 0; kk < kKk; ++kk)
#pragma unroll
                            for (int b = 0; b < 2; ++b) {
                                const Vec a = __builtin_bit_cast(
                                    Vec, *reinterpret_cast<const uint4*>(kt + (row0 + 16 * b) * kRowBytes + (k_read ^ (kk << 6))));
#pragma unroll
                                for (int k = 0; k < 3; ++k) s[b] = M::mma(a, qb[k][kk], s[b]);
                            }
                    }
                    if (bad || seg_end - token0 < kStep) {
#pragma unroll
                        for (int b = 0; b < kSubs; ++b)
#pragma unroll
                            for (int r = 0; r < 4; ++r) {
                                const std::uint32_t token = token0 + 16 * b + 4 * quad + r;
                                bool live = token < seg_end;
                                if (bad && live) live = table_row[p.block_size.div(token)] < p.num_blocks;
                                s[b][r] = live ? s[b][r] : -INFINITY;
                            }
                    }
                    float top = -INFINITY;
#pragma unroll
                    for (int b = 0; b < kSubs; ++b) top = max3(top, max3(s[b][0], s[b][1], s[b][2]), s[b][3]);
                    if (__builtin_expect(__builtin_amdgcn_ballot_w64(top > lazy) != 0, 0)) {
                        top = max_across_quads(top);
                        const bool moves = top > lazy;
                        const float shift = moves ? top : 0.0f;
                        if (moves) lazy = kLazy;
                        const float alpha = __builtin_amdgcn_exp2f(fminf(-shift, 0.0f));
                        nref -= shift;
                        sum_hi *= alpha;
                        sum_lo *= alpha;
#pragma unroll
                        for (int b = 0; b < kSubs; ++b) s[b] -= shift;
#pragma unroll
                        for (int dt = 0; dt < kDt; ++dt) acc[dt] *= alpha;
                    }
                    float pr[4 * kSubs];
#pragma unroll
                    for (int e = 0; e < 4 * kSubs; ++e) pr[e] = __builtin_amdgcn_exp2f(s[e / 4][e % 4]);
                    if constexpr (kF32) {
                        two_sum_add(sum_hi, sum_lo, (pr[0] + pr[1]) + (pr[2] + pr[3]));
                        // MFMA r takes token 4 * quad + r of lane (quad, col); block
                        // 4 * mm + j of O^T is dims 64 * mm + 4 * i + j, i = 0..15.
#pragma unroll
                        for (int r = 0; r < 4; ++r)
#pragma unroll
                            for (int mm = 0; mm < kD / 64; ++mm) {
                                const float4 x = *reinterpret_cast<const float4*>(
                                    vt + (row0 + r) * kRowBytes + v_read + 256 * mm);
                                acc[4 * mm] = __builtin_amdgcn_mfma_f32_16x16x4f32(x.x, pr[r], acc[4 * mm], 0, 0, 0);
                                acc[4 * mm + 1] = __builtin_amdgcn_mfma_f32_16x16x4f32(x.y, pr[r], acc[4 * mm + 1], 0, 0, 0);
                                acc[4 * mm + 2] = __builtin_amdgcn_mfma_f32_16x16x4f32(x.z, pr[r], acc[4 * mm + 2], 0, 0, 0);
                                acc[4 * mm + 3] = __builtin_amdgcn_mfma_f32_16x16x4f32(x.w, pr[r], acc[4 * mm + 3], 0, 0, 0);
                            }
                    } else {
                        two_sum_add(sum_hi, sum_lo,
                                    ((pr[0] + pr[1]) + (pr[2] + pr[3])) + ((pr[4] + pr[5]) + (pr[6] + pr[7])));
                        std::uint32_t parts[3][4];
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            std::uint32_t x[3];
                            M::split3(pr[2 * e] * kWeightScale, pr[2 * e + 1] * kWeightScale, x);
#pragma unroll
                            for (int k = 0; k < 3; ++k) parts[k][e] = x[k];
                        }
                        Vec pb[3];
#pragma unroll
                        for (int k = 0; k < 3; ++k)
                            pb[k] = __builtin_bit_cast(Vec, make_uint4(parts[k][0], parts[k][1], parts[k][2], parts[k][3]));
                        const auto* vbase = (__attribute__((address_space(3))) char*)(
                            (__attribute__((address_space(3))) unsigned char*)vt);
#pragma unroll
                        for (int dt = 0; dt < kDt; ++dt) {
                            const std::uint32_t off = row0 * kRowBytes + (v_read ^ (dt << 5));
                            const pf_i16x4_t lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((pf_lds_i16x4_t*)(vbase + off));
                            const pf_i16x4_t hi =
                                __builtin_amdgcn_ds_read_tr16_b64_v4i16((pf_lds_i16x4_t*)(vbase + off + 16 * kRowBytes));
                            const Vec a = __builtin_bit_cast(Vec, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
#pragma unroll
                            for (int k = 0; k < 3; ++k) acc[dt] = M::mma(a, pb[k], acc[dt]);
                        }
                    }
                }
            }
        }

        // ---- the part's partials: merged over the wavefronts that shared its
        // tokens (through the buffer just computed), then to the workspace.
        float sum = sum_across_quads(sum_hi + sum_lo);
        float top = lazy == -INFINITY ? -INFINITY : -nref;
        if (shares > 1) {  // uniform
            auto* const scratch = reinterpret_cast<pf_f32x4_t*>(buffers[buffer ^ 1]);
            wait_lgkm0();
            lds_barrier();  // every wavefront is done with the buffer
            if (active && quad == 0) part_ml[wave][col] = make_float2(top, sum);
            if (active && token_share != 0) {
#pragma unroll
                for (int dt = 0; dt < kDt; ++dt)
                    scratch[((block * (shares - 1) + token_share - 1) * kDt + dt) * 64 + lane] = acc[dt];
            }
            wait_lgkm0();
            lds_barrier();
            if (active && token_share == 0) {
                float all = top;
                for (std::uint32_t o = 1; o < shares; ++o) all = fmaxf(all, part_ml[wave + o][col].x);
                const float f0 = merge_weight(top, all);
                sum *= f0;
#pragma unroll
                for (int dt = 0; dt < kDt; ++dt) acc[dt] *= f0;
                for (std::uint32_t o = 1; o < shares; ++o) {
                    const float2 ml = part_ml[wave + o][col];
                    const float f = merge_weight(ml.x, all);
                    sum = fmaf(ml.y, f, sum);
#pragma unroll
                    for (int dt = 0; dt < kDt; ++dt) {
                        const pf_f32x4_t x = scratch[((block * (shares - 1) + o - 1) * kDt + dt) * 64 + lane];
#pragma unroll
                        for (int r = 0; r < 4; ++r) acc[dt][r] = fmaf(x[r], f, acc[dt][r]);
                    }
                }
                top = all;
            }
        }
        if (active && token_share == 0 && my_col < cols) {
            const std::uint64_t at = is_prefix ? static_cast<std::uint64_t>(slot_of_part) * kCols + my_col
                                               : static_cast<std::uint64_t>(slot_of_part) * p.row_cols + my_col;
            float* out = (is_prefix ? p.prefix_acc : p.row_acc) + at * kD;
            if (quad == 0)
                *reinterpret_cast<float2*>((is_prefix ? p.prefix_ml : p.row_ml) + 2 * at) = make_float2(top, sum);
            if constexpr (kF32) {
#pragma unroll
                for (int mm = 0; mm < kD / 64; ++mm)
#pragma unroll
                    for (int r = 0; r < 4; ++r)
                        *reinterpret_cast<float4*>(out + 64 * mm + 16 * quad + 4 * r) =
                            make_float4(acc[4 * mm][r], acc[4 * mm + 1][r], acc[4 * mm + 2][r], acc[4 * mm + 3][r]);
            } else {
#pragma unroll
                for (int dt = 0; dt < kDt; ++dt) {
                    const pf_f32x4_t x = acc[dt] * (1.0f / kWeightScale);  // a power of two: exact
                    *reinterpret_cast<float4*>(out + 16 * dt + 4 * quad) = make_float4(x[0], x[1], x[2], x[3]);
                }
            }
        }
    }
}

// Merges the partials of every (row, query head): those of its prefix's stream
// and of its own, in the order of the workgroups that left them. Both streams'
// workgroups are neighbours, from the one whose share their first tile starts
// in to the one of their last; a workgroup in between has a partial where a
// tile of the stream starts in its share.
constexpr int kMergeThreads = 128;
template <int kD>
__global__ __launch_bounds__(kMergeThreads) void shared_merge_kernel(SharedParams p) {
    constexpr std::uint32_t kMost = 2 * kWorkgroups;
    constexpr std::uint32_t kLanes = kD / 4, kGroups = kMergeThreads / kLanes;
    __shared__ float weight[kMost];  // the part's factor; below 0: no partial
    __shared__ float wave_value[2][kMergeThreads / 64];
    __shared__ float4 sums[kMergeThreads];
    const std::uint32_t row = blockIdx.x / p.query_heads, head = blockIdx.x % p.query_heads;
    const std::uint32_t tid = threadIdx.x, wave = tid / 64, lane = tid % 64;
    const std::uint64_t total = *p.total;
    const RowPlan plan = p.plans[row];
    const std::uint32_t kvh = p.group.div(head), g = head - kvh * p.group.divisor;

    // A stream's partials: workgroups first .. first + count - 1.
    struct Stream {
        std::uint64_t cost;
        std::uint32_t tiles, weight, first, count;
        std::uint64_t slot;  // partial of workgroup w: row slot + w * step of the arrays
        std::uint32_t step;
    };
    const auto span = [&](Stream& s) {
        s.first = s.count = 0;
        if (s.tiles == 0) return;
        s.first = static_cast<std::uint32_t>(s.cost * kWorkgroups / total);
        const std::uint64_t last = s.cost + static_cast<std::uint64_t>(s.tiles - 1) * s.weight;
        s.count = static_cast<std::uint32_t>(last * kWorkgroups / total) - s.first + 1;
    };
    Stream prefix, own;
    {
        const std::uint32_t c = (row - plan.first_row) * p.group.divisor + g;  // column of the prefix
        const std::uint32_t stream = kvh * plan.prefix_col_tiles + c / kCols;
        prefix.tiles = plan.prefix_tiles;
        prefix.weight = plan.prefix_weight;
        prefix.cost = plan.prefix_cost + static_cast<std::uint64_t>(stream) * prefix.tiles * prefix.weight;
        prefix.slot = static_cast<std::uint64_t>(plan.prefix_stream + stream) * kCols + c % kCols;
        prefix.step = kCols;
        span(prefix);
    }
    {
        const std::uint32_t stream = kvh * p.row_tiles + g / kCols;
        own.tiles = plan.own_tiles;
        own.weight = plan.own_weight;
        own.cost = plan.own_cost + static_cast<std::uint64_t>(stream) * own.tiles * own.weight;
        own.slot = (static_cast<std::uint64_t>(row) * p.heads * p.row_tiles + stream) * p.row_cols + g % kCols;
        own.step = p.row_cols;
        span(own);
    }
    const std::uint32_t parts = prefix.count + own.count;
    const auto partial = [&](std::uint32_t i, const float** acc) {  // its (m, sum), and its place
        const bool of_prefix = i < prefix.count;
        const Stream& s = of_prefix ? prefix : own;
        const std::uint32_t w = s.first + (of_prefix ? i : i - prefix.count);
        const std::uint64_t at = s.slot + static_cast<std::uint64_t>(w) * s.step;
        *acc = (of_prefix ? p.prefix_acc : p.row_acc) + at * kD;
        return (of_prefix ? p.prefix_ml : p.row_ml) + 2 * at;
    };
    const auto exists = [&](std::uint32_t i) {
        const bool of_prefix = i < prefix.count;
        const Stream& s = of_prefix ? prefix : own;
        const std::uint32_t w = s.first + (of_prefix ? i : i - prefix.count);
        const std::uint64_t begin = share_begin(total, w), end = share_begin(total, w + 1);
        const std::uint64_t t = begin > s.cost ? (begin - s.cost + s.weight - 1) / s.weight : 0;
        return t < s.tiles && s.cost + t * s.weight < end;
    };

    float top = -INFINITY;
    for (std::uint32_t i = tid; i < parts; i += kMergeThreads) {
        const float* acc;
        const float* ml = partial(i, &acc);
        if (exists(i)) top = fmaxf(top, ml[0]);
    }
#pragma unroll
    for (int x = 1; x < 64; x <<= 1) top = fmaxf(top, __shfl_xor(top, x));
    if (lane == 0) wave_value[0][wave] = top;
    __syncthreads();
    top = fmaxf(wave_value[0][0], wave_value[0][1]);
    float sum = 0.0f;
    for (std::uint32_t i = tid; i < parts; i += kMergeThreads) {
        const float* acc;
        const float* ml = partial(i, &acc);
        float f = -1.0f;
        if (exists(i)) {
            f = merge_weight(ml[0], top);
            sum = fmaf(ml[1], f, sum);
        }
        weight[i] = f;
    }
#pragma unroll
    for (int x = 1; x < 64; x <<= 1) sum += __shfl_xor(sum, x);
    if (lane == 0) wave_value[1][wave] = sum;
    __syncthreads();
    sum = wave_value[1][0] + wave_value[1][1];
    const std::uint32_t part0 = tid / kLanes, d4 = tid % kLanes;
    float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    for (std::uint32_t i = part0; i < parts; i += kGroups) {
        const float f = weight[i];
        if (f < 0.0f) continue;
        const float* acc;
        partial(i, &acc);
        const float4 x = *reinterpret_cast<const float4*>(acc + 4 * d4);
        o.x = fmaf(x.x, f, o.x);
        o.y = fmaf(x.y, f, o.y);
        o.z = fmaf(x.z, f, o.z);
        o.w = fmaf(x.w, f, o.w);
    }
    sums[tid] = o;
    __syncthreads();
    if (tid >= kLanes) return;
#pragma unroll
    for (std::uint32_t k = 1; k < kGroups; ++k) {
        const float4 x = sums[k * kLanes + d4];
        o.x += x.x;
        o.y += x.y;
        o.z += x.z;
        o.w += x.w;
    }
    const float inv = sum > 0.0f ? 1.0f / sum : 0.0f;
    float* out = p.output + static_cast<std::uint64_t>(blockIdx.x) * kD + 4 * d4;
    out[0] = o.x * inv;
    out[1] = o.y * inv;
    out[2] = o.z * inv;
    out[3] = o.w * inv;
}

// ---------------------------------------------------------------- dispatch

// Bytes of the workspace's parts, each a multiple of 256.
struct Layout {
    std::uint64_t total = 0, plans = 0, prefix_acc = 0, prefix_ml = 0, row_acc = 0, row_ml = 0, bytes = 0;
};

// Whether the shared kernel takes the call; if not it runs as an ordinary
// decode batch (the same results: a shared page is only read more often).
bool takes(std::uint64_t rows, std::uint64_t kv_len, std::uint64_t kv_heads, std::uint64_t query_heads,
           std::uint64_t block_size, std::uint64_t head_size, int dtype, std::uint64_t groups) {
    if (groups == 0 || groups > kMaxGroups || rows > kMaxRows) return false;
    if (head_size != 64 && head_size != 128 && (head_size != 256 || dtype == KVFLUX_DTYPE_F32)) return false;
    return kv_len < 0x80000000ULL && block_size < 0x80000000ULL && kv_heads <= 65535 && query_heads <= 65535 &&
           rows * query_heads < (1ULL << 24);  // workgroups of the merge
}

Layout layout_of(std::uint64_t rows, std::uint64_t kv_heads, std::uint64_t query_heads, std::uint64_t head_size,
                 std::uint64_t groups) {
    const auto whole = [](std::uint64_t bytes) { return (bytes + 255) & ~std::uint64_t{255}; };
    const std::uint64_t group = query_heads / kv_heads;
    const std::uint64_t prefix_slots = (groups + rows * group / kCols) * kv_heads + kWorkgroups;
    const std::uint64_t row_slots = rows * kv_heads * ((group + kCols - 1) / kCols) + kWorkgroups;
    const std::uint64_t row_cols = group < kCols ? group : kCols;
    Layout l;
    l.plans = 256;
    l.prefix_acc = l.plans + whole(rows * sizeof(RowPlan));
    l.prefix_ml = l.prefix_acc + whole(prefix_slots * kCols * head_size * sizeof(float));
    l.row_acc = l.prefix_ml + whole(prefix_slots * kCols * 2 * sizeof(float));
    l.row_ml = l.row_acc + whole(row_slots * row_cols * head_size * sizeof(float));
    l.bytes = l.row_ml + whole(row_slots * row_cols * 2 * sizeof(float));
    return l;
}

template <typename E, int kD>
int launch(const SharedParams& p, hipStream_t s) {
    hipLaunchKernelGGL((shared_attention_kernel<E, kD>), dim3(kWorkgroups), dim3(kThreads), 0, s, p);
    const int status = launch_status("shared_attention_kernel");
    if (status != KVFLUX_OK) return status;
    hipLaunchKernelGGL((shared_merge_kernel<kD>), dim3(p.rows * p.query_heads), dim3(kMergeThreads), 0, s, p);
    return launch_status("shared_merge_kernel");
}

template <typename E>
int launch_size(const SharedParams& p, std::uint64_t head_size, hipStream_t s) {
    if (head_size == 64) return launch<E, 64>(p, s);
    if constexpr (!std::is_same<E, ShF32>::value) {
        if (head_size == 256) return launch<E, 256>(p, s);
    }
    return launch<E, 128>(p, s);
}

int check_shape(std::uint64_t num_kv_heads, std::uint64_t block_size, std::uint64_t head_size, int dtype,
                std::uint64_t query_heads) {
    if (dtype_bytes(dtype) == 0) return fail(KVFLUX_ERR_INVALID_ARGUMENT, "unknown dtype %d", dtype);
    if (num_kv_heads == 0 || block_size == 0 || head_size == 0 || query_heads == 0 || query_heads % num_kv_heads != 0)
        return fail(KVFLUX_ERR_INVALID_ARGUMENT, "shared attention: invalid shape");
    return KVFLUX_OK;
}

} // namespace
} // namespace kvflux_hip

using namespace kvflux_hip;

extern "C" int kvflux_paged_attention_shared_workspace_size(uint64_t num_rows, uint64_t kv_len, uint64_t num_kv_heads,
                                                            uint64_t query_heads, uint64_t block_size,
                                                            uint64_t head_size, int dtype, uint64_t num_groups,
                                                            size_t* bytes) {
    if (!bytes) return fail(KVFLUX_ERR_INVALID_ARGUMENT, "bytes is null");
    *bytes = 0;
    const int status = check_shape(num_kv_heads, block_size, head_size, dtype, query_heads);
    if (status != KVFLUX_OK) return status;
    if (!takes(num_rows, kv_len, num_kv_heads, query_heads, block_size, head_size, dtype, num_groups))
        return kvflux_paged_attention_workspace_size(num_rows, kv_len, num_kv_heads, query_heads, block_size, head_size,
                                                     bytes);
    *bytes = layout_of(num_rows, num_kv_heads, query_heads, head_size, num_groups).bytes;
    return KVFLUX_OK;
}

extern "C" int kvflux_paged_attention_shared(const void* key_cache, const void* value_cache, uint64_t num_blocks,
                                             uint64_t num_kv_heads, uint64_t block_size, uint64_t head_size, int dtype,
                                             const uint64_t* block_table, uint64_t max_blocks_per_seq,
                                             const uint64_t* seq_lens, uint64_t kv_len, uint64_t num_rows,
                                             uint64_t query_heads, const uint64_t* group_starts,
                                             const uint64_t* group_prefixes, uint64_t num_groups,
                                             uint64_t max_prefix, const float* query, float* output, void* workspace,
                                             size_t workspace_bytes, void* stream) {
    if (num_rows == 0) return KVFLUX_OK;
    int status = check_shape(num_kv_heads, block_size, head_size, dtype, query_heads);
    if (status != KVFLUX_OK) return status;
    if (!key_cache || !value_cache || !block_table || !seq_lens || !query || !output ||
        (num_groups != 0 && (!group_starts || !group_prefixes)))
        return fail(KVFLUX_ERR_INVALID_ARGUMENT, "shared attention: null pointer");
    if (num_blocks == 0 || max_blocks_per_seq == 0)
        return fail(KVFLUX_ERR_INVALID_ARGUMENT, "shared attention: invalid shape");
    if (!takes(num_rows, kv_len, num_kv_heads, query_heads, block_size, head_size, dtype, num_groups))
        return kvflux_paged_attention(key_cache, value_cache, num_blocks, num_kv_heads, block_size, head_size, dtype,
                                      block_table, max_blocks_per_seq, seq_lens, kv_len, num_rows, query_heads, query,
                                      output, workspace, workspace_bytes, stream);
    const Layout l = layout_of(num_rows, num_kv_heads, query_heads, head_size, num_groups);
    if (!workspace || workspace_bytes < l.bytes)
        return fail(KVFLUX_ERR_INVALID_ARGUMENT, "shared attention: workspace needs %llu bytes",
                    static_cast<unsigned long long>(l.bytes));
    const void* vectors[3] = {key_cache, value_cache, workspace};
    if (copy_width(16, vectors, 3) != 16)
        return fail(KVFLUX_ERR_INVALID_ARGUMENT, "shared attention: caches and workspace must be aligned to 16 bytes");
    SharedParams p{};
    p.key_cache = key_cache;
    p.value_cache = value_cache;
    p.num_blocks = num_blocks;
    p.heads = static_cast<std::uint32_t>(num_kv_heads);
    p.block_size = FastDiv(static_cast<std::uint32_t>(block_size));
    p.table = block_table;
    p.width = max_blocks_per_seq;
    p.lens = seq_lens;
    // Tokens past the table have no page: they drop out as missing ones do.
    p.kv_len = static_cast<std::uint32_t>(
        max_blocks_per_seq < (kv_len + block_size - 1) / block_size ? max_blocks_per_seq * block_size : kv_len);
    p.rows = static_cast<std::uint32_t>(num_rows);
    p.query_heads = static_cast<std::uint32_t>(query_heads);
    p.group = FastDiv(static_cast<std::uint32_t>(query_heads / num_kv_heads));
    p.starts = group_starts;
    p.prefixes = group_prefixes;
    p.groups = static_cast<std::uint32_t>(num_groups);
    p.max_prefix = max_prefix < p.kv_len ? static_cast<std::uint32_t>(max_prefix) : p.kv_len;
    p.query = query;
    p.output = output;
    p.scale_log2 = static_cast<float>(1.4426950408889634 / std::sqrt(static_cast<double>(head_size)));
    char* base = static_cast<char*>(workspace);
    p.total = reinterpret_cast<std::uint64_t*>(base);
    p.plans = reinterpret_cast<RowPlan*>(base + l.plans);
    p.prefix_acc = reinterpret_cast<float*>(base + l.prefix_acc);
    p.prefix_ml = reinterpret_cast<float*>(base + l.prefix_ml);
    p.row_acc = reinterpret_cast<float*>(base + l.row_acc);
    p.row_ml = reinterpret_cast<float*>(base + l.row_ml);
    p.row_cols = p.group.divisor < kCols ? p.group.divisor : kCols;
    p.row_tiles = (p.group.divisor + kCols - 1) / kCols;
    const hipStream_t s = as_stream(stream);
    switch (dtype) {
    case KVFLUX_DTYPE_BF16: return launch_size<PfBf16Exact>(p, head_size, s);
    case KVFLUX_DTYPE_F16: return launch_size<PfF16Exact>(p, head_size, s);
    default: return launch_size<ShF32>(p, head_size, s);
    }
}
