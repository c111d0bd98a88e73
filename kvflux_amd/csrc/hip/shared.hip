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
// in) and the weights as three 16-bit parts each: products as exact as
// FP32's, sums FP32. FP32 caches: v_mfma_f32_16x16x4_f32 on the values as they are.
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
constexpr std::uint32_t kMaxRows = 2048;    // rows and groups whose plan is in LDS
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
    // Blocks of 16 columns that a wavefront may hold: with two, every K and V
    // operand read from LDS feeds twice the MFMAs. Head sizes 128 and 256 have no
    // registers for two; FP32 MFMAs are slow enough for one.
    static constexpr std::uint32_t kMostBlocks = kF32 || kD >= 128 ? 1 : 2;
    // The fewest wavefronts side by side over columns: with fewer, the others
    // would not have a step of the tile's tokens each.
    static constexpr std::uint32_t kLeastAcross = kSteps >= kWaves ? 1 : kWaves / kSteps;
    static constexpr int kLoads = kBufferBytes / 2 / (kThreads * 16);  // loads of a thread, K and V each
    // spread_of doubles the wavefronts side by side until they hold a stream's
    // columns: more of them than there are would leave no shares of a tile.
    static_assert(kCols <= 16 * kWaves && kLeastAcross <= kWaves && (kWaves & (kWaves - 1)) == 0, "columns of a stream");
};

// How the wavefronts take a stream of `cols` columns: `across` of them side by
// side with `blocks` blocks of 16 columns each; kWaves / across groups of such
// share a tile's tokens.
struct Spread {
    std::uint32_t across, blocks;
};
template <typename E, int kD>
__device__ inline Spread spread_of(std::uint32_t cols) {
    using S = Shape<E, kD>;
    const std::uint32_t need = (cols + 15) / 16;
    Spread s{S::kLeastAcross, 1};
    while (s.across < need) {
        // Two blocks where the merge of the shares' accumulators fits a buffer.
        if (S::kMostBlocks == 2 && s.across * 2 >= need && (kWaves - s.across) * 2 * kD * 64 <= kBufferBytes) {
            s.blocks = 2;
            break;
        }
        s.across *= 2;
    }
    return s;
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
    // Workspace: the rows' plans for the merge, partials.
    struct RowPlan* plans;
    float* prefix_acc;  // [prefix_place][D]
    float* prefix_ml;   // [prefix_place][2]
    float* row_acc;     // [slot][row_cols][D]
    float* row_ml;      // [slot][row_cols][2]
    std::uint32_t row_cols;   // min(group, kCols)
    std::uint32_t row_tiles;  // ceil(group / kCols): streams of a row for each kv head
};

// What the merge needs of a row.
struct RowPlan {
    std::uint32_t prefix_cost, own_cost;  // costs before the segments
    std::uint32_t prefix_tiles, prefix_weight, prefix_cols;
    std::uint32_t first_row, own_tiles, own_weight, total;
};

// Cost of a tile in about 1000 cycles, by the blocks of 16 columns it is computed
// for (rounded up to a power of two, as the wavefronts are laid out): what any
// tile takes, to be loaded, and its products, which a tile of a fixed size in
// bytes has as many of at every head size. A part starts with its queries and
// ends with its partials: kPartCost, in the stream's first tile.
constexpr std::uint32_t kPartCost = 4, kTileCost = 4, kMostTileCost = kTileCost + 3 * kCols / 16;
template <typename E, int kD>
__device__ inline std::uint32_t tile_cost(std::uint32_t cols) {
    const std::uint32_t blocks = cols > 64 ? 8 : cols > 32 ? 4 : cols > 16 ? 2 : 1;
    return kTileCost + (Shape<E, kD>::kF32 ? 3 : 1) * blocks;
}

// A segment: the columns (of row first_row on), the tokens [begin, end) of
// table row `table_row`, its tiles and the cost of one.
struct Segment {
    std::uint32_t first_row, table_row, cols, col_tiles, begin, end, tiles, weight;
    __device__ std::uint32_t stream_cost() const { return tiles != 0 ? tiles * weight + kPartCost : 0; }
    __device__ std::uint32_t cost(std::uint32_t heads) const { return stream_cost() * (heads * col_tiles); }
};

template <typename E, int kD>
__device__ inline Segment make_segment(std::uint32_t first_row, std::uint32_t cols, std::uint32_t begin, std::uint32_t end) {
    constexpr std::uint32_t kTile = Shape<E, kD>::kTile;
    Segment s{first_row, first_row, cols, (cols + kCols - 1) / kCols, begin, end, 0, 0};
    s.tiles = end > begin ? (end - begin - 1) / kTile + 1 : 0;
    s.weight = tile_cost<E, kD>(cols);
    return s;
}

// Inclusive scans over a wavefront by lane moves within rows of 16 and their
// broadcasts to the rows behind (six shuffles through LDS: 700 cycles more).
template <int kCtrl, int kRows>
__device__ inline std::uint32_t moved(std::uint32_t x) {  // 0 where no lane is moved from
    return static_cast<std::uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(x), kCtrl, kRows, 0xf, false));
}
template <typename Op>
__device__ inline std::uint32_t wave_scan(std::uint32_t x, Op op) {
    x = op(x, moved<0x111, 0xf>(x));  // 1, 2, 4 and 8 lanes below, in a row
    x = op(x, moved<0x112, 0xf>(x));
    x = op(x, moved<0x114, 0xf>(x));
    x = op(x, moved<0x118, 0xf>(x));
    x = op(x, moved<0x142, 0xa>(x));  // lane 15 of a row into rows 1 and 3
    x = op(x, moved<0x143, 0xc>(x));  // lane 31 into rows 2 and 3
    return x;
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

// Where workgroup w's partials of a prefix's stream go, in columns: its columns lie
// behind those of all streams before it (the groups' in order, a group's kv heads
// in order), and another kCols on for every workgroup. Streams are taken up in that
// order, so no two parts meet.
__device__ inline std::uint32_t prefix_place(const SharedParams& p, std::uint32_t first_row, std::uint32_t cols,
                                             std::uint32_t kvh, std::uint32_t col, std::uint32_t w) {
    return first_row * p.query_heads + kvh * cols + col + w * kCols;
}

// Where the share of workgroup w begins, ceil(total * w / kWorkgroups), in 32 bits.
__device__ inline std::uint32_t share_begin(std::uint32_t total, std::uint32_t w) {
    return total / kWorkgroups * w + (total % kWorkgroups * w + kWorkgroups - 1) / kWorkgroups;
}
// Where tile t of a stream starts, behind the stream's start; and the tiles
// before the first that starts at `at` or behind it.
__device__ inline std::uint32_t tile_start(std::uint32_t t, std::uint32_t weight) {
    return t == 0 ? 0 : t * weight + kPartCost;
}
__device__ inline std::uint32_t tiles_before(std::uint32_t at, std::uint32_t weight) {
    return at == 0 ? 0 : at <= weight + kPartCost ? 1 : (at - kPartCost + weight - 1) / weight;
}

// exp2(m - top) for merging partials: 0 for a part that saw no key.
__device__ inline float merge_weight(float m, float top) {
    return m == -INFINITY ? 0.0f : m == top ? 1.0f : __builtin_amdgcn_exp2f(m - top);
}

__device__ __attribute__((aligned(16))) unsigned char sh_zero_row[512];

// kWhole: pages of a multiple of 16 tokens. Then 16 neighbouring rows of a tile
// that starts at a multiple of 16 lie in one page, and a wavefront's loads are
// one scalar address and constant lane offsets; else every lane looks up the
// page of each of its rows.
template <typename E, int kD, bool kWhole>
__global__ __launch_bounds__(kThreads) void shared_attention_kernel(SharedParams p) {
    using S = Shape<E, kD>;
    constexpr bool kF32 = S::kF32;
    using M = typename std::conditional<kF32, PfBf16Exact, E>::type;
    using Vec = typename M::Vec;
    constexpr std::uint32_t kTile = S::kTile, kStep = S::kStep;
    constexpr int kRowBytes = S::kRowBytes, kCpr = S::kCpr, kLoads = S::kLoads;
    constexpr int kBlocks = static_cast<int>(S::kMostBlocks);
    constexpr int kKk = kD / 32;   // 16-bit: K steps of S^T
    constexpr int kDt = kD / 16;   // accumulator tiles of O^T
    // 16-bit parts of a query value and of a weight: three hold all 24 bits of an
    // FP32 value, as in the ordinary decode (two FP16 parts miss its last: 48 rows
    // behind 60000 tokens in FP16 216 us, and 254 with three).
    constexpr int kParts = 3;
    // FP16 parts end at 2^-24 and at 65504, whatever the query's size: a column's
    // queries are split times the power of two that brings the largest into
    // [2^14, 2^15), so only values below 2^-16 of it lose bits. Its scores, the
    // reference among them, carry that factor up to the exponentials (exact).
    constexpr bool kScaled = std::is_same<E, PfF16Exact>::value;
    constexpr float kWeightScale = kF32 ? 1.0f : M::kWeightScale;
    constexpr float kLazy = kF32 ? 8.0f : M::kLazyLog2;
    // Where the weighted sums gather before they are added to the part's: an MFMA
    // rounds a sum with a large accumulator to fewer bits and toward zero, and
    // thousands of weights of 2^-25 behind one large one lost 2e-5 that way (FP32
    // caches 9e-5). Over a tile, in registers of their own, where those are there
    // (48 rows behind 60000 tokens 262 -> 249 us, head size 64 51.4 -> 50.3); over a
    // step at head size 256, and on FP16 caches, whose reference moves too often
    // to scale two sets of sums (64 rows behind 8192, head size 64: 56.5, else 59).
    constexpr bool kTileSums = !kScaled && kD <= 128;
    static_assert(!kScaled || kLazy == 0.0f, "a scaled score is compared with kLazy");

    __shared__ __attribute__((aligned(16))) unsigned char buffers[2][kBufferBytes];
    __shared__ std::uint32_t first_of[kMaxGroups + 1];  // first row of a group, and the end
    __shared__ std::uint32_t prefix_of[kMaxGroups];     // its prefix (0: past the bound)
    __shared__ std::uint32_t begin_of[kMaxRows], end_of[kMaxRows];  // a row's own tokens
    __shared__ float2 part_ml[kWaves][kBlocks][16];
    __shared__ std::uint32_t bad_tile[2];               // the serial number of a tile with a missing page
    __shared__ std::uint32_t found[2];                  // the segment this share starts in, the cost before it

    const int tid = threadIdx.x, lane = tid % 64;
    const auto uniform = [](std::uint32_t x) {
        return static_cast<std::uint32_t>(__builtin_amdgcn_readfirstlane(static_cast<int>(x)));
    };
    const int wave = static_cast<int>(uniform(tid / 64));
    const int col = lane % 16, quad = lane / 16;

    // ---- plan: the groups (starts made monotone, whatever the caller gave),
    // every row's own tokens, and the sum of costs over all segments: groups
    // first, then rows. All loads of it are in one round trip.
    for (std::uint32_t r = tid; r < p.rows; r += kThreads) {
        const std::uint64_t n = p.lens[r];
        end_of[r] = n < p.kv_len ? static_cast<std::uint32_t>(n) : p.kv_len;
    }
    for (std::uint32_t g = tid; g < p.groups; g += kThreads) {
        const std::uint64_t n = p.prefixes[g];
        prefix_of[g] = n <= p.max_prefix ? static_cast<std::uint32_t>(n) : 0u;
    }
    if (wave == 0) {
        std::uint32_t carry = 0;
#pragma unroll 1
        for (std::uint32_t base = 0; base <= p.groups; base += 64) {
            const std::uint32_t g = base + lane;
            std::uint32_t v = 0;
            if (g <= p.groups) {
                const std::uint64_t s = p.starts[g];
                v = s < p.rows ? static_cast<std::uint32_t>(s) : p.rows;
            }
            v = wave_scan(v, [](std::uint32_t a, std::uint32_t b) { return a > b ? a : b; });
            v = v > carry ? v : carry;
            if (g <= p.groups) first_of[g] = v;
            carry = static_cast<std::uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(v), 63));
        }
    }
    if (tid < 2) bad_tile[tid] = 0;
    if (tid == 0) found[0] = ~0u;
    __syncthreads();
    // Tokens that the rows of a group share, in steps of 16 where pages are whole
    // ones: none with fewer than two rows. A row shorter than the prefix takes no
    // part in it.
    const auto shared_tokens = [&](std::uint32_t g) {
        return first_of[g + 1] - first_of[g] >= 2 ? prefix_of[g] & (kWhole ? ~15u : ~0u) : 0u;
    };
    const auto segment = [&](std::uint32_t s) {
        const bool group = s < p.groups;
        const std::uint32_t r = s - p.groups;
        return make_segment<E, kD>(group ? first_of[s] : r, (group ? first_of[s + 1] - first_of[s] : 1u) * p.group.divisor,
                                   group ? 0u : begin_of[r], group ? shared_tokens(s) : end_of[r]);
    };
    const std::uint32_t segments = p.groups + p.rows;
    // The buffers hold no tile yet: every segment's cost, then the costs before
    // it, and wave totals. A thread's segments are neighbours.
    auto* const cost_of = reinterpret_cast<std::uint32_t*>(buffers[0]);
    auto* const wave_cost = reinterpret_cast<std::uint32_t*>(buffers[1]);
    static_assert((kMaxRows + kMaxGroups) * 4 <= kBufferBytes, "costs fit a buffer");
    const std::uint32_t per = (segments + kThreads - 1) / kThreads;
    std::uint32_t mine = 0;
#pragma unroll 1
    for (std::uint32_t s = tid * per; s < (tid + 1) * per && s < segments; ++s) {
        if (s >= p.groups) {
            const std::uint32_t r = s - p.groups, g = group_of(first_of, p.groups, r);
            begin_of[r] = g < p.groups && prefix_of[g] <= end_of[r] ? shared_tokens(g) : 0u;
        }
        const std::uint32_t cost = segment(s).cost(p.heads);
        cost_of[s] = cost;
        mine += cost;
    }
    const std::uint32_t upto = wave_scan(mine, [](std::uint32_t a, std::uint32_t b) { return a + b; });
    if (lane == 63) wave_cost[wave] = upto;
    __syncthreads();
    std::uint32_t before = upto - mine, total = 0;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
        before += w < wave ? wave_cost[w] : 0;
        total += wave_cost[w];
    }
    total = uniform(total);
    // Neighbouring shares on one XCD (workgroups go round the 8 XCDs), so the
    // streams of a kv head meet in its L2.
    const std::uint32_t w = (blockIdx.x % 8) * (kWorkgroups / 8) + blockIdx.x / 8;
    const std::uint32_t share = share_begin(total, w), share_end = share_begin(total, w + 1);
#pragma unroll 1
    for (std::uint32_t s = tid * per; s < (tid + 1) * per && s < segments; ++s) {
        const std::uint32_t cost = cost_of[s];
        cost_of[s] = before;
        if (before <= share && share < before + cost) {  // one segment at most
            found[0] = s;
            found[1] = before;
        }
        before += cost;
    }
    __syncthreads();
    if (w == 0) {  // uniform: the rows' plans for the merge
        for (std::uint32_t r = tid; r < p.rows; r += kThreads) {
            const Segment own = segment(p.groups + r);
            RowPlan plan{0, cost_of[p.groups + r], 0, 0, 0, 0, own.tiles, own.weight, total};
            if (own.begin != 0) {
                const std::uint32_t g = group_of(first_of, p.groups, r);
                const Segment prefix = segment(g);
                plan.prefix_cost = cost_of[g];
                plan.prefix_tiles = prefix.tiles;
                plan.prefix_weight = prefix.weight;
                plan.prefix_cols = prefix.cols;
                plan.first_row = prefix.first_row;
            }
            p.plans[r] = plan;
        }
    }
    // A tile: its segment, stream (kv head and tile of columns) and number, and
    // the cost before the stream. `ok`: there is one, in this share.
    struct Cursor {
        Segment s;
        std::uint32_t seg, kvh, col_tile, tile, cost;
        bool ok;
    };
    const auto uniform_segment = [&](std::uint32_t s) {
        const Segment x = segment(s);
        // A prefix is read through the first of its rows that reach it: a shorter
        // row's table need not have those pages.
        std::uint32_t table_row = uniform(x.first_row);
        if (s < p.groups) {
            const std::uint32_t end = uniform(first_of[s + 1]);
#pragma unroll 1
            for (std::uint32_t base = table_row; base < end; base += 64) {
                const std::uint32_t r = base + lane;
                const std::uint64_t reach = __builtin_amdgcn_ballot_w64(r < end && begin_of[r] != 0);
                if (reach == 0) continue;
                table_row = base + static_cast<std::uint32_t>(__builtin_ctzll(reach));
                break;
            }
        }
        return Segment{uniform(x.first_row), table_row, uniform(x.cols), uniform(x.col_tiles), uniform(x.begin), uniform(x.end),
                       uniform(x.tiles), uniform(x.weight)};
    };
    Cursor ahead;  // the tile whose page ids are fetched next
    ahead.seg = uniform(found[0]);
    if (share >= share_end || ahead.seg == ~0u) return;  // uniform: an empty share
    ahead.s = uniform_segment(ahead.seg);                 // has tiles: its cost is above 0
    ahead.cost = uniform(found[1]);
    {
        const std::uint32_t stream = (share - ahead.cost) / ahead.s.stream_cost();
        ahead.cost += stream * ahead.s.stream_cost();
        ahead.kvh = stream / ahead.s.col_tiles;
        ahead.col_tile = stream - ahead.kvh * ahead.s.col_tiles;
    }
    ahead.tile = tiles_before(share - ahead.cost, ahead.s.weight);
    // A cursor past its stream's end moves on to the next tile there is.
    const auto settle = [&](Cursor& c) {
#pragma unroll 1
        while (true) {
            if (c.tile < c.s.tiles) {
                c.ok = c.cost + tile_start(c.tile, c.s.weight) < share_end;
                return;
            }
            c.cost += c.s.stream_cost();
            c.tile = 0;
            c.ok = false;
            if (c.cost >= share_end) return;
            if (++c.col_tile < c.s.col_tiles) continue;
            c.col_tile = 0;
            if (++c.kvh < p.heads) continue;
            c.kvh = 0;
            do {
                if (++c.seg >= segments) return;
                c.s = uniform_segment(c.seg);
            } while (c.s.tiles == 0);
        }
    };
    __syncthreads();  // cost_of is read: the buffers are free

    // ---- tile loads. A wavefront fills 4 KiB of K and of V, kWaveRows rows, in
    // loads of 1 KiB in lane order: chunk i * 64 + lane is slot % kCpr of row
    // / kCpr. Which chunk of the row a lane fetches sets the swizzle that keeps
    // the reads below free of bank conflicts.
    constexpr std::uint32_t kWaveRows = 4096 / kRowBytes;
    constexpr int kIds = kWhole ? (kWaveRows > 16 ? kWaveRows / 16 : 1) : kLoads;
    const auto kswz = [](int row) { return kCpr >= 16 ? (row & 15) : ((row >> 1) & 7); };
    const auto vswz = [](int row) { return kF32 ? 0 : kCpr / 8 * (row & 7); };
    const std::uint32_t bs = p.block_size.divisor;
    const std::uint32_t wave_row = wave * kWaveRows;  // first row of the tile
    const auto row_of = [&](int i) { return wave_row + (i * 64 + lane) / kCpr; };
    // Byte of its row at which the lane's chunk of load i starts.
    const auto chunk = [&](int i, bool of_key) {
        const int row = row_of(i);
        return static_cast<std::uint32_t>(((lane % kCpr) ^ (of_key ? kswz(row) : vswz(row))) * 16);
    };
    const auto first_token = [](const Cursor& c) { return c.s.begin + c.tile * kTile; };
    // The page ids of a tile's rows are fetched a tile before its loads go out.
    std::uint64_t ids[kIds];
    const auto fetch_ids = [&](const Cursor& c) {
        const std::uint64_t* const table = p.table + static_cast<std::uint64_t>(c.s.table_row) * p.width;
#pragma unroll
        for (int i = 0; i < kIds; ++i) {
            const std::uint32_t token = first_token(c) + (kWhole ? wave_row + 16 * i : row_of(i));
            ids[i] = table[p.block_size.div(token < c.s.end ? token : c.s.end - 1)];
        }
    };
    const auto issue = [&](const Cursor& c, std::uint32_t buffer, std::uint32_t serial) {
        // The ids are here (all loads before the barrier are); the compiler's own
        // wait for them must not fall between the loads below, which it does not
        // count.
#pragma unroll
        for (int i = 0; i < kIds; ++i) asm volatile("" : "+v"(ids[i]));
        const std::uint32_t to = uniform(lds_address(buffers[0]) + buffer * kBufferBytes + wave * 4096);
        const auto key = reinterpret_cast<std::uint64_t>(p.key_cache), value = reinterpret_cast<std::uint64_t>(p.value_cache);
        const std::uint32_t first = first_token(c), end = c.s.end;
        bool direct = false;
        if constexpr (kWhole) {
            direct = first + wave_row + kWaveRows <= end;
#pragma unroll
            for (int j = 0; j < kIds; ++j) {
                ids[j] = static_cast<std::uint64_t>(uniform(static_cast<std::uint32_t>(ids[j] >> 32))) << 32 |
                         uniform(static_cast<std::uint32_t>(ids[j]));
                direct &= ids[j] < p.num_blocks;
            }
            if (direct) {  // uniform in a wavefront
#pragma unroll
                for (int j = 0; j < kIds; ++j) {
                    const std::uint32_t token = first + wave_row + 16 * j;
                    const std::uint64_t from =
                        ((ids[j] * p.heads + c.kvh) * bs + (token - p.block_size.div(token) * bs)) * kRowBytes;
#pragma unroll
                    for (int i = j * (kLoads / kIds); i < (j + 1) * (kLoads / kIds); ++i) {
                        const std::uint32_t row = ((i - j * (kLoads / kIds)) * 64 + lane) / kCpr * kRowBytes;
                        load_to_lds(key + from, row + chunk(i, true), to + i * 1024);
                        load_to_lds(value + from, row + chunk(i, false), to + kBufferBytes / 2 + i * 1024);
                    }
                }
            }
        }
        if (!direct) {
            const auto zero = reinterpret_cast<std::uint64_t>(sh_zero_row);
            std::uint64_t k[kLoads], v[kLoads];
            bool missing = false;
#pragma unroll
            for (int i = 0; i < kLoads; ++i) {
                const std::uint64_t id = ids[kWhole ? i * kIds / kLoads : i];
                const std::uint32_t token = first + row_of(i), off = token - p.block_size.div(token) * bs;
                const bool inside = token < end, present = id < p.num_blocks;
                missing |= inside && !present;
                // A token past the end, or of a missing page: zeros, under a weight of zero.
                const bool live = inside && present;
                const std::uint64_t row = ((id * p.heads + c.kvh) * bs + off) * kRowBytes;
                k[i] = (live ? key + row : zero) + chunk(i, true);
                v[i] = (live ? value + row : zero) + chunk(i, false);
            }
            if (missing) bad_tile[buffer] = serial;
#pragma unroll
            for (int i = 0; i < kLoads; ++i) {
                load_to_lds(reinterpret_cast<const void*>(k[i]), to + i * 1024);
                load_to_lds(reinterpret_cast<const void*>(v[i]), to + kBufferBytes / 2 + i * 1024);
            }
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

    // ---- the tile loop, three tiles deep: `cur` is computed while `next` is
    // loaded and the page ids of `ahead` are fetched. Its code is in one place
    // only, the first rounds doing less: a launch starts with a cold instruction
    // cache, and straight code runs at the speed of its misses.
    Cursor cur = ahead, next = ahead;
    next.ok = ahead.ok = false;
    --ahead.tile;  // the first round moves it on
    bool more = true, new_part = true;
    std::uint32_t buffer = 1, serial = 0;  // of the tile in flight
    // The part (the share's tiles of one stream) at hand: its columns and this
    // wavefront's place.
    std::uint32_t cols = 0, blocks = 1, shares = 1, across = 0, token_share = 0, first_col = 0;
    bool active = false;
    const std::uint64_t* table_row = p.table;
    Vec qb[kBlocks][kF32 ? 1 : kParts][kKk];
    float qf[kF32 ? kD / 4 : 1];
    pf_f32x4_t acc[kBlocks][kDt];
    // Minus the column's reference (in all accumulator lanes: the seed of the
    // score chains), and what a score may pass it by; -inf until the column has
    // seen a key.
    float nref[kBlocks], lazy[kBlocks], sum_hi[kBlocks], sum_lo[kBlocks];
    float down[kBlocks];  // one over the column's factor
#pragma unroll 1
    do {
        if (next.ok && new_part) {
            const Segment& part = next.s;
            const std::uint32_t col0 = next.col_tile * kCols;
            cols = part.cols - col0 < kCols ? part.cols - col0 : kCols;
            const Spread spread = spread_of<E, kD>(cols);
            blocks = spread.blocks;
            shares = kWaves / spread.across;
            across = wave / shares;
            token_share = wave % shares;
            first_col = across * blocks * 16;
            active = first_col < cols;  // uniform in a wavefront
            table_row = p.table + static_cast<std::uint64_t>(part.table_row) * p.width;
#pragma unroll
            for (int n = 0; n < kBlocks; ++n) {
                if (!active || n >= static_cast<int>(blocks)) break;
                const std::uint32_t mine = first_col + 16 * n + col, c = col0 + (mine < cols ? mine : 0);
                const std::uint32_t row_in = p.group.div(c);
                const float* q = p.query + (static_cast<std::uint64_t>(part.first_row + row_in) * p.query_heads +
                                            next.kvh * p.group.divisor + (c - row_in * p.group.divisor)) * kD;
                // All loads first: one round trip, and not one for each few.
                float4 raw[kD / 16];
#pragma unroll
                for (int m = 0; m < kD / 16; ++m)
                    raw[m] = *reinterpret_cast<const float4*>(
                        q + (kF32 ? 16 * m + 4 * quad : 32 * (m / 2) + 8 * quad + 4 * (m % 2)));
                __builtin_amdgcn_sched_barrier(0);
                if constexpr (kF32) {
#pragma unroll
                    for (int m = 0; m < kD / 16; ++m) {
                        qf[4 * m] = raw[m].x * p.scale_log2;
                        qf[4 * m + 1] = raw[m].y * p.scale_log2;
                        qf[4 * m + 2] = raw[m].z * p.scale_log2;
                        qf[4 * m + 3] = raw[m].w * p.scale_log2;
                    }
                } else {
                    float up = 1.0f;
                    if constexpr (kScaled) {
                        float largest = 0.0f;
#pragma unroll
                        for (int m = 0; m < kD / 16; ++m)
                            largest = max3(max3(largest, __builtin_fabsf(raw[m].x), __builtin_fabsf(raw[m].y)),
                                           __builtin_fabsf(raw[m].z), __builtin_fabsf(raw[m].w));
                        largest = max_across_quads(largest) * p.scale_log2;
                        const int e = split_exponent(largest);
                        up = __builtin_amdgcn_ldexpf(1.0f, e);
                        down[n] = __builtin_amdgcn_ldexpf(1.0f, -e);
                    }
#pragma unroll
                    for (int kk = 0; kk < kKk; ++kk) {
                        const float4 lo = raw[2 * kk], hi = raw[2 * kk + 1];
                        const float v[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
                        std::uint32_t parts[kParts][4];
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            std::uint32_t x[3];
                            M::split3(v[2 * e] * p.scale_log2 * up, v[2 * e + 1] * p.scale_log2 * up, x);
#pragma unroll
                            for (int k = 0; k < kParts; ++k) parts[k][e] = x[k];
                        }
#pragma unroll
                        for (int k = 0; k < kParts; ++k)
                            qb[n][k][kk] =
                                __builtin_bit_cast(Vec, make_uint4(parts[k][0], parts[k][1], parts[k][2], parts[k][3]));
                    }
                }
#pragma unroll
                for (int dt = 0; dt < kDt; ++dt) acc[n][dt] = pf_f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
                nref[n] = sum_hi[n] = sum_lo[n] = 0.0f;
                lazy[n] = -INFINITY;
            }
            new_part = false;
        }
        // The tile has landed, for every wavefront, and the other buffer is no
        // longer read.
        wait_vm<0>();
        wait_lgkm0();
        lds_barrier();
        const std::uint32_t here = buffer, here_serial = serial;
        cur = next;
        next = ahead;
        if (next.ok) {
            buffer ^= 1;
            issue(next, buffer, ++serial);
        }
        if (more) {
            ++ahead.tile;
            settle(ahead);
            more = ahead.ok;
            if (more) fetch_ids(ahead);
        }
        if (!cur.ok) continue;

        // This wavefront's share of the tile.
        const unsigned char *const kt = buffers[here], *const vt = kt + kBufferBytes / 2;
        const bool bad = bad_tile[here] == here_serial;
        const std::uint32_t first = first_token(cur), end = cur.s.end;
        const auto compute = [&](auto block_count) {
            constexpr int kN = decltype(block_count)::value;
            const std::uint32_t steps = S::kSteps / shares;
            pf_f32x4_t of_tile[kTileSums ? kN : 1][kTileSums ? kDt : 1] = {};
#pragma unroll 1
            for (std::uint32_t st = 0; st < steps; ++st) {
                const std::uint32_t row0 = (token_share * steps + st) * kStep;
                const std::uint32_t token0 = first + row0;
                if (token0 >= end) break;  // uniform in a wavefront
                constexpr int kSubs = kF32 ? 1 : 2;  // 16-token score tiles of a step
                set_priority<1>();
                pf_f32x4_t s[kN][kSubs];
#pragma unroll
                for (int n = 0; n < kN; ++n)
#pragma unroll
                    for (int b = 0; b < kSubs; ++b) s[n][b] = pf_f32x4_t{nref[n], nref[n], nref[n], nref[n]};
                if constexpr (kF32) {
#pragma unroll
                    for (int m = 0; m < kD / 16; ++m) {
                        const float4 x = *reinterpret_cast<const float4*>(kt + row0 * kRowBytes + (k_read ^ (m << 6)));
                        s[0][0] = __builtin_amdgcn_mfma_f32_16x16x4f32(x.x, qf[4 * m], s[0][0], 0, 0, 0);
                        s[0][0] = __builtin_amdgcn_mfma_f32_16x16x4f32(x.y, qf[4 * m + 1], s[0][0], 0, 0, 0);
                        s[0][0] = __builtin_amdgcn_mfma_f32_16x16x4f32(x.z, qf[4 * m + 2], s[0][0], 0, 0, 0);
                        s[0][0] = __builtin_amdgcn_mfma_f32_16x16x4f32(x.w, qf[4 * m + 3], s[0][0], 0, 0, 0);
                    }
                } else {
#pragma unroll
                    for (int kk = 0; kk < kKk; ++kk)
#pragma unroll
                        for (int b = 0; b < 2; ++b) {
                            const Vec a = __builtin_bit_cast(
                                Vec, *reinterpret_cast<const uint4*>(kt + (row0 + 16 * b) * kRowBytes + (k_read ^ (kk << 6))));
#pragma unroll
                            for (int k = 0; k < kParts; ++k)
#pragma unroll
                                for (int n = 0; n < kN; ++n) s[n][b] = M::mma(a, qb[n][k][kk], s[n][b]);
                        }
                }
                // V^T operand of dims 16 dt on. At head size 128 all of them are read
                // behind K, under the score MFMAs, and those run at a raised
                // priority, the SIMD's other wavefront in its softmax meanwhile
                // (48 rows behind 60000 tokens: 270 -> 254 us); at 256 they do not
                // fit the registers.
                constexpr bool kEarlyV = !kF32 && kD == 128;
                Vec vop[kEarlyV ? kDt : 1];
                const auto read_v = [&](int dt) {
                    const auto* base = (__attribute__((address_space(3))) char*)(
                        (__attribute__((address_space(3))) unsigned char*)vt);
                    const std::uint32_t off = row0 * kRowBytes + (v_read ^ (dt << 5));
                    const pf_i16x4_t lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((pf_lds_i16x4_t*)(base + off));
                    const pf_i16x4_t hi =
                        __builtin_amdgcn_ds_read_tr16_b64_v4i16((pf_lds_i16x4_t*)(base + off + 16 * kRowBytes));
                    return __builtin_bit_cast(Vec, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
                };
                if constexpr (kEarlyV) {
#pragma unroll
                    for (int dt = 0; dt < kDt; ++dt) vop[dt] = read_v(dt);
                    __builtin_amdgcn_sched_group_barrier(0x100, 2 * kKk, 0);       // the K reads
                    __builtin_amdgcn_sched_group_barrier(0x008, 2 * kParts * kKk * kN, 0);  // the score MFMAs
                    __builtin_amdgcn_sched_group_barrier(0x100, 2 * kDt, 0);       // the V reads
                }
                set_priority<0>();
                if (bad) {  // uniform: some page of the tile is missing
#pragma unroll
                    for (int b = 0; b < kSubs; ++b)
#pragma unroll 1
                        for (int r = 0; r < 4; ++r) {
                            const std::uint32_t token = token0 + 16 * b + 4 * quad + r;
                            const bool live = token >= end || table_row[p.block_size.div(token)] < p.num_blocks;
#pragma unroll
                            for (int n = 0; n < kN; ++n) {
#pragma unroll
                                for (int e = 0; e < 4; ++e) s[n][b][e] = live || e != r ? s[n][b][e] : -INFINITY;
                            }
                        }
                }
                if (end - token0 < kStep) {  // uniform: the last tokens
                    const std::int32_t left = static_cast<std::int32_t>(end - token0) - 4 * quad;
#pragma unroll
                    for (int b = 0; b < kSubs; ++b)
#pragma unroll
                        for (int r = 0; r < 4; ++r)
#pragma unroll
                            for (int n = 0; n < kN; ++n) s[n][b][r] = 16 * b + r < left ? s[n][b][r] : -INFINITY;
                }
                float top[kN];
                bool moves = false;
#pragma unroll
                for (int n = 0; n < kN; ++n) {
                    top[n] = -INFINITY;
#pragma unroll
                    for (int b = 0; b < kSubs; ++b)
                        top[n] = max3(top[n], max3(s[n][b][0], s[n][b][1], s[n][b][2]), s[n][b][3]);
                    moves |= top[n] > lazy[n];
                }
                if (__builtin_expect(__builtin_amdgcn_ballot_w64(moves) != 0, 0)) {
#pragma unroll
                    for (int n = 0; n < kN; ++n) {
                        const float high = max_across_quads(top[n]);
                        const float shift = high > lazy[n] ? high : 0.0f;
                        if (high > lazy[n]) lazy[n] = kLazy;
                        const float alpha = __builtin_amdgcn_exp2f(fminf(kScaled ? -shift * down[n] : -shift, 0.0f));
                        nref[n] -= shift;
                        sum_hi[n] *= alpha;
                        sum_lo[n] *= alpha;
#pragma unroll
                        for (int b = 0; b < kSubs; ++b) s[n][b] -= shift;
#pragma unroll
                        for (int dt = 0; dt < kDt; ++dt) {
                            acc[n][dt] *= alpha;
                            if constexpr (kTileSums) of_tile[n][dt] *= alpha;
                        }
                    }
                }
                Vec pb[kN][kParts];
                float pr[kN][4 * kSubs];
#pragma unroll
                for (int n = 0; n < kN; ++n) {
#pragma unroll
                    for (int e = 0; e < 4 * kSubs; ++e)
                        pr[n][e] = __builtin_amdgcn_exp2f(kScaled ? s[n][e / 4][e % 4] * down[n] : s[n][e / 4][e % 4]);
                    float of_step = (pr[n][0] + pr[n][1]) + (pr[n][2] + pr[n][3]);
                    if constexpr (!kF32) {
                        of_step += (pr[n][4] + pr[n][5]) + (pr[n][6] + pr[n][7]);
                        std::uint32_t parts[kParts][4];
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            std::uint32_t x[3];
                            M::split3(pr[n][2 * e] * kWeightScale, pr[n][2 * e + 1] * kWeightScale, x);
#pragma unroll
                            for (int k = 0; k < kParts; ++k) parts[k][e] = x[k];
                        }
#pragma unroll
                        for (int k = 0; k < kParts; ++k)
                            pb[n][k] =
                                __builtin_bit_cast(Vec, make_uint4(parts[k][0], parts[k][1], parts[k][2], parts[k][3]));
                    }
                    two_sum_add(sum_hi[n], sum_lo[n], of_step);
                }
                // Weighted sums of the step, from zero or on the tile's.
                const auto gathered = [&](int n, int dt) {
                    if constexpr (kTileSums) return of_tile[n][dt];
                    else return pf_f32x4_t{};
                };
                const auto gather = [&](int n, int dt, const pf_f32x4_t& x) {
                    if constexpr (kTileSums) of_tile[n][dt] = x;
                    else acc[n][dt] += x;
                };
                if constexpr (kF32) {
                    // MFMA r takes token 4 * quad + r of lane (quad, col); block
                    // 4 * mm + j of O^T is dims 64 * mm + 4 * i + j, i = 0..15.
#pragma unroll
                    for (int mm = 0; mm < kD / 64; ++mm) {
                        pf_f32x4_t o[4];
#pragma unroll
                        for (int j = 0; j < 4; ++j) o[j] = gathered(0, 4 * mm + j);
#pragma unroll
                        for (int r = 0; r < 4; ++r) {
                            const float4 x = *reinterpret_cast<const float4*>(vt + (row0 + r) * kRowBytes + v_read + 256 * mm);
                            o[0] = __builtin_amdgcn_mfma_f32_16x16x4f32(x.x, pr[0][r], o[0], 0, 0, 0);
                            o[1] = __builtin_amdgcn_mfma_f32_16x16x4f32(x.y, pr[0][r], o[1], 0, 0, 0);
                            o[2] = __builtin_amdgcn_mfma_f32_16x16x4f32(x.z, pr[0][r], o[2], 0, 0, 0);
                            o[3] = __builtin_amdgcn_mfma_f32_16x16x4f32(x.w, pr[0][r], o[3], 0, 0, 0);
                        }
#pragma unroll
                        for (int j = 0; j < 4; ++j) gather(0, 4 * mm + j, o[j]);
                    }
                } else {
#pragma unroll
                    for (int dt = 0; dt < kDt; ++dt) {
                        const Vec a = kEarlyV ? vop[kEarlyV ? dt : 0] : read_v(dt);
                        pf_f32x4_t o[kN];
#pragma unroll
                        for (int n = 0; n < kN; ++n) o[n] = gathered(n, dt);
#pragma unroll
                        for (int k = 0; k < kParts; ++k)
#pragma unroll
                            for (int n = 0; n < kN; ++n) o[n] = M::mma(a, pb[n][k], o[n]);
#pragma unroll
                        for (int n = 0; n < kN; ++n) gather(n, dt, o[n]);
                    }
                }
            }
            if constexpr (kTileSums) {
#pragma unroll
                for (int n = 0; n < kN; ++n)
#pragma unroll
                    for (int dt = 0; dt < kDt; ++dt) acc[n][dt] += of_tile[n][dt];
            }
        };
        if (active) {
            if constexpr (kBlocks > 1) {
                if (blocks > 1) compute(std::integral_constant<int, kBlocks>{});
                else compute(std::integral_constant<int, 1>{});
            } else {
                compute(std::integral_constant<int, 1>{});
            }
        }
        if (next.ok && next.seg == cur.seg && next.kvh == cur.kvh && next.col_tile == cur.col_tile) continue;

        // ---- the part's partials: merged over the wavefronts that shared its
        // tokens (through the buffer just computed), then to the workspace.
        new_part = true;
        const bool is_prefix = cur.seg < p.groups;
        // Its first column's place: a row's streams are numbered, row_cols columns each.
        const std::uint32_t place_of_part =
            is_prefix ? prefix_place(p, cur.s.first_row, cur.s.cols, cur.kvh, cur.col_tile * kCols, w)
                      : (((cur.seg - p.groups) * p.heads + cur.kvh) * p.row_tiles + cur.col_tile + w) * p.row_cols;
        float sum[kBlocks], top[kBlocks];
#pragma unroll
        for (int n = 0; n < kBlocks; ++n) {
            sum[n] = sum_across_quads(sum_hi[n] + sum_lo[n]);
            top[n] = lazy[n] == -INFINITY ? -INFINITY : kScaled ? -nref[n] * down[n] : -nref[n];
        }
        if (shares > 1) {  // uniform
            // [across][token share but the first][block][dt][lane]
            auto* const scratch = reinterpret_cast<pf_f32x4_t*>(buffers[here]) + lane;
            const auto place = [&](std::uint32_t share, int n) {
                return ((across * (shares - 1) + share - 1) * blocks + n) * kDt * 64;
            };
            wait_lgkm0();
            lds_barrier();  // every wavefront is done with the buffer
            if (active && token_share != 0) {
#pragma unroll
                for (int n = 0; n < kBlocks; ++n) {
                    if (n >= static_cast<int>(blocks)) break;
                    if (quad == 0) part_ml[wave][n][col] = make_float2(top[n], sum[n]);
#pragma unroll
                    for (int dt = 0; dt < kDt; ++dt) scratch[place(token_share, n) + dt * 64] = acc[n][dt];
                }
            }
            wait_lgkm0();
            lds_barrier();
            if (active && token_share == 0) {
#pragma unroll
                for (int n = 0; n < kBlocks; ++n) {
                    if (n >= static_cast<int>(blocks)) break;
                    float all = top[n];
                    for (std::uint32_t o = 1; o < shares; ++o) all = fmaxf(all, part_ml[wave + o][n][col].x);
                    const float f0 = merge_weight(top[n], all);
                    sum[n] *= f0;
#pragma unroll
                    for (int dt = 0; dt < kDt; ++dt) acc[n][dt] *= f0;
                    for (std::uint32_t o = 1; o < shares; ++o) {
                        const float2 ml = part_ml[wave + o][n][col];
                        const float f = merge_weight(ml.x, all);
                        sum[n] = fmaf(ml.y, f, sum[n]);
#pragma unroll
                        for (int dt = 0; dt < kDt; ++dt) {
                            const pf_f32x4_t x = scratch[place(o, n) + dt * 64];
#pragma unroll
                            for (int r = 0; r < 4; ++r) acc[n][dt][r] = fmaf(x[r], f, acc[n][dt][r]);
                        }
                    }
                    top[n] = all;
                }
            }
        }
        if (active && token_share == 0) {
#pragma unroll
            for (int n = 0; n < kBlocks; ++n) {
                const std::uint32_t mine = first_col + 16 * n + col;
                if (n >= static_cast<int>(blocks) || mine >= cols) continue;
                const std::uint64_t at = place_of_part + mine;
                float* out = (is_prefix ? p.prefix_acc : p.row_acc) + at * kD;
                if (quad == 0)
                    *reinterpret_cast<float2*>((is_prefix ? p.prefix_ml : p.row_ml) + 2 * at) = make_float2(top[n], sum[n]);
                if constexpr (kF32) {
#pragma unroll
                    for (int mm = 0; mm < kD / 64; ++mm)
#pragma unroll
                        for (int r = 0; r < 4; ++r)
                            *reinterpret_cast<float4*>(out + 64 * mm + 16 * quad + 4 * r) =
                                make_float4(acc[n][4 * mm][r], acc[n][4 * mm + 1][r], acc[n][4 * mm + 2][r],
                                            acc[n][4 * mm + 3][r]);
                } else {
#pragma unroll
                    for (int dt = 0; dt < kDt; ++dt) {
                        const pf_f32x4_t x = acc[n][dt] * (1.0f / kWeightScale);  // a power of two: exact
                        *reinterpret_cast<float4*>(out + 16 * dt + 4 * quad) = make_float4(x[0], x[1], x[2], x[3]);
                    }
                }
            }
        }
    } while (next.ok || more);
}

// Merges the partials of every (row, query head): those of its prefix's stream
// and of its own, in the order of the workgroups that left them. A stream's
// workgroups are neighbours, from the one whose share its first tile starts in
// to the one of its last; one in between has a partial where a tile of the
// stream starts in its share (a share may be shorter than a tile's cost).
// Latency is all there is to it: the plan, then the partials' (m, sum) and the
// first four accumulators of every group of lanes at once, then the others four
// at a time (20 rows of 48 parts at head size 256, one load after the other:
// 15.0 us).
// Launches of more workgroups than the chip holds at once hide the latency behind
// each other: there one wavefront does it, without barriers to wait at (4096
// workgroups: 14.6 us with 256 threads).
constexpr std::uint64_t kManyMerges = 2048;
template <int kD, int kMergeThreads>
__global__ __launch_bounds__(kMergeThreads) void shared_merge_kernel(SharedParams p) {
    constexpr std::uint32_t kMost = 2 * kWorkgroups;
    constexpr int kMergeWaves = kMergeThreads / 64, kPer = kMost / kMergeThreads;
    constexpr std::uint32_t kLanes = kD / 4, kGroups = kMergeThreads / kLanes, kAhead = 4;
    struct Stream {
        std::uint32_t cost, tiles, weight, first, count;  // partials of workgroups first .. first + count - 1
        std::uint32_t slot, step;  // of workgroup w: row slot + w * step of the arrays
    };
    __shared__ Stream streams[2];  // the prefix's, the row's own
    __shared__ float weight[kMost];  // a part's factor; below 0: there is no partial
    __shared__ float wave_value[2][kMergeWaves];
    __shared__ float4 sums[kMergeThreads];
    const std::uint32_t row = blockIdx.x / p.query_heads, head = blockIdx.x % p.query_heads;
    const std::uint32_t tid = threadIdx.x, wave = tid / 64, lane = tid % 64;
    const RowPlan plan = p.plans[row];
    const std::uint32_t total = plan.total;
    for (std::uint32_t which = wave; which < 2; which += kMergeWaves) {
        const bool of_prefix = which == 0;
        const std::uint32_t kvh = p.group.div(head), g = head - kvh * p.group.divisor;
        const std::uint32_t c = of_prefix ? (row - plan.first_row) * p.group.divisor + g : g;  // column
        const std::uint32_t stream =
            kvh * (of_prefix ? (plan.prefix_cols + kCols - 1) / kCols : p.row_tiles) + c / kCols;
        Stream s;
        s.tiles = of_prefix ? plan.prefix_tiles : plan.own_tiles;
        s.weight = of_prefix ? plan.prefix_weight : plan.own_weight;
        s.cost = (of_prefix ? plan.prefix_cost : plan.own_cost) + stream * (s.tiles * s.weight + kPartCost);
        s.step = of_prefix ? kCols : p.row_cols;
        s.slot = of_prefix ? prefix_place(p, plan.first_row, plan.prefix_cols, kvh, c, 0)
                           : (row * p.heads * p.row_tiles + stream) * p.row_cols + c % kCols;
        // The workgroup in whose share a cost lies: a guess in FP32, put right.
        const float per_cost = static_cast<float>(kWorkgroups) / static_cast<float>(total);
        const auto owner = [&](std::uint32_t at) {
            auto w = static_cast<std::uint32_t>(static_cast<float>(at) * per_cost);
            if (w >= kWorkgroups) w = kWorkgroups - 1;
            while (share_begin(total, w) > at) --w;
            while (share_begin(total, w + 1) <= at) ++w;
            return w;
        };
        s.first = s.count = 0;
        if (s.tiles != 0) {
            s.first = owner(s.cost);
            s.count = owner(s.cost + tile_start(s.tiles - 1, s.weight)) - s.first + 1;
        }
        if (lane == 0) streams[which] = s;
    }
    __syncthreads();
    const std::uint32_t prefix_parts = streams[0].count, parts = prefix_parts + streams[1].count;
    // Row of part i in its arrays (past the parts: of the last one).
    const auto place = [&](std::uint32_t i, bool* of_prefix, std::uint32_t* w) {
        if (i >= parts) i = parts - 1;
        *of_prefix = i < prefix_parts;
        const Stream& s = streams[*of_prefix ? 0 : 1];
        *w = s.first + i - (*of_prefix ? 0u : prefix_parts);
        return s.slot + static_cast<std::uint64_t>(*w) * s.step;
    };
    const std::uint32_t group = tid / kLanes, d4 = tid % kLanes;
    const auto accumulator = [&](std::uint32_t i) {
        bool of_prefix;
        std::uint32_t w;
        const std::uint64_t at = place(i, &of_prefix, &w);
        return *reinterpret_cast<const float4*>((of_prefix ? p.prefix_acc : p.row_acc) + at * kD + 4 * d4);
    };
    float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    float sum = 0.0f;
    if (parts != 0) {  // uniform
        float4 ahead[kAhead];
#pragma unroll
        for (std::uint32_t u = 0; u < kAhead; ++u) ahead[u] = accumulator(group + u * kGroups);
        float m[kPer], l[kPer];  // a thread's parts: tid + k * kMergeThreads
        float top = -INFINITY;
#pragma unroll
        for (int k = 0; k < kPer; ++k) {
            m[k] = -INFINITY;
            l[k] = -1.0f;  // sums are never negative
            if (k * kMergeThreads >= parts) break;  // uniform
            bool of_prefix;
            std::uint32_t w;
            const std::uint64_t at = place(tid + k * kMergeThreads, &of_prefix, &w);
            const float2 ml = *reinterpret_cast<const float2*>((of_prefix ? p.prefix_ml : p.row_ml) + 2 * at);
            const Stream& s = streams[of_prefix ? 0 : 1];
            const std::uint32_t begin = share_begin(total, w);
            const std::uint32_t t = tiles_before(begin > s.cost ? begin - s.cost : 0, s.weight);
            const bool there = tid + k * kMergeThreads < parts && t < s.tiles &&
                               s.cost + tile_start(t, s.weight) < share_begin(total, w + 1);
            m[k] = there ? ml.x : -INFINITY;
            l[k] = there ? ml.y : -1.0f;
            top = fmaxf(top, m[k]);
        }
#pragma unroll
        for (int x = 1; x < 64; x <<= 1) top = fmaxf(top, __shfl_xor(top, x));
        if (lane == 0) wave_value[0][wave] = top;
        __syncthreads();
#pragma unroll
        for (int x = 0; x < kMergeWaves; ++x) top = fmaxf(top, wave_value[0][x]);
#pragma unroll
        for (int k = 0; k < kPer; ++k) {
            if (k * kMergeThreads >= parts) break;  // uniform
            const float f = merge_weight(m[k], top);
            if (l[k] != -1.0f) sum = fmaf(l[k], f, sum);
            weight[tid + k * kMergeThreads] = l[k] != -1.0f ? f : -1.0f;
        }
#pragma unroll
        for (int x = 1; x < 64; x <<= 1) sum += __shfl_xor(sum, x);
        if (lane == 0) wave_value[1][wave] = sum;
        __syncthreads();
        sum = 0.0f;
#pragma unroll
        for (int x = 0; x < kMergeWaves; ++x) sum += wave_value[1][x];
#pragma unroll 1
        for (std::uint32_t i = group;; i += kAhead * kGroups) {
#pragma unroll
            for (std::uint32_t u = 0; u < kAhead; ++u) {
                const std::uint32_t part = i + u * kGroups;
                const float f = part < parts ? weight[part] : -1.0f;
                if (f >= 0.0f) {
                    o.x = fmaf(ahead[u].x, f, o.x);
                    o.y = fmaf(ahead[u].y, f, o.y);
                    o.z = fmaf(ahead[u].z, f, o.z);
                    o.w = fmaf(ahead[u].w, f, o.w);
                }
            }
            if (i + kAhead * kGroups >= parts) break;
#pragma unroll
            for (std::uint32_t u = 0; u < kAhead; ++u) ahead[u] = accumulator(i + (kAhead + u) * kGroups);
        }
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
    std::uint64_t prefix_acc = 0, prefix_ml = 0, row_acc = 0, row_ml = 0, bytes = 0;
};

// Whether the shared kernel can take a call's shape; others run as an ordinary
// decode batch (the same results: a shared page is only read more often).
bool can_take(std::uint64_t rows, std::uint64_t kv_len, std::uint64_t kv_heads, std::uint64_t query_heads,
           std::uint64_t block_size, std::uint64_t head_size, int dtype, std::uint64_t groups) {
    if (groups == 0 || groups > kMaxGroups || rows > kMaxRows) return false;
    if (head_size != 64 && head_size != 128 && (head_size != 256 || dtype == KVFLUX_DTYPE_F32)) return false;
    if (kv_len >= 0x80000000ULL || block_size >= 0x80000000ULL || kv_heads > 65535 || query_heads > 65535) return false;
    if (rows * query_heads >= (1ULL << 24)) return false;  // workgroups of the merge
    // Costs are summed in 32 bits; a tile has 64 tokens at least.
    const std::uint64_t group = query_heads / kv_heads;
    const std::uint64_t streams = kv_heads * (rows * ((group + kCols - 1) / kCols) + groups + rows * group / kCols);
    return streams * (kv_len / 64 + 1) < (1ULL << 31) / (kMostTileCost + kPartCost);
}

// Whether sharing pays: `again` is the tokens that an ordinary decode reads again,
// once for every further row of a group, from L2, at about 9 MB a microsecond; the
// shared kernel pays its plan and merge, about 5 us, and for every row
// and kv head a part of its own, of which a round of the workgroups takes about
// 4.5 us more than the ordinary decode's items. Measured, shared and ordinary:
// 17 rows in 2 groups behind 1500-2500 tokens, 28/4 heads of 128 (77 MB read again) 23.8
// and 25.3 us; 27 in 2 behind up to 7061, 32/8 (723 MB) 25.1 and 35.9; 34 in 4 behind
// 347, 24/8 (43 MB) 21.7 and 15.0; 116 in 11 behind 423, 24/8 (182 MB) 34.8 and 30.7; 60
// in 3 behind 221, 40/8 heads of 64 (26 MB) 28.9 and 9.8.
bool pays(std::uint64_t rows, double again, std::uint64_t kv_heads, std::uint64_t head_size, int dtype) {
    return again * static_cast<double>(2 * kv_heads * head_size * dtype_bytes(dtype)) >
           9e6 * (5.0 + 4.5 * static_cast<double>(rows * kv_heads) / kWorkgroups);
}
// What a caller of the attention's entry has read again at the most: every row but
// one of a group behind the longest prefix.
double most_again(std::uint64_t rows, std::uint64_t groups, std::uint64_t max_prefix, std::uint64_t kv_len) {
    if (rows <= groups) return 0.0;
    return static_cast<double>(rows - groups) * static_cast<double>(max_prefix < kv_len ? max_prefix : kv_len);
}

Layout layout_of(std::uint64_t rows, std::uint64_t kv_heads, std::uint64_t query_heads, std::uint64_t head_size) {
    const auto whole = [](std::uint64_t bytes) { return (bytes + 255) & ~std::uint64_t{255}; };
    const std::uint64_t group = query_heads / kv_heads;
    const std::uint64_t prefix_columns = rows * query_heads + kWorkgroups * kCols;
    const std::uint64_t row_slots = rows * kv_heads * ((group + kCols - 1) / kCols) + kWorkgroups;
    const std::uint64_t row_cols = group < kCols ? group : kCols;
    Layout l;
    l.prefix_acc = whole(rows * sizeof(RowPlan));  // the plans come first
    l.prefix_ml = l.prefix_acc + whole(prefix_columns * head_size * sizeof(float));
    l.row_acc = l.prefix_ml + whole(prefix_columns * 2 * sizeof(float));
    l.row_ml = l.row_acc + whole(row_slots * row_cols * head_size * sizeof(float));
    l.bytes = l.row_ml + whole(row_slots * row_cols * 2 * sizeof(float));
    return l;
}

template <typename E, int kD>
int launch(const SharedParams& p, hipStream_t s) {
    if (p.block_size.divisor % 16 == 0)
        hipLaunchKernelGGL((shared_attention_kernel<E, kD, true>), dim3(kWorkgroups), dim3(kThreads), 0, s, p);
    else
        hipLaunchKernelGGL((shared_attention_kernel<E, kD, false>), dim3(kWorkgroups), dim3(kThreads), 0, s, p);
    const int status = launch_status("shared_attention_kernel");
    if (status != KVFLUX_OK) return status;
    const unsigned merges = p.rows * p.query_heads;
    if (merges > kManyMerges)
        hipLaunchKernelGGL((shared_merge_kernel<kD, 64>), dim3(merges), dim3(64), 0, s, p);
    else
        hipLaunchKernelGGL((shared_merge_kernel<kD, 256>), dim3(merges), dim3(256), 0, s, p);
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
    int status = check_shape(num_kv_heads, block_size, head_size, dtype, query_heads);
    if (status != KVFLUX_OK) return status;
    status = kvflux_paged_attention_workspace_size(num_rows, kv_len, num_kv_heads, query_heads, block_size, head_size, bytes);
    if (status != KVFLUX_OK) return status;
    if (can_take(num_rows, kv_len, num_kv_heads, query_heads, block_size, head_size, dtype, num_groups)) {
        const std::uint64_t need = layout_of(num_rows, num_kv_heads, query_heads, head_size).bytes;
        if (need > *bytes) *bytes = need;
    }
    return KVFLUX_OK;
}

extern "C" int kvflux_paged_attention_shared_pays(uint64_t num_rows, uint64_t kv_len, uint64_t num_kv_heads,
                                                  uint64_t query_heads, uint64_t block_size, uint64_t head_size,
                                                  int dtype, uint64_t num_groups, uint64_t shared_tokens, int* result) {
    if (!result) return fail(KVFLUX_ERR_INVALID_ARGUMENT, "pays is null");
    *result = 0;
    const int status = check_shape(num_kv_heads, block_size, head_size, dtype, query_heads);
    if (status != KVFLUX_OK) return status;
    *result = can_take(num_rows, kv_len, num_kv_heads, query_heads, block_size, head_size, dtype, num_groups) &&
              pays(num_rows, static_cast<double>(shared_tokens), num_kv_heads, head_size, dtype);
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
    if (!can_take(num_rows, kv_len, num_kv_heads, query_heads, block_size, head_size, dtype, num_groups) ||
        !pays(num_rows, most_again(num_rows, num_groups, max_prefix, kv_len), num_kv_heads, head_size, dtype))
        return kvflux_paged_attention(key_cache, value_cache, num_blocks, num_kv_heads, block_size, head_size, dtype,
                                      block_table, max_blocks_per_seq, seq_lens, kv_len, num_rows, query_heads, query,
                                      output, workspace, workspace_bytes, stream);
    const Layout l = layout_of(num_rows, num_kv_heads, query_heads, head_size);
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
    p.plans = reinterpret_cast<RowPlan*>(base);
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
