// Decode attention straight from a paged cache held in 8 bits with a scale for each
// page and kv head: for a row's query head and its tokens t < len
//   s_t = ks_t (q . k_t) / sqrt(D),  o = sum_t e^(s_t - m) vs_t v_t / sum_t e^(s_t - m)
// with ks_t, vs_t the scales of the token's page. FP32 queries, sums and outputs.
//
// What bounds it is the reading of K and V, one byte a value: half the time of a
// 16-bit cache is left for the same arithmetic. So
//  * K and V are read past the caches, whole 128-byte lines by one instruction, two
//    tiles ahead, and reach the matrix instructions through a wavefront's own LDS
//    (no barrier). 128 rows of <= 32768 tokens, 8 kv heads of 128: 730 us, 6.4 TB/s,
//    where loads alone take 705. The step to it (805 to 747) was from loads in the
//    operands' own layout, which split lines; without the streaming hint it took 1611 us;
//  * bytes are widened in registers, one conversion for two values; both formats are
//    exact in FP16;
//  * the products are FP16 MFMAs with FP32 sums, on Q and the weights in two FP16
//    parts: x = hi + lo, off by at most 2^-23 of x (half a step of hi is 2^-12, and
//    lo has 11 bits of what is left), the size of FP32's own rounding;
//  * the scales are not multiplied into K and V: a score is multiplied once by its
//    page's ks, and a weight by its vs;
//  * a wavefront's tile is 32 tokens of one kv head: all query heads of the group
//    are columns (up to 16), S^T = K Q^T and O^T += V^T P^T on 16x16x32. Row i of
//    K's block b is token 8 (i / 4) + 4 b + i % 4, so that lane (quad, col) holds the
//    scores of tokens 8 quad .. 8 quad + 7: the second product's operand as it is.
//    V's operand wants eight tokens of one dim in a lane: the transposing LDS read.
//
// The work of a call is a list of streams, a row's tokens for one kv head (and up to
// 16 of its query heads), cut into equal shares: workgroup w of N takes the tiles
// whose place in the sum of all costs lies in [wT/N, (w+1)T/N). Rows of any mix of
// lengths are spread evenly; at most N - 1 streams are cut, and a second kernel
// merges the parts of those.
#include "mfma_parts.h"
#include "quant.h"

#include <cmath>
#include <type_traits>

namespace kvflux_hip {
namespace {

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / 64;
constexpr std::uint32_t kTile = 32;       // tokens of a wavefront's step
constexpr std::uint32_t kCols = 16;       // query heads of a stream
constexpr std::uint32_t kPlanRows = 2048; // rows of a launch
// Cost of a part's start and end (a chain of loads, 4 us) in tiles of a workgroup. At 4
// and at 16: 4 rows of <= 1500 tokens 14.7 and 12.3 us, 16 rows of <= 8192 27.5 and 25.3,
// 256 rows of <= 1024 80 and 67, 128 rows of <= 32768 742 and 722; 28 is behind again.
constexpr std::uint32_t kPartCost = 16;
// The least of a share: fewer workgroups start where there is less to do. 4 rows of
// <= 1500 tokens: 6 16.4 us, 8 12.3, 10 13.2, 16 13.8.
constexpr std::uint32_t kLeastShare = 8;
// Rows of at most this many tokens (half of it with heads of 256, or where tokens have a
// record each: 8 rows of <= 1000 tokens on 5-token pages 14.9 and 12.0 us) take one workgroup
// a stream and no merge; twice as many where the streams fill the GPU by themselves.
// A workgroup a stream, and shares: 1 row of <= 1024 tokens 8.9 and 11.5 us, 8 rows 13.0
// and 14.2, 256 rows 67.6 and 75.7; 32 rows of <= 2048 21.1 and 24.2, but 8 rows 20.4 and
// 14.8, and 128 rows of <= 4096 108 and 102.
constexpr std::uint64_t kOneLaunch = 1024;
constexpr std::uint64_t kFullStreams = 256;
// The weights' FP16 parts are of 2^15 times a weight of at most 1: FP16 ends at 2^-24,
// so two parts miss a weight by at most 2^-40 of the largest, or 2^-23 of itself.
constexpr float kWeightScale = 32768.0f;
// Tiles of a wavefront after which its sums are folded into a second set, with the addition's
// rounding error kept. A tile's sum is added to the accumulator in FP32: beside a dominant key's
// value one that is under half a step is lost, 2^-24 a tile at most, so 4e-6 of a row for 64
// (rows of 65536 tokens without: 3e-5). Parts that are never longer do without the registers:
// 16 rows of <= 8192 tokens 23.0 us, with the second set 24.0; 128 rows of <= 32768 722 and 723.
constexpr std::uint32_t kFold = 64;

typedef __attribute__((ext_vector_type(2))) int qd_i32x2_t;
typedef __attribute__((address_space(3))) qd_i32x2_t qd_lds_i32x2_t;

struct QuantDecodeParams {
    const std::uint8_t* key_cache;
    const std::uint8_t* value_cache;
    const float* key_scales;
    const float* value_scales;
    std::uint64_t num_blocks;
    std::uint32_t heads;          // kv heads
    std::uint32_t head_size;      // a multiple of 16, at most kD
    FastDiv block_size;
    const std::uint64_t* table;   // [rows][width]
    std::uint64_t width;
    const std::uint64_t* lens;
    std::uint32_t kv_len;         // bound of every length
    std::uint32_t row_base, rows; // of this launch
    std::uint32_t query_heads;
    std::uint32_t group;          // query heads per kv head
    std::uint32_t sets, set_heads;  // streams of a (row, kv head), query heads of each but the last
    const float* query;
    float* output;
    float scale_log2;             // log2(e) / sqrt(head_size)
    // Workspace: the streams that are cut, and two partials of every workgroup.
    std::uint32_t by_stream;      // a cut for every stream, else for every workgroup
    uint2* cuts;                  // [grid] {stream, or the workgroup that begins it; the last workgroup}, {~0, .}: none
    float* part_acc;              // [2 * grid][set_heads][kD]
    float* part_ml;               // [2 * grid][set_heads][2]
};

// exp2(m - top) for merging: 0 for a side that saw no key.
__device__ inline float merge_weight(float m, float top) {
    return m == -INFINITY ? 0.0f : m == top ? 1.0f : __builtin_amdgcn_exp2f(m - top);
}

// A caller's FP32 arrays are only known to be float-aligned.
struct Float4 { float x, y, z, w; };

// A record is what the lanes of a wavefront know of kSub tokens of a tile: where the
// first one's K and V rows lie in the caches and how many of them count (above bit 56);
// ks, and vs over the wavefront's reference times kWeightScale.
constexpr int kCountShift = 56;
constexpr std::uint64_t kOffsetMask = (std::uint64_t{1} << kCountShift) - 1;

template <int kD>
struct Shape {
    static constexpr int kSteps = kD / 32;   // MFMAs of a 16-token block of S^T for one part of Q
    static constexpr int kDt = kD / 16;      // MFMAs of O^T for one part of the weights
    static constexpr int kCpr = kD / 16;     // 16-byte chunks of a row
    static constexpr int kLoads = kCpr / 2;  // loads of a tile's K (and V) by a wavefront
    static constexpr int kRowsOf = 64 / kCpr;  // rows of a load
    static constexpr int kPad = kD + 4;      // floats of a row of the merge buffer
    // LDS of a wavefront: its tile, K then V, and at a part's end its sums.
    static constexpr int kTileBytes = 2 * static_cast<int>(kTile) * kD;
    static constexpr int kWaveBytes = kTileBytes > static_cast<int>(kCols) * kPad * 4 ? kTileBytes : static_cast<int>(kCols) * kPad * 4;
    static constexpr int kResident = kD == 256 ? 1 : 2;  // workgroups of a CU
    static constexpr std::uint32_t kGrid = 256 * kResident;
};

// kSub: tokens that share a record. 8 where pages are multiples of 8 tokens, so that
// every 8 tokens of a tile lie in one; 1 for pages of any other size.
// kWhole: a workgroup takes one whole stream (no shares, no partials).
// kFolds: a wavefront may have more than kFold tiles of a part.
// kFull: head_size is kD (as a value of the launch it cost 4 rows of <= 1500 tokens 0.5 us of 12.4).
template <typename F, int kD, int kSub, bool kWhole, int kW, bool kFolds, bool kFull>
__global__ __launch_bounds__(64 * kW, Shape<kD>::kResident) void quant_decode_kernel(QuantDecodeParams p) {
    using S = Shape<kD>;
    constexpr int kT = 64 * kW;
    using Vec = pf_f16x8_t;
    constexpr int kSteps = S::kSteps, kDt = S::kDt, kCpr = S::kCpr, kLoads = S::kLoads, kRowsOf = S::kRowsOf;
    constexpr std::uint32_t kPerTile = kTile / kSub;      // records of a tile
    constexpr std::uint32_t kBatch = 64 / kPerTile;       // tiles whose records the lanes make at once
    __shared__ std::uint64_t before[kWhole ? 1 : kPlanRows + 1];  // costs of a stream of each row before
    __shared__ std::uint32_t lens_of[kWhole ? 1 : kPlanRows];
    __shared__ std::uint64_t wave_cost[kW];
    __shared__ std::uint64_t places[kW][2][64];
    __shared__ float2 scales_of[kW][2][64];
    __shared__ __attribute__((aligned(16))) unsigned char wave_lds[kW][S::kWaveBytes];
    __shared__ float2 stats[kW][kCols];

    const int tid = threadIdx.x, lane = tid % 64;
    const auto uniform = [](std::uint32_t x) {
        return static_cast<std::uint32_t>(__builtin_amdgcn_readfirstlane(static_cast<int>(x)));
    };
    const std::uint32_t wave = uniform(tid / 64);
    const int col = lane % 16, quad = lane / 16;
    const std::uint32_t bs = p.block_size.divisor, D = kFull ? kD : p.head_size;
    const auto length = [&](std::uint32_t row) {
        const std::uint64_t n = p.lens[p.row_base + row];
        return n < p.kv_len ? static_cast<std::uint32_t>(n) : p.kv_len;
    };
    const auto tiles_of = [](std::uint32_t len) { return len == 0 ? 0u : (len - 1) / kTile + 1; };

    // One part: tiles [t0, t1) of a stream. Leaves the sums of its heads in `to`
    // (rows of kD floats): divided by the weights' sums, or with maximum and sum
    // in `ml`.
    const auto run_part = [&](std::uint32_t row, std::uint32_t len, std::uint32_t kvh, std::uint32_t set, std::uint32_t t0,
                              std::uint32_t t1, float* to, float* ml) {
        const std::uint32_t tiles = t1 - t0 > wave ? (t1 - t0 - wave + kW - 1) / kW : 0;  // of this wavefront
        const std::uint32_t first_head = set * p.set_heads;
        const std::uint32_t heads = p.group - first_head < p.set_heads ? p.group - first_head : p.set_heads;
        const std::uint64_t* const table_row = p.table + (static_cast<std::uint64_t>(p.row_base) + row) * p.width;

        pf_f32x4_t acc[kDt];
#pragma unroll
        for (int dt = 0; dt < kDt; ++dt) acc[dt] = pf_f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
        // The sums of the tiles folded so far; acc goes on from what that rounding left.
        constexpr int kFolded = kFolds ? kDt : 0;
        pf_f32x4_t base[kFolds ? kDt : 1];
#pragma unroll
        for (int dt = 0; dt < kFolded; ++dt) base[dt] = pf_f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
        float run_max = -INFINITY, run_sum = 0.0f, run_low = 0.0f;
        float value_ref = 1.0f;  // acc is in units of this over kWeightScale

        if (tiles != 0) {  // uniform in the wavefront
            // Lane l makes record l % kPerTile of tile l / kPerTile of a batch.
            const auto token_of = [&](std::uint32_t batch) {
                const std::uint32_t j = batch * kBatch + lane / kPerTile;
                // Past the wavefront's tiles: at or behind the row's end.
                return j < tiles ? (t0 + wave + kW * j) * kTile + lane % kPerTile * kSub : ~0u;
            };
            const auto fetch_page = [&](std::uint32_t batch) {
                const std::uint32_t token = token_of(batch);
                const std::uint64_t page = p.block_size.div(token);
                const bool live = token < len && page < p.width;
                const std::uint64_t id = table_row[live ? page : 0];
                return live && id < p.num_blocks ? id : ~0ull;
            };
            struct Scales { float k, v; };
            const auto fetch_scales = [&](std::uint64_t id) {
                const std::uint64_t at = (id == ~0ull ? 0 : id) * p.heads + kvh;
                return Scales{p.key_scales[at], p.value_scales[at]};
            };
            const auto put_places = [&](std::uint32_t batch, std::uint64_t id) {
                const std::uint32_t token = token_of(batch);
                std::uint64_t at = 0;
                if (id != ~0ull) {
                    const std::uint32_t count = len - token < kSub ? len - token : kSub;
                    at = ((id * p.heads + kvh) * bs + p.block_size.mod(token)) * D | static_cast<std::uint64_t>(count) << kCountShift;
                }
                places[wave][batch & 1][lane] = at;
                __builtin_amdgcn_wave_barrier();  // a wavefront's LDS accesses are in order
            };
            float next_ref = 0.0f;
            const auto put_scales = [&](std::uint32_t batch, std::uint64_t id, const Scales& s) {
                const bool live = id != ~0ull;
                const float mine = live ? s.v : 0.0f;
                next_ref = fmaxf(next_ref, wave_max(__builtin_fabsf(mine)));
                scales_of[wave][batch & 1][lane] = make_float2(live ? s.k : 0.0f, next_ref > 0.0f ? mine / next_ref * kWeightScale : mine);
                __builtin_amdgcn_wave_barrier();
            };

            struct Tile {
                uint4 k[kLoads], v[kLoads];
            };
            // Load i of a tile: kRowsOf whole rows, 16 bytes a lane; every 128-byte line is
            // read by one instruction, so both caches are streamed past the others. Every
            // load is unconditional: places past the last tile lead to the pool's first rows.
            // A lane past the head's end reads its first chunk: what is made of it meets queries
            // of 0, or is an output that is not stored.
            const std::uint32_t my_row = static_cast<std::uint32_t>(lane) / kCpr, my_chunk = static_cast<std::uint32_t>(lane) % kCpr;
            const std::uint32_t my_byte = my_chunk * 16 < D ? my_chunk * 16 : 0;
            const auto load = [&](std::uint32_t j, Tile& b) {
                const std::uint64_t* const r = places[wave][j / kBatch & 1] + j % kBatch * kPerTile;
#pragma unroll
                for (int i = 0; i < kLoads; ++i) {
                    std::uint64_t at;
                    if constexpr (kSub == 8 && kRowsOf <= 8) {  // one place for all lanes
                        const std::uint64_t x = r[i * kRowsOf / 8];
                        const std::uint32_t lo = uniform(static_cast<std::uint32_t>(x)), hi = uniform(static_cast<std::uint32_t>(x >> 32));
                        at = ((static_cast<std::uint64_t>(hi) << 32 | lo) & kOffsetMask) + i * kRowsOf % 8 * D + (my_row * D + my_byte);
                    } else {
                        const std::uint32_t token = i * kRowsOf + my_row;
                        at = (r[token / kSub] & kOffsetMask) + token % kSub * D + my_byte;
                    }
                    b.k[i] = __builtin_bit_cast(uint4, stream_load(reinterpret_cast<const V16*>(p.key_cache + at)));
                    b.v[i] = __builtin_bit_cast(uint4, stream_load(reinterpret_cast<const V16*>(p.value_cache + at)));
                }
            };
            std::uint64_t page_now = fetch_page(0);
            std::uint64_t page_next = fetch_page(1);
            put_places(0, page_now);
            Scales scales_now = fetch_scales(page_now);

            // Queries: column `col` is head col of the set (the others repeat the
            // last), lane (quad, col) holds dims 64 m + 16 quad + 8 h of step 2 m + h,
            // as K's rows are loaded. FP16 parts end at 2^-24 and 65504, so a column
            // is split times a power of two, undone with its scores' scale.
            Vec q_hi[kSteps], q_lo[kSteps];
            float down;
            Tile b0, b1;
            {
                const std::uint32_t head = kvh * p.group + first_head + (static_cast<std::uint32_t>(col) < heads ? col : heads - 1);
                const float* const src = p.query + ((static_cast<std::uint64_t>(p.row_base) + row) * p.query_heads + head) * D;
                Float4 raw[kSteps][2];
#pragma unroll
                for (int kk = 0; kk < kSteps; ++kk)
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        const std::uint32_t at = 64 * (kk / 2) + 8 * (kk % 2) + 4 * i;
                        raw[kk][i] = Float4{0.0f, 0.0f, 0.0f, 0.0f};
                        if (kFull || at + 16 * quad < D) raw[kk][i] = *reinterpret_cast<const Float4*>(src + 16 * quad + at);
                    }
                load(0, b0);
                load(1, b1);
                float largest = 0.0f;
#pragma unroll
                for (int kk = 0; kk < kSteps; ++kk)
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        const Float4 x = raw[kk][i];
                        largest = max3(largest, __builtin_fabsf(x.x), __builtin_fabsf(x.y));
                        largest = max3(largest, __builtin_fabsf(x.z), __builtin_fabsf(x.w));
                    }
                const int e = split_exponent(max_across_quads(largest) * p.scale_log2);
                const float up = __builtin_amdgcn_ldexpf(1.0f, e);
                down = __builtin_amdgcn_ldexpf(1.0f, -e);
#pragma unroll
                for (int kk = 0; kk < kSteps; ++kk) {
                    std::uint32_t hi[4], lo[4];
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        const Float4 x = raw[kk][i];
                        const float v[4] = {x.x * p.scale_log2 * up, x.y * p.scale_log2 * up, x.z * p.scale_log2 * up,
                                            x.w * p.scale_log2 * up};
#pragma unroll
                        for (int j = 0; j < 2; ++j) {
                            const pf_f32x2_t y{v[2 * j], v[2 * j + 1]};
                            const pf_f16x2_t h = __builtin_convertvector(y, pf_f16x2_t);
                            hi[2 * i + j] = __builtin_bit_cast(std::uint32_t, h);
                            const pf_f32x2_t rest = y - __builtin_convertvector(h, pf_f32x2_t);
                            lo[2 * i + j] = __builtin_bit_cast(std::uint32_t, __builtin_convertvector(rest, pf_f16x2_t));
                        }
                    }
                    q_hi[kk] = __builtin_bit_cast(Vec, make_uint4(hi[0], hi[1], hi[2], hi[3]));
                    q_lo[kk] = __builtin_bit_cast(Vec, make_uint4(lo[0], lo[1], lo[2], lo[3]));
                }
                put_scales(0, page_now, scales_now);
                if (next_ref > 0.0f) value_ref = next_ref;  // else all are 0 or NaN, in any unit
            }
            page_now = page_next;
            scales_now = fetch_scales(page_now);
            page_next = fetch_page(2);
            // Places and scales of batch `b`, and the fetches for the ones behind it.
            const auto stage = [&](std::uint32_t b) {
                put_places(b, page_now);
                put_scales(b, page_now, scales_now);
                page_now = page_next;
                scales_now = fetch_scales(page_now);
                page_next = fetch_page(b + 2);
            };

            // Rows of a tile in LDS: chunk c of row t at slot c ^ f(t), so that the rows of a
            // read fall on different banks: K 16 rows of one chunk (8 at a time, see the
            // order of tokens), V 8 rows of one chunk.
            unsigned char* const k_lds = wave_lds[wave];
            unsigned char* const v_lds = k_lds + kTile * kD;
            const auto k_slot = [](std::uint32_t t, std::uint32_t c) {
                return c ^ (kCpr == 4 ? (t >> 1 & 1) | (t >> 3 & 1) << 1 : (t & 3) | (t >> 3 & 1) << 2);
            };
            const auto v_slot = [](std::uint32_t t, std::uint32_t c) { return c ^ (kCpr == 4 ? t >> 1 & 3 : t & 7); };
            const auto compute = [&](std::uint32_t j, Tile& b) {
                const std::uint64_t* const r = places[wave][j / kBatch & 1] + j % kBatch * kPerTile;
                const float2* const rs = scales_of[wave][j / kBatch & 1] + j % kBatch * kPerTile;
                if (j % kBatch == 0 && value_ref != next_ref && next_ref > 0.0f) {  // uniform
                    const float f = value_ref / next_ref;
#pragma unroll
                    for (int dt = 0; dt < kDt; ++dt) acc[dt] *= f;
#pragma unroll
                    for (int dt = 0; dt < kFolded; ++dt) base[dt] *= f;
                    value_ref = next_ref;
                }
                // Per token of the lane's eight, or one for all of them.
                constexpr int kOwn = kSub == 8 ? 1 : 8;
                float ks[kOwn], vs[kOwn];
                std::uint32_t live = 0;  // a bit for each of the eight that count
#pragma unroll
                for (int i = 0; i < kOwn; ++i) {
                    const int at = kSub == 8 ? quad : 8 * quad + i;
                    const float2 x = rs[at];
                    const float k = x.x * down;
                    ks[i] = k > 3.0e38f ? 3.0e38f : k;  // finite: a product of 0 stays 0
                    vs[i] = x.y;
                    const std::uint32_t count = static_cast<std::uint32_t>(r[at] >> kCountShift);
                    live |= ((1u << count) - 1) << i;
                }
                const bool part = __builtin_amdgcn_ballot_w64(live != 0xffu) != 0;  // a row's end, or a missing page
#pragma unroll
                for (int i = 0; i < kLoads; ++i) {
                    const std::uint32_t t = i * kRowsOf + my_row;
                    *reinterpret_cast<uint4*>(k_lds + t * kD + 16 * k_slot(t, my_chunk)) = b.k[i];
                    *reinterpret_cast<uint4*>(v_lds + t * kD + 16 * v_slot(t, my_chunk)) = b.v[i];
                    if (part) {  // uniform; 0 * NaN would stay
                        const std::uint32_t count = static_cast<std::uint32_t>(r[kSub == 8 ? t / 8 : t] >> kCountShift);
                        if (t % kSub >= count) *reinterpret_cast<uint4*>(v_lds + t * kD + 16 * v_slot(t, my_chunk)) = make_uint4(0, 0, 0, 0);
                    }
                }
                __builtin_amdgcn_wave_barrier();
                pf_f32x4_t s[2];
#pragma unroll
                for (int blk = 0; blk < 2; ++blk) {
                    s[blk] = pf_f32x4_t{0.0f, 0.0f, 0.0f, 0.0f};
                    Vec a[kSteps];
                    const std::uint32_t t = 8 * (col / 4) + 4 * blk + col % 4;
#pragma unroll
                    for (int m = 0; m < kSteps / 2; ++m) {
                        const uint4 w = *reinterpret_cast<const uint4*>(k_lds + t * kD + 16 * k_slot(t, 4 * m + quad));
                        a[2 * m] = __builtin_bit_cast(Vec, make_uint4(F::template pair16<0>(w.x), F::template pair16<1>(w.x),
                                                                      F::template pair16<0>(w.y), F::template pair16<1>(w.y)));
                        a[2 * m + 1] = __builtin_bit_cast(Vec, make_uint4(F::template pair16<0>(w.z), F::template pair16<1>(w.z),
                                                                          F::template pair16<0>(w.w), F::template pair16<1>(w.w)));
                    }
#pragma unroll
                    for (int kk = 0; kk < kSteps; ++kk) s[blk] = PfF16::mma(a[kk], q_lo[kk], s[blk]);
#pragma unroll
                    for (int kk = 0; kk < kSteps; ++kk) s[blk] = PfF16::mma(a[kk], q_hi[kk], s[blk]);
                }
                float x[8];
#pragma unroll
                for (int t = 0; t < 8; ++t) x[t] = s[t / 4][t % 4] * ks[kSub == 8 ? 0 : t];
                if (part) {  // uniform
#pragma unroll
                    for (int t = 0; t < 8; ++t)
                        if (!(live >> t & 1)) x[t] = -INFINITY;
                }
                const float top = max3(max3(x[0], x[1], x[2]), max3(x[3], x[4], x[5]), __builtin_elementwise_maximum(x[6], x[7]));
                if (__builtin_expect(__builtin_amdgcn_ballot_w64(top > run_max) != 0, 0)) {  // uniform
                    const float all = max_across_quads(top);
                    const float next = all > run_max ? all : run_max;
                    const float f = run_max == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(run_max - next);
                    run_max = next;
                    run_sum *= f;
                    run_low *= f;
#pragma unroll
                    for (int dt = 0; dt < kDt; ++dt) acc[dt] *= f;
#pragma unroll
                    for (int dt = 0; dt < kFolded; ++dt) base[dt] *= f;
                }
                const float ref = run_max == -INFINITY ? 0.0f : run_max;
                std::uint32_t hi[4], lo[4];
                float w[8], sum = 0.0f;
#pragma unroll
                for (int t = 0; t < 8; ++t) {
                    w[t] = __builtin_amdgcn_exp2f(x[t] - ref);
                    sum += w[t];
                }
                two_sum_add(run_sum, run_low, sum);
#pragma unroll
                for (int t = 0; t < 4; ++t) {
                    const pf_f32x2_t y{w[2 * t] * vs[kSub == 8 ? 0 : 2 * t], w[2 * t + 1] * vs[kSub == 8 ? 0 : 2 * t + 1]};
                    const pf_f16x2_t h = __builtin_convertvector(y, pf_f16x2_t);
                    hi[t] = __builtin_bit_cast(std::uint32_t, h);
                    const pf_f32x2_t rest = y - __builtin_convertvector(h, pf_f32x2_t);
                    lo[t] = __builtin_bit_cast(std::uint32_t, __builtin_convertvector(rest, pf_f16x2_t));
                }
                const Vec p_hi = __builtin_bit_cast(Vec, make_uint4(hi[0], hi[1], hi[2], hi[3]));
                const Vec p_lo = __builtin_bit_cast(Vec, make_uint4(lo[0], lo[1], lo[2], lo[3]));
                // V^T: a group of 16 lanes reads 8 tokens of 16 dims and leaves lane i with the
                // tokens of dim i. A tile's products are summed from zero and added with one
                // rounding: an MFMA on an accumulator that holds a dominant key's sum drops
                // bits of the small weights, always in the same direction.
                const std::uint32_t row = 8 * quad + col / 2;
#pragma unroll
                for (int dt = 0; dt < kDt; ++dt) {
                    const auto w = __builtin_amdgcn_ds_read_tr8_b64_v2i32(
                        (qd_lds_i32x2_t*)((__attribute__((address_space(3))) unsigned char*)v_lds + row * kD + 16 * v_slot(row, dt) + col % 2 * 8));
                    const auto lo = static_cast<std::uint32_t>(w[0]), hi = static_cast<std::uint32_t>(w[1]);
                    const Vec a = __builtin_bit_cast(Vec, make_uint4(F::template pair16<0>(lo), F::template pair16<1>(lo),
                                                                     F::template pair16<0>(hi), F::template pair16<1>(hi)));
                    acc[dt] += PfF16::mma(a, p_hi, PfF16::mma(a, p_lo, pf_f32x4_t{0.0f, 0.0f, 0.0f, 0.0f}));
                }
            };

#pragma unroll 1
            for (std::uint32_t j = 0; j < tiles; j += 2) {
                compute(j, b0);
                if ((j + 2) % kBatch == 0) stage((j + 2) / kBatch);
                load(j + 2, b0);
                if (j + 1 < tiles) compute(j + 1, b1);
                load(j + 3, b1);
                if (kFolds && j % kFold == kFold - 2) {  // uniform
#pragma unroll
                    for (int dt = 0; dt < kFolded; ++dt)
#pragma unroll
                        for (int r = 0; r < 4; ++r) {
                            float sum = base[dt][r], rest = 0.0f;
                            two_sum_add(sum, rest, acc[dt][r]);
                            base[dt][r] = sum;
                            acc[dt][r] = rest;
                        }
                }
            }
#pragma unroll
            for (int dt = 0; dt < kFolded; ++dt) acc[dt] += base[dt];
        }

        // The wavefronts' sums: in units of 1, then merged. acc[dt][r] is dim 16 dt + 4 quad + r
        // of head col.
        const float total = sum_across_quads(run_sum + run_low);
        if (quad == 0) stats[wave][col] = make_float2(run_max, total);
        float unit = value_ref * (1.0f / kWeightScale);
        if (__builtin_expect(value_ref < 0x1p-111f, 0)) {  // uniform; a subnormal number would lose bits
#pragma unroll
            for (int dt = 0; dt < kDt; ++dt) acc[dt] *= 1.0f / kWeightScale;
            unit = value_ref;
        }
        if (static_cast<std::uint32_t>(col) < heads) {
            float* const row_to = reinterpret_cast<float*>(wave_lds[wave]) + col * S::kPad + 4 * quad;
#pragma unroll
            for (int dt = 0; dt < kDt; ++dt) {
                const pf_f32x4_t o = acc[dt] * unit;
                *reinterpret_cast<float4*>(row_to + 16 * dt) = make_float4(o[0], o[1], o[2], o[3]);
            }
        }
        __syncthreads();
        for (std::uint32_t i = tid; i < heads * kD; i += kT) {
            const std::uint32_t h = i / kD, d = i % kD;
            float top = -INFINITY;
#pragma unroll
            for (int w = 0; w < kW; ++w) top = fmaxf(top, stats[w][h].x);
            float sum = 0.0f, o = 0.0f;
#pragma unroll
            for (int w = 0; w < kW; ++w) {
                const float2 s = stats[w][h];
                const float f = s.y != s.y ? s.y : merge_weight(s.x, top);
                sum += s.y * f;
                o += reinterpret_cast<const float*>(wave_lds[w])[h * S::kPad + d] * f;
            }
            if (ml == nullptr) {
                if (d < D) to[h * D + d] = sum == 0.0f ? 0.0f : o / sum;
            } else {
                to[i] = o;
                if (d == 0) {
                    ml[2 * h] = top;
                    ml[2 * h + 1] = sum;
                }
            }
        }
        __syncthreads();  // the buffers and stats are used again
    };
    const auto output_of = [&](std::uint32_t row, std::uint32_t kvh, std::uint32_t set) {
        return p.output + ((static_cast<std::uint64_t>(p.row_base) + row) * p.query_heads + kvh * p.group + set * p.set_heads) * D;
    };

    if constexpr (kWhole) {
        std::uint32_t x = blockIdx.x;
        const std::uint32_t set = x % p.sets;
        x /= p.sets;
        const std::uint32_t kvh = x % p.heads, row = x / p.heads, len = length(row);
        run_part(row, len, kvh, set, 0, tiles_of(len), output_of(row, kvh, set), nullptr);
    } else {
        // ---- plan: the cost of a stream of every row, and the sums of those before.
        const std::uint32_t per = (p.rows + kT - 1) / kT;
        std::uint64_t mine = 0;
        for (std::uint32_t i = 0; i < per; ++i) {
            const std::uint32_t r = tid * per + i;
            if (r >= p.rows) break;
            const std::uint32_t n = length(r);
            lens_of[r] = n;
            mine += n != 0 ? tiles_of(n) + kPartCost : 0;
        }
        std::uint64_t upto = mine;
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            const std::uint64_t add = __shfl_up(upto, d);
            if (lane >= d) upto += add;
        }
        if (lane == 63) wave_cost[wave] = upto;
        __syncthreads();
        std::uint64_t run = upto - mine;
        for (std::uint32_t w = 0; w < wave; ++w) run += wave_cost[w];
        for (std::uint32_t i = 0; i < per; ++i) {
            const std::uint32_t r = tid * per + i;
            if (r >= p.rows) break;
            before[r] = run;
            run += lens_of[r] != 0 ? tiles_of(lens_of[r]) + kPartCost : 0;
        }
        if (tid == kT - 1) before[p.rows] = run;
        __syncthreads();
        const std::uint32_t streams = p.heads * p.sets;  // of a row
        const std::uint64_t total = before[p.rows] * streams;
        const std::uint64_t wanted = total / kLeastShare;
        const std::uint32_t shares = wanted == 0 ? 1 : wanted < gridDim.x ? static_cast<std::uint32_t>(wanted) : gridDim.x;
        const std::uint64_t each = total / shares;
        const std::uint32_t more = static_cast<std::uint32_t>(total - each * shares);  // the first shares have one more
        // Neighbouring shares, whose streams are often heads of one row, go to one XCD: the
        // scales of a page's heads share lines in its L2 (128 rows of <= 32768 tokens: 730 us
        // without, 724 with; but one row of 32768 24.9 and 25.7).
        const std::uint32_t w = p.rows > 1 && gridDim.x % 8 == 0 ? blockIdx.x % 8 * (gridDim.x / 8) + blockIdx.x / 8 : blockIdx.x;
        // Rows without tokens: zeros.
        for (std::uint32_t r = w; r < p.rows; r += gridDim.x) {
            if (lens_of[r] != 0) continue;
            if (p.by_stream)
                for (std::uint32_t i = tid; i < streams; i += kT) p.cuts[r * streams + i] = make_uint2(~0u, 0);
            float* const out = p.output + (static_cast<std::uint64_t>(p.row_base) + r) * p.query_heads * D;
            for (std::uint32_t i = tid; i < p.query_heads * D; i += kT) out[i] = 0.0f;
        }
        if (tid == 0 && !p.by_stream) p.cuts[w] = make_uint2(~0u, 0);
        if (w >= shares) return;
        const std::uint64_t begin = each * w + (w < more ? w : more), end = begin + each + (w < more ? 1 : 0);
        // The row of the first stream: the last one that begins at or before it.
        std::uint32_t row = 0;
        for (std::uint32_t step = p.rows > 64 ? 64 : 1;; step = 1) {
            const std::uint32_t r = row + lane * step;
            const std::uint64_t behind = __builtin_amdgcn_ballot_w64(r < p.rows && before[r < p.rows ? r : 0] * streams <= begin);
            row += (__builtin_popcountll(behind) - 1) * step;
            if (step == 1) break;
        }
        std::uint64_t at = begin;
        while (at < end) {
            while (row < p.rows && before[row + 1] * streams <= at) ++row;
            if (row >= p.rows) break;
            const std::uint32_t len = uniform(lens_of[row]);
            const std::uint32_t tiles = tiles_of(len), cost = tiles + kPartCost;
            const std::uint32_t stream = static_cast<std::uint32_t>((at - before[row] * streams) / cost);
            const std::uint64_t start = before[row] * streams + static_cast<std::uint64_t>(stream) * cost;
            const std::uint64_t stop = start + cost;
            const std::uint64_t until = stop < end ? stop : end;
            // A stream's cost lies before its first tile.
            const std::uint32_t t0 = at > start + kPartCost ? static_cast<std::uint32_t>(at - start - kPartCost) : 0;
            const std::uint32_t t1 = until > start + kPartCost ? static_cast<std::uint32_t>(until - start - kPartCost) : 0;
            if (t1 > t0) {
                const std::uint32_t kvh = stream / p.sets, set = stream % p.sets;
                const bool whole = t0 == 0 && t1 == tiles;
                // The part that a stream begins with takes the workgroup's second place,
                // a later one the first: a share has one of each at most.
                const std::uint32_t slot = 2 * w + (t0 == 0 ? 1 : 0);
                run_part(row, len, kvh, set, t0, t1, whole ? output_of(row, kvh, set) : p.part_acc + static_cast<std::uint64_t>(slot) * p.set_heads * kD,
                         whole ? nullptr : p.part_ml + static_cast<std::uint64_t>(slot) * p.set_heads * 2);
                if (t0 == 0 && tid == 0) {
                    const std::uint32_t index = row * streams + stream;
                    if (!whole) {
                        // The workgroup of the stream's last tile, at cost stop - 1.
                        const std::uint64_t x = stop - 1, longer = (each + 1) * more;
                        const std::uint64_t last = x < longer ? x / (each + 1) : more + (x - longer) / each;
                        p.cuts[p.by_stream ? index : w] = make_uint2(p.by_stream ? w : index, static_cast<std::uint32_t>(last));
                    } else if (p.by_stream) {
                        p.cuts[index] = make_uint2(~0u, 0);
                    }
                }
            }
            at = until;
        }
    }
}

// Merges the parts of a cut stream: the second partial of the workgroup that begins it
// and the first ones of the workgroups up to the last, in that order, so results are the
// same from call to call. blockIdx.x is the stream, or the workgroup that begins it. A block is one query head; kMergeThreads
// hold kD / 4 dims of neighbouring parts each.
template <int kD, int kMergeThreads>
__global__ __launch_bounds__(kMergeThreads) void quant_decode_merge_kernel(QuantDecodeParams p) {
    constexpr std::uint32_t kLanes = kD / 4, kGroups = kMergeThreads / kLanes;
    __shared__ float4 sums[kMergeThreads];
    __shared__ float2 ml_of[kGroups];
    const std::uint32_t h = blockIdx.y;
    const uint2 cut = p.cuts[blockIdx.x];
    if (cut.x == ~0u) return;
    const std::uint32_t w = p.by_stream ? cut.x : blockIdx.x, index = p.by_stream ? blockIdx.x : cut.x;
    const std::uint32_t streams = p.heads * p.sets;
    const std::uint32_t row = index / streams, stream = index % streams, kvh = stream / p.sets, set = stream % p.sets;
    const std::uint32_t head = set * p.set_heads + h;
    if (head >= p.group) return;
    const std::uint32_t parts = cut.y - w + 1;
    const std::uint32_t g = threadIdx.x / kLanes, d4 = threadIdx.x % kLanes;
    const auto place = [&](std::uint32_t i) {
        return static_cast<std::uint64_t>(2 * (w + i) + (i == 0 ? 1 : 0)) * p.set_heads + h;
    };
    // This group's parts: an online merge.
    float top = -INFINITY, sum = 0.0f;
    float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    constexpr int kAhead = kMergeThreads > 512 ? 2 : 4;  // the registers of 1024 threads
    for (std::uint32_t i0 = g; i0 < parts; i0 += kGroups * kAhead) {
        Float4 a[kAhead];
        float m[kAhead], l[kAhead];
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
            const std::uint32_t i = i0 + u * kGroups;
            const std::uint64_t at = place(i < parts ? i : i0);
            a[u] = *reinterpret_cast<const Float4*>(p.part_acc + at * kD + 4 * d4);
            m[u] = p.part_ml[2 * at];
            l[u] = p.part_ml[2 * at + 1];
        }
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
            if (i0 + u * kGroups >= parts) break;
            const float next = fmaxf(top, m[u]);
            const float f = merge_weight(top, next), f1 = l[u] != l[u] ? l[u] : merge_weight(m[u], next);
            o.x = o.x * f + a[u].x * f1;
            o.y = o.y * f + a[u].y * f1;
            o.z = o.z * f + a[u].z * f1;
            o.w = o.w * f + a[u].w * f1;
            sum = sum * f + l[u] * f1;
            top = next;
        }
    }
    sums[threadIdx.x] = o;
    if (d4 == 0) ml_of[g] = make_float2(top, sum);
    __syncthreads();
    if (threadIdx.x >= kLanes) return;
    float all = -INFINITY;
    for (std::uint32_t i = 0; i < kGroups; ++i) all = fmaxf(all, ml_of[i].x);
    sum = 0.0f;
    o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    for (std::uint32_t i = 0; i < kGroups; ++i) {
        const float2 s = ml_of[i];
        const float f = s.y != s.y ? s.y : merge_weight(s.x, all);
        const float4 v = sums[i * kLanes + d4];
        sum += s.y * f;
        o.x += v.x * f;
        o.y += v.y * f;
        o.z += v.z * f;
        o.w += v.w * f;
    }
    if (4 * d4 >= p.head_size) return;
    const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
    *reinterpret_cast<Float4*>(p.output + ((static_cast<std::uint64_t>(p.row_base) + row) * p.query_heads + kvh * p.group + head) * p.head_size + 4 * d4) =
        Float4{o.x * inv, o.y * inv, o.z * inv, o.w * inv};
}

// Any other head_size up to 512, and caches at any byte: a workgroup for each (query row, query
// head), a lane for each of 64 tokens of a wavefront's step, FP32 products and sums. A step's
// weighted values are summed from zero and added with the addition's rounding error kept: one
// by one beside a dominant key's value, thousands of small ones are lost (16384 tokens of
// 2^-24 each: 2.4e-4 of the row).
constexpr std::uint32_t kGenericD = 512;
template <typename F>
__global__ __launch_bounds__(kThreads) void quant_rows_kernel(QuantRows p, std::uint32_t first_row) {
    __shared__ float q[kGenericD];
    __shared__ float weight[kWaves][64];
    __shared__ std::uint64_t at_of[kWaves][64];
    __shared__ float reduce[kWaves][kGenericD];
    __shared__ float2 stats[kWaves];
    const std::uint32_t tid = threadIdx.x, wave = tid / 64, lane = tid % 64, D = p.head_size;
    const std::uint64_t row = static_cast<std::uint64_t>(first_row) + blockIdx.x / p.query_heads;
    const std::uint32_t head = blockIdx.x % p.query_heads, kvh = head / p.group;
    const std::uint64_t seq = p.query_lens ? row / p.max_query : row;
    const std::uint64_t full = p.lens[seq];
    std::uint32_t len = full < p.kv_len ? static_cast<std::uint32_t>(full) : p.kv_len;
    std::uint64_t out_row = row;
    if (p.query_lens) {
        const std::uint32_t i = static_cast<std::uint32_t>(row % p.max_query);
        const std::uint64_t queries = p.query_lens[seq];
        std::uint32_t n = queries < len ? static_cast<std::uint32_t>(queries) : len;
        if (n > p.max_query) n = p.max_query;
        if (i >= n) return;  // uniform
        len = len - n + i + 1;
        out_row = p.query_offsets[seq] + i;
    }
    out_row = out_row * p.query_heads + head;
    for (std::uint32_t d = tid; d < D; d += kThreads) q[d] = p.query[out_row * D + d] * p.scale_log2;
    __syncthreads();
    float top = -INFINITY, sum = 0.0f, sum_low = 0.0f;
    float acc[kGenericD / 64] = {}, low[kGenericD / 64] = {};
    for (std::uint64_t base = wave * 64; base < len; base += kThreads) {
        const std::uint32_t token = static_cast<std::uint32_t>(base) + lane;
        const std::uint64_t page = p.block_size.div(token);
        bool live = base + lane < len && page < p.width;
        std::uint64_t id = p.table[seq * p.width + (live ? page : 0)];
        live = live && id < p.num_blocks;
        id = live ? id : 0;
        const std::uint64_t scale_at = id * p.heads + kvh;
        const std::uint64_t at = (scale_at * p.block_size.divisor + (live ? p.block_size.mod(token) : 0)) * D;
        float dot = 0.0f, v4[4];
        for (std::uint32_t d = 0; d < D; ++d) {
            F::values4(p.key_cache[at + d], v4);
            dot = fmaf(q[d], v4[0], dot);
        }
        const float s = live ? dot * p.key_scales[scale_at] : -INFINITY;
        float next = s;
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) next = fmaxf(next, __shfl_xor(next, d));
        next = fmaxf(next, top);
        const float ref = next == -INFINITY ? 0.0f : next;
        const float f = top == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(top - ref);
        const float w = live ? __builtin_amdgcn_exp2f(s - ref) : 0.0f;
        top = next;
        sum *= f;
        sum_low *= f;
        two_sum_add(sum, sum_low, w);
        // A missing token's row is read from the pool's first page, and dropped.
        weight[wave][lane] = live ? w * p.value_scales[scale_at] : 0.0f;
        at_of[wave][lane] = live ? at : ~0ull;
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (std::uint32_t i = 0; i < kGenericD / 64; ++i) {
            if (64 * i >= D) break;  // uniform
            acc[i] *= f;
            low[i] *= f;
        }
        float step[kGenericD / 64] = {};
        constexpr int kAtOnce = 8;  // tokens whose bytes are on their way together
        for (int t = 0; t < 64; t += kAtOnce) {
#pragma unroll
            for (std::uint32_t i = 0; i < kGenericD / 64; ++i) {
                if (64 * i >= D) break;  // uniform
                const std::uint32_t d = lane + 64 * i < D ? lane + 64 * i : 0;  // past the head's end its first, not stored
                std::uint8_t raw[kAtOnce];
#pragma unroll
                for (int u = 0; u < kAtOnce; ++u) {
                    const std::uint64_t from = at_of[wave][t + u];
                    raw[u] = p.value_cache[(from == ~0ull ? 0 : from) + d];
                }
#pragma unroll
                for (int u = 0; u < kAtOnce; ++u) {
                    F::values4(raw[u], v4);
                    step[i] = fmaf(weight[wave][t + u], at_of[wave][t + u] == ~0ull ? 0.0f : v4[0], step[i]);
                }
            }
        }
#pragma unroll
        for (std::uint32_t i = 0; i < kGenericD / 64; ++i) {
            if (64 * i >= D) break;  // uniform
            two_sum_add(acc[i], low[i], step[i]);
        }
        __builtin_amdgcn_wave_barrier();
    }
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const float other = __shfl_xor(sum, d);
        sum_low += __shfl_xor(sum_low, d);
        two_sum_add(sum, sum_low, other);
    }
    sum += sum_low;
    if (lane == 0) stats[wave] = make_float2(top, sum);
#pragma unroll
    for (std::uint32_t i = 0; i < kGenericD / 64; ++i)
        if (lane + 64 * i < D) reduce[wave][lane + 64 * i] = acc[i] + low[i];
    __syncthreads();
    float all = -INFINITY, total = 0.0f;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) all = fmaxf(all, stats[w].x);
    float factor[kWaves];
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
        factor[w] = stats[w].y != stats[w].y ? stats[w].y : merge_weight(stats[w].x, all);
        total += stats[w].y * factor[w];
    }
    for (std::uint32_t d = tid; d < D; d += kThreads) {
        float o = 0.0f;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) o += reduce[w][d] * factor[w];
        p.output[out_row * D + d] = total == 0.0f ? 0.0f : o / total;
    }
}

// ---------------------------------------------------------------- dispatch
// Streams of a (row, kv head), and query heads of each.
void head_sets(std::uint64_t group, std::uint32_t* sets, std::uint32_t* heads) {
    *sets = static_cast<std::uint32_t>((group + kCols - 1) / kCols);
    *heads = static_cast<std::uint32_t>((group + *sets - 1) / *sets);
}

// Workgroups of a launch over `rows` rows; 0: one for each stream.
std::uint32_t decode_grid(std::uint64_t rows, std::uint64_t kv_len, std::uint64_t streams, std::uint64_t block_size,
                          std::uint64_t head_size) {
    const std::uint64_t whole = head_size == 256 || block_size % 8 != 0 ? kOneLaunch / 2 : kOneLaunch;
    if (kv_len <= whole || (kv_len <= 2 * whole && rows * streams >= kFullStreams)) return 0;
    const std::uint64_t most = head_size == 256 ? Shape<256>::kGrid : Shape<128>::kGrid;
    const std::uint64_t tiles = (kv_len + kTile - 1) / kTile + kPartCost;
    const std::uint64_t shares = tiles > most * kLeastShare ? most : rows * streams * tiles / kLeastShare + 1;
    return static_cast<std::uint32_t>(shares < most ? shares : most);
}
// Rows of a launch: what the plan holds, and what a grid counts (query_heads < 2^20).
std::uint64_t decode_slice(std::uint64_t rows, std::uint64_t streams) {
    const std::uint64_t most = kMostWorkgroups / streams < kPlanRows ? kMostWorkgroups / streams : kPlanRows;
    return rows < most ? rows : most;
}
std::size_t decode_workspace(std::uint32_t grid, std::uint32_t set_heads, std::uint64_t head_size) {
    return 2ull * grid * set_heads * (head_size + 2) * sizeof(float) + grid * sizeof(uint2);
}

template <typename F, int kD, int kSub, bool kFull>
int launch_decode(QuantDecodeParams& p, std::uint32_t grid, hipStream_t stream) {
    const std::uint64_t streams = static_cast<std::uint64_t>(p.heads) * p.sets;
    if (grid == 0) {
        const dim3 workgroups(static_cast<unsigned>(p.rows * streams));
        // Eight wavefronts where a CU has a stream at most (at 256 the registers are those of
        // four), and each more than a tile or two. 8 rows of <= 1000 tokens: 12.7 us with
        // four, 11.6 with eight; one of <= 300: 6.6 and 7.2.
        if constexpr (kD <= 128 && kFull) {
            if (p.rows * streams <= kFullStreams && p.kv_len > kOneLaunch / 2) {
                quant_decode_kernel<F, kD, kSub, true, 2 * kWaves, false, kFull><<<workgroups, dim3(2 * kThreads), 0, stream>>>(p);
                return launch_status("quant_decode_kernel");
            }
        }
        quant_decode_kernel<F, kD, kSub, true, kWaves, false, kFull><<<workgroups, dim3(kThreads), 0, stream>>>(p);
        return launch_status("quant_decode_kernel");
    }
    // The merge takes the shorter list: streams of a few rows, or the workgroups' cuts.
    // 16 rows of 2 kv heads with 16 query heads each: 40 us by workgroup, 19 by stream.
    const std::uint32_t cuts = p.rows * streams < grid ? static_cast<std::uint32_t>(p.rows * streams) : grid;
    p.by_stream = cuts < grid;
    // The longest part's tiles: a row's, or a share's.
    const std::uint64_t tiles = (static_cast<std::uint64_t>(p.kv_len) + kTile - 1) / kTile;
    const std::uint64_t share = p.rows * streams * (tiles + kPartCost) / grid + 1;
    if ((tiles < share ? tiles : share) > kFold * kWaves)
        quant_decode_kernel<F, kD, kSub, false, kWaves, true, kFull><<<dim3(grid), dim3(kThreads), 0, stream>>>(p);
    else
        quant_decode_kernel<F, kD, kSub, false, kWaves, false, kFull><<<dim3(grid), dim3(kThreads), 0, stream>>>(p);
    if (const int s = launch_status("quant_decode_kernel")) return s;
    // Parts of a stream: many where there are few streams. With 1024 threads and with 128:
    // 64 parts 25.3 and 26.6 us (the whole call), 18 parts 16.2 and 13.2.
    if (grid > 32 * p.rows * streams)
        quant_decode_merge_kernel<kD, 1024><<<dim3(cuts, p.set_heads), dim3(1024), 0, stream>>>(p);
    else
        quant_decode_merge_kernel<kD, 128><<<dim3(cuts, p.set_heads), dim3(128), 0, stream>>>(p);
    return launch_status("quant_decode_merge_kernel");
}
template <typename F, int kD>
int launch_decode_pages(QuantDecodeParams& p, std::uint32_t grid, hipStream_t s) {
    if (p.head_size == kD)
        return p.block_size.divisor % 8 == 0 ? launch_decode<F, kD, 8, true>(p, grid, s) : launch_decode<F, kD, 1, true>(p, grid, s);
    return p.block_size.divisor % 8 == 0 ? launch_decode<F, kD, 8, false>(p, grid, s) : launch_decode<F, kD, 1, false>(p, grid, s);
}
template <typename F>
int launch_decode_format(QuantDecodeParams& p, std::uint64_t head_size, std::uint32_t grid, hipStream_t s) {
    switch (head_size) {
    case 64: return launch_decode_pages<F, 64>(p, grid, s);
    case 128: return launch_decode_pages<F, 128>(p, grid, s);
    default: return launch_decode_pages<F, 256>(p, grid, s);
    }
}

int check_shape(const char* op, std::uint64_t num_rows, std::uint64_t kv_len, std::uint64_t heads,
                std::uint64_t query_heads, std::uint64_t block_size, std::uint64_t head_size) {
    if (heads == 0 || block_size == 0 || head_size == 0 || query_heads == 0 || query_heads % heads != 0)
        return fail(KVFLUX_ERR_INVALID_ARGUMENT, "%s: invalid shape", op);
    if (heads > 65535 || head_size > kGenericD || block_size > 0x7fffffffULL / head_size || query_heads > 0xfffffULL ||
        num_rows > 0xffffffffULL || kv_len > 0xffffffffULL - 2 * kTile)
        return fail(KVFLUX_ERR_UNSUPPORTED, "%s: shape too large", op);
    return KVFLUX_OK;
}

} // namespace

int launch_quant_rows(const QuantRows& p, std::uint64_t rows, int format, hipStream_t stream) {
    const std::uint64_t at_once = kMostWorkgroups / p.query_heads;
    for (std::uint64_t first = 0; first < rows; first += at_once) {
        const dim3 grid(static_cast<unsigned>((rows - first < at_once ? rows - first : at_once) * p.query_heads));
        if (format == KVFLUX_QUANT_E4M3)
            quant_rows_kernel<QuantE4m3><<<grid, dim3(kThreads), 0, stream>>>(p, static_cast<std::uint32_t>(first));
        else
            quant_rows_kernel<QuantInt8><<<grid, dim3(kThreads), 0, stream>>>(p, static_cast<std::uint32_t>(first));
        if (const int s = launch_status("quant_rows_kernel")) return s;
    }
    return KVFLUX_OK;
}

} // namespace kvflux_hip

using namespace kvflux_hip;

extern "C" int kvflux_quant_attention_workspace_size(uint64_t num_rows, uint64_t kv_len, uint64_t num_kv_heads,
                                                     uint64_t query_heads, uint64_t block_size, uint64_t head_size,
                                                     size_t* bytes) {
    if (!bytes) return fail(KVFLUX_ERR_INVALID_ARGUMENT, "quant attention workspace: null pointer");
    *bytes = 0;
    if (const int s = check_shape("quant attention workspace", num_rows, kv_len, num_kv_heads, query_heads, block_size, head_size))
        return s;
    head_size = padded_head_size(head_size);
    if (num_rows == 0 || head_size == 0) return KVFLUX_OK;
    std::uint32_t sets, set_heads;
    head_sets(query_heads / num_kv_heads, &sets, &set_heads);
    const std::uint64_t streams = num_kv_heads * sets;
    std::uint64_t rows = decode_slice(num_rows, streams);
    // Enough for fewer rows as well, where those are cut into shares and these not.
    if (decode_grid(rows, kv_len, streams, block_size, head_size) == 0) {
        const std::uint64_t fewer = (kFullStreams - 1) / streams;
        if (fewer < rows) rows = fewer;
    }
    if (rows == 0) return KVFLUX_OK;
    *bytes = decode_workspace(decode_grid(rows, kv_len, streams, block_size, head_size), set_heads, head_size);
    return KVFLUX_OK;
}

extern "C" int kvflux_quant_attention(const void* key_cache, const void* value_cache, const float* key_scales,
                                      const float* value_scales, uint64_t num_blocks, uint64_t num_kv_heads,
                                      uint64_t block_size, uint64_t head_size, int format, const uint64_t* block_table,
                                      uint64_t max_blocks_per_seq, const uint64_t* seq_lens, uint64_t kv_len,
                                      uint64_t num_rows, uint64_t query_heads, const float* query, float* output,
                                      void* workspace, size_t workspace_bytes, void* stream) {
    if (num_rows == 0) return KVFLUX_OK;
    if (const int s = check_quant_cache("quant attention", key_cache, value_cache, key_scales, value_scales, num_blocks,
                                        num_kv_heads, block_size, head_size, format))
        return s;
    if (!block_table || !seq_lens || !query || !output)
        return fail(KVFLUX_ERR_INVALID_ARGUMENT, "quant attention: null pointer");
    if (max_blocks_per_seq == 0) return fail(KVFLUX_ERR_INVALID_ARGUMENT, "quant attention: empty table rows");
    if (const int s = check_shape("quant attention", num_rows, kv_len, num_kv_heads, query_heads, block_size, head_size))
        return s;
    if (!aligned(4, {query, output}) || !aligned(8, {block_table, seq_lens}))
        return fail(KVFLUX_ERR_INVALID_ARGUMENT, "quant attention: misaligned array");
    const float scale_log2 = static_cast<float>(1.4426950408889634 / std::sqrt(static_cast<double>(head_size)));
    const std::uint64_t padded = padded_head_size(head_size);
    if (padded == 0 || !aligned(16, {key_cache, value_cache})) {
        QuantRows rows{};
        rows.key_cache = static_cast<const std::uint8_t*>(key_cache);
        rows.value_cache = static_cast<const std::uint8_t*>(value_cache);
        rows.key_scales = key_scales;
        rows.value_scales = value_scales;
        rows.num_blocks = num_blocks;
        rows.heads = static_cast<std::uint32_t>(num_kv_heads);
        rows.head_size = static_cast<std::uint32_t>(head_size);
        rows.block_size = FastDiv(static_cast<std::uint32_t>(block_size));
        rows.table = block_table;
        rows.width = max_blocks_per_seq;
        rows.lens = seq_lens;
        rows.kv_len = static_cast<std::uint32_t>(kv_len);
        rows.query_heads = static_cast<std::uint32_t>(query_heads);
        rows.group = static_cast<std::uint32_t>(query_heads / num_kv_heads);
        rows.query = query;
        rows.output = output;
        rows.scale_log2 = scale_log2;
        return launch_quant_rows(rows, num_rows, format, as_stream(stream));
    }
    QuantDecodeParams p{};
    p.key_cache = static_cast<const std::uint8_t*>(key_cache);
    p.value_cache = static_cast<const std::uint8_t*>(value_cache);
    p.key_scales = key_scales;
    p.value_scales = value_scales;
    p.num_blocks = num_blocks;
    p.heads = static_cast<std::uint32_t>(num_kv_heads);
    p.head_size = static_cast<std::uint32_t>(head_size);
    p.block_size = FastDiv(static_cast<std::uint32_t>(block_size));
    p.table = block_table;
    p.width = max_blocks_per_seq;
    p.lens = seq_lens;
    p.kv_len = static_cast<std::uint32_t>(kv_len);
    p.query_heads = static_cast<std::uint32_t>(query_heads);
    p.group = static_cast<std::uint32_t>(query_heads / num_kv_heads);
    head_sets(p.group, &p.sets, &p.set_heads);
    p.query = query;
    p.output = output;
    p.scale_log2 = scale_log2;
    const std::uint64_t streams = num_kv_heads * p.sets;
    const std::uint64_t slice = decode_slice(num_rows, streams);
    const std::uint32_t grid = decode_grid(slice, kv_len, streams, block_size, padded);
    if (grid != 0) {
        if (!workspace || workspace_bytes < decode_workspace(grid, p.set_heads, padded))
            return fail(KVFLUX_ERR_INVALID_ARGUMENT, "quant attention: workspace too small");
        if (!aligned(8, {workspace})) return fail(KVFLUX_ERR_INVALID_ARGUMENT, "quant attention: misaligned workspace");
        p.cuts = static_cast<uint2*>(workspace);
        p.part_acc = reinterpret_cast<float*>(p.cuts + grid);
        p.part_ml = p.part_acc + 2ull * grid * p.set_heads * padded;
    }
    for (std::uint64_t base = 0; base < num_rows; base += slice) {
        p.row_base = static_cast<std::uint32_t>(base);
        p.rows = static_cast<std::uint32_t>(num_rows - base < slice ? num_rows - base : slice);
        const int s = format == KVFLUX_QUANT_E4M3
                          ? launch_decode_format<QuantE4m3>(p, padded, grid, as_stream(stream))
                          : launch_decode_format<QuantInt8>(p, padded, grid, as_stream(stream));
        if (s != KVFLUX_OK) return s;
    }
    return KVFLUX_OK;
}
