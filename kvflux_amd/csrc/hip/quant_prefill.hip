// Causal attention of prompts, or of a prompt's next tokens behind its cached ones,
// straight from a paged cache held in 8 bits with a scale for each page and kv head:
// for query i of a sequence's last n of len tokens and keys t <= len - n + i
//   s_t = ks_t (q_i . k_t) / sqrt(D),  o_i = sum_t e^(s_t - m) vs_t v_t / sum_t e^(s_t - m).
//
// Bound by the matrix instructions: FP16 MFMAs on K and V as FP16 (exact) and on Q and
// the weights in two FP16 parts each (off by at most 2^-23), so two products where a
// rounded kernel has one. 32x32x16, whose operands feed twice the products of a
// 16x16x32's for the same bytes from LDS.
//  * A workgroup owns one kv head and 32 rows a wavefront, a row being a (query token,
//    query head) pair of the heads of that kv head.
//  * Keys go through LDS in tiles of 64: a thread loads 16 bytes of the next tile's K
//    and V into registers while this one is computed, widens them to FP16 once for all
//    wavefronts and stores them to the other buffer; one barrier a tile.
//  * S^T = K Q^T leaves lane (row, half) with keys 8 i + 4 half .. + 3 of the row:
//    O^T += V^T P^T takes them as they are when V's tokens are read in that order
//    (ds_read_b64_tr_b16, four tokens of a dim a lane).
//  * The scales stay out of K and V: ks joins the score's subtraction (one FMA), vs
//    multiplies the weight.
//  * The tile's weighted values are summed from zero and added with one rounding: an
//    MFMA on a large accumulator drops bits of small weights, always in one direction.
// A call whose workgroups would leave CUs idle (a short chunk behind a long prefix)
// spreads each one's keys over several, merged by a second kernel.
#include "mfma_parts.h"
#include "quant.h"

#include <cmath>
#include <type_traits>

namespace kvflux_hip {
namespace {

typedef __attribute__((ext_vector_type(16))) float qp_f32x16_t;

constexpr std::uint32_t kTile = 64;     // keys of a tile
constexpr std::uint32_t kWindow = 2048; // pages whose ids and scales are in LDS at a time
constexpr std::uint32_t kMissing = 0x80000000u;
constexpr float kWeightScale = 32768.0f;  // as in the decode: parts of 2^15 times a weight of at most 1

template <int kD>
struct Shape {
    // The registers of two wavefronts a SIMD hold Q and the sums of 32 rows up to D = 128.
    static constexpr int kWaves = kD == 256 ? 4 : 8;
    static constexpr int kThreads = 64 * kWaves;
    static constexpr std::uint32_t kRows = 32 * kWaves;
};

struct QuantPrefillParams {
    const std::uint8_t* key_cache;
    const std::uint8_t* value_cache;
    const float* key_scales;
    const float* value_scales;
    std::uint64_t num_blocks;
    std::uint32_t heads;
    FastDiv block_size;
    const std::uint64_t* table;
    std::uint64_t width;
    const std::uint64_t* kv_lens;
    const std::uint64_t* query_lens;
    const std::uint64_t* query_offsets;
    std::uint32_t num_seqs, max_query, max_kv;
    std::uint32_t query_heads, group;
    std::uint32_t first, heads_of;     // of the group's query heads, those of this launch
    FastDiv heads_div;                 // heads_of
    std::uint32_t tokens;              // query tokens of a workgroup
    std::uint32_t blocks;              // workgroups along max_query
    std::uint32_t splits, split_tiles;
    std::uint32_t window_tiles;        // tiles whose pages fit kWindow
    const float* query;
    float* output;
    float scale_log2;
    float* part_acc;  // [splits][num_seqs * max_query][query_heads][D]
    float* part_ml;   // [splits][num_seqs * max_query][query_heads][2]
};

// kUniform: pages are multiples of 16 tokens, so 16 neighbouring keys of a tile share
// their scales, which are then one value for a wavefront.
template <typename F, int kD, bool kUniform>
__global__ __launch_bounds__(Shape<kD>::kThreads, kD == 256 ? 1 : 2) void quant_prefill_kernel(QuantPrefillParams p) {
    using S = Shape<kD>;
    using Vec = pf_f16x8_t;
    constexpr int kThreads = S::kThreads;
    constexpr int kSteps = kD / 16;            // MFMAs of a 32-key block of S^T for one part of Q
    constexpr int kDb = kD / 32;               // dim blocks of O^T
    constexpr int kRowBytes = kD * 2;          // a key's row in LDS
    constexpr int kCpr = kRowBytes / 16;
    constexpr int kTileBytes = static_cast<int>(kTile) * kRowBytes;
    constexpr int kChunks = static_cast<int>(kTile) * kD / 16;  // 16-byte chunks of a tile in the cache
    constexpr int kLoads = 2 * kChunks / kThreads;              // of a thread: K's chunks, then V's
    static_assert(2 * kChunks % kThreads == 0, "tile split");
    __shared__ __attribute__((aligned(16))) unsigned char tiles_lds[2][2][kTileBytes];  // [buffer][K, V]
    __shared__ std::uint32_t page_id[kWindow];
    __shared__ float page_ks[kWindow], page_vs[kWindow];
    // Of a buffer's tile: scales of its keys (vs over the reference), which of them
    // count, and the reference.
    __shared__ __attribute__((aligned(16))) float tile_ks[2][kTile];
    __shared__ __attribute__((aligned(16))) float tile_vs[2][kTile];
    __shared__ std::uint64_t tile_live[2];
    __shared__ float tile_ref[2];
    __shared__ float wave_top[S::kWaves];

    const int tid = threadIdx.x, lane = tid % 64;
    const std::uint32_t wave = static_cast<std::uint32_t>(__builtin_amdgcn_readfirstlane(tid / 64));
    const int col = lane % 32, half = lane / 32;
    // Heaviest query blocks first; neighbouring workgroups take the kv heads in turn.
    std::uint32_t x = blockIdx.x;
    const std::uint32_t kvh = x % p.heads;
    x /= p.heads;
    const std::uint32_t split = x % p.splits;
    x /= p.splits;
    const std::uint32_t seq = x % p.num_seqs, qb = p.blocks - 1 - x / p.num_seqs;
    const std::uint64_t full_len = p.kv_lens[seq], full_q = p.query_lens[seq];
    const std::uint32_t kv_len = full_len < p.max_kv ? static_cast<std::uint32_t>(full_len) : p.max_kv;
    std::uint32_t tq = full_q < kv_len ? static_cast<std::uint32_t>(full_q) : kv_len;
    if (tq > p.max_query) tq = p.max_query;
    const std::uint32_t t0 = qb * p.tokens;
    if (t0 >= tq) return;  // uniform
    const std::uint32_t t_end = t0 + p.tokens < tq ? t0 + p.tokens : tq;
    const std::uint32_t past = kv_len - tq;
    const std::uint32_t tile_count = (past + t_end - 1) / kTile + 1;
    const std::uint32_t tile_begin = split * p.split_tiles < tile_count ? split * p.split_tiles : tile_count;
    const std::uint32_t tile_end = tile_begin + p.split_tiles < tile_count ? tile_begin + p.split_tiles : tile_count;
    const std::uint64_t* const table = p.table + seq * p.width;

    // This lane's row.
    const std::uint32_t r = 32 * wave + static_cast<std::uint32_t>(col);
    const std::uint32_t token = t0 + p.heads_div.div(r), head = p.first + p.heads_div.mod(r);
    const bool row_live = r < p.tokens * p.heads_of && token < t_end;
    const bool wave_live = __builtin_amdgcn_ballot_w64(row_live) != 0;
    const std::uint64_t q_row = (p.query_offsets[seq] + (row_live ? token : t0)) * p.query_heads + kvh * p.group + (row_live ? head : p.first);
    const float* const q_src = p.query + q_row * kD + 8 * half;
    struct Float4 { float x, y, z, w; };  // float-aligned
    Float4 raw[kSteps][2];
#pragma unroll
    for (int kk = 0; kk < kSteps; ++kk)
#pragma unroll
        for (int i = 0; i < 2; ++i) raw[kk][i] = *reinterpret_cast<const Float4*>(q_src + 16 * kk + 4 * i);

    // ---- the window's pages: ids, scales, the largest |vs|.
    std::uint32_t window = tile_begin / p.window_tiles;  // tiles [window * window_tiles, + window_tiles)
    std::uint32_t window_page = 0;                       // page of page_id[0]
    float reference = 0.0f;
    const auto stage = [&] {
        const std::uint32_t tile0 = window * p.window_tiles;
        const std::uint32_t tile1 = tile0 + p.window_tiles < tile_count ? tile0 + p.window_tiles : tile_count;
        window_page = p.block_size.div(tile0 * kTile);
        const std::uint32_t last = p.block_size.div(tile1 * kTile - 1);
        float top = 0.0f;
        for (std::uint32_t i = tid; window_page + i <= last; i += kThreads) {
            const std::uint64_t page = window_page + i;
            const bool in_row = page < p.width && page * p.block_size.divisor < kv_len;
            const std::uint64_t id = table[in_row ? page : 0];
            const bool live = in_row && id < p.num_blocks;
            const std::uint64_t at = (live ? id : 0) * p.heads + kvh;
            float ks = live ? p.key_scales[at] : 0.0f, vs = live ? p.value_scales[at] : 0.0f;
            if (vs != vs) {  // what sees these values is NaN by its score, what does not is left alone
                ks = vs;
                vs = 0.0f;
            }
            page_id[i] = live ? static_cast<std::uint32_t>(id) : kMissing;
            page_ks[i] = ks;
            page_vs[i] = vs;
            top = fmaxf(top, __builtin_fabsf(vs));
        }
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) top = fmaxf(top, __shfl_xor(top, d));
        if (lane == 0) wave_top[wave] = top;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < S::kWaves; ++w) reference = fmaxf(reference, wave_top[w]);
    };

    // ---- loads: chunk e of a tile is 16 values of key e * 16 / D.
    uint4 held[kLoads];
    const std::uint64_t head_bytes = static_cast<std::uint64_t>(p.block_size.divisor) * kD;
    const auto page_of = [&](std::uint32_t key, std::uint32_t& in_page) {
        const std::uint32_t page = p.block_size.div(key);
        in_page = key - page * p.block_size.divisor;
        return page - window_page;
    };
    const auto chunk_key = [](int e) { return static_cast<std::uint32_t>(e * 16 / kD % static_cast<int>(kTile)); };
    const auto fetch = [&](std::uint32_t tile) {
#pragma unroll
        for (int i = 0; i < kLoads; ++i) {
            const int e = i * kThreads + tid;
            const std::uint8_t* const cache = e < kChunks ? p.key_cache : p.value_cache;
            const std::uint32_t key = tile * kTile + chunk_key(e);
            std::uint32_t in_page;
            const std::uint32_t id = page_id[page_of(key, in_page)];
            // Missing pages: the pool's first row.
            const std::uint64_t at = id & kMissing ? 0 : (static_cast<std::uint64_t>(id) * p.heads + kvh) * head_bytes + in_page * kD;
            held[i] = *reinterpret_cast<const uint4*>(cache + at + e * 16 % kD);
        }
    };
    // Swizzled slot of a row's 16-byte chunk: rows of one read fall on different banks.
    const auto k_slot = [](std::uint32_t row, std::uint32_t c) { return c ^ (kCpr >= 16 ? row & 15 : (row >> 1) & 7); };
    const auto v_slot = [](std::uint32_t row, std::uint32_t c) { return c ^ (kCpr / 8 * (row & 7)); };
    const auto put = [&](std::uint32_t tile, int buf) {
#pragma unroll
        for (int i = 0; i < kLoads; ++i) {
            const int e = i * kThreads + tid;
            const bool value = e >= kChunks;
            const std::uint32_t row = chunk_key(e), c = static_cast<std::uint32_t>(e * 16 % kD) / 8;
            const std::uint32_t key = tile * kTile + row;
            std::uint32_t in_page;
            const bool live = key < kv_len && !(page_id[page_of(key, in_page)] & kMissing);
            uint4 w = held[i];
            if (value && !live) w = make_uint4(0, 0, 0, 0);  // 0 * NaN would stay
            unsigned char* const to = tiles_lds[buf][value ? 1 : 0] + row * kRowBytes;
            const uint4 lo = make_uint4(F::template pair16<0>(w.x), F::template pair16<1>(w.x), F::template pair16<0>(w.y), F::template pair16<1>(w.y));
            const uint4 hi = make_uint4(F::template pair16<0>(w.z), F::template pair16<1>(w.z), F::template pair16<0>(w.w), F::template pair16<1>(w.w));
            *reinterpret_cast<uint4*>(to + 16 * (value ? v_slot(row, c) : k_slot(row, c))) = lo;
            *reinterpret_cast<uint4*>(to + 16 * (value ? v_slot(row, c + 1) : k_slot(row, c + 1))) = hi;
        }
        if (wave == 0) {
            const std::uint32_t key = tile * kTile + lane;
            std::uint32_t in_page;
            const std::uint32_t i = page_of(key, in_page);
            const bool live = key < kv_len && !(page_id[i] & kMissing);
            const std::uint64_t all = __builtin_amdgcn_ballot_w64(live);
            tile_ks[buf][lane] = page_ks[i];
            tile_vs[buf][lane] = reference > 0.0f ? page_vs[i] / reference * kWeightScale : page_vs[i];
            if (lane == 0) {
                tile_live[buf] = all;
                tile_ref[buf] = reference > 0.0f ? reference : 1.0f;
            }
        }
    };

    qp_f32x16_t acc[kDb];
#pragma unroll
    for (int db = 0; db < kDb; ++db) acc[db] = qp_f32x16_t{};
    // A score moves the reference when it passes it by `threshold`: the row's first key
    // does, whatever its score.
    float ref = 0.0f, threshold = -INFINITY, sum = 0.0f, low = 0.0f;
    float unit = 0.0f;  // acc is in units of this over kWeightScale; 0: nothing there yet
    // Queries in two parts, times a power of two that the scores carry.
    Vec q_hi[kSteps], q_lo[kSteps];
    float down;
    {
        float largest = 0.0f;
#pragma unroll
        for (int kk = 0; kk < kSteps; ++kk)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const Float4 v = raw[kk][i];
                largest = max3(largest, __builtin_fabsf(v.x), __builtin_fabsf(v.y));
                largest = max3(largest, __builtin_fabsf(v.z), __builtin_fabsf(v.w));
            }
        const auto swapped = __builtin_amdgcn_permlane32_swap(__float_as_uint(largest), __float_as_uint(largest), false, false);
        largest = __builtin_elementwise_maximum(__uint_as_float(swapped[0]), __uint_as_float(swapped[1]));
        const int e = split_exponent(largest * p.scale_log2);
        const float up = __builtin_amdgcn_ldexpf(1.0f, e);
        down = __builtin_amdgcn_ldexpf(1.0f, -e);
#pragma unroll
        for (int kk = 0; kk < kSteps; ++kk) {
            std::uint32_t hi[4], lo[4];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const Float4 v = raw[kk][i];
                const float y[4] = {v.x * p.scale_log2 * up, v.y * p.scale_log2 * up, v.z * p.scale_log2 * up, v.w * p.scale_log2 * up};
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const pf_f32x2_t z{y[2 * j], y[2 * j + 1]};
                    const pf_f16x2_t h = __builtin_convertvector(z, pf_f16x2_t);
                    hi[2 * i + j] = __builtin_bit_cast(std::uint32_t, h);
                    const pf_f32x2_t rest = z - __builtin_convertvector(h, pf_f32x2_t);
                    lo[2 * i + j] = __builtin_bit_cast(std::uint32_t, __builtin_convertvector(rest, pf_f16x2_t));
                }
            }
            q_hi[kk] = __builtin_bit_cast(Vec, make_uint4(hi[0], hi[1], hi[2], hi[3]));
            q_lo[kk] = __builtin_bit_cast(Vec, make_uint4(lo[0], lo[1], lo[2], lo[3]));
        }
    }
    const std::uint32_t limit = past + (row_live ? token : t0);  // the row's last key
    const std::uint32_t least_limit = past + t0;

    // Score i of a lane in block kb is key 32 kb + 8 (i / 4) + 4 half + i % 4 of the tile.
    const auto compute = [&](std::uint32_t tile, int buf) {
        const float now = tile_ref[buf];
        if (now != unit) {  // uniform: the reference of the weights moved up
            const float f = unit / now;
#pragma unroll
            for (int db = 0; db < kDb; ++db) acc[db] *= f;
            unit = now;
        }
        const std::uint64_t live = tile_live[buf];
        const std::uint32_t key0 = tile * kTile;
        const bool masked = live != ~0ull || key0 + kTile - 1 > least_limit;  // uniform
        qp_f32x16_t s[2];
#pragma unroll
        for (int kb = 0; kb < 2; ++kb) {
            s[kb] = qp_f32x16_t{};
            const std::uint32_t row = 32 * kb + col;
            const unsigned char* const from = tiles_lds[buf][0] + row * kRowBytes;
#pragma unroll
            for (int kk = 0; kk < kSteps; ++kk) {
                const Vec a = __builtin_bit_cast(Vec, *reinterpret_cast<const uint4*>(from + 16 * k_slot(row, 2 * kk + half)));
                s[kb] = __builtin_amdgcn_mfma_f32_32x32x16_f16(a, q_lo[kk], s[kb], 0, 0, 0);
                s[kb] = __builtin_amdgcn_mfma_f32_32x32x16_f16(a, q_hi[kk], s[kb], 0, 0, 0);
            }
        }
        // Scores to s ks - ref in place: ks times the row's factor, finite (a product of
        // 0 stays 0; NaN stays).
        const auto finite = [](float y) { return y > 3.0e38f ? 3.0e38f : y; };
        const auto one = [](float y) { return __int_as_float(__builtin_amdgcn_readfirstlane(__float_as_int(y))); };
        float top = -INFINITY;
#pragma unroll
        for (int kb = 0; kb < 2; ++kb) {
            if constexpr (kUniform) {
#pragma unroll
                for (int g = 0; g < 2; ++g) {
                    const float ks = finite(one(tile_ks[buf][32 * kb + 16 * g]) * down);
#pragma unroll
                    for (int i = 0; i < 8; ++i) s[kb][8 * g + i] = fmaf(s[kb][8 * g + i], ks, -ref);
                }
            } else {
#pragma unroll
                for (int g = 0; g < 4; ++g) {
                    const float4 k4 = *reinterpret_cast<const float4*>(&tile_ks[buf][32 * kb + 8 * g + 4 * half]);
                    s[kb][4 * g] = fmaf(s[kb][4 * g], finite(k4.x * down), -ref);
                    s[kb][4 * g + 1] = fmaf(s[kb][4 * g + 1], finite(k4.y * down), -ref);
                    s[kb][4 * g + 2] = fmaf(s[kb][4 * g + 2], finite(k4.z * down), -ref);
                    s[kb][4 * g + 3] = fmaf(s[kb][4 * g + 3], finite(k4.w * down), -ref);
                }
            }
            if (masked) {  // uniform
                const std::uint32_t bits = static_cast<std::uint32_t>(live >> (32 * kb)) >> (4 * half);
                const int room = static_cast<int>(limit) - static_cast<int>(key0 + 32 * kb + 4 * half);
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    const int k = 8 * (i / 4) + i % 4;
                    if (k > room || !(bits >> k & 1)) s[kb][i] = -INFINITY;
                }
            }
#pragma unroll
            for (int i = 0; i < 16; i += 2) top = max3(top, s[kb][i], s[kb][i + 1]);
        }
        if (__builtin_expect(__builtin_amdgcn_ballot_w64(top > threshold) != 0, 0)) {  // uniform
            const auto swapped = __builtin_amdgcn_permlane32_swap(__float_as_uint(top), __float_as_uint(top), false, false);
            const float all = __builtin_elementwise_maximum(__uint_as_float(swapped[0]), __uint_as_float(swapped[1]));
            const bool moves = all > threshold;
            const float next = moves ? ref + all : ref, shift = next - ref;  // exact: what ref really moves by
            const float f = threshold == 0.0f ? __builtin_amdgcn_exp2f(-shift) : 1.0f;  // nothing there before
            if (moves) threshold = 0.0f;
            ref = next;
            sum *= f;
            low *= f;
#pragma unroll
            for (int db = 0; db < kDb; ++db) acc[db] *= f;
#pragma unroll
            for (int kb = 0; kb < 2; ++kb)
#pragma unroll
                for (int i = 0; i < 16; ++i) s[kb][i] -= shift;
        }
        // Weights, and their two parts: operand j of block kb holds scores 8 j .. 8 j + 7.
        Vec p_hi[2][2], p_lo[2][2];
#pragma unroll
        for (int kb = 0; kb < 2; ++kb) {
            float part = 0.0f;
#pragma unroll
            for (int i = 0; i < 16; ++i) s[kb][i] = __builtin_amdgcn_exp2f(s[kb][i]);
#pragma unroll
            for (int i = 0; i < 16; i += 4) part += (s[kb][i] + s[kb][i + 1]) + (s[kb][i + 2] + s[kb][i + 3]);
            two_sum_add(sum, low, part);
#pragma unroll
            for (int g = 0; g < (kUniform ? 2 : 4); ++g) {
                if constexpr (kUniform) {
                    const float vs = one(tile_vs[buf][32 * kb + 16 * g]);
#pragma unroll
                    for (int i = 0; i < 8; ++i) s[kb][8 * g + i] *= vs;
                } else {
                    const float4 v4 = *reinterpret_cast<const float4*>(&tile_vs[buf][32 * kb + 8 * g + 4 * half]);
                    s[kb][4 * g] *= v4.x;
                    s[kb][4 * g + 1] *= v4.y;
                    s[kb][4 * g + 2] *= v4.z;
                    s[kb][4 * g + 3] *= v4.w;
                }
            }
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                std::uint32_t hi[4], lo[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int n = 8 * j + 2 * i;
                    const pf_f32x2_t y{s[kb][n], s[kb][n + 1]};
                    const pf_f16x2_t h = __builtin_convertvector(y, pf_f16x2_t);
                    hi[i] = __builtin_bit_cast(std::uint32_t, h);
                    const pf_f32x2_t rest = y - __builtin_convertvector(h, pf_f32x2_t);
                    lo[i] = __builtin_bit_cast(std::uint32_t, __builtin_convertvector(rest, pf_f16x2_t));
                }
                p_hi[kb][j] = __builtin_bit_cast(Vec, make_uint4(hi[0], hi[1], hi[2], hi[3]));
                p_lo[kb][j] = __builtin_bit_cast(Vec, make_uint4(lo[0], lo[1], lo[2], lo[3]));
            }
        }
        // V^T: a group of 16 lanes transposes 4 tokens of 16 dims.
        const std::uint32_t in16 = lane % 16, token_in = 4 * half + in16 / 4;
        const std::uint32_t dim_chunk = 2 * (lane / 16 % 2) + in16 % 4 / 2;  // 16-byte chunk within a dim block's 64 bytes
        const std::uint32_t in_chunk = in16 % 2 * 8;
#pragma unroll
        for (int db = 0; db < kDb; ++db) {
            qp_f32x16_t o{};
#pragma unroll
            for (int kb = 0; kb < 2; ++kb)
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const auto read = [&](int more) {
                        const std::uint32_t row = 32 * kb + 16 * j + more + token_in;
                        const unsigned char* const at = tiles_lds[buf][1] + row * kRowBytes + 16 * v_slot(row, 4 * db + dim_chunk) + in_chunk;
                        return __builtin_amdgcn_ds_read_tr16_b64_v4i16((pf_lds_i16x4_t*)((__attribute__((address_space(3))) const unsigned char*)at));
                    };
                    const pf_i16x4_t a0 = read(0), a1 = read(8);
                    const Vec a = __builtin_bit_cast(Vec, __builtin_shufflevector(a0, a1, 0, 1, 2, 3, 4, 5, 6, 7));
                    o = __builtin_amdgcn_mfma_f32_32x32x16_f16(a, p_lo[kb][j], o, 0, 0, 0);
                    o = __builtin_amdgcn_mfma_f32_32x32x16_f16(a, p_hi[kb][j], o, 0, 0, 0);
                }
            acc[db] += o;
        }
    };

    if (tile_begin < tile_end) {  // uniform
        stage();
        __syncthreads();
        fetch(tile_begin);
        put(tile_begin, 0);
        __syncthreads();
        int buf = 0;
        for (std::uint32_t tile = tile_begin; tile < tile_end; ++tile) {
            const bool more = tile + 1 < tile_end;
            if (more) {
                if ((tile + 1) / p.window_tiles != window) {  // uniform
                    // Every wavefront is past its reads of the old pages: the last were
                    // before the barrier that ended the step.
                    ++window;
                    stage();
                    __syncthreads();
                }
                fetch(tile + 1);
            }
            if (wave_live) compute(tile, buf);
            if (more) put(tile + 1, buf ^ 1);
            __syncthreads();
            buf ^= 1;
        }
    }

    // Row `col`: dims 32 db + 8 g + 4 half .. + 3 in acc[db][4 g ..].
    sum += low;
    const auto swapped = __builtin_amdgcn_permlane32_swap(__float_as_uint(sum), __float_as_uint(sum), false, false);
    sum = __uint_as_float(swapped[0]) + __uint_as_float(swapped[1]);
    if (!row_live) return;
    const bool whole = p.splits == 1;
    const std::uint32_t head_at = kvh * p.group + head;
    const std::uint64_t part_row = ((static_cast<std::uint64_t>(split) * p.num_seqs + seq) * p.max_query + token) * p.query_heads + head_at;
    float* const to = whole ? p.output + ((p.query_offsets[seq] + token) * p.query_heads + head_at) * kD : p.part_acc + part_row * kD;
    const float inv = whole && sum != 0.0f ? 1.0f / sum : 1.0f, in_ones = unit * (1.0f / kWeightScale);
#pragma unroll
    for (int db = 0; db < kDb; ++db)
#pragma unroll
        for (int g = 0; g < 4; ++g)
            *reinterpret_cast<Float4*>(to + 32 * db + 8 * g + 4 * half) =
                Float4{acc[db][4 * g] * inv * in_ones, acc[db][4 * g + 1] * inv * in_ones, acc[db][4 * g + 2] * inv * in_ones,
                       acc[db][4 * g + 3] * inv * in_ones};
    if (!whole && half == 0) {
        p.part_ml[2 * part_row] = ref;
        p.part_ml[2 * part_row + 1] = sum;
    }
}

// Merges the splits of a (sequence, query token, head): a block is a query token's
// row and as many heads as fit, a thread 4 dims of one.
template <int kD>
__global__ __launch_bounds__(256) void quant_prefill_merge_kernel(QuantPrefillParams p) {
    struct Float4 { float x, y, z, w; };
    constexpr std::uint32_t kLanes = kD / 4;
    const std::uint32_t seq = blockIdx.y, per = 256 / kLanes;
    const std::uint64_t full_len = p.kv_lens[seq], full_q = p.query_lens[seq];
    const std::uint64_t len = full_len < p.max_kv ? full_len : p.max_kv, tq = full_q < len ? full_q : len;
    const std::uint64_t i = static_cast<std::uint64_t>(blockIdx.x) * per + threadIdx.x / kLanes;  // token * heads + head
    const std::uint64_t live = (tq < p.max_query ? tq : p.max_query) * p.query_heads;
    if (i >= live) return;
    const std::uint32_t d4 = threadIdx.x % kLanes;
    const std::uint64_t stride = static_cast<std::uint64_t>(p.num_seqs) * p.max_query * p.query_heads;
    const std::uint64_t at = static_cast<std::uint64_t>(seq) * p.max_query * p.query_heads + i;
    float top = -INFINITY, sum = 0.0f;
    Float4 o{0.0f, 0.0f, 0.0f, 0.0f};
    for (std::uint32_t s = 0; s < p.splits; ++s) {
        const float m = p.part_ml[2 * (s * stride + at)], l = p.part_ml[2 * (s * stride + at) + 1];
        if (l == 0.0f) continue;  // saw no key
        const Float4 v = *reinterpret_cast<const Float4*>(p.part_acc + (s * stride + at) * kD + 4 * d4);
        const float next = m > top ? m : top;
        // NaN sums stay NaN; the first split has nothing before it.
        const float f = top == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(top - next), g = __builtin_amdgcn_exp2f(m - next);
        o = Float4{o.x * f + v.x * g, o.y * f + v.y * g, o.z * f + v.z * g, o.w * f + v.w * g};
        sum = sum * f + l * g;
        top = next;
    }
    const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
    *reinterpret_cast<Float4*>(p.output + (p.query_offsets[seq] * p.query_heads + i) * kD + 4 * d4) =
        Float4{o.x * inv, o.y * inv, o.z * inv, o.w * inv};
}

// ---------------------------------------------------------------- dispatch
struct PrefillPlan {
    std::uint32_t rows;      // of a workgroup
    std::uint32_t heads_of;  // query heads of a launch: the largest divisor of the group that fits
    std::uint32_t tokens, blocks, splits, split_tiles;
};
constexpr std::uint32_t kCus = 256;
constexpr std::uint32_t kLeastTiles = 4;  // of a split

PrefillPlan prefill_plan(std::uint64_t num_seqs, std::uint64_t max_query, std::uint64_t max_kv, std::uint64_t heads,
                         std::uint64_t group, std::uint64_t head_size) {
    PrefillPlan plan{};
    plan.rows = head_size == 256 ? Shape<256>::kRows : Shape<128>::kRows;
    plan.heads_of = static_cast<std::uint32_t>(group < plan.rows ? group : plan.rows);
    while (group % plan.heads_of != 0) --plan.heads_of;
    plan.tokens = plan.rows / plan.heads_of;
    plan.blocks = static_cast<std::uint32_t>((max_query + plan.tokens - 1) / plan.tokens);
    const std::uint64_t workgroups = num_seqs * plan.blocks * heads, tiles = (max_kv + kTile - 1) / kTile;
    std::uint64_t splits = workgroups < kCus ? kCus / workgroups : 1;
    if (splits > tiles / kLeastTiles) splits = tiles / kLeastTiles;
    if (splits < 1) splits = 1;
    plan.split_tiles = static_cast<std::uint32_t>((tiles + splits - 1) / splits);
    plan.splits = static_cast<std::uint32_t>((tiles + plan.split_tiles - 1) / plan.split_tiles);
    return plan;
}
std::uint64_t prefill_workspace(const PrefillPlan& plan, std::uint64_t num_seqs, std::uint64_t max_query,
                                std::uint64_t query_heads, std::uint64_t head_size) {
    return plan.splits == 1 ? 0 : plan.splits * num_seqs * max_query * query_heads * (head_size + 2) * sizeof(float);
}

template <typename F, int kD>
int launch_prefill(QuantPrefillParams& p, hipStream_t stream) {
    const dim3 grid(p.heads * p.splits * p.num_seqs * p.blocks), threads(Shape<kD>::kThreads);
    for (p.first = 0; p.first < p.group; p.first += p.heads_of) {
        if (p.block_size.divisor % 16 == 0) quant_prefill_kernel<F, kD, true><<<grid, threads, 0, stream>>>(p);
        else quant_prefill_kernel<F, kD, false><<<grid, threads, 0, stream>>>(p);
        if (const int s = launch_status("quant_prefill_kernel")) return s;
    }
    if (p.splits == 1) return KVFLUX_OK;
    const std::uint64_t per = 256 / (kD / 4);
    quant_prefill_merge_kernel<kD><<<dim3(static_cast<unsigned>((static_cast<std::uint64_t>(p.max_query) * p.query_heads + per - 1) / per), p.num_seqs),
                                     dim3(256), 0, stream>>>(p);
    return launch_status("quant_prefill_merge_kernel");
}
template <typename F>
int launch_prefill_head_size(QuantPrefillParams& p, std::uint64_t head_size, hipStream_t s) {
    switch (head_size) {
    case 64: return launch_prefill<F, 64>(p, s);
    case 128: return launch_prefill<F, 128>(p, s);
    default: return launch_prefill<F, 256>(p, s);
    }
}

bool fast_head_size(std::uint64_t head_size) { return head_size == 64 || head_size == 128 || head_size == 256; }

int check_prefill(const char* op, std::uint64_t num_seqs, std::uint64_t max_query, std::uint64_t max_kv,
                  std::uint64_t heads, std::uint64_t query_heads, std::uint64_t block_size, std::uint64_t head_size) {
    if (heads == 0 || block_size == 0 || head_size == 0 || query_heads == 0 || query_heads % heads != 0)
        return fail(KVFLUX_ERR_INVALID_ARGUMENT, "%s: invalid shape", op);
    if (max_query > max_kv) return fail(KVFLUX_ERR_INVALID_ARGUMENT, "%s: more queries than tokens", op);
    // Workgroups, query rows and keys are counted in 31 bits.
    if (heads > 65535 || head_size > 512 || block_size > 0x7fffffffULL / head_size || query_heads > 0xfffffULL ||
        num_seqs > 65535 || max_kv > 0x7fffff00ULL || num_seqs * max_query > 0x7fffffffULL / query_heads)
        return fail(KVFLUX_ERR_UNSUPPORTED, "%s: shape too large", op);
    return KVFLUX_OK;
}

} // namespace
} // namespace kvflux_hip

using namespace kvflux_hip;

extern "C" int kvflux_quant_prefill_workspace_size(uint64_t num_seqs, uint64_t max_query_tokens, uint64_t max_kv_len,
                                                   uint64_t num_kv_heads, uint64_t query_heads, uint64_t block_size,
                                                   uint64_t head_size, size_t* bytes) {
    if (!bytes) return fail(KVFLUX_ERR_INVALID_ARGUMENT, "quant prefill workspace: null pointer");
    *bytes = 0;
    if (const int s = check_prefill("quant prefill workspace", num_seqs, max_query_tokens, max_kv_len, num_kv_heads,
                                    query_heads, block_size, head_size))
        return s;
    if (num_seqs == 0 || max_query_tokens == 0 || !fast_head_size(head_size)) return KVFLUX_OK;
    const PrefillPlan plan = prefill_plan(num_seqs, max_query_tokens, max_kv_len, num_kv_heads, query_heads / num_kv_heads, head_size);
    *bytes = prefill_workspace(plan, num_seqs, max_query_tokens, query_heads, head_size);
    return KVFLUX_OK;
}

extern "C" int kvflux_quant_prefill(const void* key_cache, const void* value_cache, const float* key_scales,
                                    const float* value_scales, uint64_t num_blocks, uint64_t num_kv_heads,
                                    uint64_t block_size, uint64_t head_size, int format, const uint64_t* block_table,
                                    uint64_t max_blocks_per_seq, const uint64_t* kv_lens, const uint64_t* query_lens,
                                    const uint64_t* query_offsets, uint64_t num_seqs, uint64_t max_query_tokens,
                                    uint64_t max_kv_len, uint64_t query_heads, const float* query, float* output,
                                    void* workspace, size_t workspace_bytes, void* stream) {
    if (num_seqs == 0 || max_query_tokens == 0) return KVFLUX_OK;
    if (const int s = check_quant_cache("quant prefill", key_cache, value_cache, key_scales, value_scales, num_blocks,
                                        num_kv_heads, block_size, head_size, format))
        return s;
    if (!block_table || !kv_lens || !query_lens || !query_offsets || !query || !output)
        return fail(KVFLUX_ERR_INVALID_ARGUMENT, "quant prefill: null pointer");
    if (max_blocks_per_seq == 0) return fail(KVFLUX_ERR_INVALID_ARGUMENT, "quant prefill: empty table rows");
    if (const int s = check_prefill("quant prefill", num_seqs, max_query_tokens, max_kv_len, num_kv_heads, query_heads, block_size, head_size))
        return s;
    if (num_blocks >= kMissing) return fail(KVFLUX_ERR_UNSUPPORTED, "quant prefill: too many pages");
    if (!aligned(4, {query, output}) || !aligned(8, {block_table, kv_lens, query_lens, query_offsets}))
        return fail(KVFLUX_ERR_INVALID_ARGUMENT, "quant prefill: misaligned array");
    const std::uint64_t group = query_heads / num_kv_heads;
    const float scale_log2 = static_cast<float>(1.4426950408889634 / std::sqrt(static_cast<double>(head_size)));
    if (!fast_head_size(head_size) || !aligned(16, {key_cache, value_cache})) {
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
        rows.lens = kv_lens;
        rows.kv_len = static_cast<std::uint32_t>(max_kv_len);
        rows.query_lens = query_lens;
        rows.query_offsets = query_offsets;
        rows.max_query = static_cast<std::uint32_t>(max_query_tokens);
        rows.query_heads = static_cast<std::uint32_t>(query_heads);
        rows.group = static_cast<std::uint32_t>(group);
        rows.query = query;
        rows.output = output;
        rows.scale_log2 = scale_log2;
        return launch_quant_rows(rows, num_seqs * max_query_tokens, format, as_stream(stream));
    }
    const PrefillPlan plan = prefill_plan(num_seqs, max_query_tokens, max_kv_len, num_kv_heads, group, head_size);
    QuantPrefillParams p{};
    p.key_cache = static_cast<const std::uint8_t*>(key_cache);
    p.value_cache = static_cast<const std::uint8_t*>(value_cache);
    p.key_scales = key_scales;
    p.value_scales = value_scales;
    p.num_blocks = num_blocks;
    p.heads = static_cast<std::uint32_t>(num_kv_heads);
    p.block_size = FastDiv(static_cast<std::uint32_t>(block_size));
    p.table = block_table;
    p.width = max_blocks_per_seq;
    p.kv_lens = kv_lens;
    p.query_lens = query_lens;
    p.query_offsets = query_offsets;
    p.num_seqs = static_cast<std::uint32_t>(num_seqs);
    p.max_query = static_cast<std::uint32_t>(max_query_tokens);
    p.max_kv = static_cast<std::uint32_t>(max_kv_len);
    p.query_heads = static_cast<std::uint32_t>(query_heads);
    p.group = static_cast<std::uint32_t>(group);
    p.heads_of = plan.heads_of;
    p.heads_div = FastDiv(plan.heads_of);
    p.tokens = plan.tokens;
    p.blocks = plan.blocks;
    p.splits = plan.splits;
    p.split_tiles = plan.split_tiles;
    // A window of n tiles has at most n * kTile / block_size + 2 pages.
    const std::uint64_t window = (kWindow - 2) * block_size / kTile;
    p.window_tiles = static_cast<std::uint32_t>(window < 0x7fffffffULL ? window : 0x7fffffffULL);
    p.query = query;
    p.output = output;
    p.scale_log2 = scale_log2;
    if (static_cast<std::uint64_t>(p.heads) * p.splits * p.num_seqs * p.blocks > 0x7fffffffULL)
        return fail(KVFLUX_ERR_UNSUPPORTED, "quant prefill: shape too large");
    if (plan.splits > 1) {
        if (!workspace || workspace_bytes < prefill_workspace(plan, num_seqs, max_query_tokens, query_heads, head_size))
            return fail(KVFLUX_ERR_INVALID_ARGUMENT, "quant prefill: workspace too small");
        if (!aligned(4, {workspace})) return fail(KVFLUX_ERR_INVALID_ARGUMENT, "quant prefill: misaligned workspace");
        p.part_acc = static_cast<float*>(workspace);
        p.part_ml = p.part_acc + static_cast<std::uint64_t>(plan.splits) * num_seqs * max_query_tokens * query_heads * head_size;
    }
    return format == KVFLUX_QUANT_E4M3 ? launch_prefill_head_size<QuantE4m3>(p, head_size, as_stream(stream))
                                       : launch_prefill_head_size<QuantInt8>(p, head_size, as_stream(stream));
}
