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
//  * Keys go through LDS in tiles of 64: a thread loads its bytes of the next tile's K
//    and V into registers while this one is computed, widens them to FP16 once for all
//    wavefronts and stores them to the other buffer.
//  * Eight wavefronts work in phases: of a SIMD's two, one multiplies while the other works
//    out weights (512 tokens behind 32768 506 us without the phases, 490 with them: 14 %
//    fewer cycles, of which the lower clock under that load gives most back).
//  * S^T = K Q^T leaves lane (row, half) with keys 8 i + 4 half .. + 3 of the row:
//    O^T += V^T P^T takes them as they are when V's tokens are read in that order
//    (ds_read_b64_tr_b16, four tokens of a dim a lane).
//  * The scales stay out of K and V: ks joins the score's subtraction (one FMA), vs
//    multiplies the weight.
//  * The tile's weighted values are summed from zero and added with one rounding: an
//    MFMA on a large accumulator drops bits of small weights, always in one direction.
//  * Where workgroups are few, two sets of four wavefronts on the same rows take every other
//    tile and are merged in LDS; where CUs would be left idle (a short chunk behind a long
//    prefix) a block's keys go to several workgroups, merged by a second kernel.
//  * Every 144 tiles a row's sums are folded into its place in the output, so that a row
//    which one key dominates loses nothing of the others (kFold).
//
// 32 query heads, 8 kv heads of 128: 512 tokens behind 32768 479 us, 1157 TFLOP/s of the
// two parts' products, where a large library product in FP16 reaches 1174; 8 prompts of
// 4096 2.00 ms, 1097 TFLOP/s, the diagonal tiles' masked half counted out. What is left is
// the arithmetic beside the matrix instructions, some 400 VALU instructions of a tile and
// wavefront to 64 MFMAs, and the power that both draw.
#include "mfma_parts.h"
#include "quant.h"

#include <cmath>
#include <type_traits>

namespace kvflux_hip {
namespace {

typedef __attribute__((ext_vector_type(16))) float qp_f32x16_t;

constexpr std::uint32_t kTile = 64;     // keys of a tile
constexpr std::uint32_t kWindow = 1024; // pages whose ids and scales are in LDS at a time
constexpr std::uint32_t kUnread = 0x80000000u;  // a page whose bytes are not read, in place of its id
constexpr std::uint32_t kMissing = ~0u;         // one that is not there
constexpr std::uint32_t kBand = 16;       // powers of two of |vs| worked on at once, see `present`
// Tiles after which a row's sums are folded into its place in the output, with the addition's
// rounding error kept. A tile's sum is added to the accumulator in FP32: beside a dominant key's
// value one that is under half a step is lost, 2^-24 a tile at most, so 9e-6 of a row for 144
// (rows of 32768 tokens without: 3e-5; the contract is 1e-5).
constexpr std::uint32_t kFold = 144;
constexpr float kWeightScale = 32768.0f;  // as in the decode: parts of 2^15 times a weight of at most 1

// How a workgroup's wavefronts share its work: four of 32 rows each; eight that take turns;
// or two sets of four on the same 128 rows, which take every other tile and are merged.
enum class Order { Four, Turns, Halves };

template <int kD, Order kOrder, bool kUniform>
struct Shape {
    static constexpr int kWaves = kOrder == Order::Four ? 4 : 8;
    static constexpr int kSets = kOrder == Order::Halves ? 2 : 1;
    static constexpr int kThreads = 64 * kWaves;
    static constexpr int kLoaders = kThreads / kSets;  // threads that load a tile
    static constexpr std::uint32_t kRows = 32 * kWaves / kSets;
    // Wavefronts of a SIMD: the registers of two hold Q and the sums of 32 rows up to D = 128,
    // of three at 64 (8 prompts of 2048: two 181 us, three 167), but not with scales that
    // differ within 16 keys.
    static constexpr int kPerSimd = kD == 256 ? 1 : kD == 64 && kUniform && kOrder == Order::Four ? 3 : 2;
};

struct QuantPrefillParams {
    const std::uint8_t* key_cache;
    const std::uint8_t* value_cache;
    const float* key_scales;
    const float* value_scales;
    std::uint64_t num_blocks;
    std::uint32_t heads, head_size;    // a multiple of 16, at most kD
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
    std::uint32_t splits, split_tiles; // workgroups of a block of queries at most, tiles of each
    std::uint32_t window_tiles;        // tiles whose pages fit kWindow; at most kFold where sums are folded
    std::uint32_t fold_windows;        // windows that are folded together
    const float* query;
    float* output;
    float scale_log2;
    float* part_acc;  // [splits][num_seqs * max_query][query_heads][kD]
    float* part_ml;   // [splits][num_seqs * max_query][query_heads][2]
};

// How many workgroups share a block of queries whose last sees `tile_count` tiles, at
// most `most` each, and the tiles of one.
struct Split {
    std::uint32_t count, tiles;
};
__device__ inline Split split_of(std::uint32_t tile_count, std::uint32_t most) {
    const std::uint32_t count = (tile_count - 1) / most + 1;
    return {count, (tile_count - 1) / count + 1};
}

// kUniform: pages are multiples of 16 tokens, so 16 neighbouring keys of a tile share
// their scales, which are then one value for a wavefront.
// kFolds: a workgroup may have more than kFold tiles (and is not in two sets).
template <typename F, int kD, Order kOrder, bool kUniform, bool kFolds>
__global__ __launch_bounds__((Shape<kD, kOrder, kUniform>::kThreads), (Shape<kD, kOrder, kUniform>::kPerSimd)) void quant_prefill_kernel(QuantPrefillParams p) {
    using S = Shape<kD, kOrder, kUniform>;
    using Vec = pf_f16x8_t;
    constexpr int kThreads = S::kThreads, kWaves = S::kWaves, kSets = S::kSets, kLoaders = S::kLoaders;
    constexpr int kSteps = kD / 16;            // MFMAs of a 32-key block of S^T for one part of Q
    constexpr int kDb = kD / 32;               // dim blocks of O^T
    constexpr int kRowBytes = kD * 2;          // a key's row in LDS
    constexpr int kCpr = kRowBytes / 16;
    constexpr int kTileBytes = static_cast<int>(kTile) * kRowBytes;
    // Bytes of K, and as many of V, that a thread loads of a tile: of one key.
    constexpr int kBytes = static_cast<int>(kTile) * kD / kLoaders;
    constexpr int kKeyThreads = kD / kBytes;   // threads of a key
    constexpr int kWords = kBytes / 4;
    static_assert(kBytes % 16 == 0 && kD % kBytes == 0, "tile split");
    // [set][buffer][K, V]; at the end of two sets the second one's sums.
    constexpr int kPad = kD + 4;
    __shared__ __attribute__((aligned(16))) unsigned char tiles_lds[kSets][2][2][kTileBytes];
    static_assert(kSets == 1 || sizeof(tiles_lds) >= S::kRows * kPad * sizeof(float), "merge buffer");
    __shared__ float2 stats[kSets == 1 ? 1 : S::kRows];
    __shared__ std::uint32_t page_id[kWindow];
    __shared__ float page_ks[kWindow], page_vs[kWindow];  // vs over the reference, times kWeightScale
    // Where the scales differ within 16 keys: those of a buffer's keys.
    __shared__ __attribute__((aligned(16))) float key_ks[kSets][kUniform ? 1 : 2][kUniform ? 4 : kTile];
    __shared__ __attribute__((aligned(16))) float key_vs[kSets][kUniform ? 1 : 2][kUniform ? 4 : kTile];
    __shared__ float wave_top[kWaves], wave_least[kWaves];
    __shared__ std::uint32_t wave_missing[kWaves], wave_bands[kWaves];
    static_assert(!kFolds || kSets == 1, "a set has no place to fold into");
    __shared__ float* place_of[kFolds ? kThreads : 1];
    __shared__ float fold_ref[kFolds ? S::kRows : 1], fold_unit;  // of the sums folded so far: ref, -INFINITY for none, and unit

    const int tid = threadIdx.x, lane = tid % 64;
    const std::uint32_t wave = static_cast<std::uint32_t>(__builtin_amdgcn_readfirstlane(tid / 64));
    const int col = lane % 32, half = lane / 32;
    // Heaviest query blocks first; neighbouring workgroups take the kv heads in turn, then the
    // sequences, at every block from another one on: workgroups go to the shader engines in
    // turn, and the longest sequence's are not to meet on one (16 prompts of up to 2048 tokens,
    // 8 kv heads: 658 us without, 473 with).
    std::uint32_t x = blockIdx.x;
    const std::uint32_t kvh = x % p.heads;
    x /= p.heads;
    const std::uint32_t split = x % p.splits;
    x /= p.splits;
    const std::uint32_t level = x / p.num_seqs, qb = p.blocks - 1 - level, seq = (x + level) % p.num_seqs;
    const std::uint64_t full_len = p.kv_lens[seq], full_q = p.query_lens[seq];
    const std::uint32_t kv_len = full_len < p.max_kv ? static_cast<std::uint32_t>(full_len) : p.max_kv;
    std::uint32_t tq = full_q < kv_len ? static_cast<std::uint32_t>(full_q) : kv_len;
    if (tq > p.max_query) tq = p.max_query;
    const std::uint32_t t0 = qb * p.tokens;
    if (t0 >= tq) return;  // uniform
    const std::uint32_t t_end = t0 + p.tokens < tq ? t0 + p.tokens : tq;
    const std::uint32_t past = kv_len - tq;
    const std::uint32_t tile_count = (past + t_end - 1) / kTile + 1;
    const Split mine = split_of(tile_count, p.split_tiles);
    if (split >= mine.count) return;  // uniform
    const std::uint32_t tile_begin = split * mine.tiles < tile_count ? split * mine.tiles : tile_count;
    const std::uint32_t tile_end = tile_begin + mine.tiles < tile_count ? tile_begin + mine.tiles : tile_count;
    const std::uint64_t* const table = p.table + seq * p.width;

    // This lane's row.
    const std::uint32_t set = kSets == 1 ? 0 : wave / 4;  // uniform
    const std::uint32_t r = 32 * (kSets == 1 ? wave : wave % 4) + static_cast<std::uint32_t>(col);
    const std::uint32_t token = t0 + p.heads_div.div(r), head = p.first + p.heads_div.mod(r);
    const bool row_live = r < p.tokens * p.heads_of && token < t_end;
    const bool wave_live = __builtin_amdgcn_ballot_w64(row_live) != 0;
    const std::uint64_t q_row = (p.query_offsets[seq] + (row_live ? token : t0)) * p.query_heads + kvh * p.group + (row_live ? head : p.first);
    const std::uint32_t D = p.head_size, head_at = kvh * p.group + head;
    // A live row's place: in the output where one workgroup sees all its keys, else a partial.
    const auto row_place = [&] {
        const std::uint64_t part = ((static_cast<std::uint64_t>(split) * p.num_seqs + seq) * p.max_query + token) * p.query_heads + head_at;
        return mine.count == 1 ? p.output + ((p.query_offsets[seq] + token) * p.query_heads + head_at) * D : p.part_acc + part * kD;
    };
    const float* const q_src = p.query + q_row * D;
    struct Float4 { float x, y, z, w; };  // float-aligned
    Float4 raw[kSteps][2];
#pragma unroll
    for (int kk = 0; kk < kSteps; ++kk)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const std::uint32_t d = 16 * kk + 8 * half + 4 * i;
            raw[kk][i] = *reinterpret_cast<const Float4*>(q_src + (d < D ? d : 0));
            if (d >= D) raw[kk][i] = Float4{0.0f, 0.0f, 0.0f, 0.0f};
        }

    const auto one = [](float y) { return __int_as_float(__builtin_amdgcn_readfirstlane(__float_as_int(y))); };

    // ---- the window's pages: ids, scales, the largest |vs| so far (the weights' reference).
    std::uint32_t window = 0;              // window_tiles tiles each, from tile_begin on
    std::uint32_t window_page = 0;         // page of page_id[0]
    float reference = 0.0f, floor = 0.0f;  // floor: of the windows before
    bool missing = false;                  // a page of the window is
    // A query need not see the window's largest |vs|: a weight's parts, relative to that, would
    // lose bits of what it sees (2^15 times a weight over 2^16 is 2^-1, and FP16 ends at
    // 2^-24). So pages whose |vs| is under 2^-16 of the largest are worked on in a pass of their
    // own, in a smaller unit, and so on from the smallest up: the sums' unit only grows. Such a pass
    // takes the tiles that have a page of its band, run by run; the last one takes all, and counts
    // the weights. (512 tokens behind 16384 302 us; with 2 pages of zeros, whose scale is the least
    // there is, 304; with 20 339.) What sees a page of this window sees all of the windows before,
    // so no unit need be smaller than `floor`.
    std::uint32_t present = 1;                    // bits of the bands that have a page, and of the last pass's, 0
    float now = 1.0f, counted = 1.0f;             // the pass's unit; whether its weights count (1 or 0)
    const auto stage = [&](std::uint32_t band) {  // ~0: of the window's first pass. Returns the pass's band
        const std::uint32_t tile0 = tile_begin + window * p.window_tiles;
        const std::uint32_t tile1 = tile0 + p.window_tiles < tile_end ? tile0 + p.window_tiles : tile_end;
        window_page = p.block_size.div(tile0 * kTile);
        const std::uint32_t pages = p.block_size.div(tile1 * kTile - 1) - window_page + 1;
        float top = 0.0f, least = INFINITY;
        bool lost = false;
        for (std::uint32_t i = tid; i < pages; i += kThreads) {
            const std::uint64_t page = window_page + i;
            const bool in_row = page < p.width && page * p.block_size.divisor < kv_len;
            const std::uint64_t id = table[in_row ? page : 0];
            const bool live = in_row && id < p.num_blocks;
            const std::uint64_t at = (live ? id : 0) * p.heads + kvh;
            float ks = live ? p.key_scales[at] : 0.0f, vs = live ? p.value_scales[at] : 0.0f;
            page_id[i] = live ? static_cast<std::uint32_t>(id) : kMissing;
            // What sees these values is NaN by its score. What does not is left alone: their
            // bytes may be NaN as well, and a weight of 0 times that is.
            if (!(__builtin_fabsf(vs) < INFINITY)) {
                ks = __builtin_nanf("");
                vs = 0.0f;
                page_id[i] = kUnread;
            }
            page_ks[i] = ks;
            page_vs[i] = vs;
            top = fmaxf(top, __builtin_fabsf(vs));
            if (vs != 0.0f) least = fminf(least, __builtin_fabsf(vs));
            lost |= !live && page * p.block_size.divisor < kv_len;  // behind that no query sees
        }
        top = wave_max(top);
        least = -wave_max(-least);
        const bool any_lost = __builtin_amdgcn_ballot_w64(lost) != 0;
        if (lane == 0) {
            wave_top[wave] = top;
            wave_least[wave] = least;
            wave_missing[wave] = any_lost;
        }
        __syncthreads();
        std::uint32_t lost_all = 0;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) {
            top = fmaxf(top, wave_top[w]);
            least = fminf(least, wave_least[w]);
            lost_all |= wave_missing[w];
        }
        reference = one(fmaxf(reference, top));
        missing = __builtin_amdgcn_readfirstlane(static_cast<int>(lost_all)) != 0;
        now = reference > 0.0f ? reference : 1.0f;
        // Exponents of a float that is not 0 lie between -148 and 128.
        const int tallest = __builtin_amdgcn_frexp_expf(now), lowest = floor > 0.0f ? __builtin_amdgcn_frexp_expf(floor) : -1024;
        const auto band_of = [&](float vs) {
            const int e = __builtin_amdgcn_frexp_expf(vs);
            return static_cast<std::uint32_t>(tallest - (e > lowest ? e : lowest)) / kBand;
        };
        const bool one_band = __builtin_amdgcn_readfirstlane(top == 0.0f || band_of(least) == 0);
        if (__builtin_expect(one_band, 1)) {
            present = 1;
            band = 0;
        } else {
            std::uint32_t seen = 0;
            for (std::uint32_t i = tid; i < pages; i += kThreads)
                if (page_vs[i] != 0.0f) seen |= 1u << band_of(page_vs[i]);
            seen = over_wave(seen, [](std::uint32_t a, std::uint32_t b) { return a | b; });
            if (lane == 0) wave_bands[wave] = seen;
            __syncthreads();
            present = 1;
#pragma unroll 1
            for (int w = 0; w < kWaves; ++w) present |= wave_bands[w];
            present = static_cast<std::uint32_t>(__builtin_amdgcn_readfirstlane(static_cast<int>(present)));
            if (band == ~0u) band = 31 - __builtin_clz(present);
            // |vs| of a band are under 2^(1 - kBand * band) of the largest.
            if (band != 0) now = one(__builtin_amdgcn_ldexpf(now, 1 - static_cast<int>(kBand * band)));
            for (std::uint32_t i = tid; i < pages; i += kThreads)
                if (band_of(page_vs[i]) != band) page_vs[i] = 0.0f;
        }
        counted = band == 0 ? 1.0f : 0.0f;
        for (std::uint32_t i = tid; i < pages; i += kThreads) page_vs[i] = page_vs[i] / now * kWeightScale;
        __syncthreads();
        return band;
    };
    // Whether a tile has a page of the pass's band; the same in every wavefront.
    const auto band_tile = [&](std::uint32_t tile) {
        return __builtin_amdgcn_ballot_w64(page_vs[p.block_size.div(tile * kTile + lane) - window_page] != 0.0f) != 0;
    };

    // ---- loads: a thread's kBytes of K and of V of one key of a tile, at the same place.
    const std::uint32_t loader = static_cast<std::uint32_t>(tid) % kLoaders;
    const std::uint32_t my_row = loader / kKeyThreads, my_col = loader % kKeyThreads * kBytes;
    const std::uint64_t head_bytes = static_cast<std::uint64_t>(p.block_size.divisor) * D;
    std::uint32_t held[2][kWords];
    bool held_live = false;  // V's
    const auto fetch_one = [&](int which, std::uint32_t tile) {
        const std::uint32_t key = tile * kTile + my_row, page = p.block_size.div(key);
        const std::uint32_t id = page_id[page - window_page];
        if (which) held_live = !(id & kUnread) && key < kv_len;
        // In place of a page that is not read: the pool's first row.
        const std::uint64_t at = id & kUnread ? 0 : (static_cast<std::uint64_t>(id) * p.heads + kvh) * head_bytes +
                                                        (key - page * p.block_size.divisor) * D;
        const std::uint8_t* const row = (which ? p.value_cache : p.key_cache) + at;
#pragma unroll
        for (int i = 0; i < kBytes / 16; ++i) {
            // Past the head's end its first bytes: they meet queries of 0, or make outputs that
            // are not stored.
            const std::uint32_t c = my_col + 16 * i;
            __builtin_memcpy(held[which] + 4 * i, __builtin_assume_aligned(row + (c < D ? c : 0), 16), 16);
        }
    };
    // Swizzled slots of a row's 16-byte chunks (LDS repeats its banks every 128 bytes). K is
    // read 16 rows of one chunk at a time, V 4 rows of 32 bytes.
    const auto k_slot = [](std::uint32_t row, std::uint32_t c) { return c ^ (row & (kCpr >= 16 ? 15 : 7)); };
    const auto v_slot = [](std::uint32_t row, std::uint32_t c) { return c ^ (2 * (row & 3)); };
    const auto put_one = [&](int which, unsigned char* buf) {  // buf: K's tile, V's behind it
#pragma unroll
        for (int i = 0; i < kWords; i += 2) {  // eight values: one chunk of K or V
            std::uint32_t w0 = held[which][i], w1 = held[which][i + 1];
            if (which && !held_live) w0 = w1 = 0;  // 0 * NaN would stay
            const std::uint32_t c = my_col / 8 + i / 2;
            *reinterpret_cast<uint4*>(buf + which * kTileBytes + my_row * kRowBytes + 16 * (which ? v_slot(my_row, c) : k_slot(my_row, c))) =
                make_uint4(F::template pair16<0>(w0), F::template pair16<1>(w0), F::template pair16<0>(w1), F::template pair16<1>(w1));
        }
    };
    // Scales of a tile's keys where those of 16 neighbours differ; missing pages' are 0.
    const auto put_scales = [&](std::uint32_t tile, float* ks, float* vs) {
        if (kUniform || loader >= kTile) return;
        const std::uint32_t i = p.block_size.div(tile * kTile + loader) - window_page;
        ks[loader] = page_ks[i];
        vs[loader] = page_vs[i];
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

    // Of a tile's four groups of 16 keys: the scales (kUniform), and which keys count.
    struct Marks {
        float ks[4], vs[4];
        std::uint64_t live;
    };
    const auto marks_of = [&](std::uint32_t tile) {
        Marks m;
        if constexpr (kUniform) {
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const std::uint32_t i = p.block_size.div(tile * kTile + 16 * g) - window_page;
                m.ks[g] = one(page_ks[i]);
                m.vs[g] = one(page_vs[i]);
            }
        }
        m.live = ~0ull;
        if (missing) m.live = __builtin_amdgcn_ballot_w64(page_id[p.block_size.div(tile * kTile + lane) - window_page] != kMissing);
        return m;
    };

    // Score i of a lane in block kb is key 32 kb + 8 (i / 4) + 4 half + i % 4 of the tile.
    struct Scores {
        qp_f32x16_t of[2];
    };
    struct Weights {  // operand j of block kb holds those of scores 8 j .. 8 j + 7, in two parts
        Vec hi[2][2], lo[2][2];
    };
    const auto scores = [&](const unsigned char* buf) {
        Scores out;
        auto& s = out.of;
#pragma unroll
        for (int kb = 0; kb < 2; ++kb) {
            s[kb] = qp_f32x16_t{};
            const std::uint32_t row = 32 * kb + col;
            const unsigned char* const from = buf + row * kRowBytes;
#pragma unroll
            for (int kk = 0; kk < kSteps; ++kk) {
                const Vec a = __builtin_bit_cast(Vec, *reinterpret_cast<const uint4*>(from + 16 * k_slot(row, 2 * kk + half)));
                s[kb] = __builtin_amdgcn_mfma_f32_32x32x16_f16(a, q_lo[kk], s[kb], 0, 0, 0);
                s[kb] = __builtin_amdgcn_mfma_f32_32x32x16_f16(a, q_hi[kk], s[kb], 0, 0, 0);
            }
        }
        // Operands of the next products on their way while these are computed.
        __builtin_amdgcn_sched_group_barrier(0x100, 3, 0);
#pragma unroll
        for (int i = 0; i < 2 * kSteps - 3; ++i) {
            __builtin_amdgcn_sched_group_barrier(0x008, 2, 0);
            __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
        }
        __builtin_amdgcn_sched_group_barrier(0x008, 2 * 3, 0);
        return out;
    };
    const auto weights = [&](Scores scores_of, std::uint32_t tile, const Marks& marks, const float* key_k, const float* key_v) {
        auto& s = scores_of.of;
        if (now != unit) {  // uniform: the reference of the weights moved up
            const float f = unit / now;
#pragma unroll
            for (int db = 0; db < kDb; ++db) acc[db] *= f;
            unit = now;
        }
        const std::uint64_t live = marks.live;
        const std::uint32_t key0 = tile * kTile;
        const bool masked = live != ~0ull || key0 + kTile - 1 > least_limit;  // uniform; keys past the sequence are past every limit
        // Scores to s ks - ref in place: ks times the row's factor, finite (a product of
        // 0 stays 0; NaN stays).
        const auto finite = [](float y) { return y > 3.0e38f ? 3.0e38f : y; };
        float top = -INFINITY;
#pragma unroll
        for (int kb = 0; kb < 2; ++kb) {
            if constexpr (kUniform) {
#pragma unroll
                for (int g = 0; g < 2; ++g) {
                    const float ks = finite(marks.ks[2 * kb + g] * down);
#pragma unroll
                    for (int i = 0; i < 8; ++i) s[kb][8 * g + i] = fmaf(s[kb][8 * g + i], ks, -ref);
                }
            } else {
#pragma unroll
                for (int g = 0; g < 4; ++g) {
                    const float4 k4 = *reinterpret_cast<const float4*>(key_k + 32 * kb + 8 * g + 4 * half);
                    s[kb][4 * g] = fmaf(s[kb][4 * g], finite(k4.x * down), -ref);
                    s[kb][4 * g + 1] = fmaf(s[kb][4 * g + 1], finite(k4.y * down), -ref);
                    s[kb][4 * g + 2] = fmaf(s[kb][4 * g + 2], finite(k4.z * down), -ref);
                    s[kb][4 * g + 3] = fmaf(s[kb][4 * g + 3], finite(k4.w * down), -ref);
                }
            }
        }
        if (__builtin_expect(masked, 0)) {  // uniform
            asm volatile("");               // a branch: as selects it would cost every tile 130 instructions
#pragma unroll
            for (int kb = 0; kb < 2; ++kb) {
                const std::uint32_t bits = static_cast<std::uint32_t>(live >> (32 * kb)) >> (4 * half);
                const int room = static_cast<int>(limit) - static_cast<int>(key0 + 32 * kb + 4 * half);
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    const int k = 8 * (i / 4) + i % 4;
                    if (k > room || !(bits >> k & 1)) s[kb][i] = -INFINITY;
                }
            }
        }
#pragma unroll
        for (int kb = 0; kb < 2; ++kb)
#pragma unroll
            for (int i = 0; i < 16; i += 2) top = max3(top, s[kb][i], s[kb][i + 1]);
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
        Weights out;
#pragma unroll
        for (int kb = 0; kb < 2; ++kb) {
            float part = 0.0f;
#pragma unroll
            for (int i = 0; i < 16; ++i) s[kb][i] = __builtin_amdgcn_exp2f(s[kb][i]);
#pragma unroll
            for (int i = 0; i < 16; i += 4) part += (s[kb][i] + s[kb][i + 1]) + (s[kb][i + 2] + s[kb][i + 3]);
            two_sum_add(sum, low, part * counted);
#pragma unroll
            for (int g = 0; g < (kUniform ? 2 : 4); ++g) {
                if constexpr (kUniform) {
                    const float vs = marks.vs[2 * kb + g];
#pragma unroll
                    for (int i = 0; i < 8; ++i) s[kb][8 * g + i] *= vs;
                } else {
                    const float4 v4 = *reinterpret_cast<const float4*>(key_v + 32 * kb + 8 * g + 4 * half);
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
                out.hi[kb][j] = __builtin_bit_cast(Vec, make_uint4(hi[0], hi[1], hi[2], hi[3]));
                out.lo[kb][j] = __builtin_bit_cast(Vec, make_uint4(lo[0], lo[1], lo[2], lo[3]));
            }
        }
        return out;
    };
    const auto weigh = [&](const Weights& w, const unsigned char* buf) {
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
                        const unsigned char* const at = buf + kTileBytes + row * kRowBytes + 16 * v_slot(row, 4 * db + dim_chunk) + in_chunk;
                        return __builtin_amdgcn_ds_read_tr16_b64_v4i16((pf_lds_i16x4_t*)((__attribute__((address_space(3))) const unsigned char*)at));
                    };
                    const pf_i16x4_t a0 = read(0), a1 = read(8);
                    const Vec a = __builtin_bit_cast(Vec, __builtin_shufflevector(a0, a1, 0, 1, 2, 3, 4, 5, 6, 7));
                    o = __builtin_amdgcn_mfma_f32_32x32x16_f16(a, w.lo[kb][j], o, 0, 0, 0);
                    o = __builtin_amdgcn_mfma_f32_32x32x16_f16(a, w.hi[kb][j], o, 0, 0, 0);
                }
#pragma unroll
            for (int i = 0; i < 16; ++i) acc[db][i] += o[i];
        }
        __builtin_amdgcn_sched_group_barrier(0x100, 2 * 2, 0);
#pragma unroll
        for (int i = 0; i < 4 * kDb - 2; ++i) {
            __builtin_amdgcn_sched_group_barrier(0x008, 2, 0);
            __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
        }
        __builtin_amdgcn_sched_group_barrier(0x008, 2 * 2, 0);
    };

    if constexpr (kFolds) place_of[tid] = row_live ? row_place() + 4 * half : nullptr;
    // What fold needs of a lane comes from LDS and the lane's number: registers held over the
    // loop for it undo the order of the products' reads (4 x 512 tokens behind 32768 5 %).
    const auto this_lane = [] { return __builtin_amdgcn_mbcnt_hi(~0u, __builtin_amdgcn_mbcnt_lo(~0u, 0u)); };
    // What the sums folded so far count now.
    const auto folded = [&] { return __builtin_amdgcn_exp2f(fold_ref[32 * wave + this_lane() % 32] - ref) * (fold_unit / unit); };
    const auto fold = [&] {
        const bool begun = window >= p.fold_windows;
        if (float* const at = place_of[64 * wave + this_lane()]) {
            const float f = begun ? folded() : 0.0f;
#pragma unroll
            for (int db = 0; db < kDb; ++db)
#pragma unroll
                for (int g = 0; g < 4; ++g) {
                    if (32 * db + 8 * g >= static_cast<int>(D)) break;  // uniform
                    Float4* const held = reinterpret_cast<Float4*>(at + 32 * db + 8 * g);
                    Float4 v{0.0f, 0.0f, 0.0f, 0.0f};
                    if (begun) v = *held;
                    float sums[4] = {v.x * f, v.y * f, v.z * f, v.w * f};
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        float rest = 0.0f;
                        two_sum_add(sums[i], rest, acc[db][4 * g + i]);
                        acc[db][4 * g + i] = rest;
                    }
                    *held = Float4{sums[0], sums[1], sums[2], sums[3]};
                }
        }
        __builtin_amdgcn_wave_barrier();  // a row's two lanes have read the ones before
        fold_ref[32 * wave + this_lane() % 32] = threshold == 0.0f ? ref : -INFINITY;
        __syncthreads();  // every wavefront has read the unit before
        fold_unit = now;  // what `unit` is where a wavefront has rows
    };

    if (tile_begin < tile_end) {  // uniform
        const auto key_ks_of = [&](std::uint32_t tile) { return key_ks[set][kUniform ? 0 : tile / kSets & 1]; };
        const auto key_vs_of = [&](std::uint32_t tile) { return key_vs[set][kUniform ? 0 : tile / kSets & 1]; };
        const auto buffer = [&](std::uint32_t tile) { return tiles_lds[set][tile / kSets & 1][0]; };
        const auto work = [&](std::uint32_t from, std::uint32_t to) {  // tiles [from, to), from < to
            if constexpr (kOrder == Order::Turns) {
                fetch_one(0, from);
                // Two wavefronts a SIMD take turns: one multiplies (a tile's weighted values and
                // the next one's scores) while the other works out weights, for whole phases. The
                // second half's is a phase behind, and fills the buffers a tile ahead.
                const std::uint32_t ahead = wave / 4;  // uniform
                // V of `tile` and K of the next one; behind the last tile that one again, into
                // buffers that nothing reads any more.
                const auto fill = [&](std::uint32_t tile) {
                    put_one(0, buffer(tile + 1));
                    put_one(1, buffer(tile));
                    fetch_one(0, tile + 2 < to ? tile + 2 : to - 1);
                    fetch_one(1, tile + 1 < to ? tile + 1 : to - 1);
                };
                const auto phase = [&] {
                    __builtin_amdgcn_sched_barrier(0);
                    wait_lgkm0();
                    lds_barrier();
                    __builtin_amdgcn_sched_barrier(0);
                };
                put_one(0, buffer(from));
                put_scales(from, key_ks_of(from), key_vs_of(from));
                fetch_one(1, from);
                fetch_one(0, from + 1 < to ? from + 1 : from);
                phase();
                if (ahead) {
                    fill(from);
                    phase();
                }
                const auto fill_step = [&](std::uint32_t tile) {
                    fill(tile + ahead);
                    if constexpr (!kUniform)
                        if (tile + 1 < to) put_scales(tile + 1, key_ks_of(tile + 1), key_vs_of(tile + 1));
                };
                for (std::uint32_t tile = from; tile < to; ++tile) {
                    const Scores of = scores(buffer(tile));
                    set_priority<0>();
                    phase();
                    fill_step(tile);
                    const Weights w = weights(of, tile, marks_of(tile), key_ks_of(tile), key_vs_of(tile));
                    phase();
                    set_priority<1>();
                    weigh(w, buffer(tile));
                }
                if (!ahead) phase();
                phase();
            } else {
                const auto fetch = [&](std::uint32_t tile) {
                    fetch_one(0, tile);
                    fetch_one(1, tile);
                };
                const auto put = [&](std::uint32_t tile) {
                    put_one(0, buffer(tile));
                    put_one(1, buffer(tile));
                    put_scales(tile, key_ks_of(tile), key_vs_of(tile));
                };
                if (from + set < to) {
                    fetch(from + set);
                    put(from + set);
                }
                __syncthreads();
                for (std::uint32_t step = from; step < to; step += kSets) {
                    const std::uint32_t tile = step + set;
                    const bool more = tile + kSets < to;
                    if (more) fetch(tile + kSets);
                    if (wave_live && (kSets == 1 || tile < to)) {
                        const auto finish = [&](const Scores& of, const Marks& marks) {
                            weigh(weights(of, tile, marks, key_ks_of(tile), key_vs_of(tile)), buffer(tile));
                        };
                        if constexpr (kSets == 2) {
                            // Marks before the products, whose reads of LDS would wait for each of
                            // theirs in turn (one prompt of 1000 tokens 42.2 us and 41.0).
                            const Marks marks = marks_of(tile);
                            __builtin_amdgcn_sched_barrier(0);
                            finish(scores(buffer(tile)), marks);
                        } else {
                            const Scores of = scores(buffer(tile));
                            finish(of, marks_of(tile));
                        }
                    }
                    if (more) put(tile + kSets);
                    __syncthreads();
                }
            }
        };
        std::uint32_t band = ~0u;
        for (std::uint32_t from = tile_begin;;) {
            band = stage(band);
            const std::uint32_t behind = tile_begin + (window + 1) * p.window_tiles, last = behind < tile_end ? behind : tile_end;
            std::uint32_t to = last;
            if (__builtin_expect(band != 0, 0)) {
                // The next run of the pass's tiles, over gaps of two: a run's start costs as much.
                while (from < last && !band_tile(from)) ++from;
                to = from;
                for (std::uint32_t next = from; next < last && next < to + 3; ++next)
                    if (band_tile(next)) to = next + 1;
                __syncthreads();  // every wavefront has looked for them
            }
            if (__builtin_expect(from < to, 1)) work(from, to);
            from = to;
            if (__builtin_expect(band != 0, 0)) {
                if (to == last) {  // the window's next pass
                    band = 31 - __builtin_clz(present & ((1u << band) - 1));
                    from = tile_begin + window * p.window_tiles;
                }
                continue;
            }
            if (to == tile_end) break;
            if constexpr (kFolds)
                if ((window + 1) % p.fold_windows == 0) fold();
            band = ~0u;
            floor = reference;
            ++window;
        }
    }

    // Row `col`: dims 32 db + 8 g + 4 half .. + 3 in acc[db][4 g ..].
    sum += low;
    const auto swapped = __builtin_amdgcn_permlane32_swap(__float_as_uint(sum), __float_as_uint(sum), false, false);
    sum = __uint_as_float(swapped[0]) + __uint_as_float(swapped[1]);
    float* place = nullptr;  // of a live row
    if constexpr (kFolds) place = place_of[64 * wave + this_lane()];
    if (kFolds && window >= p.fold_windows && place) {
        const float f = folded();
#pragma unroll
        for (int db = 0; db < kDb; ++db)
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                if (32 * db + 8 * g >= static_cast<int>(D)) break;  // uniform
                const Float4 v = *reinterpret_cast<const Float4*>(place + 32 * db + 8 * g);
                acc[db][4 * g] += v.x * f;
                acc[db][4 * g + 1] += v.y * f;
                acc[db][4 * g + 2] += v.z * f;
                acc[db][4 * g + 3] += v.w * f;
            }
    }
    float in_ones = unit * (1.0f / kWeightScale);
    if (__builtin_expect(unit < 0x1p-111f && unit != 0.0f, 0)) {  // uniform; a subnormal number would lose bits
#pragma unroll
        for (int db = 0; db < kDb; ++db) acc[db] *= 1.0f / kWeightScale;
        in_ones = unit;
    }
    if constexpr (kSets == 2) {
        float m = threshold == 0.0f ? ref : -INFINITY;  // -INFINITY: no key seen
        if (set == 1) {
            if (half == 0) stats[r] = make_float2(m, sum);
            float* const to = reinterpret_cast<float*>(tiles_lds) + r * kPad + 4 * half;
#pragma unroll
            for (int db = 0; db < kDb; ++db)
#pragma unroll
                for (int g = 0; g < 4; ++g)
                    *reinterpret_cast<float4*>(to + 32 * db + 8 * g) =
                        make_float4(acc[db][4 * g] * in_ones, acc[db][4 * g + 1] * in_ones, acc[db][4 * g + 2] * in_ones, acc[db][4 * g + 3] * in_ones);
        }
        __syncthreads();
        if (set == 1) return;
        const float2 other = stats[r];
        const float top = fmaxf(m, other.x);
        // NaN sums stay NaN.
        const auto share = [&](float of, float total) {
            return total != total ? total : of == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(of - top);
        };
        const float f0 = share(m, sum), f1 = share(other.x, other.y);
        const float* const from = reinterpret_cast<const float*>(tiles_lds) + r * kPad + 4 * half;
#pragma unroll
        for (int db = 0; db < kDb; ++db)
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const float4 v = *reinterpret_cast<const float4*>(from + 32 * db + 8 * g);
                acc[db][4 * g] = acc[db][4 * g] * in_ones * f0 + v.x * f1;
                acc[db][4 * g + 1] = acc[db][4 * g + 1] * in_ones * f0 + v.y * f1;
                acc[db][4 * g + 2] = acc[db][4 * g + 2] * in_ones * f0 + v.z * f1;
                acc[db][4 * g + 3] = acc[db][4 * g + 3] * in_ones * f0 + v.w * f1;
            }
        sum = sum * f0 + other.y * f1;
        ref = top == -INFINITY ? 0.0f : top;
        in_ones = 1.0f;
    }
    if constexpr (!kFolds) place = row_live ? row_place() + 4 * half : nullptr;
    if (!place) return;
    const bool whole = mine.count == 1;
    const float inv = whole && sum != 0.0f ? 1.0f / sum : 1.0f;
#pragma unroll
    for (int db = 0; db < kDb; ++db)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            if (32 * db + 8 * g >= static_cast<int>(D)) break;  // uniform; parts: not read
            *reinterpret_cast<Float4*>(place + 32 * db + 8 * g) =
                Float4{acc[db][4 * g] * inv * in_ones, acc[db][4 * g + 1] * inv * in_ones, acc[db][4 * g + 2] * inv * in_ones,
                       acc[db][4 * g + 3] * inv * in_ones};
        }
    const std::uint64_t part = static_cast<std::uint64_t>(place - p.part_acc) / kD;  // half 0's
    if (!whole && (kFolds ? this_lane() < 32 : half == 0)) {
        p.part_ml[2 * part] = ref;
        p.part_ml[2 * part + 1] = sum;
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
    // The block of queries that this one was in, and its splits.
    const std::uint32_t queries = static_cast<std::uint32_t>(live / p.query_heads), token = static_cast<std::uint32_t>(i / p.query_heads);
    const std::uint32_t behind = (token / p.tokens + 1) * p.tokens;
    const std::uint32_t last = static_cast<std::uint32_t>(len) - queries + (behind < queries ? behind : queries) - 1;
    const std::uint32_t splits = split_of(last / kTile + 1, p.split_tiles).count;
    if (splits == 1) return;
    const std::uint32_t d4 = threadIdx.x % kLanes;
    if (4 * d4 >= p.head_size) return;
    const std::uint64_t stride = static_cast<std::uint64_t>(p.num_seqs) * p.max_query * p.query_heads;
    const std::uint64_t at = static_cast<std::uint64_t>(seq) * p.max_query * p.query_heads + i;
    float top = -INFINITY, sum = 0.0f;
    Float4 o{0.0f, 0.0f, 0.0f, 0.0f};
    constexpr std::uint32_t kAhead = 8;  // loads in flight
    for (std::uint32_t s0 = 0; s0 < splits; s0 += kAhead) {
        Float4 v[kAhead];
        float m[kAhead], l[kAhead];
#pragma unroll
        for (std::uint32_t u = 0; u < kAhead; ++u) {
            const std::uint64_t part = (s0 + u < splits ? s0 + u : s0) * stride + at;
            m[u] = p.part_ml[2 * part];
            l[u] = p.part_ml[2 * part + 1];
            v[u] = *reinterpret_cast<const Float4*>(p.part_acc + part * kD + 4 * d4);
        }
#pragma unroll
        for (std::uint32_t u = 0; u < kAhead; ++u) {
            if (s0 + u >= splits || l[u] == 0.0f) continue;  // l 0: saw no key
            const float next = m[u] > top ? m[u] : top;
            // NaN sums stay NaN; the first split has nothing before it.
            const float f = top == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(top - next), g = __builtin_amdgcn_exp2f(m[u] - next);
            o = Float4{o.x * f + v[u].x * g, o.y * f + v[u].y * g, o.z * f + v[u].z * g, o.w * f + v[u].w * g};
            sum = sum * f + l[u] * g;
            top = next;
        }
    }
    const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
    *reinterpret_cast<Float4*>(p.output + (p.query_offsets[seq] * p.query_heads + i) * p.head_size + 4 * d4) =
        Float4{o.x * inv, o.y * inv, o.z * inv, o.w * inv};
}

// ---------------------------------------------------------------- dispatch
struct PrefillPlan {
    Order order;
    std::uint32_t heads_of;  // query heads of a launch: the largest divisor of the group that fits
    std::uint32_t tokens, blocks, splits, split_tiles;
};
constexpr std::uint32_t kCus = 256;
constexpr std::uint64_t kLeastTiles = 4;  // of a split

PrefillPlan prefill_plan(std::uint64_t num_seqs, std::uint64_t max_query, std::uint64_t max_kv, std::uint64_t heads,
                         std::uint64_t group, std::uint64_t head_size) {
    PrefillPlan plan{};
    const auto shape = [&](Order order) {
        plan.order = order;
        const std::uint64_t rows = order == Order::Turns ? 256 : 128;
        plan.heads_of = static_cast<std::uint32_t>(group < rows ? group : rows);
        while (group % plan.heads_of != 0) --plan.heads_of;
        plan.tokens = static_cast<std::uint32_t>(rows / plan.heads_of);
        plan.blocks = static_cast<std::uint32_t>((max_query + plan.tokens - 1) / plan.tokens);
        return num_seqs * plan.blocks * heads;
    };
    // Turns: eight wavefronts share a tile's loads and conversions; two workgroups of four a
    // CU are filled by fewer rows and wait less at barriers. Head size 128, eight and four:
    // 512 tokens behind 32768 490 and 541 us; 8 x 4096 2060 and 2189; 16 prompts of up to
    // 4096 2000 and 2108, of up to 2048 675 and 656, of up to 1000 191 and 169; 8 x 2048 573
    // and 606; 64 tokens behind 2000 34 and 27. Head size 64: 8 x 2048 199 and 167. At 256
    // the registers are those of four.
    std::uint64_t workgroups = shape(head_size == 128 ? Order::Turns : Order::Four);
    if (plan.order == Order::Turns && (max_query * group <= 128 || max_kv < 4096)) workgroups = shape(Order::Four);
    // Halves: half as many steps for the longest workgroups where there are few, one a CU.
    // Halves and four: 7 prompts of up to 700, heads of 64, 20.6 and 24.3 us; one prompt of
    // 1000 45.7 and 53.5, of 2000 86 and 93; 8 x 128 tokens behind up to 3000 104 and 134; but
    // 16 prompts of up to 700, heads of 64, 37 and 30. A workgroup of one wavefront's rows
    // leaves the CU to others: 16 x 4 tokens behind up to 9000 127 and 96.
    if (plan.order == Order::Four && head_size != 256 && workgroups <= 2 * kCus && max_kv > 4 * kTile &&
        (max_query * group > 32 || max_kv <= 32 * kTile))
        plan.order = Order::Halves;
    const std::uint64_t tiles = (max_kv + kTile - 1) / kTile;
    if (plan.order != Order::Four || head_size == 256) {
        // One workgroup a CU: the keys of each go to as many as fill the CUs once (1024 tokens
        // behind 16384: 504 us, in shares of the mean 701).
        std::uint64_t most = workgroups < kCus ? kCus / workgroups : 1;
        if (tiles <= 2 * kLeastTiles) most = 1;
        if (most > (tiles + kLeastTiles - 1) / kLeastTiles) most = (tiles + kLeastTiles - 1) / kLeastTiles;
        // Two sets have no place to fold sums into: kFold tiles each.
        if (plan.order == Order::Halves && most * 2 * kFold < tiles) most = (tiles + 2 * kFold - 1) / (2 * kFold);
        plan.split_tiles = static_cast<std::uint32_t>((tiles + most - 1) / most);
    } else {
        // Where the heaviest block of queries would run on alone, its keys go to several
        // workgroups, none with more tiles than its share of all (bounds standing for
        // lengths). Two workgroups of a CU take 3.1 us a tile each, one by itself 1.7 (head
        // size 128), so a block may have twice the share.
        const std::uint64_t first = max_query < plan.tokens ? max_query : plan.tokens;
        const std::uint64_t lightest = (max_kv - max_query + first + kTile - 1) / kTile;
        std::uint64_t share = (workgroups * (tiles + lightest) / 2 + 2 * kCus - 1) / (2 * kCus);
        if (share < kLeastTiles) share = kLeastTiles;
        plan.split_tiles = static_cast<std::uint32_t>(2 * share + share / 4 < tiles ? share : tiles);
    }
    plan.splits = static_cast<std::uint32_t>((tiles + plan.split_tiles - 1) / plan.split_tiles);
    return plan;
}
std::uint64_t prefill_workspace(const PrefillPlan& plan, std::uint64_t num_seqs, std::uint64_t max_query,
                                std::uint64_t query_heads, std::uint64_t head_size) {
    return plan.splits == 1 ? 0 : plan.splits * num_seqs * max_query * query_heads * (head_size + 2) * sizeof(float);
}

// Whether the merge's threads, four dims each, fit a grid.
bool merge_fits(const PrefillPlan& plan, std::uint64_t max_query, std::uint64_t query_heads, std::uint64_t head_size) {
    return plan.splits == 1 || max_query * query_heads <= kMostWorkgroups * (256 / (head_size / 4));
}

template <typename F, int kD, Order kOrder>
int launch_prefill(QuantPrefillParams& p, hipStream_t stream) {
    const dim3 grid(p.heads * p.splits * p.num_seqs * p.blocks), threads(Shape<kD, kOrder, true>::kThreads);
    for (p.first = 0; p.first < p.group; p.first += p.heads_of) {
        const bool uniform = p.block_size.divisor % 16 == 0;
        bool folds = false;
        if constexpr (kOrder != Order::Halves) {
            folds = p.split_tiles > kFold;
            if (folds) {
                if (uniform) quant_prefill_kernel<F, kD, kOrder, true, true><<<grid, threads, 0, stream>>>(p);
                else quant_prefill_kernel<F, kD, kOrder, false, true><<<grid, threads, 0, stream>>>(p);
            }
        }
        if (!folds) {
            if (uniform) quant_prefill_kernel<F, kD, kOrder, true, false><<<grid, threads, 0, stream>>>(p);
            else quant_prefill_kernel<F, kD, kOrder, false, false><<<grid, threads, 0, stream>>>(p);
        }
        if (const int s = launch_status("quant_prefill_kernel")) return s;
    }
    if (p.splits == 1) return KVFLUX_OK;
    const std::uint64_t per = 256 / (kD / 4);
    quant_prefill_merge_kernel<kD><<<dim3(static_cast<unsigned>((static_cast<std::uint64_t>(p.max_query) * p.query_heads + per - 1) / per), p.num_seqs),
                                     dim3(256), 0, stream>>>(p);
    return launch_status("quant_prefill_merge_kernel");
}
template <typename F>
int launch_prefill_head_size(QuantPrefillParams& p, std::uint64_t head_size, Order order, hipStream_t s) {
    switch (head_size) {
    case 64: return order == Order::Four ? launch_prefill<F, 64, Order::Four>(p, s) : launch_prefill<F, 64, Order::Halves>(p, s);
    case 128:
        switch (order) {
        case Order::Four: return launch_prefill<F, 128, Order::Four>(p, s);
        case Order::Turns: return launch_prefill<F, 128, Order::Turns>(p, s);
        default: return launch_prefill<F, 128, Order::Halves>(p, s);
        }
    default: return launch_prefill<F, 256, Order::Four>(p, s);
    }
}

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
    head_size = padded_head_size(head_size);
    if (num_seqs == 0 || max_query_tokens == 0 || head_size == 0) return KVFLUX_OK;
    const PrefillPlan plan = prefill_plan(num_seqs, max_query_tokens, max_kv_len, num_kv_heads, query_heads / num_kv_heads, head_size);
    if (!merge_fits(plan, max_query_tokens, query_heads, head_size))
        return fail(KVFLUX_ERR_UNSUPPORTED, "quant prefill workspace: shape too large");
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
    if (num_blocks >= kUnread) return fail(KVFLUX_ERR_UNSUPPORTED, "quant prefill: too many pages");
    if (!aligned(4, {query, output}) || !aligned(8, {block_table, kv_lens, query_lens, query_offsets}))
        return fail(KVFLUX_ERR_INVALID_ARGUMENT, "quant prefill: misaligned array");
    const std::uint64_t group = query_heads / num_kv_heads;
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
    const PrefillPlan plan = prefill_plan(num_seqs, max_query_tokens, max_kv_len, num_kv_heads, group, padded);
    QuantPrefillParams p{};
    p.key_cache = static_cast<const std::uint8_t*>(key_cache);
    p.value_cache = static_cast<const std::uint8_t*>(value_cache);
    p.key_scales = key_scales;
    p.value_scales = value_scales;
    p.num_blocks = num_blocks;
    p.head_size = static_cast<std::uint32_t>(head_size);
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
    const std::uint64_t window = (kWindow - 2) * block_size / kTile, longest = plan.order == Order::Halves ? 2 * kFold : kFold;
    p.window_tiles = static_cast<std::uint32_t>(window < longest ? window : longest);
    p.fold_windows = kFold / p.window_tiles;  // read where sums are folded
    p.query = query;
    p.output = output;
    p.scale_log2 = scale_log2;
    if (static_cast<std::uint64_t>(p.heads) * p.splits * p.num_seqs * p.blocks > kMostWorkgroups / 2 ||
        !merge_fits(plan, max_query_tokens, query_heads, padded))
        return fail(KVFLUX_ERR_UNSUPPORTED, "quant prefill: shape too large");
    if (plan.splits > 1) {
        if (!workspace || workspace_bytes < prefill_workspace(plan, num_seqs, max_query_tokens, query_heads, padded))
            return fail(KVFLUX_ERR_INVALID_ARGUMENT, "quant prefill: workspace too small");
        if (!aligned(4, {workspace})) return fail(KVFLUX_ERR_INVALID_ARGUMENT, "quant prefill: misaligned workspace");
        p.part_acc = static_cast<float*>(workspace);
        p.part_ml = p.part_acc + static_cast<std::uint64_t>(plan.splits) * num_seqs * max_query_tokens * query_heads * padded;
    }
    return format == KVFLUX_QUANT_E4M3 ? launch_prefill_head_size<QuantE4m3>(p, padded, plan.order, as_stream(stream))
                                       : launch_prefill_head_size<QuantInt8>(p, padded, plan.order, as_stream(stream));
}
