// From the projection's output to the attention's inputs in one pass: the RMS
// norm of every query and key head, the position rotation, queries as the FP32
// rows the attention takes, keys and values into their pages.
//
// For a row x of D values (one head of one token) with weight w:
//   n = x / sqrt(mean(x^2) + eps) * w          (w null: n = x)
// and over the first R of the D dims, with angle_j = position * inv_freq[j]:
//   (y_a, y_b) = (n_a cos - n_b sin, n_b cos + n_a sin)
// for the pairs (a, b) = (j, j + R/2), or (2j, 2j + 1) when interleaved. Values
// are neither normed nor rotated. All arithmetic is FP32, the angle FP64 (in
// turns, reduced exactly): at position 131071 an FP32 angle is off by 2^-8.
// Keys are rounded once, to the cache's type; values with the cache's type are
// copied bit by bit.
#include "common.h"

#include <cmath>
#include <type_traits>

namespace kvflux_hip {
namespace {

constexpr std::uint64_t kMaxHead = 512;

typedef __attribute__((ext_vector_type(4))) float f32x4_t;

struct Bf16 { using Storage = std::uint16_t; };
struct F16 { using Storage = std::uint16_t; };
struct F32 { using Storage = std::uint32_t; };

template <typename E>
__device__ inline float to_float(typename E::Storage x) {
    if constexpr (std::is_same<E, F32>::value) return __uint_as_float(x);
    if constexpr (std::is_same<E, F16>::value) return static_cast<float>(__builtin_bit_cast(_Float16, x));
    return __uint_as_float(static_cast<std::uint32_t>(x) << 16);
}
// Rounded to nearest even (the only rounding a key meets after the FP32 steps).
template <typename E>
__device__ inline typename E::Storage from_float(float x) {
    if constexpr (std::is_same<E, F32>::value) return __float_as_uint(x);
    else if constexpr (std::is_same<E, F16>::value) return __builtin_bit_cast(std::uint16_t, static_cast<_Float16>(x));
    else return __builtin_bit_cast(std::uint16_t, static_cast<__bf16>(x));
}

struct Params {
    const void* query_in;
    const void* key_in;
    const void* value_in;
    std::uint64_t query_stride, key_stride, value_stride;  // elements from a token to the next
    void* key_cache;
    void* value_cache;
    std::uint64_t slot_count;
    FastDiv block_size;       // slots below 2^32; wide: 64-bit divisions
    bool wide;
    std::uint64_t head_step;  // block_size * head_dim
    std::uint32_t kv_heads, query_heads, head_dim;
    FastDiv token_rows;       // query_heads + 2 * kv_heads: rows of a token, queries, keys, values
    std::uint32_t rows;       // num_tokens * token_rows
    std::uint32_t tokens;
    const float* query_norm;  // null: no norm
    const float* key_norm;
    float eps, inv_dim;       // inv_dim = 1 / head_dim
    const double* inv_freq;   // [rotary / 2]
    std::uint32_t rotary;
    FastDiv half;             // rotary / 2 (1 without a rotation)
    bool interleaved;
    float* query_out;
};

// Where a token's position and slot come from: arrays, or the place just
// appended to a sequence, read from a device batch block table (position
// len - 1 of row n). No slot: ~0. A token without a place at all (an empty row)
// is not `live`: nothing of it is written.
struct Listed {
    const std::uint64_t* positions;
    const std::uint64_t* slots;
    __device__ bool live(std::uint32_t) const { return true; }
    __device__ std::uint64_t position(std::uint32_t n) const { return positions[n]; }
    __device__ std::uint64_t slot(std::uint32_t n) const { return slots[n]; }
};
struct Tail {
    const std::uint64_t* table;
    std::uint64_t width;
    const std::uint64_t* lens;
    std::uint64_t block_size, num_blocks;
    __device__ bool live(std::uint32_t n) const { return lens[n] != 0; }
    __device__ std::uint64_t position(std::uint32_t n) const { return lens[n] - 1; }
    __device__ std::uint64_t slot(std::uint32_t n) const {
        const std::uint64_t len = lens[n];
        if (len == 0) return ~0ULL;
        const std::uint64_t b = (len - 1) / block_size;
        if (b >= width) return ~0ULL;
        const std::uint64_t page = table[static_cast<std::uint64_t>(n) * width + b];
        return page < num_blocks ? page * block_size + (len - 1) % block_size : ~0ULL;
    }
};

// cos and sin of position * inv_freq. In turns the reduction is exact: the
// quarter turn nearest is taken off in FP64, so FP32 sees at most an eighth of
// a turn (its rounding is 2^-27 turns), and the quarters swap and negate.
__device__ inline void rotation(std::uint64_t position, double inv_freq, float* c, float* s) {
    const double quarters = static_cast<double>(position) * (inv_freq * 0.63661977236758134308);  // 2 / pi
    const double nearest = rint(quarters);
    float sn, cs;
    sincospif(static_cast<float>(0.5 * (quarters - nearest)), &sn, &cs);
    const int k = static_cast<int>(nearest - 4.0 * floor(0.25 * nearest));  // nearest mod 4 (NaN for an angle past FP64: garbage in)
    *c = k == 0 ? cs : k == 1 ? -sn : k == 2 ? -cs : sn;
    *s = k == 0 ? sn : k == 1 ? cs : k == 2 ? -sn : -cs;
}

// Element of a cache where head 0 of `slot` starts (head h: h * head_step on),
// or kNowhere.
constexpr std::uint64_t kNowhere = ~0ULL;
__device__ inline std::uint64_t cache_place(const Params& p, std::uint64_t slot) {
    if (slot >= p.slot_count) return kNowhere;
    std::uint64_t page, offset;
    if (p.wide) {
        page = slot / p.block_size.divisor;
        offset = slot - page * p.block_size.divisor;
    } else {
        const auto s = static_cast<std::uint32_t>(slot);
        page = p.block_size.div(s);
        offset = s - static_cast<std::uint32_t>(page) * p.block_size.divisor;
    }
    return page * p.kv_heads * p.head_step + offset * p.head_dim;
}

// Sum over aligned groups of `lanes` lanes (a power of two, uniform), in every
// lane of the group: lane moves within 16, a swizzle and a shuffle beyond.
__device__ inline float row_sum(float x, std::uint32_t lanes) {
    const auto moved = [](float v, auto ctrl) {
        return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), decltype(ctrl)::value, 0xf, 0xf, true));
    };
    if (lanes >= 2) x += moved(x, std::integral_constant<int, 0xb1>{});    // lanes 1 apart
    if (lanes >= 4) x += moved(x, std::integral_constant<int, 0x4e>{});    // lanes 2 apart
    if (lanes >= 8) x += moved(x, std::integral_constant<int, 0x141>{});   // the other half of 8
    if (lanes >= 16) x += moved(x, std::integral_constant<int, 0x128>{});  // the other half of 16
    if (lanes >= 32) x += __int_as_float(__builtin_amdgcn_ds_swizzle(__float_as_int(x), 0x401f));
    if (lanes >= 64) x += __shfl_xor(x, 32);
    return x;
}

// Rows whose squares or their mean leave FP32's normal range (a mean under 2^-100,
// which a tiny eps leaves there; a sum of 2^120 and more, up to infinity): the
// reciprocal root takes no denormals, and a sum that overflowed has none. Such a
// row is normed times f^2 = 2^100 or 2^-100, with eps times f^4, and scaled in two
// steps of f, so no step leaves the range.
__device__ inline bool out_of_range(float mean, float square) { return mean < 0x1p-100f || square >= 0x1p120f; }
__device__ inline float range_factor(float mean) { return mean < 0x1p-100f ? 0x1p50f : 0x1p-50f; }
// What (x * f) is multiplied by, `square` being the sum of the squares of x f^2.
__device__ inline float ranged_scale(float square, float inv_dim, float eps, float f) {
    return __builtin_amdgcn_rsqf(fmaf(square, inv_dim, eps * (f * f) * (f * f))) * f;
}

// Four values of a row: 8 bytes of a 16-bit type, 16 of FP32.
template <typename E>
using Four = typename std::conditional<std::is_same<E, F32>::value, V16, V8>::type;
template <typename E>
__device__ inline void widen(const Four<E>& v, float (&x)[4]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if constexpr (std::is_same<E, F32>::value) x[i] = __uint_as_float(v.w[i]);
        else x[i] = to_float<E>(static_cast<std::uint16_t>(v.w[i / 2] >> (16 * (i % 2))));
    }
}
template <typename E>
__device__ inline Four<E> narrow(const float (&x)[4]) {
    Four<E> v;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if constexpr (std::is_same<E, F32>::value) v.w[i] = __float_as_uint(x[i]);
        else if (i % 2 == 0)
            v.w[i / 2] = from_float<E>(x[i]) | static_cast<std::uint32_t>(from_float<E>(x[i + 1])) << 16;
    }
    return v;
}

// The fast kernel, for vectors of four values (head size and rotation
// multiples of 8, aligned rows). 2^lane_shift lanes hold a row, each lane two vectors:
// values 4l and 4l + R/2 on of the rotated part in the half form, so a pair's
// two values are in one lane, and 8l and 8l + 4 on elsewhere. A workgroup
// takes kUnroll * 256 / lanes consecutive rows (token by token: queries, keys,
// values), so any number of heads fills it; cos and sin of its tokens, and the
// place of each in the caches, are worked out once into LDS while the rows'
// loads are in flight.
//
// Bound: HBM, and the launch below about 300 tokens. BF16, 32/8 heads of 128, MI355X:
// 4096 tokens (134 MB) 22 to 25 us, 5.4 to 6.05 TB/s; 64/8 heads, 16384 tokens (940 MB)
// 159 us, 5.9 TB/s; 64 tokens 4.2 us. What it took:
//  * a wavefront a row, a sincos a value: 120 and 775 us;
//  * this layout, with the slot's page found by each row: 46 and 270 us, about 500
//    instructions a row, the divisions the larger part; found once a token: 30 and 168;
//  * non-temporal stores (each row is written once, in whole lines): 22.1 and 159 us;
//    non-temporal loads as well: 26 and 159;
//  * rows of a thread (kUnroll): one 23-25 and 171 us, two 22.2 and 158, four 22.1 and
//    158 but 5.2 us instead of 4.2 for 64 tokens. Two everywhere.
constexpr int kThreads = 256;
constexpr int kUnroll = 2;
// Rows of a workgroup are at most kThreads * kUnroll (one lane a row, head size
// 8), their values 8 * kThreads * kUnroll, and a token has three rows at least:
// the tokens they touch, and those tokens' rotated values.
constexpr int kSpanTokens = kThreads * kUnroll / 3 + 2;
constexpr int kSpanRotated = 8 * kThreads * kUnroll / 3 + 2 * static_cast<int>(kMaxHead);

template <typename In, typename Cache, typename Place>
__global__ __launch_bounds__(kThreads) void norm_rope_write_kernel(Params p, Place place, std::uint32_t lane_shift) {
    __shared__ __attribute__((aligned(16))) float turn[kSpanRotated];  // [token][cos R/2, sin R/2]
    __shared__ std::uint64_t places[kSpanTokens];
    __shared__ bool live[kSpanTokens];
    using Vec = Four<In>;
    const std::uint32_t tid = threadIdx.x, lanes = 1u << lane_shift, l = tid & (lanes - 1);
    const std::uint32_t pass_rows = kThreads >> lane_shift;
    const std::uint32_t first = blockIdx.x * pass_rows * kUnroll;
    const std::uint32_t last = first + pass_rows * kUnroll < p.rows ? first + pass_rows * kUnroll - 1 : p.rows - 1;
    const bool inside = 8 * l < p.head_dim;
    const bool rotated = 8 * l < p.rotary;
    const std::uint32_t a = rotated && !p.interleaved ? 4 * l : 8 * l;
    const std::uint32_t b = rotated && !p.interleaved ? 4 * l + p.rotary / 2 : 8 * l + 4;

    // Every row's loads, unconditional (a lane past a row's values rereads its
    // first vectors, a row past the last one the last).
    Vec va[kUnroll], vb[kUnroll];
    std::uint32_t token[kUnroll], row[kUnroll];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
        const std::uint32_t item = first + u * pass_rows + (tid >> lane_shift);
        const std::uint32_t at = item < p.rows ? item : p.rows - 1;
        token[u] = p.token_rows.div(at);
        row[u] = at - token[u] * p.token_rows.divisor;
        const bool is_query = row[u] < p.query_heads, is_key = row[u] < p.query_heads + p.kv_heads;
        const void* in = is_query ? p.query_in : is_key ? p.key_in : p.value_in;
        const std::uint64_t stride = is_query ? p.query_stride : is_key ? p.key_stride : p.value_stride;
        const std::uint32_t head = is_query ? row[u] : row[u] - p.query_heads - (is_key ? 0u : p.kv_heads);
        const auto* src = static_cast<const typename In::Storage*>(in) + token[u] * stride +
                          static_cast<std::uint64_t>(head) * p.head_dim;
        va[u] = *reinterpret_cast<const Vec*>(src + (inside ? a : 0u));
        vb[u] = *reinterpret_cast<const Vec*>(src + (inside ? b : 4u));
        if (item >= p.rows) row[u] = ~0u;
    }
    const auto weights = [&](const float* norm, std::uint32_t at) {
        return norm ? *reinterpret_cast<const f32x4_t*>(norm + at) : f32x4_t{1.0f, 1.0f, 1.0f, 1.0f};  // uniform
    };
    const f32x4_t wqa = weights(p.query_norm, inside ? a : 0u), wqb = weights(p.query_norm, inside ? b : 4u);
    const f32x4_t wka = weights(p.key_norm, inside ? a : 0u), wkb = weights(p.key_norm, inside ? b : 4u);

    const std::uint32_t token0 = p.token_rows.div(first), tokens = p.token_rows.div(last) - token0 + 1;
    const std::uint32_t half = p.rotary / 2;
    for (std::uint32_t i = tid; i < tokens * half; i += kThreads) {
        const std::uint32_t t = p.half.div(i), j = i - t * half;
        rotation(place.position(token0 + t), p.inv_freq[j], &turn[t * p.rotary + j], &turn[t * p.rotary + half + j]);
    }
    for (std::uint32_t t = tid; t < tokens; t += kThreads) {
        places[t] = cache_place(p, place.slot(token0 + t));
        live[t] = place.live(token0 + t);
    }
    __syncthreads();

    auto finish = [&](const Vec& row_a, const Vec& row_b, std::uint32_t token_u, std::uint32_t row_u) {
        float xa[4], xb[4], square = 0.0f;
        widen<In>(row_a, xa);
        widen<In>(row_b, xb);
#pragma unroll
        for (int i = 0; i < 4; ++i) square = fmaf(xa[i], xa[i], fmaf(xb[i], xb[i], square));
        if (!inside) square = 0.0f;
        square = row_sum(square, lanes);
        const bool is_query = row_u < p.query_heads, is_key = row_u < p.query_heads + p.kv_heads;
        const bool normed = is_query ? p.query_norm != nullptr : is_key && p.key_norm != nullptr;
        const float mean = fmaf(square, p.inv_dim, p.eps);
        float scale = __builtin_amdgcn_rsqf(mean);
        const bool odd = normed && out_of_range(mean, square);
        if (__builtin_expect(__builtin_amdgcn_ballot_w64(odd) != 0, 0)) {  // uniform
            const float f = range_factor(mean);
            float again = 0.0f;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float ya = xa[i] * f * f, yb = xb[i] * f * f;
                again = fmaf(ya, ya, fmaf(yb, yb, again));
            }
            again = row_sum(inside ? again : 0.0f, lanes);
            if (odd) {
                const float by = ranged_scale(again, p.inv_dim, p.eps, f);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    xa[i] = xa[i] * f * by;
                    xb[i] = xb[i] * f * by;
                }
                scale = 1.0f;
            }
        }
        if (row_u == ~0u || !inside) return;
        const std::uint32_t t = token_u - token0;
        const std::uint64_t at = places[t];
        if (is_query ? !live[t] : at == kNowhere) return;
        const std::uint32_t head = row_u - (is_query ? 0u : is_key ? p.query_heads : p.query_heads + p.kv_heads);
        if (!is_query && !is_key) {
            auto* dst = static_cast<typename Cache::Storage*>(p.value_cache) + at + head * p.head_step;
            Four<Cache> ca, cb;
            if constexpr (std::is_same<In, Cache>::value) {
                ca = row_a;
                cb = row_b;
            } else {
                ca = narrow<Cache>(xa);
                cb = narrow<Cache>(xb);
            }
            stream_store(reinterpret_cast<Four<Cache>*>(dst + a), ca);
            stream_store(reinterpret_cast<Four<Cache>*>(dst + b), cb);
            return;
        }
        if (normed) {
            const f32x4_t wa = is_query ? wqa : wka, wb = is_query ? wqb : wkb;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                xa[i] *= scale * wa[i];
                xb[i] *= scale * wb[i];
            }
        }
        if (rotated) {
            const float4 c4 = *reinterpret_cast<const float4*>(turn + t * p.rotary + 4 * l);
            const float4 s4 = *reinterpret_cast<const float4*>(turn + t * p.rotary + half + 4 * l);
            const float c[4] = {c4.x, c4.y, c4.z, c4.w}, s[4] = {s4.x, s4.y, s4.z, s4.w};
            if (p.interleaved) {
#pragma unroll
                for (int i = 0; i < 4; i += 2) {
                    const float ya = xa[i] * c[i / 2] - xa[i + 1] * s[i / 2];
                    xa[i + 1] = xa[i + 1] * c[i / 2] + xa[i] * s[i / 2];
                    xa[i] = ya;
                    const float yb = xb[i] * c[2 + i / 2] - xb[i + 1] * s[2 + i / 2];
                    xb[i + 1] = xb[i + 1] * c[2 + i / 2] + xb[i] * s[2 + i / 2];
                    xb[i] = yb;
                }
            } else {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float y = xa[i] * c[i] - xb[i] * s[i];
                    xb[i] = xb[i] * c[i] + xa[i] * s[i];
                    xa[i] = y;
                }
            }
        }
        if (is_query) {
            float* dst = p.query_out + (static_cast<std::uint64_t>(token_u) * p.query_heads + head) * p.head_dim;
            stream_store(reinterpret_cast<V16*>(dst + a), narrow<F32>(xa));
            stream_store(reinterpret_cast<V16*>(dst + b), narrow<F32>(xb));
        } else {
            auto* dst = static_cast<typename Cache::Storage*>(p.key_cache) + at + head * p.head_step;
            stream_store(reinterpret_cast<Four<Cache>*>(dst + a), narrow<Cache>(xa));
            stream_store(reinterpret_cast<Four<Cache>*>(dst + b), narrow<Cache>(xb));
        }
    };
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) finish(va[u], vb[u], token[u], row[u]);
}

// One wavefront a row; any head size up to kMaxHead, any even rotation, any
// alignment. Bound by its instructions, a sincos a value among them: 4096 tokens of
// 32/8 heads of 80, 20 dims rotated, 81 us, 1.0 TB/s; heads of 128 an element off
// their alignment 94 us.
template <typename In, typename Cache, typename Place>
__global__ __launch_bounds__(64) void norm_rope_write_generic_kernel(Params p, Place place) {
    constexpr int kPer = static_cast<int>(kMaxHead) / 64;
    __shared__ float normed[kMaxHead];
    const std::uint32_t token = p.token_rows.div(blockIdx.x);
    const std::uint32_t row = blockIdx.x - token * p.token_rows.divisor;
    const int lane = threadIdx.x;
    if (!place.live(token)) return;  // uniform
    const bool is_query = row < p.query_heads;
    const bool is_value = row >= p.query_heads + p.kv_heads;
    const std::uint32_t head = is_query ? row : is_value ? row - p.query_heads - p.kv_heads : row - p.query_heads;
    const void* in = is_query ? p.query_in : is_value ? p.value_in : p.key_in;
    const std::uint64_t stride = is_query ? p.query_stride : is_value ? p.value_stride : p.key_stride;
    const auto* src = static_cast<const typename In::Storage*>(in) + token * stride +
                      static_cast<std::uint64_t>(head) * p.head_dim;
    std::uint64_t at = 0;
    if (!is_query) {
        at = cache_place(p, place.slot(token));
        if (at == kNowhere) return;
        at += head * p.head_step;
    }
    if (is_value) {
        auto* dst = static_cast<typename Cache::Storage*>(p.value_cache) + at;
        for (std::uint32_t d = lane; d < p.head_dim; d += 64) {
            if constexpr (std::is_same<In, Cache>::value) dst[d] = src[d];
            else dst[d] = from_float<Cache>(to_float<In>(src[d]));
        }
        return;
    }
    const float* norm = is_query ? p.query_norm : p.key_norm;
    float x[kPer], square = 0.0f;
#pragma unroll
    for (int k = 0; k < kPer; ++k) {
        const std::uint32_t d = lane + 64 * k;
        x[k] = d < p.head_dim ? to_float<In>(src[d]) : 0.0f;
        square = fmaf(x[k], x[k], square);
    }
#pragma unroll
    for (int m = 1; m < 64; m <<= 1) square += __shfl_xor(square, m);
    const float mean = fmaf(square, p.inv_dim, p.eps);
    float scale = __builtin_amdgcn_rsqf(mean);
    if (norm && out_of_range(mean, square)) {  // uniform
        const float f = range_factor(mean);
        square = 0.0f;
#pragma unroll
        for (int k = 0; k < kPer; ++k) {
            const float y = x[k] * f * f;
            square = fmaf(y, y, square);
            x[k] *= f;
        }
#pragma unroll
        for (int m = 1; m < 64; m <<= 1) square += __shfl_xor(square, m);
        scale = ranged_scale(square, p.inv_dim, p.eps, f);
    }
#pragma unroll
    for (int k = 0; k < kPer; ++k) {
        const std::uint32_t d = lane + 64 * k;
        if (d < p.head_dim) normed[d] = norm ? x[k] * scale * norm[d] : x[k];
    }
    __syncthreads();
    const std::uint64_t position = place.position(token);
    const std::uint32_t half = p.rotary / 2;
    for (std::uint32_t d = lane; d < p.head_dim; d += 64) {
        float y = normed[d];
        if (d < p.rotary) {
            const std::uint32_t j = p.interleaved ? d / 2 : d < half ? d : d - half;
            const bool first = p.interleaved ? d % 2 == 0 : d < half;
            const float other = normed[p.interleaved ? d ^ 1u : first ? d + half : d - half];
            float c, s;
            rotation(position, p.inv_freq[j], &c, &s);
            y = first ? y * c - other * s : y * c + other * s;
        }
        if (is_query)
            p.query_out[(static_cast<std::uint64_t>(token) * p.query_heads + head) * p.head_dim + d] = y;
        else
            static_cast<typename Cache::Storage*>(p.key_cache)[at + d] = from_float<Cache>(y);
    }
}

// Whether rows can be read and written in vectors of four values.
template <typename In, typename Cache>
bool in_vectors(const Params& p) {
    if (p.head_dim % 8 != 0 || p.rotary % 8 != 0) return false;
    if ((p.query_stride | p.key_stride | p.value_stride) % 4 != 0) return false;
    const void* in[3] = {p.query_in, p.key_in, p.value_in};
    const void* cache[2] = {p.key_cache, p.value_cache};
    const void* floats[3] = {p.query_out, p.query_norm, p.key_norm};
    return copy_width(sizeof(Four<In>), in, 3) == sizeof(Four<In>) &&
           copy_width(sizeof(Four<Cache>), cache, 2) == sizeof(Four<Cache>) && copy_width(16, floats, 3) == 16;
}

template <typename In, typename Cache, typename Place>
int launch(const Params& p, const Place& place, hipStream_t s) {
    if (in_vectors<In, Cache>(p)) {
        std::uint32_t lane_shift = 0;
        while ((8u << lane_shift) < p.head_dim) ++lane_shift;
        const std::uint32_t rows = (kThreads >> lane_shift) * kUnroll;
        hipLaunchKernelGGL((norm_rope_write_kernel<In, Cache, Place>), dim3((p.rows + rows - 1) / rows), dim3(kThreads),
                           0, s, p, place, lane_shift);
        return launch_status("norm_rope_write_kernel");
    }
    hipLaunchKernelGGL((norm_rope_write_generic_kernel<In, Cache, Place>), dim3(p.rows), dim3(64), 0, s, p, place);
    return launch_status("norm_rope_write_generic_kernel");
}

template <typename In, typename Place>
int launch_cache(const Params& p, int dtype, const Place& place, hipStream_t s) {
    switch (dtype) {
    case KVFLUX_DTYPE_BF16: return launch<In, Bf16>(p, place, s);
    case KVFLUX_DTYPE_F16: return launch<In, F16>(p, place, s);
    default: return launch<In, F32>(p, place, s);
    }
}

// Checks and launch shared by both entry points.
template <typename Place>
int norm_rope_write(void* key_cache, void* value_cache, uint64_t num_blocks, uint64_t num_kv_heads,
                    uint64_t block_size, uint64_t head_size, int dtype, const void* query_in, const void* key_in,
                    const void* value_in, int input_dtype, uint64_t query_stride, uint64_t key_stride,
                    uint64_t value_stride, uint64_t query_heads, const float* query_norm, const float* key_norm,
                    float eps, const double* inv_freq, uint64_t rotary_dim, int interleaved, const Place& place,
                    uint64_t num_tokens, float* query_out, void* stream) {
    const std::size_t in_bytes = dtype_bytes(input_dtype), cache_bytes = dtype_bytes(dtype);
    if (cache_bytes == 0) return fail(KVFLUX_ERR_INVALID_ARGUMENT, "unknown dtype %d", dtype);
    if (in_bytes == 0) return fail(KVFLUX_ERR_INVALID_ARGUMENT, "unknown input dtype %d", input_dtype);
    if (!key_cache || !value_cache || !query_in || !key_in || !value_in || !query_out)
        return fail(KVFLUX_ERR_INVALID_ARGUMENT, "norm, rotation and write: null pointer");
    if (num_blocks == 0 || num_kv_heads == 0 || block_size == 0 || head_size == 0 || query_heads == 0)
        return fail(KVFLUX_ERR_INVALID_ARGUMENT, "norm, rotation and write: zero dimension");
    if (rotary_dim % 2 != 0 || rotary_dim > head_size)
        return fail(KVFLUX_ERR_INVALID_ARGUMENT, "norm, rotation and write: rotary_dim %llu of head_size %llu",
                    static_cast<unsigned long long>(rotary_dim), static_cast<unsigned long long>(head_size));
    if (rotary_dim != 0 && !inv_freq)
        return fail(KVFLUX_ERR_INVALID_ARGUMENT, "norm, rotation and write: null inv_freq");
    if (!(eps >= 0.0f) || eps == INFINITY)
        return fail(KVFLUX_ERR_INVALID_ARGUMENT, "norm, rotation and write: eps is negative or not finite");
    if (head_size > kMaxHead)
        return fail(KVFLUX_ERR_UNSUPPORTED, "norm, rotation and write: head_size %llu > %llu",
                    static_cast<unsigned long long>(head_size), static_cast<unsigned long long>(kMaxHead));
    if (num_blocks > (~0ULL) / block_size)
        return fail(KVFLUX_ERR_OVERFLOW, "norm, rotation and write: size overflow");
    // Rows of a launch: a wavefront each in the generic kernel, and fewer than 2^32 threads.
    constexpr std::uint64_t limit = (1ULL << 26) - 1;
    if (query_heads > limit || num_kv_heads > limit || block_size > 0x7fffffffULL ||
        num_tokens > limit / (query_heads + 2 * num_kv_heads))
        return fail(KVFLUX_ERR_UNSUPPORTED, "norm, rotation and write: dimension too large");
    if (query_stride < query_heads * head_size || key_stride < num_kv_heads * head_size ||
        value_stride < num_kv_heads * head_size)
        return fail(KVFLUX_ERR_INVALID_ARGUMENT, "norm, rotation and write: a stride is shorter than a token's heads");
    const auto misaligned = [](const void* ptr, std::size_t bytes) {
        return reinterpret_cast<std::uintptr_t>(ptr) % bytes != 0;
    };
    if (misaligned(query_in, in_bytes) || misaligned(key_in, in_bytes) || misaligned(value_in, in_bytes) ||
        misaligned(key_cache, cache_bytes) || misaligned(value_cache, cache_bytes) ||
        misaligned(query_out, sizeof(float)) || misaligned(query_norm, sizeof(float)) ||
        misaligned(key_norm, sizeof(float)) || misaligned(inv_freq, sizeof(double)))
        return fail(KVFLUX_ERR_INVALID_ARGUMENT, "norm, rotation and write: misaligned buffers");

    Params p{};
    p.query_in = query_in;
    p.key_in = key_in;
    p.value_in = value_in;
    p.query_stride = query_stride;
    p.key_stride = key_stride;
    p.value_stride = value_stride;
    p.key_cache = key_cache;
    p.value_cache = value_cache;
    p.slot_count = num_blocks * block_size;
    p.block_size = FastDiv(static_cast<std::uint32_t>(block_size));
    p.head_step = block_size * head_size;
    p.wide = p.slot_count > 0xffffffffULL;
    p.kv_heads = static_cast<std::uint32_t>(num_kv_heads);
    p.query_heads = static_cast<std::uint32_t>(query_heads);
    p.head_dim = static_cast<std::uint32_t>(head_size);
    p.token_rows = FastDiv(static_cast<std::uint32_t>(query_heads + 2 * num_kv_heads));
    p.tokens = static_cast<std::uint32_t>(num_tokens);
    p.rows = p.tokens * p.token_rows.divisor;
    p.query_norm = query_norm;
    p.key_norm = key_norm;
    p.eps = eps;
    p.inv_dim = 1.0f / static_cast<float>(head_size);
    p.inv_freq = inv_freq;
    p.rotary = static_cast<std::uint32_t>(rotary_dim);
    p.half = FastDiv(p.rotary != 0 ? p.rotary / 2 : 1);
    p.interleaved = interleaved != 0;
    p.query_out = query_out;
    const hipStream_t s = as_stream(stream);
    switch (input_dtype) {
    case KVFLUX_DTYPE_BF16: return launch_cache<Bf16>(p, dtype, place, s);
    case KVFLUX_DTYPE_F16: return launch_cache<F16>(p, dtype, place, s);
    default: return launch_cache<F32>(p, dtype, place, s);
    }
}

} // namespace
} // namespace kvflux_hip

using namespace kvflux_hip;

extern "C" int kvflux_norm_rope_write(void* key_cache, void* value_cache, uint64_t num_blocks, uint64_t num_kv_heads,
                                      uint64_t block_size, uint64_t head_size, int dtype, const void* query_in,
                                      const void* key_in, const void* value_in, int input_dtype,
                                      uint64_t query_stride, uint64_t key_stride, uint64_t value_stride,
                                      uint64_t query_heads, const float* query_norm, const float* key_norm, float eps,
                                      const double* inv_freq, uint64_t rotary_dim, int interleaved,
                                      const uint64_t* positions, const uint64_t* slots, uint64_t num_tokens,
                                      float* query_out, void* stream) {
    if (num_tokens == 0) return KVFLUX_OK;
    if (!positions || !slots) return fail(KVFLUX_ERR_INVALID_ARGUMENT, "norm, rotation and write: null pointer");
    return norm_rope_write(key_cache, value_cache, num_blocks, num_kv_heads, block_size, head_size, dtype, query_in,
                           key_in, value_in, input_dtype, query_stride, key_stride, value_stride, query_heads,
                           query_norm, key_norm, eps, inv_freq, rotary_dim, interleaved, Listed{positions, slots},
                           num_tokens, query_out, stream);
}

extern "C" int kvflux_norm_rope_write_tail(void* key_cache, void* value_cache, uint64_t num_blocks,
                                           uint64_t num_kv_heads, uint64_t block_size, uint64_t head_size, int dtype,
                                           const void* query_in, const void* key_in, const void* value_in,
                                           int input_dtype, uint64_t query_stride, uint64_t key_stride,
                                           uint64_t value_stride, uint64_t query_heads, const float* query_norm,
                                           const float* key_norm, float eps, const double* inv_freq,
                                           uint64_t rotary_dim, int interleaved, const uint64_t* block_table,
                                           uint64_t table_width, const uint64_t* seq_lens, uint64_t num_rows,
                                           float* query_out, void* stream) {
    if (num_rows == 0) return KVFLUX_OK;
    if (!block_table || !seq_lens || table_width == 0)
        return fail(KVFLUX_ERR_INVALID_ARGUMENT, "norm, rotation and tail write: null table");
    if (num_rows > (~0ULL) / table_width)
        return fail(KVFLUX_ERR_OVERFLOW, "norm, rotation and tail write: size overflow");
    return norm_rope_write(key_cache, value_cache, num_blocks, num_kv_heads, block_size, head_size, dtype, query_in,
                           key_in, value_in, input_dtype, query_stride, key_stride, value_stride, query_heads,
                           query_norm, key_norm, eps, inv_freq, rotary_dim, interleaved,
                           Tail{block_table, table_width, seq_lens, block_size, num_blocks}, num_rows, query_out,
                           stream);
}
