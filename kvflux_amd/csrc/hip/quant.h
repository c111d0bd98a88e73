// The formats of an 8-bit cache: what a byte stands for, and the scale of the
// values that share one.
//
// A value is q * s with s = 2^k, the smallest power of two that brings the largest
// magnitude to the format's top (448 or 127). Powers of two, not top / largest:
// dividing by s is exact, so rounding happens once and is the same whoever
// computes it; raising the scale of a page that has tokens moves E4M3 values by
// whole exponents (exact above their subnormals), where another factor would round
// all of them anew at each step. E4M3 loses nothing by it (its relative precision
// is the same at every size), integers at most one bit of seven.
#pragma once

#include "common.h"

#include <initializer_list>

namespace kvflux_hip {

// Attention of any shape, a workgroup for each (query row, query head): quant_rows_kernel.
struct QuantRows {
    const std::uint8_t* key_cache;
    const std::uint8_t* value_cache;
    const float* key_scales;
    const float* value_scales;
    std::uint64_t num_blocks;
    std::uint32_t heads, head_size;
    FastDiv block_size;
    const std::uint64_t* table;
    std::uint64_t width;
    const std::uint64_t* lens;
    std::uint32_t kv_len;  // bound of every length
    // Null: row r is the one query of sequence r. Else row r is query r % max_query of
    // sequence r / max_query's last query_lens[.], at row query_offsets[.] on.
    const std::uint64_t* query_lens;
    const std::uint64_t* query_offsets;
    std::uint32_t max_query;
    std::uint32_t query_heads, group;
    const float* query;
    float* output;
    float scale_log2;
};
int launch_quant_rows(const QuantRows& p, std::uint64_t rows, int format, hipStream_t stream);

namespace {

typedef __attribute__((ext_vector_type(2))) float qt_f32x2_t;
typedef __attribute__((ext_vector_type(2))) _Float16 qt_f16x2_t;

// hold4: four values, divided by their scale, to bytes (nearest, ties to even).
// values4: what four bytes stand for. pair16: bytes 2 * half and 2 * half + 1 of a word as two
// FP16 values, exactly (448 and 2^-9 are normal there; bytes up to -128 are whole).
struct QuantE4m3 {
    static constexpr int kTopLog2 = 9;                     // 448 = 0.875 * 2^9
    static constexpr std::uint32_t kTopMantissa = 0x600000u;  // of 1.75
    __device__ static std::uint32_t hold4(float a, float b, float c, float d) {
        const int lo = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
        return static_cast<std::uint32_t>(__builtin_amdgcn_cvt_pk_fp8_f32(c, d, lo, true));
    }
    __device__ static void values4(std::uint32_t w, float (&out)[4]) {
        const qt_f32x2_t lo = __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(w), false);
        const qt_f32x2_t hi = __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(w), true);
        out[0] = lo[0];
        out[1] = lo[1];
        out[2] = hi[0];
        out[3] = hi[1];
    }
    template <int kHalf>
    __device__ static std::uint32_t pair16(std::uint32_t w) {
        return __builtin_bit_cast(std::uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, kHalf != 0));
    }
};
struct QuantInt8 {
    static constexpr int kTopLog2 = 7;                     // 127 = (127 / 128) * 2^7
    static constexpr std::uint32_t kTopMantissa = 0x7e0000u;  // of 127 / 64
    __device__ static std::uint32_t hold4(float a, float b, float c, float d) {
        const auto byte = [](float x) { return static_cast<std::uint32_t>(static_cast<int>(__builtin_rintf(x))) & 0xffu; };
        return byte(a) | byte(b) << 8 | byte(c) << 16 | byte(d) << 24;
    }
    __device__ static void values4(std::uint32_t w, float (&out)[4]) {
#pragma unroll
        for (int i = 0; i < 4; ++i) out[i] = static_cast<float>(static_cast<int>(w << (24 - 8 * i)) >> 24);
    }
    // The byte plus 128 is the mantissa of an FP16 of 1024 to 1279.
    template <int kHalf>
    __device__ static std::uint32_t pair16(std::uint32_t w) {
        const std::uint32_t m = __builtin_amdgcn_perm(0x64646464u, w ^ 0x80808080u, kHalf == 0 ? 0x04010400u : 0x04030402u);
        const qt_f16x2_t base{static_cast<_Float16>(-1152.0f), static_cast<_Float16>(-1152.0f)};
        return __builtin_bit_cast(std::uint32_t, __builtin_bit_cast(qt_f16x2_t, m) + base);
    }
};

// op over a wavefront's 64 values, the same in every lane: lane permutations of the
// VALU, a few cycles a step where a shuffle through LDS takes some 60.
template <typename T, typename Op>
__device__ inline T over_wave(T x, Op op) {
    static_assert(sizeof(T) == 4, "a register");
    const auto with = [&](int bits) { x = op(x, __builtin_bit_cast(T, bits)); };
    const auto bits = [&] { return __builtin_bit_cast(int, x); };
    with(__builtin_amdgcn_update_dpp(0, bits(), 0xb1, 0xf, 0xf, true));   // quad_perm: lane ^ 1
    with(__builtin_amdgcn_update_dpp(0, bits(), 0x4e, 0xf, 0xf, true));   // quad_perm: lane ^ 2
    with(__builtin_amdgcn_update_dpp(0, bits(), 0x141, 0xf, 0xf, true));  // row_half_mirror
    with(__builtin_amdgcn_update_dpp(0, bits(), 0x140, 0xf, 0xf, true));  // row_mirror
    // The pair's values are copied out: a bit cast of a vector's element reads the first.
    const auto a = __builtin_amdgcn_permlane16_swap(static_cast<unsigned>(bits()), static_cast<unsigned>(bits()), false, false);
    const unsigned a0 = a[0], a1 = a[1];
    x = op(__builtin_bit_cast(T, a0), __builtin_bit_cast(T, a1));
    const auto b = __builtin_amdgcn_permlane32_swap(static_cast<unsigned>(bits()), static_cast<unsigned>(bits()), false, false);
    const unsigned b0 = b[0], b1 = b[1];
    return op(__builtin_bit_cast(T, b0), __builtin_bit_cast(T, b1));
}
__device__ inline float wave_max(float x) {  // of what is no NaN
    return over_wave(x, [](float a, float b) { return fmaxf(a, b); });
}

// The scale for values whose largest magnitude has the FP32 bits `largest`; NaN for
// an infinity or NaN. 2^-110 at least: every value of either format times it is a
// normal FP32 number (2^-9 * 2^-110 > 2^-126), zeros apart.
constexpr int kLeastScaleLog2 = -110;
template <typename F>
__device__ inline float quant_scale(std::uint32_t largest) {
    int k = static_cast<int>(largest >> 23) - 126 - F::kTopLog2 + ((largest & 0x7fffffu) > F::kTopMantissa ? 1 : 0);
    if (k < kLeastScaleLog2) k = kLeastScaleLog2;
    return __uint_as_float(largest >= 0x7f800000u ? 0x7fc00000u : static_cast<std::uint32_t>(k + 127) << 23);
}

// Head size of the attention kernels that a head size runs on, the least that holds it; 0:
// the generic kernel's.
inline std::uint64_t padded_head_size(std::uint64_t head_size) {
    if (head_size % 16 != 0 || head_size > 256) return 0;
    return head_size <= 64 ? 64 : head_size <= 128 ? 128 : 256;
}

// Workgroups of a launch: HIP counts the threads of a grid, 256 a workgroup here, in 32 bits.
constexpr std::uint64_t kMostWorkgroups = 0xffffffffULL / 256;

inline bool aligned(std::uint64_t bytes, std::initializer_list<const void*> pointers) {
    for (const void* x : pointers)
        if (reinterpret_cast<std::uintptr_t>(x) % bytes != 0) return false;
    return true;
}

// What every call on an 8-bit cache checks.
inline int check_quant_cache(const char* op, const void* key_cache, const void* value_cache, const void* key_scales,
                             const void* value_scales, std::uint64_t num_blocks, std::uint64_t heads,
                             std::uint64_t block_size, std::uint64_t head_size, int format) {
    if (format != KVFLUX_QUANT_E4M3 && format != KVFLUX_QUANT_INT8)
        return fail(KVFLUX_ERR_INVALID_ARGUMENT, "%s: unknown format %d", op, format);
    if (!key_cache || !value_cache || !key_scales || !value_scales)
        return fail(KVFLUX_ERR_INVALID_ARGUMENT, "%s: null cache pointer", op);
    if (num_blocks == 0 || heads == 0 || block_size == 0 || head_size == 0)
        return fail(KVFLUX_ERR_INVALID_ARGUMENT, "%s: empty cache shape", op);
    if (!aligned(4, {key_scales, value_scales}))
        return fail(KVFLUX_ERR_INVALID_ARGUMENT, "%s: misaligned scales", op);
    if (heads > 65535 || head_size > 0x7fffffffULL || block_size > 0x7fffffffULL / head_size)
        return fail(KVFLUX_ERR_UNSUPPORTED, "%s: a page is too large", op);
    if (num_blocks > (std::uint64_t{1} << 56) / (heads * block_size * head_size))
        return fail(KVFLUX_ERR_OVERFLOW, "%s: cache size", op);
    return KVFLUX_OK;
}

} // namespace
} // namespace kvflux_hip
