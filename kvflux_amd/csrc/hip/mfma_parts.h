// What the MFMA attention kernels on 16-bit caches share: operand types and the
// splits of an FP32 value into 16-bit parts, maxima and sums across the quads of
// a column, and loads from global memory straight into LDS with their waits.
#pragma once

#include "common.h"

namespace kvflux_hip {
namespace {

typedef __attribute__((ext_vector_type(8))) __bf16 pf_bf16x8_t;
typedef __attribute__((ext_vector_type(8))) _Float16 pf_f16x8_t;
typedef __attribute__((ext_vector_type(4))) float pf_f32x4_t;
typedef short pf_i16x4_t __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) pf_i16x4_t pf_lds_i16x4_t;

typedef __attribute__((ext_vector_type(2))) float pf_f32x2_t;
typedef __attribute__((ext_vector_type(2))) __bf16 pf_bf16x2_t;
typedef __attribute__((ext_vector_type(2))) _Float16 pf_f16x2_t;

// pack(a, b): a in the low half, b in the high half, each rounded to nearest
// even (one v_cvt_pk_{bf16,f16}_f32). split3(a, b): the same pair as three
// 16-bit parts whose sum is a and b (each part the rounded remainder of the
// ones before; the differences are exact in FP32), so an MFMA over the three
// parts against 16-bit cache values forms FP32-exact products.
struct PfBf16 {
    using Vec = pf_bf16x8_t;
    // Weights enter the split scaled by kWeightScale (undone exactly in the
    // epilogue); the running reference moves once a score passes it by
    // 2^kLazyLog2, so weights stay <= 2^kLazyLog2.
    static constexpr float kWeightScale = 1.0f;
    static constexpr float kLazyLog2 = 8.0f;
    static constexpr bool kExact = false;
    static constexpr std::uint32_t kOnes = 0x3f803f80u;  // two 1.0
    __device__ static std::uint32_t pack(float a, float b) {
        return __builtin_bit_cast(std::uint32_t, __builtin_convertvector(pf_f32x2_t{a, b}, pf_bf16x2_t));
    }
    __device__ static void split3(float a, float b, std::uint32_t (&w)[3]) {
        pf_f32x2_t x{a, b};
#pragma unroll
        for (int i = 0; i < 3; ++i) {
            const pf_bf16x2_t h = __builtin_convertvector(x, pf_bf16x2_t);
            w[i] = __builtin_bit_cast(std::uint32_t, h);
            x -= __builtin_convertvector(h, pf_f32x2_t);
        }
    }
    __device__ static pf_f32x4_t mma(const Vec& a, const Vec& b, const pf_f32x4_t& c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
    }
};
struct PfF16 {
    using Vec = pf_f16x8_t;
    static constexpr float kWeightScale = 1.0f;
    static constexpr float kLazyLog2 = 8.0f;
    static constexpr bool kExact = false;
    static constexpr std::uint32_t kOnes = 0x3c003c00u;  // two 1.0
    __device__ static std::uint32_t pack(float a, float b) {
        return __builtin_bit_cast(std::uint32_t, __builtin_convertvector(pf_f32x2_t{a, b}, pf_f16x2_t));
    }
    __device__ static void split3(float a, float b, std::uint32_t (&w)[3]) {
        pf_f32x2_t x{a, b};
#pragma unroll
        for (int i = 0; i < 3; ++i) {
            const pf_f16x2_t h = __builtin_convertvector(x, pf_f16x2_t);
            w[i] = __builtin_bit_cast(std::uint32_t, h);
            x -= __builtin_convertvector(h, pf_f32x2_t);
        }
    }
    __device__ static pf_f32x4_t mma(const Vec& a, const Vec& b, const pf_f32x4_t& c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
    }
};
// The exact variants: Q and the softmax weights enter the MFMAs as three
// 16-bit parts each (FP32-exact products, FP32 accumulation), the row sums
// are FP32 sums of the weights, and a wavefront holds one row block.
struct PfBf16Exact : PfBf16 {
    static constexpr bool kExact = true;
};
// FP16's exponent stops at 2^-24: an unscaled weight below that would
// vanish from the numerator while still counting in the FP32 row sum. The
// FP16 exact variant therefore keeps every weight <= 1 (the reference moves
// with every new row maximum) and splits 2^15 times the weight (<= 32768, in
// range): a leading part loses bits to FP16's subnormals only below 2^-29
// of the row maximum and vanishes only below 2^-39, where 2^15 such keys
// together weigh under 2^-24 of the row; the epilogue multiplies by 2^-15
// (exact).
struct PfF16Exact : PfF16 {
    static constexpr bool kExact = true;
    static constexpr float kWeightScale = 32768.0f;
    static constexpr float kLazyLog2 = 0.0f;
};
// Exponent of the power of two by which a row of scaled queries is split into FP16
// parts, whose range is fixed: it takes the `largest` into [2^14, 2^15), so only
// values below 2^-16 of that lose bits of FP32's 24. 0 for zero,
// NaN, infinity and what passes 2^100 (whose scores could pass FP32), and 126 at
// most, as 2^-126 is the last normal number.
__device__ inline int split_exponent(float largest) {
    const int e = largest > 0.0f && largest < 0x1p100f ? 15 - __builtin_amdgcn_frexp_expf(largest) : 0;
    return e < 126 ? e : 126;
}
// NaN-propagating maximum of three (one v_maximum3_f32).
__device__ inline float max3(float a, float b, float c) {
    return __builtin_elementwise_maximum(__builtin_elementwise_maximum(a, b), c);
}
// Sum over the four lanes l, l^16, l^32, l^48, the same in all four (each
// level adds a pair in either order).
__device__ inline float sum_across_quads(float x) {
    const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = __uint_as_float(a[0]) + __uint_as_float(a[1]);
    const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}
// Maximum over the four lanes l, l^16, l^32, l^48 (the four quads of a
// column) with two cross-row lane swaps, no LDS round trip.
__device__ inline float max_across_quads(float x) {
    const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = __builtin_elementwise_maximum(__uint_as_float(a[0]), __uint_as_float(a[1]));
    const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return __builtin_elementwise_maximum(__uint_as_float(b[0]), __uint_as_float(b[1]));
}

// s_waitcnt immediates (gfx9 encoding): vmcnt(n) alone, lgkmcnt(0) alone.
template <int kN>
__device__ inline void wait_vm() {
    static_assert(kN >= 0 && kN < 64, "vmcnt range");
    __builtin_amdgcn_s_waitcnt((kN & 15) | ((kN >> 4) << 14) | (7 << 4) | (15 << 8));
}
__device__ inline void wait_lgkm0() { __builtin_amdgcn_s_waitcnt(0xF | (3 << 14) | (7 << 4)); }
// One 16-byte-per-lane load from global memory straight into LDS at
// m0 + lane * 16 (m0 wave-uniform). Issued as inline assembly so the
// compiler's wait-count tracking does not treat it as an LDS write (it would
// then wait for every such load before any LDS read); completion is ordered
// by the explicit vmcnt waits before the barriers.
__device__ inline void load_to_lds(const void* src, std::uint32_t lds_byte) {
    asm volatile("global_load_lds_dwordx4 %0, off" ::"v"(src), "{m0}"(lds_byte) : "memory");
}
// The same from `base` (wave-uniform) and a byte offset of each lane.
__device__ inline void load_to_lds(std::uint64_t base, std::uint32_t offset, std::uint32_t lds_byte) {
    asm volatile("global_load_lds_dwordx4 %0, %1" ::"v"(offset), "s"(base), "{m0}"(lds_byte) : "memory");
}
__device__ inline std::uint32_t lds_address(const void* p) {
    return static_cast<std::uint32_t>(reinterpret_cast<std::uintptr_t>((__attribute__((address_space(3))) const char*)p));
}
// Workgroup barrier without the release fence of __syncthreads (which would
// also wait for the tile loads still in flight); LDS visibility is ordered by
// the explicit waits before it.
__device__ inline void lds_barrier() {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}
// Wave priority (s_setprio) pinned in place: raised while a wave issues its
// QK^T MFMAs, so a SIMD's other wave runs its softmax in the meantime.
template <short kLevel>
__device__ inline void set_priority() {
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_setprio(kLevel);
    __builtin_amdgcn_sched_barrier(0);
}

} // namespace
} // namespace kvflux_hip
