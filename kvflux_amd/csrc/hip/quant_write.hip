// Writes to and reads from a paged cache held in 8 bits with a scale for each
// page and kv head:
//   write  s' = max(s if the page has earlier tokens, 2^ceil(log2(max|x| / top)))
//          q = round(x / s'), and q' = round(q s / s') of those earlier tokens
//          (the quotients in FP32: exact, unless a scale of another origin is no power of two)
//   read   x = q s
//
// Both are bound by memory, and small calls by the chain of dependent loads: a
// row's length, its table entry, the page's scale. A unit of the write is the part
// of one page, head and cache that takes new tokens: its values are read once into
// registers (their largest magnitude is needed before the first of them can be
// rounded) and written once. A wavefront takes a unit of up to 2048 values (16
// tokens of 128), so nothing waits at a barrier; a workgroup takes a larger one
// (8192 in registers, what is behind them is read again from the L2). 4096 tokens of
// BF16, 8 kv heads of 128 (25 MB): 6.4 us a call, 5.7 to 6.9 in the kernel (7.2 with
// shuffles through LDS); one token each of 8 rows 3.4 in the kernel, 6.0 a call.
#include "quant.h"

#include <type_traits>

namespace kvflux_hip {
namespace {

constexpr int kThreads = 256;

struct InF16 {
    using T = std::uint16_t;
    __device__ static float value(std::uint16_t x) { return static_cast<float>(__builtin_bit_cast(_Float16, x)); }
};
struct InBf16 {
    using T = std::uint16_t;
    __device__ static float value(std::uint16_t x) { return __uint_as_float(static_cast<std::uint32_t>(x) << 16); }
};
struct InF32 {
    using T = float;
    __device__ static float value(float x) { return x; }
};

// kV neighbouring values of a row: 16 or 32 bytes, or a single one.
template <typename In, int kV>
struct alignas(sizeof(typename In::T) * kV < 16 ? sizeof(typename In::T) * kV : 16) Group {
    typename In::T x[kV];
};

struct WriteParams {
    std::uint8_t* cache[2];
    float* scales[2];
    const void* rows[2];
    std::uint64_t stride[2];
    std::uint64_t num_blocks;
    FastDiv heads;
    std::uint32_t block_size;
    int bs_shift;             // log2(block_size), or -1
    std::uint32_t head_size;
    FastDiv row_groups;       // head_size / kV
    const std::uint64_t* table;
    std::uint64_t width;
    const std::uint64_t* kv_lens;
    const std::uint64_t* new_lens;  // null: one token a sequence, input row = sequence
    const std::uint64_t* offsets;
    std::uint32_t max_new;    // bound of new_lens
    FastDiv pages;            // pages a sequence may touch
    std::uint32_t units;
};

// kWaves wavefronts for a unit; unit = ((sequence * pages + page) * 2 + cache) *
// heads + head, so neighbouring wavefronts read neighbouring heads of a token.
template <typename In, typename F, int kV, int kWaves>
__global__ __launch_bounds__(kThreads) void quant_write_kernel(WriteParams p) {
    using G = Group<In, kV>;
    constexpr std::uint32_t kT = 64 * kWaves;
    constexpr int kHeld = 4;  // groups of a thread in registers
    __shared__ std::uint32_t largest_of[kWaves];
    const auto uniform = [](std::uint32_t x) {
        return static_cast<std::uint32_t>(__builtin_amdgcn_readfirstlane(static_cast<int>(x)));
    };
    const std::uint32_t unit = kWaves == 1 ? blockIdx.x * (kThreads / 64) + uniform(threadIdx.x / 64) : blockIdx.x;
    if (unit >= p.units) return;  // uniform in the unit
    const std::uint32_t tid = threadIdx.x % kT;
    std::uint32_t rest = p.heads.div(unit);
    const std::uint32_t head = unit - rest * p.heads.divisor;
    const std::uint32_t kv = rest & 1;
    rest >>= 1;
    const std::uint32_t seq = p.pages.div(rest);
    const std::uint32_t page_of_new = rest - seq * p.pages.divisor;

    const std::uint64_t full = p.kv_lens[seq];
    std::uint64_t fresh = p.new_lens ? p.new_lens[seq] : 1;
    const std::uint64_t offset = p.offsets ? p.offsets[seq] : seq;
    if (fresh > full) fresh = full;
    if (fresh == 0) return;
    const std::uint64_t start = full - fresh, len = fresh < p.max_new ? full : start + p.max_new;
    const std::uint64_t page = (p.bs_shift >= 0 ? start >> p.bs_shift : start / p.block_size) + page_of_new;
    const std::uint64_t at = page * p.block_size;  // position of the page's first token
    if (at >= len || page >= p.width) return;
    const std::uint64_t entry = p.table[seq * p.width + page];
    const std::uint32_t first = start > at ? static_cast<std::uint32_t>(start - at) : 0;
    const std::uint32_t last = len - at < p.block_size ? static_cast<std::uint32_t>(len - at) : p.block_size;

    // Group c of the page and head is kV values of its token c / row_groups; `base`
    // is where token 0's row would lie among the inputs (formed without it).
    const std::uint32_t cpr = p.row_groups.divisor;
    const typename In::T* const rows = static_cast<const typename In::T*>(p.rows[kv]) + static_cast<std::uint64_t>(head) * p.head_size;
    const std::uint64_t first_row = offset + (at + first - start);
    const auto input = [&](std::uint32_t c) {
        const std::uint32_t t = p.row_groups.div(c);
        return reinterpret_cast<const G*>(rows + (first_row + (t - first)) * p.stride[kv] + (c - t * cpr) * kV);
    };
    const std::uint32_t begin = first * cpr, end = last * cpr;
    G held[kHeld];
    std::uint32_t largest = 0;
    const auto weigh = [&](const G& g) {
#pragma unroll
        for (int i = 0; i < kV; ++i) {
            const std::uint32_t bits = __float_as_uint(In::value(g.x[i])) & 0x7fffffffu;
            largest = bits > largest ? bits : largest;
        }
    };
#pragma unroll
    for (int i = 0; i < kHeld; ++i) {
        const std::uint32_t c = begin + tid + i * kT;
        held[i] = *input(c < end ? c : end - 1);
    }
    // The input needs no page: it is on its way while the table is read. (A page that is
    // not there: the first one's scale, and no store.)
    const bool there = entry < p.num_blocks;
    const std::uint64_t id = there ? entry : 0;
    float* const scale_at = p.scales[kv] + (id * p.heads.divisor + head);
    const float before = *scale_at;
#pragma unroll
    for (int i = 0; i < kHeld; ++i) weigh(held[i]);  // past the end: the last group again
    for (std::uint32_t c = begin + tid + kHeld * kT; c < end; c += kT) weigh(*input(c));
    largest = over_wave(largest, [](std::uint32_t a, std::uint32_t b) { return a > b ? a : b; });
    if constexpr (kWaves > 1) {
        if (tid % 64 == 0) largest_of[tid / 64] = largest;
        __syncthreads();  // every wavefront has read the scale as well
#pragma unroll
        for (int w = 0; w < kWaves; ++w) largest = largest_of[w] > largest ? largest_of[w] : largest;
    }
    if (!there) return;  // uniform in the unit
    float scale = quant_scale<F>(largest);
    // A scale of another origin may be negative: it is its size that has to do.
    if (first != 0 && !(scale > __builtin_fabsf(before))) scale = before != before || scale == scale ? before : scale;
    const float inverse = 1.0f / scale;

    std::uint8_t* const held_at = p.cache[kv] + (id * p.heads.divisor + head) * p.block_size * static_cast<std::uint64_t>(p.head_size);
    const auto put = [&](std::uint32_t c, const float (&y)[kV]) {
        if constexpr (kV == 1) {
            held_at[c] = static_cast<std::uint8_t>(F::hold4(y[0], 0.0f, 0.0f, 0.0f));
        } else {
            *reinterpret_cast<V8*>(held_at + static_cast<std::uint64_t>(c) * 8) =
                V8{{F::hold4(y[0], y[1], y[2], y[3]), F::hold4(y[4], y[5], y[6], y[7])}};
        }
    };
    const auto write = [&](std::uint32_t c, const G& g) {
        float y[kV];
#pragma unroll
        for (int i = 0; i < kV; ++i) y[i] = In::value(g.x[i]) * inverse;
        // A kept scale of another origin may be no power of two: its reciprocal is rounded.
        if (__builtin_expect((__float_as_uint(scale) & 0x7fffffu) != 0, 0)) {  // uniform in the unit
#pragma unroll
            for (int i = 0; i < kV; ++i) y[i] = In::value(g.x[i]) / scale;
        }
        put(c, y);
    };
#pragma unroll
    for (int i = 0; i < kHeld; ++i) {
        const std::uint32_t c = begin + tid + i * kT;
        if (c < end) write(c, held[i]);
    }
    for (std::uint32_t c = begin + tid + kHeld * kT; c < end; c += kT) write(c, *input(c));
    if (first != 0 && scale != before) {  // the earlier tokens, to the new scale
        const float ratio = before * inverse;
        for (std::uint32_t c = tid; c < begin; c += kT) {
            float q[4], y[kV];
            if constexpr (kV == 1) {
                F::values4(held_at[c], q);
                y[0] = q[0] * ratio;
            } else {
                const V8 w = *reinterpret_cast<const V8*>(held_at + static_cast<std::uint64_t>(c) * 8);
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    F::values4(w.w[h], q);
#pragma unroll
                    for (int i = 0; i < 4; ++i) y[4 * h + i] = q[i] * ratio;
                }
            }
            put(c, y);
        }
    }
    if (tid == 0) *scale_at = scale;
}

template <typename In, typename F, int kV>
int launch_write(WriteParams& p, hipStream_t stream) {
    p.row_groups = FastDiv(p.head_size / kV);
    if (kV > 1 && p.head_size * static_cast<std::uint64_t>(p.block_size) <= 2048) {
        const std::uint32_t units = kThreads / 64;
        quant_write_kernel<In, F, kV, 1><<<dim3((p.units - 1) / units + 1), dim3(kThreads), 0, stream>>>(p);
    } else {
        quant_write_kernel<In, F, kV, kThreads / 64><<<dim3(p.units), dim3(kThreads), 0, stream>>>(p);
    }
    return launch_status("quant_write_kernel");
}

template <typename In>
int launch_write_format(WriteParams& p, int format, bool wide, hipStream_t stream) {
    if (format == KVFLUX_QUANT_E4M3)
        return wide ? launch_write<In, QuantE4m3, 8>(p, stream) : launch_write<In, QuantE4m3, 1>(p, stream);
    return wide ? launch_write<In, QuantInt8, 8>(p, stream) : launch_write<In, QuantInt8, 1>(p, stream);
}

int write(const char* op, void* key_cache, void* value_cache, float* key_scales, float* value_scales,
          std::uint64_t num_blocks, std::uint64_t heads, std::uint64_t block_size, std::uint64_t head_size, int format,
          const void* key_new, const void* value_new, int input_dtype, std::uint64_t key_stride,
          std::uint64_t value_stride, const std::uint64_t* table, std::uint64_t width, const std::uint64_t* kv_lens,
          const std::uint64_t* new_lens, const std::uint64_t* offsets, std::uint64_t num_seqs,
          std::uint64_t max_new, void* stream) {
    if (const int s = check_quant_cache(op, key_cache, value_cache, key_scales, value_scales, num_blocks, heads, block_size,
                                  head_size, format))
        return s;
    const std::uint64_t element = dtype_bytes(input_dtype);
    if (element == 0) return fail(KVFLUX_ERR_INVALID_ARGUMENT, "%s: unknown dtype %d", op, input_dtype);
    if (!key_new || !value_new || !table || !kv_lens) return fail(KVFLUX_ERR_INVALID_ARGUMENT, "%s: null pointer", op);
    if (!aligned(element, {key_new, value_new}) || !aligned(8, {table, kv_lens, new_lens, offsets}))
        return fail(KVFLUX_ERR_INVALID_ARGUMENT, "%s: misaligned array", op);
    if (width == 0) return fail(KVFLUX_ERR_INVALID_ARGUMENT, "%s: empty table rows", op);
    const std::uint64_t row = heads * head_size;
    if (num_seqs > 1 || max_new > 1) {
        if (key_stride < row || value_stride < row)
            return fail(KVFLUX_ERR_INVALID_ARGUMENT, "%s: a stride is shorter than a token's heads", op);
    }
    // A run of n tokens touches at most (n + block_size - 2) / block_size + 1 pages.
    const std::uint64_t pages = max_new > 0x7fffffffULL ? ~0ULL : (max_new + block_size - 2) / block_size + 1;
    if (num_seqs > 0x7fffffffULL || pages > 0x7fffffffULL || pages * num_seqs > kMostWorkgroups / (2 * heads))
        return fail(KVFLUX_ERR_UNSUPPORTED, "%s: too many new tokens", op);
    WriteParams p{};
    p.cache[0] = static_cast<std::uint8_t*>(key_cache);
    p.cache[1] = static_cast<std::uint8_t*>(value_cache);
    p.scales[0] = key_scales;
    p.scales[1] = value_scales;
    p.rows[0] = key_new;
    p.rows[1] = value_new;
    p.stride[0] = key_stride;
    p.stride[1] = value_stride;
    p.num_blocks = num_blocks;
    p.heads = FastDiv(static_cast<std::uint32_t>(heads));
    p.block_size = static_cast<std::uint32_t>(block_size);
    p.bs_shift = -1;
    if (is_pow2(block_size)) p.bs_shift = __builtin_ctzll(block_size);
    p.head_size = static_cast<std::uint32_t>(head_size);
    p.table = table;
    p.width = width;
    p.kv_lens = kv_lens;
    p.new_lens = new_lens;
    p.offsets = offsets;
    p.max_new = static_cast<std::uint32_t>(max_new);
    p.pages = FastDiv(static_cast<std::uint32_t>(pages));
    p.units = static_cast<std::uint32_t>(pages * num_seqs * 2 * heads);
    const bool wide = head_size % 8 == 0 && key_stride % 8 == 0 && value_stride % 8 == 0 &&
                      aligned(16, {key_new, value_new}) && aligned(8, {key_cache, value_cache});
    const hipStream_t s = as_stream(stream);
    switch (input_dtype) {
    case KVFLUX_DTYPE_F16: return launch_write_format<InF16>(p, format, wide, s);
    case KVFLUX_DTYPE_BF16: return launch_write_format<InBf16>(p, format, wide, s);
    default: return launch_write_format<InF32>(p, format, wide, s);
    }
}

// ---------------------------------------------------------------- read
struct ReadParams {
    const std::uint8_t* cache[2];
    const float* scales[2];
    void* out[2];
    std::uint64_t num_blocks;
    std::uint32_t heads, block_size, head_size;
    FastDiv token_groups;  // groups of an output token
    FastDiv row_groups;    // groups of a (token, head) row
    const std::uint64_t* table;
    std::uint64_t width;
    const std::uint64_t* lens;
    const std::uint64_t* offsets;
    const std::uint64_t* page_starts;
    std::uint32_t num_seqs;
    FastDiv parts;         // parts of a page
    std::uint32_t units;
};

struct OutF16 {
    using T = std::uint16_t;
    __device__ static std::uint16_t hold(float x) { return __builtin_bit_cast(std::uint16_t, static_cast<_Float16>(x)); }
};
struct OutBf16 {
    using T = std::uint16_t;
    __device__ static std::uint16_t hold(float x) { return __builtin_bit_cast(std::uint16_t, static_cast<__bf16>(x)); }
};
struct OutF32 {
    using T = float;
    __device__ static float hold(float x) { return x; }
};

constexpr int kReadGroups = 4;  // groups of a thread

// A workgroup takes one part of one (page, cache): groups of kV values numbered as
// they lie in the output, so every store of a wavefront is one run of memory and a
// page's missing tokens are its last groups.
// 64 sequences of up to 16384 tokens, 8 kv heads of 128, to BF16 (3.55 GB): 613 us, 5.8
// TB/s; with the streaming hint on the loads too 621, without it on the stores 635, with
// 2 and 8 groups a thread 640 and 649, a whole page a workgroup 613.
template <typename F, typename Out, int kV>
__global__ __launch_bounds__(kThreads) void quant_gather_kernel(ReadParams p) {
    using Raw = typename std::conditional<kV == 8, V8, std::uint8_t>::type;
    const std::uint32_t w = p.parts.div(blockIdx.x);
    const std::uint32_t part = blockIdx.x - w * p.parts.divisor;
    const std::uint32_t kv = blockIdx.y;
    const std::uint32_t seq = __builtin_amdgcn_readfirstlane(find_sequence(p.page_starts, p.num_seqs, w));
    const std::uint64_t first_page = p.page_starts[seq];
    if (w < first_page) return;  // malformed scan
    const std::uint64_t logical = w - first_page;
    if (logical >= p.width) return;
    const std::uint64_t id = p.table[seq * p.width + logical];
    const std::uint64_t len = p.lens[seq], offset = p.offsets[seq];
    const std::uint64_t at = logical * p.block_size;
    if (at >= len || id >= p.num_blocks) return;
    const std::uint32_t valid = len - at < p.block_size ? static_cast<std::uint32_t>(len - at) : p.block_size;
    const std::uint32_t live = valid * p.token_groups.divisor;
    const std::uint32_t cpr = p.row_groups.divisor;
    const std::uint8_t* const src = p.cache[kv] + id * p.heads * p.block_size * static_cast<std::uint64_t>(p.head_size);
    const float* const scales = p.scales[kv] + id * p.heads;
    typename Out::T* const dst = static_cast<typename Out::T*>(p.out[kv]) + (offset + at) * p.heads * static_cast<std::uint64_t>(p.head_size);
    const std::uint32_t begin = part * (kThreads * kReadGroups) + threadIdx.x;
    Raw raw[kReadGroups];
    float scale[kReadGroups];
#pragma unroll
    for (int u = 0; u < kReadGroups; ++u) {
        const std::uint32_t j = begin + u * kThreads < live ? begin + u * kThreads : 0;
        const std::uint32_t token = p.token_groups.div(j), in_token = j - token * p.token_groups.divisor;
        const std::uint32_t head = p.row_groups.div(in_token);
        const std::uint64_t c = (static_cast<std::uint64_t>(head) * p.block_size + token) * cpr + (in_token - head * cpr);
        raw[u] = reinterpret_cast<const Raw*>(src)[c];
        scale[u] = scales[head];
    }
#pragma unroll
    for (int u = 0; u < kReadGroups; ++u) keep_in_registers(raw[u]);
#pragma unroll
    for (int u = 0; u < kReadGroups; ++u) {
        const std::uint32_t j = begin + u * kThreads;
        if (j >= live) continue;
        float q[4];
        if constexpr (kV == 1) {
            F::values4(raw[u], q);
            dst[j] = Out::hold(q[0] * scale[u]);
        } else {
            struct alignas(16) { typename Out::T x[8]; } out;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                F::values4(raw[u].w[h], q);
#pragma unroll
                for (int i = 0; i < 4; ++i) out.x[4 * h + i] = Out::hold(q[i] * scale[u]);
            }
            V16 v[sizeof(out) / 16];
            __builtin_memcpy(v, &out, sizeof(out));
            V16* const to = reinterpret_cast<V16*>(dst + static_cast<std::uint64_t>(j) * 8);
#pragma unroll
            for (unsigned i = 0; i < sizeof(out) / 16; ++i) stream_store(to + i, v[i]);
        }
    }
}

template <typename F, typename Out, int kV>
int launch_gather(ReadParams& p, std::uint64_t pages, hipStream_t stream) {
    const std::uint64_t row_groups = p.head_size / kV, token_groups = row_groups * p.heads;
    const std::uint64_t page_groups = token_groups * p.block_size;
    const std::uint64_t parts = (page_groups - 1) / (kThreads * kReadGroups) + 1;
    if (page_groups > 0xffffffffULL || parts > kMostWorkgroups / pages)
        return fail(KVFLUX_ERR_UNSUPPORTED, "quant gather: too many pages");
    p.row_groups = FastDiv(static_cast<std::uint32_t>(row_groups));
    p.token_groups = FastDiv(static_cast<std::uint32_t>(token_groups));
    p.parts = FastDiv(static_cast<std::uint32_t>(parts));
    quant_gather_kernel<F, Out, kV><<<dim3(static_cast<unsigned>(pages * parts), 2), dim3(kThreads), 0, stream>>>(p);
    return launch_status("quant_gather_kernel");
}

template <typename F>
int launch_gather_format(ReadParams& p, int dtype, bool wide, std::uint64_t pages, hipStream_t s) {
    switch (dtype) {
    case KVFLUX_DTYPE_F16: return wide ? launch_gather<F, OutF16, 8>(p, pages, s) : launch_gather<F, OutF16, 1>(p, pages, s);
    case KVFLUX_DTYPE_BF16: return wide ? launch_gather<F, OutBf16, 8>(p, pages, s) : launch_gather<F, OutBf16, 1>(p, pages, s);
    default: return wide ? launch_gather<F, OutF32, 8>(p, pages, s) : launch_gather<F, OutF32, 1>(p, pages, s);
    }
}

} // namespace
} // namespace kvflux_hip

using namespace kvflux_hip;

extern "C" int kvflux_quant_write(void* key_cache, void* value_cache, float* key_scales, float* value_scales,
                                  uint64_t num_blocks, uint64_t num_kv_heads, uint64_t block_size, uint64_t head_size,
                                  int format, const void* key_new, const void* value_new, int input_dtype,
                                  uint64_t key_stride, uint64_t value_stride, const uint64_t* block_table,
                                  uint64_t table_width, const uint64_t* kv_lens, const uint64_t* new_lens,
                                  const uint64_t* new_offsets, uint64_t num_seqs, uint64_t max_new_tokens,
                                  void* stream) {
    if (num_seqs == 0 || max_new_tokens == 0) return KVFLUX_OK;
    if (!new_lens || !new_offsets) return fail(KVFLUX_ERR_INVALID_ARGUMENT, "quant write: null pointer");
    return write("quant write", key_cache, value_cache, key_scales, value_scales, num_blocks, num_kv_heads, block_size,
                 head_size, format, key_new, value_new, input_dtype, key_stride, value_stride, block_table, table_width,
                 kv_lens, new_lens, new_offsets, num_seqs, max_new_tokens, stream);
}

extern "C" int kvflux_quant_write_tail(void* key_cache, void* value_cache, float* key_scales, float* value_scales,
                                       uint64_t num_blocks, uint64_t num_kv_heads, uint64_t block_size,
                                       uint64_t head_size, int format, const void* key_new, const void* value_new,
                                       int input_dtype, uint64_t key_stride, uint64_t value_stride,
                                       const uint64_t* block_table, uint64_t table_width, const uint64_t* seq_lens,
                                       uint64_t num_rows, void* stream) {
    if (num_rows == 0) return KVFLUX_OK;
    return write("quant write tail", key_cache, value_cache, key_scales, value_scales, num_blocks, num_kv_heads,
                 block_size, head_size, format, key_new, value_new, input_dtype, key_stride, value_stride, block_table,
                 table_width, seq_lens, nullptr, nullptr, num_rows, 1, stream);
}

extern "C" int kvflux_quant_gather(const void* key_cache, const void* value_cache, const float* key_scales,
                                   const float* value_scales, uint64_t num_blocks, uint64_t num_kv_heads,
                                   uint64_t block_size, uint64_t head_size, int format, const uint64_t* block_table,
                                   uint64_t max_blocks_per_seq, const uint64_t* seq_lens, const uint64_t* out_offsets,
                                   const uint64_t* page_starts, uint64_t num_seqs, uint64_t total_pages, void* key_out,
                                   void* value_out, int output_dtype, void* stream) {
    if (num_seqs == 0 || total_pages == 0) return KVFLUX_OK;
    if (const int s = check_quant_cache("quant gather", key_cache, value_cache, key_scales, value_scales, num_blocks,
                                  num_kv_heads, block_size, head_size, format))
        return s;
    const std::uint64_t element = dtype_bytes(output_dtype);
    if (element == 0) return fail(KVFLUX_ERR_INVALID_ARGUMENT, "quant gather: unknown dtype %d", output_dtype);
    if (!block_table || !seq_lens || !out_offsets || !page_starts || !key_out || !value_out)
        return fail(KVFLUX_ERR_INVALID_ARGUMENT, "quant gather: null pointer");
    if (!aligned(element, {key_out, value_out}) || !aligned(8, {block_table, seq_lens, out_offsets, page_starts}))
        return fail(KVFLUX_ERR_INVALID_ARGUMENT, "quant gather: misaligned array");
    if (max_blocks_per_seq == 0) return fail(KVFLUX_ERR_INVALID_ARGUMENT, "quant gather: empty table rows");
    if (num_seqs > 0x7fffffffULL || total_pages > 0x7fffffffULL)
        return fail(KVFLUX_ERR_UNSUPPORTED, "quant gather: too many pages");
    ReadParams p{};
    p.cache[0] = static_cast<const std::uint8_t*>(key_cache);
    p.cache[1] = static_cast<const std::uint8_t*>(value_cache);
    p.scales[0] = key_scales;
    p.scales[1] = value_scales;
    p.out[0] = key_out;
    p.out[1] = value_out;
    p.num_blocks = num_blocks;
    p.heads = static_cast<std::uint32_t>(num_kv_heads);
    p.block_size = static_cast<std::uint32_t>(block_size);
    p.head_size = static_cast<std::uint32_t>(head_size);
    p.table = block_table;
    p.width = max_blocks_per_seq;
    p.lens = seq_lens;
    p.offsets = out_offsets;
    p.page_starts = page_starts;
    p.num_seqs = static_cast<std::uint32_t>(num_seqs);
    const bool wide = head_size % 8 == 0 && aligned(16, {key_out, value_out}) && aligned(8, {key_cache, value_cache});
    const hipStream_t s = as_stream(stream);
    return format == KVFLUX_QUANT_E4M3 ? launch_gather_format<QuantE4m3>(p, output_dtype, wide, total_pages, s)
                                       : launch_gather_format<QuantInt8>(p, output_dtype, wide, total_pages, s);
}
