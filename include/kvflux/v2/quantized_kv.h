#pragma once
// A paged KV cache held in 8 bits, a scale for each page and kv head, and the calls
// on it: what PagedKVStorage, write_paged_kv, read_paged_kv_batch, paged_attention and
// decode_step are for caches of 16 and 32 bits. No counterpart in the reference
// (include/kvflux/v2/paged_kv_layout.h:12-40 knows FP16, BF16 and FP32). Half the memory of a
// 16-bit cache, so twice the tokens, and half the bytes of every attention.

#include "kvflux/v2/device_batch_table.h"
#include "kvflux/v2/paged_kv_storage.h"
#include "kvflux/v2/sequence_state.h"

#include <cstddef>
#include <memory>
#include <utility>
#include <vector>

namespace kvflux::v2 {

// What a value is held as: 8-bit floats (4 exponent and 3 mantissa bits, up to 448), or
// integers of -127 to 127; times the scale of its page and head, a power of two.
// E4M3 keeps small values of a page as exact as its large ones (2^-4 of each), Int8
// has the smaller error where values of a page are of one size (2^-7 of the largest, at
// worst 2^-6).
enum class QuantFormat { E4M3, Int8 };

// Bytes K[num_blocks][num_kv_heads][block_size][head_size], V of the same shape, then the
// scales of K and of V, float [num_blocks][num_kv_heads] each.
class QuantizedKVLayout {
public:
    QuantizedKVLayout(std::size_t num_blocks, std::size_t num_kv_heads, std::size_t block_size, std::size_t head_size,
                      QuantFormat format);

    std::size_t num_blocks() const noexcept { return blocks_; }
    std::size_t num_kv_heads() const noexcept { return heads_; }
    std::size_t block_size() const noexcept { return block_size_; }
    std::size_t head_size() const noexcept { return head_size_; }
    QuantFormat format() const noexcept { return format_; }
    std::size_t page_bytes() const noexcept { return page_bytes_; }       // of one cache, without its scales
    std::size_t cache_bytes() const noexcept { return cache_bytes_; }     // of K, or of V
    std::size_t scale_bytes() const noexcept { return scale_bytes_; }     // of K's scales, or of V's
    std::size_t total_bytes() const noexcept { return 2 * cache_stride_ + 2 * scale_bytes_; }
    // From K to V, a multiple of 256 bytes.
    std::size_t cache_stride() const noexcept { return cache_stride_; }

private:
    std::size_t blocks_, heads_, block_size_, head_size_;
    QuantFormat format_;
    std::size_t page_bytes_, cache_bytes_, cache_stride_, scale_bytes_;
};

class QuantizedKVStorage {
public:
    QuantizedKVStorage(PhysicalBlockPool& pool, std::size_t num_kv_heads, std::size_t head_size, QuantFormat format,
                       int device = 0);
    ~QuantizedKVStorage();
    QuantizedKVStorage(const QuantizedKVStorage&) = delete;
    QuantizedKVStorage& operator=(const QuantizedKVStorage&) = delete;

    const QuantizedKVLayout& layout() const noexcept { return layout_; }
    int device() const noexcept { return device_; }
    bool uses_pool(const BlockTable& table) const noexcept { return table.uses_pool(pool_); }
    // Device addresses (not dereferenceable on the host).
    void* key_base() const;
    void* value_base() const;
    float* key_scales() const;
    float* value_scales() const;

    // As PagedKVStorage::copy_blocks, the pages' scales with them.
    void copy_blocks(const std::vector<std::pair<PhysicalBlockHandle, PhysicalBlockHandle>>& pairs) const;

    // Library-internal: reusable device buffers for per-call metadata.
    detail::DeviceScratch& scratch() const { return *scratch_; }

private:
    PhysicalBlockPool& pool_;
    QuantizedKVLayout layout_;
    int device_;
    void* arena_ = nullptr;
    std::unique_ptr<detail::DeviceScratch> scratch_;
};

// New K and V rows: device arrays [tokens][num_kv_heads][head_size] of `dtype`, `*_stride`
// elements from one token to the next (0: the rows follow each other). They may be
// parts of one array, as a projection leaves them.
struct NewRows {
    const void* key = nullptr;
    const void* value = nullptr;
    DType dtype = DType::BFloat16;
    std::size_t key_stride = 0;
    std::size_t value_stride = 0;
};

// Quantises and writes the last new_tokens[i] tokens of sequences[i] (appended before),
// whose rows follow each other in input order. A page's scale is that of the largest
// magnitude among its tokens; where new ones raise it, the page's earlier tokens are
// rounded again (kvflux_quant_write). std::invalid_argument: a null sequence or one of
// another pool, more new tokens than tokens, as many counts as sequences not given, two
// sequences writing to the same page (fork_shared before append_tokens_cow), null, host,
// foreign or misaligned rows, a stride below a token's heads, rows overlapping the cache.
// std::length_error: a sequence whose new tokens touch 2^24 pages and more, counted for each
// head of K and V. No new tokens: no-op. Returns after completion.
void write_quantized_kv(QuantizedKVStorage& storage, const std::vector<const SequenceState*>& sequences,
                        const std::vector<std::size_t>& new_tokens, const NewRows& rows);

// Every sequence's K and V back as `dtype`, packed in input order (checks as
// read_paged_kv_batch): what the cache holds, rounded once.
void read_quantized_kv(const QuantizedKVStorage& storage, const std::vector<const SequenceState*>& sequences, DType dtype,
                       void* key_out_device, void* value_out_device);

// Batch decode, one query a sequence; contract and checks as the calls of the same name on a
// PagedKVStorage.
void paged_attention_batch(const QuantizedKVStorage& storage, const std::vector<const SequenceState*>& sequences,
                           const float* query_device, float* output_device, std::size_t query_heads);
void paged_attention_batch(const QuantizedKVStorage& storage, const DeviceBatchTable& batch, const float* query_device,
                           float* output_device, std::size_t query_heads);

// Causal attention of the last query_tokens[i] tokens of every sequence i (whole prompts, or
// their next chunks), in one launch: Q/O device FP32 [sum of query_tokens][query_heads]
// [head_size], in input order. Within 1e-5, as paged_attention's Exact; checks as there.
void paged_attention_prompts(const QuantizedKVStorage& storage, const std::vector<const SequenceState*>& sequences,
                             const std::vector<std::size_t>& query_tokens, const float* query_device,
                             float* output_device, std::size_t query_heads);

// As the calls of the same names on a PagedKVStorage (copy_on_write.h, device_batch_table.h):
// appends with copies of shared partial tails, and a whole decode step, whose new rows
// are quantised as they are written.
std::vector<TokenLocation> append_tokens_cow(const QuantizedKVStorage& storage,
                                             const std::vector<SequenceState*>& sequences);
std::vector<TokenLocation> decode_step(QuantizedKVStorage& storage, DeviceBatchTable& batch, const NewRows& rows,
                                       const float* query_device, float* output_device, std::size_t query_heads);

} // namespace kvflux::v2
