// The 8-bit paged cache (quantized_kv.h): its layout and storage, and the calls whose
// metadata is built from sequences. Each call validates on the host, uploads its metadata
// once, launches through the C ABI and waits for the default stream, as the calls on
// PagedKVStorage do (paged_kv_ops.cpp); the decode step is in decode_step.cpp.
#include "kvflux/v2/quantized_kv.h"

#include "kvflux/v2/batch_block_table.h"

#include "device_runtime.h"
#include "row_checks.h"

#include <algorithm>
#include <limits>
#include <stdexcept>
#include <unordered_set>

namespace kvflux::v2 {

using detail::check;
using detail::mul_checked;

QuantizedKVLayout::QuantizedKVLayout(std::size_t num_blocks, std::size_t num_kv_heads, std::size_t block_size,
                                     std::size_t head_size, QuantFormat format)
    : blocks_(num_blocks), heads_(num_kv_heads), block_size_(block_size), head_size_(head_size), format_(format) {
    if (num_blocks == 0 || num_kv_heads == 0 || block_size == 0 || head_size == 0) {
        throw std::invalid_argument("quantised KV layout dimensions must be positive");
    }
    (void)detail::abi_format(format);
    constexpr const char* too_large = "quantised KV layout size overflow";
    page_bytes_ = mul_checked(mul_checked(num_kv_heads, block_size, too_large), head_size, too_large);
    cache_bytes_ = mul_checked(num_blocks, page_bytes_, too_large);
    scale_bytes_ = mul_checked(mul_checked(num_blocks, num_kv_heads, too_large), sizeof(float), too_large);
    if (cache_bytes_ > std::numeric_limits<std::size_t>::max() / 4 ||
        scale_bytes_ > std::numeric_limits<std::size_t>::max() / 8) {
        throw std::overflow_error(too_large);
    }
    cache_stride_ = (cache_bytes_ + 255) & ~std::size_t{255};
}

QuantizedKVStorage::QuantizedKVStorage(PhysicalBlockPool& pool, std::size_t num_kv_heads, std::size_t head_size,
                                       QuantFormat format, int device)
    : pool_(pool), layout_(pool.capacity(), num_kv_heads, pool.block_size(), head_size, format), device_(device),
      scratch_(std::make_unique<detail::DeviceScratch>()) {
    int count = 0;
    check(kvflux_device_count(&count), "count devices");
    if (device < 0 || device >= count) throw std::invalid_argument("invalid GPU device");
    detail::DeviceGuard guard(device_);
    check(kvflux_device_malloc(&arena_, layout_.total_bytes()), "allocate quantised KV arena");
}

QuantizedKVStorage::~QuantizedKVStorage() {
    // Scratch buffers and the arena belong to device_; free them there.
    int previous = 0;
    const bool switched = kvflux_get_device(&previous) == KVFLUX_OK &&
                          (previous == device_ || kvflux_set_device(device_) == KVFLUX_OK);
    scratch_.reset();
    if (arena_) (void)kvflux_device_free(arena_);
    if (switched && previous != device_) (void)kvflux_set_device(previous);
}

void* QuantizedKVStorage::key_base() const { return arena_; }
void* QuantizedKVStorage::value_base() const { return static_cast<unsigned char*>(arena_) + layout_.cache_stride(); }
float* QuantizedKVStorage::key_scales() const {
    return reinterpret_cast<float*>(static_cast<unsigned char*>(arena_) + 2 * layout_.cache_stride());
}
float* QuantizedKVStorage::value_scales() const {
    return reinterpret_cast<float*>(reinterpret_cast<unsigned char*>(key_scales()) + layout_.scale_bytes());
}

void QuantizedKVStorage::copy_blocks(
    const std::vector<std::pair<PhysicalBlockHandle, PhysicalBlockHandle>>& pairs) const {
    if (pairs.empty()) return;
    std::vector<std::uint64_t> ids;
    ids.reserve(2 * pairs.size());
    std::unordered_set<PhysicalBlockID> destinations;
    for (const auto& [source, destination] : pairs) {
        const auto from = pool_.id(source);
        const auto to = pool_.id(destination);
        if (from == to || pool_.ref_count(destination) != 1 || pool_.is_published(destination) ||
            !destinations.insert(to).second) {
            throw std::invalid_argument("copy destination must be a private, unpublished page");
        }
        ids.push_back(from);
        ids.push_back(to);
    }
    for (std::size_t i = 0; i < ids.size(); i += 2) {
        if (destinations.count(ids[i])) {
            throw std::invalid_argument("a copy source is also a destination of the batch");
        }
    }
    detail::DeviceGuard guard(device_);
    const auto dev = scratch_->upload({{ids.data(), ids.size() * sizeof(std::uint64_t)}});
    try {
        detail::copy_quantized_pages(*this, dev[0], pairs.size());
        check(kvflux_stream_synchronize(nullptr), "synchronize KV page copy");
    } catch (...) {
        (void)kvflux_stream_synchronize(nullptr);
        throw;
    }
}

namespace detail {

int abi_format(QuantFormat format) {
    switch (format) {
    case QuantFormat::E4M3: return KVFLUX_QUANT_E4M3;
    case QuantFormat::Int8: return KVFLUX_QUANT_INT8;
    }
    throw std::invalid_argument("unsupported quantised KV format");
}

std::pair<std::size_t, std::size_t> check_new_rows(const QuantizedKVStorage& storage, const NewRows& rows,
                                                   std::size_t tokens) {
    constexpr const char* too_large = "new rows size overflow";
    const auto& layout = storage.layout();
    const std::size_t element = abi_dtype(rows.dtype) == KVFLUX_DTYPE_F32 ? 4 : 2;
    if (!rows.key || !rows.value) throw std::invalid_argument("K_new and V_new device pointers are required");
    const auto row = mul_checked(layout.num_kv_heads(), layout.head_size(), too_large);
    const std::size_t strides[2] = {rows.key_stride ? rows.key_stride : row, rows.value_stride ? rows.value_stride : row};
    const void* const data[2] = {rows.key, rows.value};
    const char* const names[2] = {"K_new", "V_new"};
    for (int i = 0; i < 2; ++i) {
        if (strides[i] < row) throw std::invalid_argument("a stride is shorter than a token's heads");
        const auto before = mul_checked(tokens - 1, strides[i], too_large);
        if (before > std::numeric_limits<std::size_t>::max() - row) throw std::overflow_error(too_large);
        const auto bytes = mul_checked(before + row, element, too_large);
        require_device_pointer(data[i], storage.device(), names[i]);
        if (reinterpret_cast<std::uintptr_t>(data[i]) % element != 0) {
            throw std::invalid_argument(std::string("misaligned ") + names[i]);
        }
        if (overlaps(data[i], bytes, storage.key_base(), layout.total_bytes())) {
            throw std::invalid_argument(std::string(names[i]) + " must not overlap the KV cache");
        }
    }
    return {strides[0], strides[1]};
}

void copy_quantized_pages(const QuantizedKVStorage& storage, const std::uint64_t* pairs, std::size_t count) {
    const auto& layout = storage.layout();
    check(kvflux_copy_pages(storage.key_base(), storage.value_base(), layout.num_blocks(), layout.page_bytes(), pairs,
                            count, nullptr),
          "copy KV pages");
    check(kvflux_copy_pages(storage.key_scales(), storage.value_scales(), layout.num_blocks(),
                            layout.num_kv_heads() * sizeof(float), pairs, count, nullptr),
          "copy KV scales");
}

// What a write counts in 24 bits: pages that a launch's sequences may touch, for each head of K and V.
std::size_t pages_of_a_launch(const QuantizedKVStorage& storage) {
    constexpr std::size_t most = (std::size_t{1} << 24) - 1;
    return most / (2 * storage.layout().num_kv_heads());
}

void enqueue_quantized_tails(const QuantizedKVStorage& storage, const NewRows& rows,
                             const std::pair<std::size_t, std::size_t>& strides, const std::uint64_t* table,
                             std::size_t width, const std::uint64_t* lengths, std::size_t count) {
    const auto& layout = storage.layout();
    const std::size_t element = abi_dtype(rows.dtype) == KVFLUX_DTYPE_F32 ? 4 : 2;
    const std::size_t at_once = std::max<std::size_t>(1, pages_of_a_launch(storage));  // none: refused below
    for (std::size_t first = 0; first < count; first += at_once) {
        check(kvflux_quant_write_tail(storage.key_base(), storage.value_base(), storage.key_scales(),
                                      storage.value_scales(), layout.num_blocks(), layout.num_kv_heads(),
                                      layout.block_size(), layout.head_size(), abi_format(layout.format()),
                                      static_cast<const unsigned char*>(rows.key) + first * strides.first * element,
                                      static_cast<const unsigned char*>(rows.value) + first * strides.second * element,
                                      abi_dtype(rows.dtype), strides.first, strides.second, table + first * width,
                                      width, lengths + first, std::min(count - first, at_once), nullptr),
              "quantised KV tail write kernel launch");
    }
}

std::pair<void*, std::size_t> quantized_decode_workspace(const QuantizedKVStorage& storage, std::size_t max_len,
                                                         std::size_t rows, std::size_t query_heads) {
    const auto& layout = storage.layout();
    std::size_t bytes = 0;
    check(kvflux_quant_attention_workspace_size(rows, max_len, layout.num_kv_heads(), query_heads, layout.block_size(),
                                                layout.head_size(), &bytes),
          "attention workspace size");
    return {bytes ? storage.scratch().workspace.reserve(bytes) : nullptr, bytes};
}

void enqueue_quantized_decode(const QuantizedKVStorage& storage, const std::uint64_t* table, std::size_t width,
                              const std::uint64_t* lengths, std::size_t max_len, std::size_t rows, const float* query,
                              float* output, std::size_t query_heads) {
    const auto& layout = storage.layout();
    const auto [workspace, bytes] = quantized_decode_workspace(storage, max_len, rows, query_heads);
    check(kvflux_quant_attention(storage.key_base(), storage.value_base(), storage.key_scales(), storage.value_scales(),
                                 layout.num_blocks(), layout.num_kv_heads(), layout.block_size(), layout.head_size(),
                                 abi_format(layout.format()), table, width, lengths, max_len, rows, query_heads, query,
                                 output, workspace, bytes, nullptr),
          "quantised attention batch kernel launch");
}

} // namespace detail

namespace {

// Table, lengths and row offsets of a batch of sequences on the device, and what bounds them.
struct Batch {
    BatchBlockTable table;
    std::vector<std::uint64_t> lengths, counts, offsets;
    std::size_t total = 0, most = 0, longest = 0;  // of counts; of lengths
};

// `counts`: tokens of each sequence that the call is about (its last ones).
Batch collect(const QuantizedKVStorage& storage, const std::vector<const SequenceState*>& sequences,
              const std::vector<std::size_t>& counts, const char* what) {
    if (counts.size() != sequences.size()) throw std::invalid_argument("as many token counts as sequences are required");
    const auto& layout = storage.layout();
    Batch b;
    b.table = build_batch_block_table(sequences);
    for (std::size_t r = 0; r < sequences.size(); ++r) {
        if (!storage.uses_pool(sequences[r]->block_table()) || sequences[r]->block_size() != layout.block_size()) {
            throw std::invalid_argument("sequence and KV storage must use one physical pool");
        }
        const std::size_t length = b.table.sequence_lengths()[r];
        if (counts[r] > length) throw std::invalid_argument(std::string("more ") + what + " than tokens of a sequence");
        b.lengths.push_back(length);
        b.counts.push_back(counts[r]);
        b.offsets.push_back(b.total);
        if (counts[r] > std::numeric_limits<std::size_t>::max() - b.total) throw std::overflow_error("batch size overflow");
        b.total += counts[r];
        b.most = std::max(b.most, counts[r]);
        b.longest = std::max(b.longest, length);
    }
    for (const auto block : b.table.block_table()) {
        if (block != BatchBlockTable::invalid_block() && block >= layout.num_blocks()) {
            throw std::out_of_range("KV block out of range");
        }
    }
    return b;
}

std::size_t q_bytes(const QuantizedKVStorage& storage, std::size_t rows, std::size_t query_heads) {
    const auto& layout = storage.layout();
    if (query_heads == 0 || query_heads % layout.num_kv_heads() != 0) {
        throw std::invalid_argument("invalid attention head count");
    }
    constexpr const char* too_large = "paged attention size overflow";
    return mul_checked(mul_checked(mul_checked(rows, query_heads, too_large), layout.head_size(), too_large), sizeof(float),
                       too_large);
}

std::vector<std::size_t> all_tokens(const std::vector<const SequenceState*>& sequences) {
    std::vector<std::size_t> counts;
    for (const auto* s : sequences) counts.push_back(s ? s->num_tokens() : 0);
    return counts;
}

} // namespace

void write_quantized_kv(QuantizedKVStorage& storage, const std::vector<const SequenceState*>& sequences,
                        const std::vector<std::size_t>& new_tokens, const NewRows& rows) {
    const auto& layout = storage.layout();
    const Batch b = collect(storage, sequences, new_tokens, "new tokens");
    if (b.total == 0) return;
    std::unordered_set<PhysicalBlockID> touched;
    const auto width = b.table.max_blocks_per_sequence();
    for (std::size_t r = 0; r < sequences.size(); ++r) {
        if (b.counts[r] == 0) continue;
        for (std::size_t page = (b.lengths[r] - b.counts[r]) / layout.block_size(); page * layout.block_size() < b.lengths[r]; ++page) {
            if (!touched.insert(b.table.block_table()[r * width + page]).second) {
                throw std::invalid_argument("two sequences write to one page");
            }
        }
    }
    // A launch has room for as many pages of each of its sequences as the longest may touch: runs of
    // sequences that fit one, so that a long prompt beside many single tokens does not count for each.
    struct Run {
        std::size_t first, count, most;
    };
    std::vector<Run> runs;
    const auto room = detail::pages_of_a_launch(storage);
    const auto pages = [&](std::size_t tokens) { return (tokens + layout.block_size() - 2) / layout.block_size() + 1; };
    for (std::size_t r = 0; r < sequences.size(); ++r) {
        if (b.counts[r] == 0) continue;
        if (pages(b.counts[r]) > room) throw std::length_error("too many new tokens of a sequence");
        if (!runs.empty()) {
            auto& last = runs.back();
            const std::size_t most = std::max<std::size_t>(last.most, b.counts[r]), count = r + 1 - last.first;
            if (pages(most) <= room / count) {
                last.count = count;
                last.most = most;
                continue;
            }
        }
        runs.push_back({r, 1, b.counts[r]});
    }
    detail::DeviceGuard guard(storage.device());
    const auto strides = detail::check_new_rows(storage, rows, b.total);
    const auto dev = storage.scratch().upload({{b.table.block_table().data(), b.table.block_table().size() * 8},
                                               {b.lengths.data(), b.lengths.size() * 8},
                                               {b.counts.data(), b.counts.size() * 8},
                                               {b.offsets.data(), b.offsets.size() * 8}});
    for (const auto& run : runs) {
        check(kvflux_quant_write(storage.key_base(), storage.value_base(), storage.key_scales(), storage.value_scales(),
                                 layout.num_blocks(), layout.num_kv_heads(), layout.block_size(), layout.head_size(),
                                 detail::abi_format(layout.format()), rows.key, rows.value, detail::abi_dtype(rows.dtype),
                                 strides.first, strides.second, dev[0] + run.first * width, width, dev[1] + run.first,
                                 dev[2] + run.first, dev[3] + run.first, run.count, run.most, nullptr),
              "quantised KV write kernel launch");
    }
    check(kvflux_stream_synchronize(nullptr), "quantised KV write synchronize");
}

void read_quantized_kv(const QuantizedKVStorage& storage, const std::vector<const SequenceState*>& sequences, DType dtype,
                       void* key_out_device, void* value_out_device) {
    const auto& layout = storage.layout();
    const Batch b = collect(storage, sequences, all_tokens(sequences), "tokens");
    const std::size_t element = detail::abi_dtype(dtype) == KVFLUX_DTYPE_F32 ? 4 : 2;
    if (b.total == 0) return;
    if (!key_out_device || !value_out_device) {
        throw std::invalid_argument("K and V output device pointers are required");
    }
    constexpr const char* too_large = "quantised KV read size overflow";
    const auto out_bytes = mul_checked(mul_checked(mul_checked(b.total, layout.num_kv_heads(), too_large), layout.head_size(), too_large),
                                       element, too_large);
    detail::DeviceGuard guard(storage.device());
    detail::require_device_pointer(key_out_device, storage.device(), "K_out");
    detail::require_device_pointer(value_out_device, storage.device(), "V_out");
    if (detail::overlaps(key_out_device, out_bytes, value_out_device, out_bytes) ||
        detail::overlaps(key_out_device, out_bytes, storage.key_base(), layout.total_bytes()) ||
        detail::overlaps(value_out_device, out_bytes, storage.key_base(), layout.total_bytes())) {
        throw std::invalid_argument("KV read outputs must not overlap each other or the cache");
    }
    std::vector<std::uint64_t> page_starts;
    std::uint64_t pages = 0;
    for (const auto length : b.lengths) {
        page_starts.push_back(pages);
        pages += (length + layout.block_size() - 1) / layout.block_size();
    }
    const auto dev = storage.scratch().upload({{b.table.block_table().data(), b.table.block_table().size() * 8},
                                               {b.lengths.data(), b.lengths.size() * 8},
                                               {b.offsets.data(), b.offsets.size() * 8},
                                               {page_starts.data(), page_starts.size() * 8}});
    check(kvflux_quant_gather(storage.key_base(), storage.value_base(), storage.key_scales(), storage.value_scales(),
                              layout.num_blocks(), layout.num_kv_heads(), layout.block_size(), layout.head_size(),
                              detail::abi_format(layout.format()), dev[0], b.table.max_blocks_per_sequence(), dev[1],
                              dev[2], dev[3], sequences.size(), pages, key_out_device, value_out_device,
                              detail::abi_dtype(dtype), nullptr),
          "quantised KV read kernel launch");
    check(kvflux_stream_synchronize(nullptr), "quantised KV read synchronize");
}

void paged_attention_batch(const QuantizedKVStorage& storage, const std::vector<const SequenceState*>& sequences,
                           const float* query_device, float* output_device, std::size_t query_heads) {
    const auto tensor_bytes = q_bytes(storage, sequences.size(), query_heads);
    const Batch b = collect(storage, sequences, all_tokens(sequences), "tokens");
    if (std::find(b.lengths.begin(), b.lengths.end(), 0) != b.lengths.end()) {
        throw std::invalid_argument("invalid batch attention sequence");
    }
    if (sequences.empty()) return;
    if (!query_device || !output_device) {
        throw std::invalid_argument("Q and attention output device pointers are required");
    }
    detail::DeviceGuard guard(storage.device());
    detail::validate_q_o(storage, query_device, output_device, tensor_bytes);
    const auto dev = storage.scratch().upload({{b.table.block_table().data(), b.table.block_table().size() * 8},
                                               {b.lengths.data(), b.lengths.size() * 8}});
    detail::enqueue_quantized_decode(storage, dev[0], b.table.max_blocks_per_sequence(), dev[1], b.longest,
                                     sequences.size(), query_device, output_device, query_heads);
    check(kvflux_stream_synchronize(nullptr), "paged attention batch synchronize");
}

void paged_attention_prompts(const QuantizedKVStorage& storage, const std::vector<const SequenceState*>& sequences,
                             const std::vector<std::size_t>& query_tokens, const float* query_device,
                             float* output_device, std::size_t query_heads) {
    const auto& layout = storage.layout();
    const Batch b = collect(storage, sequences, query_tokens, "queries");
    const auto tensor_bytes = q_bytes(storage, b.total, query_heads);
    if (b.total == 0) return;
    if (!query_device || !output_device) {
        throw std::invalid_argument("Q and attention output device pointers are required");
    }
    detail::DeviceGuard guard(storage.device());
    detail::validate_q_o(storage, query_device, output_device, tensor_bytes);
    std::size_t bytes = 0;
    check(kvflux_quant_prefill_workspace_size(sequences.size(), b.most, b.longest, layout.num_kv_heads(), query_heads,
                                              layout.block_size(), layout.head_size(), &bytes),
          "prefill workspace size");
    void* const workspace = bytes ? storage.scratch().workspace.reserve(bytes) : nullptr;
    const auto dev = storage.scratch().upload({{b.table.block_table().data(), b.table.block_table().size() * 8},
                                               {b.lengths.data(), b.lengths.size() * 8},
                                               {b.counts.data(), b.counts.size() * 8},
                                               {b.offsets.data(), b.offsets.size() * 8}});
    check(kvflux_quant_prefill(storage.key_base(), storage.value_base(), storage.key_scales(), storage.value_scales(),
                               layout.num_blocks(), layout.num_kv_heads(), layout.block_size(), layout.head_size(),
                               detail::abi_format(layout.format()), dev[0], b.table.max_blocks_per_sequence(), dev[1],
                               dev[2], dev[3], sequences.size(), b.most, b.longest, query_heads, query_device,
                               output_device, workspace, bytes, nullptr),
          "quantised prefill kernel launch");
    check(kvflux_stream_synchronize(nullptr), "quantised prefill synchronize");
}

} // namespace kvflux::v2
