// Library-internal: grouping of a batch's rows by their shared pages, the checks of
// projected and of new rows, and what the calls on an 8-bit cache share, for
// shared_prefix.h, norm_rope_write.h and quantized_kv.h.
#pragma once

#include "kvflux/v2/norm_rope_write.h"
#include "kvflux/v2/quantized_kv.h"
#include "kvflux/v2/shared_prefix.h"

#include <cstddef>
#include <cstdint>
#include <utility>
#include <vector>

namespace kvflux::v2::detail {

// A row's page ids, and how many of them are full.
struct RowPages {
    const std::uint64_t* ids;
    std::size_t whole;
};

// The grouping of neighbouring rows that shares the most tokens.
SharedPrefixGroups group_rows(const std::vector<RowPages>& rows, std::size_t block_size);

// Tokens that the groups' further rows need not have read again: the sum of
// (rows - 1) * prefix.
std::uint64_t shared_tokens(const SharedPrefixGroups& groups);

// Whether the shared attention serves a batch better than the ordinary one; and
// whether it could, whatever the rows (one at least) share.
bool sharing_pays(const PagedKVStorage& storage, std::size_t rows, std::size_t kv_len, std::size_t query_heads,
                  std::size_t groups, std::uint64_t shared_tokens);
bool sharing_could_pay(const PagedKVStorage& storage, std::size_t rows, std::size_t kv_len, std::size_t query_heads);

// Elements from one token of a projection to the next.
struct ProjectionStrides {
    std::size_t query, key, value;
};

// Throws std::invalid_argument (std::overflow_error for sizes) unless `rows` can
// be normed, rotated and written; the current device is the storage's.
ProjectionStrides check_projection(const PagedKVStorage& storage, const ProjectedRows& rows, const NormRope& form,
                                   std::size_t query_heads, std::size_t tokens, const float* query_out);

// kvflux_quant_format of a format.
int abi_format(QuantFormat format);

// Strides of K and V rows (never 0); throws std::invalid_argument (std::overflow_error for
// sizes) unless `tokens` such rows can be written. The current device is the storage's.
std::pair<std::size_t, std::size_t> check_new_rows(const QuantizedKVStorage& storage, const NewRows& rows,
                                                   std::size_t tokens);

// Enqueues the copies of {source, destination} pages (a device array) and of their scales.
void copy_quantized_pages(const QuantizedKVStorage& storage, const std::uint64_t* pairs, std::size_t count);

// Enqueues the writes of one new token for each of `count` rows of a device table.
void enqueue_quantized_tails(const QuantizedKVStorage& storage, const NewRows& rows,
                             const std::pair<std::size_t, std::size_t>& strides, const std::uint64_t* table,
                             std::size_t width, const std::uint64_t* lengths, std::size_t count);

// Workspace of the decode attention of `rows` rows of at most max_len tokens, and its bytes;
// null where none is needed. Throws for shapes that the attention refuses.
std::pair<void*, std::size_t> quantized_decode_workspace(const QuantizedKVStorage& storage, std::size_t max_len,
                                                         std::size_t rows, std::size_t query_heads);

// Enqueues the decode attention of `rows` rows of a device table.
void enqueue_quantized_decode(const QuantizedKVStorage& storage, const std::uint64_t* table, std::size_t width,
                              const std::uint64_t* lengths, std::size_t max_len, std::size_t rows, const float* query,
                              float* output, std::size_t query_heads);

} // namespace kvflux::v2::detail
