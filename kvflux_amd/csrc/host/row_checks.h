// Library-internal: grouping of a batch's rows by their shared pages, and the
// checks of projected rows, for the calls of shared_prefix.h and norm_rope_write.h.
#pragma once

#include "kvflux/v2/norm_rope_write.h"
#include "kvflux/v2/shared_prefix.h"

#include <cstddef>
#include <cstdint>
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

} // namespace kvflux::v2::detail
