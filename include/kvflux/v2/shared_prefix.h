#pragma once
// Decode attention that computes shared prefixes once. The reference shares
// prefix pages between requests (src/v2/prefix_cache.cpp:7-57,
// SequenceState::fork_shared) but its batch attention reads them for every row
// (src/v2/paged_attention.cu:130-153).

#include "kvflux/v2/device_batch_table.h"
#include "kvflux/v2/norm_rope_write.h"
#include "kvflux/v2/paged_kv_storage.h"
#include "kvflux/v2/sequence_state.h"

#include <cstddef>
#include <cstdint>
#include <vector>

namespace kvflux::v2 {

// Groups of neighbouring rows of a batch: group g is rows starts[g] ..
// starts[g + 1], which have the pages of their first prefixes[g] tokens in common
// (whole pages). Empty: no two neighbouring rows share a page.
struct SharedPrefixGroups {
    std::vector<std::uint64_t> starts;    // groups + 1 entries, or none
    std::vector<std::uint64_t> prefixes;  // groups entries
    std::size_t groups() const noexcept { return prefixes.size(); }
};

// The grouping of the rows, in their order, that shares the most tokens. Rows
// that share pages should be neighbours. Null sequences, or ones of several pools
// or block sizes: std::invalid_argument.
SharedPrefixGroups find_shared_prefixes(const std::vector<const SequenceState*>& sequences);

// paged_attention_batch with every group's prefix computed once (see
// kvflux_paged_attention_shared); groups from find_shared_prefixes. Same contract:
// FP32 Q and O, Exact, the same exceptions. Results agree with
// paged_attention_batch to 1e-5; where sharing, as the groups really share, does not
// pay they are its bits.
void paged_attention_batch_shared(const PagedKVStorage& storage,
                                  const std::vector<const SequenceState*>& sequences,
                                  const float* query_device, float* output_device,
                                  std::size_t query_heads);

// The same over a refreshed device table, whose groups are found at the first
// such call that they could pay for and stay: rows only ever append pages behind
// the whole ones.
void paged_attention_batch_shared(const PagedKVStorage& storage, DeviceBatchTable& batch,
                                  const float* query_device, float* output_device,
                                  std::size_t query_heads);

// One decode step from the projection's output: appends one token to each
// sequence of `batch` (copy-on-write as decode_step), norms, rotates and writes
// row r of `rows` at its new position, and computes each row's attention, shared
// prefixes once. The queries as the attention took them are left in
// query_device ([rows][query_heads][head_size], as output_device). One
// synchronisation. Exceptions and what a failure leaves: as decode_step.
std::vector<TokenLocation> decode_step_projected(PagedKVStorage& storage, DeviceBatchTable& batch,
                                                 const ProjectedRows& rows, const NormRope& form,
                                                 float* query_device, float* output_device,
                                                 std::size_t query_heads);

} // namespace kvflux::v2
