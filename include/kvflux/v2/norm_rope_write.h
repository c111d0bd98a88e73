#pragma once
// From a projection's output to the attention's inputs in one pass: RMS norms
// of queries and keys for each head, the position rotation, K and V into their
// pages. No counterpart in the reference, whose write_paged_kv
// (src/v2/paged_kv_write.cu:101-139) takes finished K/V rows.

#include "kvflux/kv_layout.h"
#include "kvflux/v2/paged_kv_storage.h"

#include <cstddef>
#include <cstdint>
#include <vector>

namespace kvflux::v2 {

// New tokens as a projection leaves them: device arrays of `dtype` (any of the
// three, whatever the storage's), queries [tokens][query_heads][head_size], keys
// and values [tokens][num_kv_heads][head_size], with `*_stride` elements from one
// token to the next (0: the rows follow each other). The three may be parts of
// one array.
struct ProjectedRows {
    const void* query = nullptr;
    const void* key = nullptr;
    const void* value = nullptr;
    DType dtype = DType::BFloat16;
    std::size_t query_stride = 0;
    std::size_t key_stride = 0;
    std::size_t value_stride = 0;
};

// What is done to query and key rows. query_norm, key_norm: device float
// [head_size], the RMS norm's weights (null: no norm). inv_freq: device double
// [rotary_dim / 2], the angle of a pair for each position; rotary_dim 0: no
// rotation. Pairs are dims (j, j + rotary_dim / 2), or (2j, 2j + 1) when interleaved.
struct NormRope {
    const float* query_norm = nullptr;
    const float* key_norm = nullptr;
    float eps = 1e-6f;
    const double* inv_freq = nullptr;
    std::size_t rotary_dim = 0;
    bool interleaved = false;
};

// Token n, at positions[n], goes to slot_mapping[n]; its query to query_out
// (device float [tokens][query_heads][head_size], as the attention takes it).
// Checks and exceptions as write_paged_kv; positions and slots differing in
// number, a position of 2^53 or more, a query head count that is no multiple of the kv heads, a stride below
// a token's heads, an odd rotary_dim or one above head_size, a negative eps,
// misaligned arrays, or query_out overlapping the inputs or the cache:
// std::invalid_argument. A head_size above 512, or 2^26 heads of all tokens:
// std::runtime_error. Empty mapping: no-op. Returns after completion.
void norm_rope_write(PagedKVStorage& storage, const ProjectedRows& rows, const NormRope& form,
                     std::size_t query_heads, const std::vector<std::uint64_t>& positions,
                     const SlotMapping& slot_mapping, float* query_out);

} // namespace kvflux::v2
