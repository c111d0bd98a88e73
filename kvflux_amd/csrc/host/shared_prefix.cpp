// Shared prefixes of a decode batch: finding them, and the attention over a list
// of sequences that computes each once (shared_prefix.h).
#include "kvflux/v2/shared_prefix.h"

#include "kvflux/v2/batch_block_table.h"

#include "device_runtime.h"
#include "row_checks.h"

#include <algorithm>
#include <stdexcept>

namespace kvflux::v2 {
namespace detail {

SharedPrefixGroups group_rows(const std::vector<RowPages>& rows, std::size_t block_size) {
    const std::size_t n = rows.size();
    // common[r]: whole pages that rows r and r + 1 start with. The rows of a
    // segment have the least of theirs in common.
    std::vector<std::size_t> common(n, 0);
    for (std::size_t r = 0; r + 1 < n; ++r) {
        const std::size_t most = std::min(rows[r].whole, rows[r + 1].whole);
        std::size_t k = 0;
        while (k < most && rows[r].ids[k] == rows[r + 1].ids[k]) ++k;
        common[r] = k;
    }
    // A cut between two rows of a run of equal `common` gains nothing over one at the
    // run's end: moved by a row, one segment wins what it shares and the other loses
    // what it does, until one of them is past the run. So segments start only next to
    // where `common` changes: the work grows with those places, not with the rows
    // (2048 rows behind one prefix: 1.1 ms otherwise).
    std::vector<std::size_t> at{0};
    for (std::size_t r = 1; r < n; ++r) {
        const bool inside = r >= 2 && r + 1 < n && common[r - 2] == common[r - 1] && common[r - 1] == common[r];
        if (!inside) at.push_back(r);
    }
    if (n != 0) at.push_back(n);
    // best[i]: pages not computed again in rows [0, at[i]) under their best grouping,
    // whose last segment starts at at[from[i]]. A row that shares nothing with the one
    // before it starts a segment, so a segment never reaches across such a place.
    std::vector<std::size_t> best(at.size(), 0), from(at.size(), 0);
    for (std::size_t end = 1; end < at.size(); ++end) {
        best[end] = best[end - 1];
        from[end] = end - 1;
        std::size_t least = static_cast<std::size_t>(-1);
        for (std::size_t begin = end; begin-- > 0;) {
            // The rows at[begin] .. at[begin + 1] join: what they have in common, and
            // with the rows behind them.
            if (at[begin] + 1 < at[begin + 1]) least = std::min(least, common[at[begin]]);
            if (begin + 1 != end) least = std::min(least, common[at[begin + 1] - 1]);
            if (least == 0) break;
            const std::size_t rows_saved = at[end] - at[begin] - 1;
            const std::size_t saved = best[begin] + (rows_saved != 0 ? rows_saved * least : 0);
            if (saved > best[end]) {
                best[end] = saved;
                from[end] = begin;
            }
        }
    }
    SharedPrefixGroups out;
    if (best.back() == 0) return out;
    std::vector<std::size_t> cuts;
    for (std::size_t i = at.size() - 1; i != 0; i = from[i]) cuts.push_back(at[from[i]]);
    std::reverse(cuts.begin(), cuts.end());
    for (std::size_t g = 0; g < cuts.size(); ++g) {
        const std::size_t begin = cuts[g], end = g + 1 < cuts.size() ? cuts[g + 1] : n;
        std::size_t least = end - begin > 1 ? static_cast<std::size_t>(-1) : 0;
        for (std::size_t r = begin; r + 1 < end; ++r) least = std::min(least, common[r]);
        // Rows that share nothing are one group without a prefix.
        if (least == 0 && !out.prefixes.empty() && out.prefixes.back() == 0) continue;
        out.starts.push_back(begin);
        out.prefixes.push_back(least * block_size);
    }
    out.starts.push_back(n);
    return out;
}

std::uint64_t shared_tokens(const SharedPrefixGroups& groups) {
    std::uint64_t sum = 0;
    for (std::size_t g = 0; g < groups.groups(); ++g)
        sum += (groups.starts[g + 1] - groups.starts[g] - 1) * groups.prefixes[g];
    return sum;
}

bool sharing_pays(const PagedKVStorage& storage, std::size_t rows, std::size_t kv_len, std::size_t query_heads,
                  std::size_t groups, std::uint64_t shared_tokens) {
    const auto& layout = storage.layout();
    int pays = 0;
    check(kvflux_paged_attention_shared_pays(rows, kv_len, layout.num_kv_heads(), query_heads, layout.block_size(),
                                             layout.head_size(), abi_dtype(layout.dtype()), groups, shared_tokens,
                                             &pays),
          "shared attention");
    return pays != 0;
}

bool sharing_could_pay(const PagedKVStorage& storage, std::size_t rows, std::size_t kv_len, std::size_t query_heads) {
    std::uint64_t most = 0;  // one group of all rows that is all prefix; an overflow is past what the kernel takes
    return !__builtin_mul_overflow(static_cast<std::uint64_t>(rows - 1), static_cast<std::uint64_t>(kv_len), &most) &&
           sharing_pays(storage, rows, kv_len, query_heads, 1, most);
}

} // namespace detail

SharedPrefixGroups find_shared_prefixes(const std::vector<const SequenceState*>& sequences) {
    std::vector<std::vector<PhysicalBlockID>> ids(sequences.size());
    std::vector<detail::RowPages> rows(sequences.size());
    static_assert(sizeof(PhysicalBlockID) == sizeof(std::uint64_t), "page ids are 64-bit");
    for (std::size_t r = 0; r < sequences.size(); ++r) {
        const SequenceState* s = sequences[r];
        if (!s) throw std::invalid_argument("null sequence");
        if (s->block_size() != sequences[0]->block_size() ||
            &s->block_table().pool() != &sequences[0]->block_table().pool()) {
            throw std::invalid_argument("shared prefixes need sequences of one physical pool");
        }
        ids[r].resize(s->num_allocated_blocks());
        s->physical_block_ids(ids[r].data());
        rows[r] = {reinterpret_cast<const std::uint64_t*>(ids[r].data()), s->num_tokens() / s->block_size()};
    }
    return detail::group_rows(rows, sequences.empty() ? 1 : sequences[0]->block_size());
}

void paged_attention_batch_shared(const PagedKVStorage& storage, const std::vector<const SequenceState*>& sequences,
                                  const float* query_device, float* output_device, std::size_t query_heads) {
    const auto& layout = storage.layout();
    if (query_heads == 0 || query_heads % layout.num_kv_heads() != 0) {
        throw std::invalid_argument("invalid batch attention head count");
    }
    const auto batch = build_batch_block_table(sequences);
    for (std::size_t r = 0; r < sequences.size(); ++r) {
        if (!storage.uses_pool(sequences[r]->block_table()) ||
            sequences[r]->block_size() != layout.block_size() || batch.sequence_lengths()[r] == 0) {
            throw std::invalid_argument("invalid batch attention sequence");
        }
    }
    for (const auto block : batch.block_table()) {
        if (block != BatchBlockTable::invalid_block() && block >= layout.num_blocks()) {
            throw std::out_of_range("batch attention block out of range");
        }
    }
    const auto elements = detail::mul_checked(
        detail::mul_checked(sequences.size(), query_heads, "paged attention size overflow"), layout.head_size(),
        "paged attention size overflow");
    const auto tensor_bytes = detail::mul_checked(elements, sizeof(float), "paged attention size overflow");
    if (sequences.empty()) return;
    if (!query_device || !output_device) {
        throw std::invalid_argument("Q and attention output device pointers are required");
    }
    const auto table_bytes = detail::mul_checked(batch.block_table().size(), sizeof(PhysicalBlockID),
                                                 "paged attention size overflow");
    const std::vector<std::uint64_t> lengths(batch.sequence_lengths().begin(), batch.sequence_lengths().end());
    const auto max_len = *std::max_element(lengths.begin(), lengths.end());
    SharedPrefixGroups groups;
    if (detail::sharing_could_pay(storage, sequences.size(), max_len, query_heads)) {
        std::vector<detail::RowPages> rows(sequences.size());
        for (std::size_t r = 0; r < rows.size(); ++r) {
            rows[r] = {reinterpret_cast<const std::uint64_t*>(batch.block_table().data()) + r * batch.max_blocks_per_sequence(),
                       lengths[r] / layout.block_size()};
        }
        groups = detail::group_rows(rows, layout.block_size());
    }
    const bool pays = detail::sharing_pays(storage, sequences.size(), max_len, query_heads, groups.groups(),
                                           detail::shared_tokens(groups));
    detail::DeviceGuard guard(storage.device());
    detail::validate_q_o(storage, query_device, output_device, tensor_bytes);
    const auto dev = storage.scratch().upload({{batch.block_table().data(), table_bytes},
                                               {lengths.data(), lengths.size() * 8},
                                               {groups.starts.data(), groups.starts.size() * 8},
                                               {groups.prefixes.data(), groups.prefixes.size() * 8}});
    std::size_t ws_bytes = 0;
    if (pays) {
        const auto most = *std::max_element(groups.prefixes.begin(), groups.prefixes.end());
        void* ws = detail::shared_attention_workspace(storage, sequences.size(), max_len, query_heads, groups.groups(),
                                                      &ws_bytes);
        detail::check(kvflux_paged_attention_shared(
                          storage.key_base(), storage.value_base(), layout.num_blocks(), layout.num_kv_heads(),
                          layout.block_size(), layout.head_size(), detail::abi_dtype(layout.dtype()), dev[0],
                          batch.max_blocks_per_sequence(), dev[1], max_len, sequences.size(), query_heads, dev[2],
                          dev[3], groups.groups(), most, query_device, output_device, ws, ws_bytes, nullptr),
                      "shared attention batch kernel launch");
    } else {
        void* ws = detail::attention_workspace(storage, sequences.size(), max_len, query_heads, &ws_bytes);
        detail::check(kvflux_paged_attention(storage.key_base(), storage.value_base(), layout.num_blocks(),
                                             layout.num_kv_heads(), layout.block_size(), layout.head_size(),
                                             detail::abi_dtype(layout.dtype()), dev[0],
                                             batch.max_blocks_per_sequence(), dev[1], max_len, sequences.size(),
                                             query_heads, query_device, output_device, ws, ws_bytes, nullptr),
                      "paged attention batch kernel launch");
    }
    detail::check(kvflux_stream_synchronize(nullptr), "paged attention batch synchronize");
}

} // namespace kvflux::v2
