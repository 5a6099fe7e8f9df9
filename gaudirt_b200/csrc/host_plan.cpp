// Host side of the C ABI: status text, pool geometry, paged-metadata validation and the
// length-aware split-KV schedule.  Nothing here touches the device, and nothing leaves a C entry by exception: lists that do
// not fit into memory end as GK_ERR_CAPACITY.
#include "../../include/gaudirt_b200.h"

#include <algorithm>
#include <array>
#include <climits>
#include <cmath>
#include <functional>
#include <cstdint>
#include <numeric>
#include <unordered_map>
#include <vector>

namespace {
thread_local const char* g_metadata_error = "";     // always one of the messages below: nothing is allocated

int metadata_fail(const char* message) {
  g_metadata_error = message;
  return GK_ERR_METADATA;
}

inline int64_t round_up(int64_t v, int64_t m) { return (v + m - 1) / m * m; }
}  // namespace

namespace gk {
extern thread_local int g_last_cuda_error;
}

extern "C" const char* gk_status_string(int status) {
  switch (status) {
    case GK_OK: return "ok";
    case GK_ERR_INVALID_ARGUMENT: return "invalid argument (null pointer, negative size, misaligned pointer or stride)";
    case GK_ERR_UNSUPPORTED: return "unsupported geometry";
    case GK_ERR_CUDA: return "CUDA launch failed";
    case GK_ERR_CAPACITY: return "output array or scratch area too small";
    case GK_ERR_METADATA: return "paged metadata rejected";
    default: return "unknown status";
  }
}

extern "C" int gk_abi_version(void) { return 1; }
extern "C" int gk_last_cuda_error(void) { return gk::g_last_cuda_error; }
extern "C" const char* gk_metadata_error(void) { return g_metadata_error; }

extern "C" int gk_paged_kv_pool_bytes(int64_t layers, int64_t slots, int64_t kv_heads, int64_t head_dim,
                                      uint64_t* bytes_out) {
  if (!bytes_out) return GK_ERR_INVALID_ARGUMENT;
  // Geometry limits of allocate_paged_kv (src/bridge/paged_kv_pool.cpp:16-20) without its
  // 131072-slot descriptor cap; slots stay addressable by int32 slot ids.
  if (layers <= 0 || layers > 4096 || slots <= 0 || slots > INT32_MAX || kv_heads <= 0 || kv_heads > 256 ||
      (head_dim != 64 && head_dim != 128 && head_dim != 256))
    return GK_ERR_UNSUPPORTED;
  const uint64_t layer = 2ull * (uint64_t)slots * (uint64_t)kv_heads * (uint64_t)head_dim * 2ull;
  if (layer > UINT64_MAX / (uint64_t)layers) return GK_ERR_UNSUPPORTED;
  *bytes_out = layer * (uint64_t)layers;
  return GK_OK;
}

extern "C" int gk_paged_metadata_validate(const int32_t* locations, const int32_t* requests, const int32_t* positions,
                                          int64_t rows, const int32_t* mapping, int64_t n_requests, int64_t context,
                                          int64_t slots, int32_t* seq_out, int64_t* n_seq_out,
                                          int32_t* page_tokens_out) try {
  if (!locations || !requests || !positions || !mapping || !seq_out || !n_seq_out) return GK_ERR_INVALID_ARGUMENT;
  if (rows <= 0 || rows > INT32_MAX || slots <= 0 || slots > INT32_MAX || n_requests <= 0 || n_requests > INT32_MAX ||
      context <= 0 || context > INT32_MAX || n_requests * context > INT32_MAX)
    return metadata_fail("GaudiRT: paged metadata dimensions outside supported range");
  const int64_t cells = n_requests * context;
  for (int64_t i = 0; i < cells; ++i)
    if (mapping[i] < -1 || mapping[i] >= slots) return metadata_fail("GaudiRT: request-to-token slot is out of range");

  std::vector<int32_t> reach(n_requests, -1);
  std::unordered_map<int32_t, std::pair<int32_t, int32_t>> target;   // output slot -> (request, position)
  target.reserve((size_t)rows * 2);
  // One bit per slot in front of the map: the prefix walk below touches every visible position,
  // almost none of which is an output slot of this step.
  std::vector<uint64_t> is_target(static_cast<size_t>(slots / 64 + 1), 0);
  int64_t n_seq = 0;
  for (int64_t i = 0; i < rows; ++i) {
    const int64_t slot = locations[i], request = requests[i], position = positions[i];
    if (slot < 0 || slot >= slots || request < 0 || request >= n_requests || position < 0 || position >= context)
      return metadata_fail("GaudiRT: paged metadata index is out of range");
    if (mapping[request * context + position] != slot)
      return metadata_fail("GaudiRT: output slot does not match request-to-token mapping");
    if (!target.emplace((int32_t)slot, std::make_pair((int32_t)request, (int32_t)position)).second)
      return metadata_fail("GaudiRT: duplicate output KV slot");
    is_target[static_cast<size_t>(slot >> 6)] |= 1ull << (slot & 63);
    const bool continues = i > 0 && requests[i - 1] == request && positions[i - 1] + 1 == position;
    if (continues) {
      ++seq_out[(n_seq - 1) * 4 + 1];
    } else {
      int32_t* s = seq_out + n_seq * 4;
      s[0] = (int32_t)i;
      s[1] = 1;
      s[2] = (int32_t)position;
      s[3] = (int32_t)request;
      ++n_seq;
    }
    reach[request] = std::max(reach[request], (int32_t)position);
  }
  int page = 128;
  for (int64_t request = 0; request < n_requests; ++request) {
    const int32_t* row = mapping + request * context;
    for (int32_t position = 0; position <= reach[request]; ++position) {
      const int32_t slot = row[position];
      if (slot < 0) return metadata_fail("GaudiRT: missing KV slot in a visible prefix");
      if (is_target[static_cast<size_t>(slot >> 6)] >> (slot & 63) & 1) {
        const auto hit = target.find(slot);
        if (hit != target.end() && (hit->second.first != request || hit->second.second != position))
          return metadata_fail("GaudiRT: output KV slot aliases another visible prefix position");
      }
      // A break in slot contiguity at `position` only allows pages that end there.
      if (position > 0 && slot != row[position - 1] + 1) page = std::min(page, position & -position);
    }
  }
  *n_seq_out = n_seq;
  if (page_tokens_out) *page_tokens_out = page;
  return GK_OK;
} catch (...) {
  return GK_ERR_CAPACITY;
}

// Host half of slot allocation (src/bridge/paged_slot_allocator.cpp:95-128): the argument checks
// and one {prefix, length, first token, first fresh page} record per request.
extern "C" int gk_paged_slots_layout(const int64_t* prefixes, const int64_t* lengths, int64_t n_requests,
                                     int64_t page_size, int64_t free_page_count, int32_t* records_out,
                                     int64_t* total_out, int64_t* pages_out) {
  if (!prefixes || !lengths || !total_out || !pages_out) return GK_ERR_INVALID_ARGUMENT;
  if (page_size < 1 || page_size > INT32_MAX || n_requests <= 0 || n_requests > (int64_t{1} << 30))
    return metadata_fail("GaudiRT paged allocator: unsupported page size or request count");
  int64_t total = 0, pages = 0;
  for (int64_t i = 0; i < n_requests; ++i) {
    const int64_t prefix = prefixes[i], length = lengths[i];
    if (prefix < 0 || length < 0 || prefix > INT32_MAX || length > INT32_MAX || prefix + length > INT32_MAX)
      return metadata_fail("GaudiRT paged allocator: invalid request lengths");
    if (records_out && total <= INT32_MAX && pages <= INT32_MAX) {
      int32_t* r = records_out + i * 4;
      r[0] = (int32_t)prefix;
      r[1] = (int32_t)length;
      r[2] = (int32_t)total;
      r[3] = (int32_t)pages;
    }
    total += length;
    pages += (prefix + length + page_size - 1) / page_size - (prefix + page_size - 1) / page_size;
  }
  if (total <= 0 || total > (int64_t{1} << 30) || pages > (int64_t{1} << 30) || pages > free_page_count)
    return metadata_fail("GaudiRT paged allocator: invalid token count or insufficient free pages");
  *total_out = total;
  *pages_out = pages;
  return GK_OK;
}

namespace {
// What a step may say about its sequences beyond their records (any pointer may be null):
//   kv_from       first key of the sequence that its own work records cover (the keys before it are the shared
//                 prefix, attended to elsewhere)
//   parts_before  partial states of those keys that stand in front of the sequence's own splits
//   two_way       keys below it are visible to every row of the sequence, not only to the rows behind them
//   row_entry     out, [rows*2]: {first entry (query head 0), entries between two parts} of every row with parts_before
struct SequenceExtras {
  const int32_t* kv_from = nullptr;
  const int32_t* parts_before = nullptr;
  const int32_t* two_way = nullptr;
  int32_t* row_entry = nullptr;
};

int attention_plan_build(const int32_t* seq, int64_t n_seq, const SequenceExtras& extras, int q_heads, int kv_heads,
                         int head_dim, int window, int sm_count, int split_tokens, int32_t* work_out, int64_t work_cap,
                         int64_t* n_work_out, int32_t* combine_out, int64_t combine_cap, int64_t* n_combine_out,
                         int64_t* partial_entries_out) {
  if (!seq || n_seq <= 0 || !n_work_out || !n_combine_out || !partial_entries_out || sm_count <= 0 ||
      split_tokens < 0 || (window != -1 && window <= 0))
    return GK_ERR_INVALID_ARGUMENT;
  if (q_heads <= 0 || q_heads > 256 || kv_heads <= 0 || kv_heads > 256 || q_heads % kv_heads != 0 ||
      (head_dim != 64 && head_dim != 128 && head_dim != 256) || q_heads / kv_heads > GK_MAX_PACKED_ROWS)
    return GK_ERR_UNSUPPORTED;
  const int group = q_heads / kv_heads;
  const int block_rows = std::max(1, GK_MAX_PACKED_ROWS / group);

  struct Block { int32_t first_row, n_rows, first_pos, table_row, lo, hi, before; };
  std::vector<Block> blocks;
  int64_t total_span = 0;
  for (int64_t s = 0; s < n_seq; ++s) {
    const int32_t* r = seq + s * 4;
    if (r[1] <= 0 || r[2] < 0 || r[0] < 0 || r[3] < 0) return GK_ERR_INVALID_ARGUMENT;
    const int32_t from = extras.kv_from ? extras.kv_from[s] : 0, before = extras.parts_before ? extras.parts_before[s] : 0;
    const int32_t two_way = extras.two_way ? extras.two_way[s] : 0;
    if (from < 0 || from > r[2] || before < 0 || two_way < 0 || (int64_t)two_way > (int64_t)r[2] + r[1])
      return GK_ERR_INVALID_ARGUMENT;
    for (int32_t done = 0; done < r[1]; done += block_rows) {
      const int32_t n = std::min<int32_t>(block_rows, r[1] - done);
      const int64_t first_pos = (int64_t)r[2] + done;
      if (first_pos + n > INT32_MAX) return GK_ERR_UNSUPPORTED;
      const int32_t lo = std::max(from, window > 0 ? (int32_t)std::max<int64_t>(0, first_pos - window + 1) : 0);
      blocks.push_back({r[0] + done, n, (int32_t)first_pos, r[3], lo, std::max((int32_t)(first_pos + n), two_way), before});
      total_span += blocks.back().hi - lo;
    }
  }
  // How a block's KV range is cut for a given longest-range limit.  Even cut: equal pieces, multiples
  // of the 64 tokens four warps eat, and no cut for ranges within 25 % of the limit.  Uneven cut: pieces
  // of exactly `chunk` tokens and the remainder as the last piece (a remainder under 64 tokens stays with
  // the piece before it).  The uneven cut is what fills the machine when a few hundred equal ranges meet
  // a slightly larger number of resident CTA slots: every range gives up its tail, and the tails fill
  // the slots that would have idled for the whole launch.
  auto cut = [](int64_t span, int64_t chunk, bool uneven, int64_t& splits, int64_t& per) {
    splits = 1;
    per = span;
    if (uneven) {
      if (span >= chunk + 64) {
        per = chunk;
        splits = (span + per - 1) / per;
        if (span - (splits - 1) * per < 64) --splits;
      }
      return;
    }
    if (span > chunk + chunk / 4) {
      splits = (span + chunk - 1) / chunk;
      per = round_up((span + splits - 1) / splits, 64);
      splits = (span + per - 1) / per;
    }
  };
  // Longest KV range of one work item.  The grid is (work items x KV heads) CTAs, two resident
  // per SM, handed out longest first by the hardware scheduler; the cost of a candidate limit is
  // the makespan of that list schedule (a CTA costs its tokens plus a fixed prologue/epilogue)
  // plus the split-state traffic of the combine.  Candidates: the throughput heuristic (about
  // four CTAs per resident slot), the longest range divided by small integers, and uneven cuts a
  // little below the longest range.
  int64_t chunk = split_tokens;
  bool uneven = false;
  // The count-only call and the filling call of one plan see the same input: remember the
  // last choice per thread instead of searching twice.
  struct Memo { uint64_t key = 0; int64_t chunk = 0; bool uneven = false; };
  thread_local Memo memo;
  uint64_t key = 1469598103934665603ull;
  auto mix = [&key](uint64_t v) { key = (key ^ v) * 1099511628211ull; };
  for (const Block& b : blocks) { mix((uint64_t)b.n_rows << 32 | (uint32_t)b.lo); mix((uint64_t)b.before << 32 | (uint32_t)b.hi); }
  mix(q_heads); mix(kv_heads); mix(head_dim); mix((uint32_t)window); mix(sm_count);
  if (chunk == 0 && memo.key == key && memo.chunk > 0) {
    chunk = memo.chunk;
    uneven = memo.uneven;
  } else if (chunk == 0) {
    const int64_t slots_resident = (int64_t)sm_count * 2;
    const int64_t want = slots_resident * 4;
    chunk = round_up(std::max<int64_t>(256, (total_span * kv_heads + want - 1) / want), 64);
    int64_t longest = 0;
    for (const Block& b : blocks) longest = std::max<int64_t>(longest, b.hi - b.lo);
    if ((int64_t)blocks.size() * kv_heads < 16 * slots_resident) {
      constexpr double kCtaOverheadTokens = 150.0;    // ~3.5 us of prologue + merge at 23 ns/token
      constexpr double kCombineLaunchTokens = 130.0;  // ~3 us
      constexpr double kLoneSpeedup = 1.5;
      auto estimate = [&](int64_t limit, bool odd) {
        std::vector<int32_t> pieces;
        double combine_bytes = 0.0;
        for (const Block& b : blocks) {
          int64_t splits, per;
          cut(b.hi - b.lo, limit, odd, splits, per);
          for (int64_t i = 0; i < splits; ++i)
            pieces.push_back((int32_t)((i + 1 == splits ? (int64_t)b.hi : b.lo + (i + 1) * per) - (b.lo + i * per)));
          if (splits > 1) combine_bytes += 2.0 * splits * b.n_rows * q_heads * (head_dim + 2) * 4;
        }
        std::sort(pieces.begin(), pieces.end(), std::greater<int32_t>());
        // While CTAs are still queued every slot streams its fair share of the memory bandwidth (rate 1).
        // Once the queue is empty the CTAs that are left speed up as slots fall idle, up to kLoneSpeedup
        // (measured: 36 GB/s for a CTA on an otherwise idle GPU, 23.4 GB/s with all 296 slots busy).
        std::vector<double> heap((size_t)slots_resident, 0.0);       // min-heap of slot finish times at rate 1
        auto later = std::greater<double>();
        double last_start = 0.0;
        for (int32_t len : pieces)
          for (int h = 0; h < kv_heads; ++h) {
            std::pop_heap(heap.begin(), heap.end(), later);
            last_start = heap.back();
            heap.back() += len + kCtaOverheadTokens;
            std::push_heap(heap.begin(), heap.end(), later);
          }
        std::vector<double> left;
        for (double finish : heap)
          if (finish > last_start) left.push_back(finish - last_start);
        std::sort(left.begin(), left.end());
        double makespan = last_start, done = 0.0;
        for (size_t k = 0; k < left.size(); ++k) {
          const double active = (double)(left.size() - k);
          makespan += (left[k] - done) / std::min(kLoneSpeedup, (double)slots_resident / active);
          done = left[k];
        }
        const double token_bytes = 2.0 * head_dim * 2;
        return makespan + combine_bytes / token_bytes / slots_resident + (combine_bytes > 0 ? kCombineLaunchTokens : 0.0);
      };
      double best = estimate(chunk, false);
      for (int k : {1, 2, 3, 4, 6, 8, 12, 16}) {
        const int64_t candidate = round_up((longest + k - 1) / k, 64);
        if (candidate < 256) break;
        // finer cuts than ~12 CTAs per resident slot only add overhead: stop searching there
        int64_t ctas = 0;
        for (const Block& b : blocks) {
          int64_t splits, per;
          cut(b.hi - b.lo, candidate, false, splits, per);
          ctas += splits * kv_heads;
        }
        if (ctas > 12 * slots_resident) break;
        const double cost = estimate(candidate, false);
        if (cost < best * 0.995) {
          best = cost;
          chunk = candidate;
          uneven = false;
        }
      }
      // Uneven cuts: only worth a look while the whole grid is a few waves (that is where idle slots cost most).
      if ((int64_t)blocks.size() * kv_heads <= 4 * slots_resident)
        for (int percent : {97, 94, 91, 88, 85, 80, 75, 70, 65, 60, 55}) {
          const int64_t candidate = round_up(longest * percent / 100, 64);
          if (candidate < 256 || candidate >= longest) continue;
          const double cost = estimate(candidate, true);
          if (cost < best * 0.98) {
            best = cost;
            chunk = candidate;
            uneven = true;
          }
        }
    }
    memo.key = key;
    memo.chunk = chunk;
    memo.uneven = uneven;
  }
  chunk = std::max<int64_t>(chunk, 16);

  struct Item { int32_t w[GK_WORK_WORDS]; };
  std::vector<Item> items;
  std::vector<std::array<int32_t, GK_COMBINE_WORDS>> merges;
  int64_t entries = 0;
  for (const Block& b : blocks) {
    const int64_t span = b.hi - b.lo;
    int64_t splits, per;
    cut(span, chunk, uneven, splits, per);
    const int64_t parts = b.before + splits;         // states to merge: the ones in front, then the block's own splits
    if (parts > 0x7fff) return GK_ERR_CAPACITY;      // the split index shares a record word with the count
    int64_t base = -1;
    if (parts > 1) {
      base = entries;
      entries += parts * b.n_rows * q_heads;
      if (entries > INT32_MAX) return GK_ERR_CAPACITY;
      merges.push_back({b.first_row, b.n_rows, (int32_t)base, (int32_t)parts});
      if (b.before > 0 && extras.row_entry)
        for (int32_t r = 0; r < b.n_rows; ++r) {
          extras.row_entry[2 * (int64_t)(b.first_row + r)] = (int32_t)(base + (int64_t)r * q_heads);
          extras.row_entry[2 * (int64_t)(b.first_row + r) + 1] = b.n_rows * q_heads;
        }
    }
    for (int64_t s = 0; s < splits; ++s) {
      Item it{};
      it.w[0] = b.first_row;
      it.w[1] = b.n_rows;
      it.w[2] = b.first_pos;
      it.w[3] = b.table_row;
      it.w[4] = (int32_t)(b.lo + s * per);
      it.w[5] = s + 1 == splits ? b.hi : (int32_t)(b.lo + (s + 1) * per);
      const int64_t part = b.before + s;
      it.w[6] = base < 0 ? -1 : (int32_t)(base + part * b.n_rows * q_heads);
      it.w[7] = (int32_t)(parts | (part << 16));   // low half: states of the block to merge, high half: which one
      items.push_back(it);
    }
  }
  *n_work_out = (int64_t)items.size();
  *n_combine_out = (int64_t)merges.size();
  *partial_entries_out = entries;
  if (!work_out) return GK_OK;
  if (work_cap < (int64_t)items.size() || combine_cap < (int64_t)merges.size() || (!merges.empty() && !combine_out))
    return GK_ERR_CAPACITY;
  std::stable_sort(items.begin(), items.end(),
                   [](const Item& a, const Item& b) { return a.w[5] - a.w[4] > b.w[5] - b.w[4]; });
  for (size_t i = 0; i < items.size(); ++i) std::copy(items[i].w, items[i].w + GK_WORK_WORDS, work_out + i * GK_WORK_WORDS);
  for (size_t i = 0; i < merges.size(); ++i)
    std::copy(merges[i].begin(), merges[i].end(), combine_out + i * GK_COMBINE_WORDS);
  return GK_OK;
}

}  // namespace

extern "C" int gk_attention_plan_build(const int32_t* seq, int64_t n_seq, int q_heads, int kv_heads, int head_dim,
                                       int window, int sm_count, int split_tokens, int32_t* work_out,
                                       int64_t work_cap, int64_t* n_work_out, int32_t* combine_out,
                                       int64_t combine_cap, int64_t* n_combine_out, int64_t* partial_entries_out) try {
  return attention_plan_build(seq, n_seq, SequenceExtras{}, q_heads, kv_heads, head_dim, window, sm_count, split_tokens,
                              work_out, work_cap, n_work_out, combine_out, combine_cap, n_combine_out, partial_entries_out);
} catch (...) {
  return GK_ERR_CAPACITY;
}

// Sequences whose rows see a two-way prefix and, by group, read a common prefix together.
extern "C" int gk_shared_prefix_plan_build(const int32_t* seq, int64_t n_seq, const int32_t* two_way, const int32_t* groups,
                                           const int32_t* prefix_tokens, int64_t n_groups, int q_heads, int kv_heads,
                                           int head_dim, int window, int sm_count, int split_tokens,
                                           int prefix_split_tokens, int64_t min_saved_bytes, int* form_out,
                                           int32_t* work_out,
                                           int64_t work_cap, int64_t* n_work_out, int32_t* combine_out,
                                           int64_t combine_cap, int64_t* n_combine_out, int64_t* partial_entries_out,
                                           int32_t* prefix_work_out, int64_t prefix_work_cap, int64_t* n_prefix_work_out,
                                           int32_t* prefix_rows_out, int64_t prefix_rows_cap,
                                           int64_t* n_prefix_rows_out) try {
  if (!seq || n_seq <= 0 || n_groups < 0 || (n_groups > 0 && (!groups || !prefix_tokens)) || prefix_split_tokens < 0 ||
      min_saved_bytes < 0 || !form_out || !n_prefix_work_out || !n_prefix_rows_out || sm_count <= 0 || (window != -1 && window <= 0))
    return GK_ERR_INVALID_ARGUMENT;
  if (q_heads <= 0 || q_heads > 256 || kv_heads <= 0 || kv_heads > 256 || q_heads % kv_heads != 0 ||
      (head_dim != 64 && head_dim != 128 && head_dim != 256) || q_heads / kv_heads > GK_MAX_PACKED_ROWS)
    return GK_ERR_UNSUPPORTED;
  const int group_heads = q_heads / kv_heads;
  const int tile = head_dim == 256 ? 64 : 128;                                    // keys of one tile of the kernel
  const int tile_rows = GK_PREFILL_TILE_ROWS / group_heads;
  const int ctas_per_record = head_dim == 256 ? 2 : 1;

  struct Group { std::vector<int32_t> members; int64_t rows = 0; int32_t lo = 0, hi = 0, seen = 0; };
  std::vector<Group> all(static_cast<size_t>(n_groups));
  int64_t last_row = 0;
  for (int64_t s = 0; s < n_seq; ++s) {
    const int32_t* r = seq + s * 4;
    if (r[1] <= 0 || r[2] < 0 || r[0] < 0 || r[3] < 0 || (int64_t)r[2] + r[1] > INT32_MAX) return GK_ERR_INVALID_ARGUMENT;
    last_row = std::max<int64_t>(last_row, (int64_t)r[0] + r[1]);
    const int32_t g = n_groups > 0 ? groups[s] : -1;
    if (g < -1 || g >= n_groups) return GK_ERR_INVALID_ARGUMENT;
    if (g < 0) continue;
    if (prefix_tokens[g] < 0 || prefix_tokens[g] > r[2]) return GK_ERR_INVALID_ARGUMENT;   // every row is behind the prefix
    all[g].members.push_back((int32_t)s);
    all[g].rows += r[1];
  }
  // Groups are attended to together when that saves enough reading to pay for the launch and for the merge of the parts.
  std::vector<Group*> shared;
  const int64_t token_bytes = (int64_t)kv_heads * head_dim * 4;
  int64_t saved = 0;
  for (int64_t g = 0; g < n_groups; ++g) {
    Group& one = all[g];
    one.hi = prefix_tokens[g];
    one.lo = one.hi;
    for (int32_t s : one.members)
      one.lo = std::min(one.lo, window > 0 ? std::max(0, seq[s * 4 + 2] - window + 1) : 0);   // first key any row sees
    if (one.members.size() < 2 || one.hi <= one.lo) continue;
    saved += (int64_t)(one.members.size() - 1) * (one.hi - one.lo) * token_bytes;
    one.seen = one.lo;
    one.lo = one.lo / tile * tile;      // cut at whole tiles; the first record says where its keys begin, the kernel masks a row's own window
    shared.push_back(&one);
  }
  if (saved < min_saved_bytes) shared.clear();
  // The form of the records (one or two query tiles) and how long a piece of the prefix one CTA takes: the cheapest by a
  // model of the two kernels side by side, in us.  A prefix CTA has an SM to itself for a fixed 7 us and 1.2 us per 128 keys
  // and one query tile, 2.4 us per two (1.0 and 1.9 at head_dim 64, 1.1 per 64 keys at 256; scores without cap or bias).  The members' own CTAs take
  // 3.5 us and 36 GB/s each, two per SM on the SMs that the prefix leaves and on all of them once it is done, never faster
  // than memory gives their bytes and never more than 50 of them in a us (2048 of 64 KB took 40 us on 84 and on 148 SMs).  Every part of a row costs its merge 0.15 us.  So the longer of the two
  // gets the SMs: measured with 256 members of 4096 + 1024 tokens, 32 CTAs of two tiles or 64 of one 108 us, 128 of one
  // 123 us; with 32 members of 2048 + 256, 32 CTAs 16.7 us, 64 of them 18.4 us, 128 of them 23.7 us.
  bool one_tile = head_dim != 256;
  int64_t piece = prefix_split_tokens;
  if (!shared.empty()) {
    constexpr double kFixed = 7.0, kTailFixed = 3.5, kTailBytes = 36e3, kMemoryBytes = 5.9e6, kTailsPerUs = 50.0,
                     kMergePart = 0.15;
    const double one_time = head_dim == 64 ? 1.0 : head_dim == 128 ? 1.2 : 1.1, two_time = head_dim == 64 ? 1.9 : 2.4;
    const double head_bytes = head_dim * 4.0;
    double all_bytes = 0.0, tail_bytes = 0.0, tail_longest = 0.0;
    int64_t tail_ctas = 0;
    std::vector<int32_t> starts(static_cast<size_t>(n_seq), 0);
    int32_t longest = 0;
    for (const Group* g : shared) {
      for (int32_t s : g->members) starts[s] = g->hi;
      longest = std::max(longest, g->hi - g->lo);
      all_bytes += (double)(g->hi - g->lo) * kv_heads * head_bytes;
    }
    for (int64_t s = 0; s < n_seq; ++s) {
      const int32_t* r = seq + s * 4;
      const int64_t from = std::max<int64_t>(starts[s], window > 0 ? std::max(0, r[2] - window + 1) : 0);
      const double bytes = (double)((int64_t)r[2] + r[1] - from) * head_bytes;
      const int64_t ctas = (r[1] + GK_MAX_PACKED_ROWS / group_heads - 1) / (GK_MAX_PACKED_ROWS / group_heads) * kv_heads;
      tail_bytes += ctas * bytes;
      tail_ctas += ctas;
      tail_longest = std::max(tail_longest, bytes);
    }
    all_bytes += tail_bytes;
    const double mean_bytes = tail_bytes / (double)tail_ctas;
    const double tail_mean = kTailFixed + mean_bytes / kTailBytes;
    tail_longest = kTailFixed + tail_longest / kTailBytes;
    auto estimate = [&](bool one, int64_t tiles) {
      int64_t ctas = 0, most_parts = 0;
      double busy = 0.0, slowest = 0.0;
      for (const Group* g : shared) {
        const int64_t rows_per_record = one ? tile_rows : GK_PREFILL_TILES_PER_ITEM * tile_rows;
        const int64_t records = (g->rows + rows_per_record - 1) / rows_per_record * kv_heads * ctas_per_record;
        const int64_t span = (g->hi - g->lo + tile - 1) / tile, pieces = (span + tiles - 1) / tiles;
        const double per_tile = one || head_dim == 256 ? one_time : g->rows > tile_rows ? two_time : 1.8 * one_time;
        ctas += records * pieces;
        busy += records * (pieces * kFixed + span * per_tile);
        slowest = std::max(slowest, kFixed + (double)((span + pieces - 1) / pieces) * per_tile);
        most_parts = std::max(most_parts, pieces);
      }
      const double waves = (double)((ctas + sm_count - 1) / sm_count);
      const double prefix = std::max(slowest, waves > 1.0 ? waves * busy / (double)ctas : 0.0);
      const double slots = 2.0 * (double)std::max<int64_t>(0, sm_count - ctas);
      double tails = tail_longest;
      if ((double)tail_ctas > slots) {
        const double beside = std::min(std::floor(prefix / tail_mean) * slots, prefix * kTailsPerUs);
        const double left = std::max(0.0, (double)tail_ctas - beside);
        tails = prefix;
        if (left > 0.0)
          tails += std::max({std::max(1.0, left / (2.0 * sm_count)) * tail_mean, left * mean_bytes / kMemoryBytes, left / kTailsPerUs});
      }
      return std::max({prefix, tails, all_bytes / kMemoryBytes}) + kMergePart * (double)most_parts;
    };
    double best = -1.0;
    const int64_t all_tiles = (longest + tile - 1) / tile, given = (piece + tile - 1) / tile;
    std::vector<int64_t> lengths;                                 // of a piece, in tiles: every one up to 16, then in steps of an eighth
    if (given > 0) lengths.push_back(given);
    for (int64_t tiles = 1; given == 0 && tiles < all_tiles; tiles += std::max<int64_t>(1, tiles < 16 ? 1 : tiles / 8)) lengths.push_back(tiles);
    if (given == 0) lengths.push_back(all_tiles);
    for (bool one : {true, false}) {
      if (one && head_dim == 256) continue;
      for (const int64_t tiles : lengths) {
        const double cost = estimate(one, tiles);
        if (best >= 0.0 && cost >= best) continue;
        best = cost;
        one_tile = one;
        if (given == 0) piece = tiles * tile;
      }
    }
    piece = round_up(std::max<int64_t>(piece, tile), tile);
  }
  const int record_rows = one_tile ? tile_rows : GK_PREFILL_TILES_PER_ITEM * tile_rows;

  std::vector<int32_t> kv_from(static_cast<size_t>(n_seq), 0), before(static_cast<size_t>(n_seq), 0);
  struct Item { int32_t w[GK_WORK_WORDS]; };
  std::vector<Item> items;
  std::vector<std::array<int32_t, 4>> rows;
  for (const Group* g : shared) {
    const int64_t span = (g->hi - g->lo + tile - 1) / tile, pieces = (span * tile + piece - 1) / piece;
    const int64_t even = (span + pieces - 1) / pieces * tile, parts = (span * tile + even - 1) / even;
    if (parts >= 0x7fff) return GK_ERR_CAPACITY;
    std::vector<std::array<int32_t, 2>> places;                   // {row, position}
    for (int32_t s : g->members) {
      kv_from[s] = g->hi;
      before[s] = (int32_t)parts;
      for (int32_t r = 0; r < seq[s * 4 + 1]; ++r) places.push_back({seq[s * 4] + r, seq[s * 4 + 2] + r});
    }
    for (size_t at = 0; at < places.size(); at += record_rows) {
      const int32_t n = (int32_t)std::min<size_t>(record_rows, places.size() - at);
      int32_t highest = 0;
      for (int32_t i = 0; i < n; ++i) highest = std::max(highest, places[at + i][1]);
      for (int64_t part = 0; part < parts; ++part)
        items.push_back({{(int32_t)(rows.size()), n, (int32_t)part, seq[g->members[0] * 4 + 3], std::max(g->seen, (int32_t)(g->lo + part * even)),
                          (int32_t)std::min<int64_t>(g->hi, g->lo + (part + 1) * even), highest, 0}});
      for (int32_t i = 0; i < n; ++i) rows.push_back({places[at + i][0], places[at + i][1], 0, 0});
    }
  }
  std::vector<int32_t> row_entry(static_cast<size_t>(last_row) * 2, 0);
  SequenceExtras extras;
  extras.kv_from = kv_from.data();
  extras.parts_before = before.data();
  extras.two_way = two_way;
  extras.row_entry = row_entry.data();
  const int built = attention_plan_build(seq, n_seq, extras, q_heads, kv_heads, head_dim, window, sm_count, split_tokens,
                                         work_out, work_cap, n_work_out, combine_out, combine_cap, n_combine_out,
                                         partial_entries_out);
  if (built != GK_OK) return built;
  // Tails of one query block each, many of them and short: two warps and four CTAs per SM instead of four warps and two,
  // so that a CTA's fixed cost (3 to 4 us of look-ups and merges) is a smaller part of its time.  Measured at head_dim 128:
  // 10-14 % faster at 1024 and 2048 CTAs of 64 to 512 tokens, even at 8192 tokens, 10-25 % slower at 128 to 512 CTAs; all
  // of that with few prefix CTAs beside them, so the rule counts every SM and not the ones that the prefix leaves.
  int64_t own_tokens = 0;
  for (int64_t s = 0; s < n_seq; ++s) own_tokens += seq[s * 4 + 2] + seq[s * 4 + 1] - kv_from[s];
  const bool short_tails = head_dim != 256 && !items.empty() && *n_work_out * kv_heads >= 6 * (int64_t)sm_count &&
                           own_tokens <= 2048 * *n_work_out;
  *form_out = items.empty() ? 0 : GK_SHARED_PREFIX | (one_tile ? GK_SHARED_ONE_TILE : 0) | (short_tails ? GK_SHARED_SHORT_TAILS : 0);
  *n_prefix_work_out = (int64_t)items.size();
  *n_prefix_rows_out = (int64_t)rows.size();
  if (!work_out) return GK_OK;
  if (prefix_work_cap < (int64_t)items.size() || prefix_rows_cap < (int64_t)rows.size() ||
      (!items.empty() && (!prefix_work_out || !prefix_rows_out)))
    return GK_ERR_CAPACITY;
  std::stable_sort(items.begin(), items.end(),
                   [](const Item& a, const Item& b) { return a.w[5] - a.w[4] > b.w[5] - b.w[4]; });
  for (size_t i = 0; i < items.size(); ++i) std::copy(items[i].w, items[i].w + GK_WORK_WORDS, prefix_work_out + i * GK_WORK_WORDS);
  for (size_t i = 0; i < rows.size(); ++i) {
    rows[i][2] = row_entry[2 * (size_t)rows[i][0]];
    rows[i][3] = row_entry[2 * (size_t)rows[i][0] + 1];
    std::copy(rows[i].begin(), rows[i].end(), prefix_rows_out + i * 4);
  }
  return GK_OK;
} catch (...) {
  return GK_ERR_CAPACITY;
}

namespace {
int prefill_plan_build(const int32_t* seq, int64_t n_seq, const int32_t* two_way, int q_heads, int kv_heads, int window,
                       int min_rows, int32_t* work_out, int64_t work_cap, int64_t* n_work_out, int32_t* rest_seq_out,
                       int64_t* n_rest_out) {
  if (!seq || n_seq <= 0 || !n_work_out || !n_rest_out || min_rows < 0 || (window != -1 && window <= 0))
    return GK_ERR_INVALID_ARGUMENT;
  if (q_heads <= 0 || kv_heads <= 0 || q_heads % kv_heads != 0 || q_heads / kv_heads > GK_PREFILL_TILE_ROWS)
    return GK_ERR_UNSUPPORTED;
  const int group = q_heads / kv_heads;
  // one record feeds both query tiles of a CTA: up to 2 x (128 / group) consecutive rows
  const int tile_rows = GK_PREFILL_TILES_PER_ITEM * (GK_PREFILL_TILE_ROWS / group);
  if (min_rows == 0) min_rows = std::max(2, (32 + group - 1) / group);
  struct Item { int32_t w[GK_WORK_WORDS]; };
  std::vector<Item> items;
  int64_t n_rest = 0;
  for (int64_t s = 0; s < n_seq; ++s) {
    const int32_t* r = seq + s * 4;
    if (r[1] <= 0 || r[2] < 0 || r[0] < 0 || r[3] < 0) return GK_ERR_INVALID_ARGUMENT;
    if (two_way && (two_way[s] < 0 || (int64_t)two_way[s] > (int64_t)r[2] + r[1])) return GK_ERR_INVALID_ARGUMENT;
    if (r[1] < min_rows) {
      if (rest_seq_out) std::copy(r, r + 4, rest_seq_out + n_rest * 4);
      ++n_rest;
      continue;
    }
    for (int32_t done = 0; done < r[1]; done += tile_rows) {
      const int32_t n = std::min<int32_t>(tile_rows, r[1] - done);
      const int64_t first_pos = (int64_t)r[2] + done;
      if (first_pos + n > INT32_MAX) return GK_ERR_UNSUPPORTED;
      Item it{};
      it.w[0] = r[0] + done;
      it.w[1] = n;
      it.w[2] = (int32_t)first_pos;
      it.w[3] = r[3];
      it.w[4] = window > 0 ? (int32_t)std::max<int64_t>(0, first_pos - window + 1) : 0;
      it.w[5] = std::max((int32_t)(first_pos + n), two_way ? two_way[s] : 0);
      it.w[6] = -1;
      it.w[7] = 1;
      items.push_back(it);
    }
  }
  *n_work_out = (int64_t)items.size();
  *n_rest_out = n_rest;
  if (!work_out) return GK_OK;
  if (work_cap < (int64_t)items.size()) return GK_ERR_CAPACITY;
  std::stable_sort(items.begin(), items.end(),
                   [](const Item& a, const Item& b) { return a.w[5] - a.w[4] > b.w[5] - b.w[4]; });
  for (size_t i = 0; i < items.size(); ++i) std::copy(items[i].w, items[i].w + GK_WORK_WORDS, work_out + i * GK_WORK_WORDS);
  return GK_OK;
}
}  // namespace

extern "C" int gk_prefill_plan_build(const int32_t* seq, int64_t n_seq, int q_heads, int kv_heads, int window,
                                     int min_rows, int32_t* work_out, int64_t work_cap, int64_t* n_work_out,
                                     int32_t* rest_seq_out, int64_t* n_rest_out) try {
  return prefill_plan_build(seq, n_seq, nullptr, q_heads, kv_heads, window, min_rows, work_out, work_cap, n_work_out,
                            rest_seq_out, n_rest_out);
} catch (...) {
  return GK_ERR_CAPACITY;
}

extern "C" int gk_prefill_plan_build_two_way(const int32_t* seq, int64_t n_seq, const int32_t* two_way, int q_heads,
                                             int kv_heads, int window, int min_rows, int32_t* work_out, int64_t work_cap,
                                             int64_t* n_work_out, int32_t* rest_seq_out, int64_t* n_rest_out) try {
  return prefill_plan_build(seq, n_seq, two_way, q_heads, kv_heads, window, min_rows, work_out, work_cap, n_work_out,
                            rest_seq_out, n_rest_out);
} catch (...) {
  return GK_ERR_CAPACITY;
}
