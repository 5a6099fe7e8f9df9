// Slot maps and table rows of a step, built on the device from the requests' lengths.
//
// Request i of the batch holds c = lengths[i] cached tokens and appends n = new_tokens[i]; its rows are the positions
// c .. c + n - 1, rows of a request side by side, requests in batch order.  With page size P the first (-c) mod P rows
// continue the open page behind slot table[request][c - 1]; the others take fresh pages,
//   slot = free_pages[used + first_i + k / P] * P + k % P,   first_i = sum over j < i of ceil((c_j + n_j) / P) - ceil(c_j / P).
// Both sums over the batch (rows and fresh pages) are exclusive scans.  What bounds it is latency, not bytes (20 bytes in
// per request, 16 out per row): up to kOneLaunchBatch requests every CTA scans the whole batch for itself in shared
// memory, so one launch is all there is; above that one CTA scans into a workspace and a second launch expands.
// The same lengths give the same bits: nothing depends on scheduling.
#include "gk_common.cuh"

#include <algorithm>

namespace gk {
namespace {

constexpr int kThreads = 1024;
constexpr int kOneLaunchBatch = 4096;      // requests whose offsets fit the one-launch form's shared memory
constexpr int64_t kMaxBatch = 65536, kMaxRequests = 262144;

struct ExtendArgs {
  int32_t* table;
  int64_t n_requests, context, table_stride;
  const int32_t* requests;
  const int64_t* lengths;
  const int32_t* new_tokens;
  int batch;
  const int64_t* free_pages;
  int64_t n_free;
  const int64_t* used;
  int64_t page, rows;
  int32_t *locations, *positions, *row_requests, *row_offsets;
  int64_t *next_lengths, *next_used;
  int32_t* status;
  int32_t* workspace;                      // two-launch form: first row [batch], first page [batch], then the verdict
};

struct Totals {
  int64_t rows, pages;
  bool bad;
};

// Exclusive scans of the batch's new rows and fresh pages into first_row / first_page, and the checks of the whole batch:
// request ids in range and each named once, lengths that fit the table, rows that fit the outputs, pages that are free.
// `seen` holds one bit per request.  Called by all threads of a CTA; the arrays are complete when it returns.
template <int kItems>
__device__ Totals scan_batch(const ExtendArgs& a, int32_t* first_row, int32_t* first_page, unsigned* seen) {
  __shared__ int64_t warp_rows[32], warp_pages[32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  for (int64_t w = threadIdx.x; w < (a.n_requests + 31) / 32; w += kThreads) seen[w] = 0;
  __syncthreads();
  Totals t{0, 0, false};
  bool bad = false;
  // kItems consecutive requests per thread and pass.  Measured: 4096 requests 9.8 us with four, 11.7 us with one; 64 requests
  // 6.2 and 5.5 us, so the launcher takes one up to 1024 requests.
  for (int base = 0; base < a.batch; base += kThreads * kItems) {
    const int first = base + threadIdx.x * kItems;
    int64_t c[kItems], n[kItems], r[kItems];
#pragma unroll
    for (int k = 0; k < kItems; ++k) {
      const bool in = first + k < a.batch;
      c[k] = in ? a.lengths[first + k] : 0;
      n[k] = in ? a.new_tokens[first + k] : 0;
      r[k] = in ? a.requests[first + k] : -1;
    }
    int64_t rows[kItems], pages[kItems], r_sum = 0, p_sum = 0;
#pragma unroll
    for (int k = 0; k < kItems; ++k) {
      rows[k] = pages[k] = 0;
      if (first + k < a.batch) {
        if (c[k] < 0 || n[k] < 0 || c[k] > a.context || n[k] > a.context - c[k] || r[k] < 0 || r[k] >= a.n_requests) {
          bad = true;
        } else {
          if (atomicOr(seen + (r[k] >> 5), 1u << (r[k] & 31)) >> (r[k] & 31) & 1) bad = true;      // the same request twice
          rows[k] = n[k];
          // lengths fit the table and with it 32 bits
          const unsigned page = (unsigned)a.page;
          pages[k] = ((unsigned)(c[k] + n[k]) + (page - 1)) / page - ((unsigned)c[k] + (page - 1)) / page;
        }
      }
      r_sum += rows[k];
      p_sum += pages[k];
    }
    const int64_t r_mine = r_sum, p_mine = p_sum;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int64_t r_up = __shfl_up_sync(0xffffffffu, r_sum, d), p_up = __shfl_up_sync(0xffffffffu, p_sum, d);
      if (lane >= d) {
        r_sum += r_up;
        p_sum += p_up;
      }
    }
    if (lane == 31) {
      warp_rows[warp] = r_sum;
      warp_pages[warp] = p_sum;
    }
    __syncthreads();
    if (warp == 0) {
      int64_t r = warp_rows[lane], p = warp_pages[lane];
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const int64_t r_up = __shfl_up_sync(0xffffffffu, r, d), p_up = __shfl_up_sync(0xffffffffu, p, d);
        if (lane >= d) {
          r += r_up;
          p += p_up;
        }
      }
      warp_rows[lane] = r;
      warp_pages[lane] = p;
    }
    __syncthreads();
    // cut to 32 bits: a batch whose totals do not fit is refused below and nothing reads these
    int64_t row = t.rows + (warp ? warp_rows[warp - 1] : 0) + r_sum - r_mine;
    int64_t page = t.pages + (warp ? warp_pages[warp - 1] : 0) + p_sum - p_mine;
#pragma unroll
    for (int k = 0; k < kItems; ++k)
      if (first + k < a.batch) {
        first_row[first + k] = (int32_t)row;
        first_page[first + k] = (int32_t)page;
        row += rows[k];
        page += pages[k];
      }
    t.rows += warp_rows[31];
    t.pages += warp_pages[31];
    __syncthreads();
  }
  const int64_t used = *a.used;
  bad |= used < 0 || used > a.n_free || t.pages > a.n_free - used || t.rows > a.rows;
  t.bad = __syncthreads_or(bad);
  return t;
}

// Everything the step writes, from the scanned batch; a refused batch leaves the table, the lengths and the used count as
// they are and blanks every row.
__device__ void expand_batch(const ExtendArgs& a, const Totals& t, const int32_t* first_row, const int32_t* first_page) {
  const int64_t used = *a.used, step = (int64_t)gridDim.x * kThreads, start = (int64_t)blockIdx.x * kThreads + threadIdx.x;
  for (int64_t i = start; i < a.batch; i += step) {
    a.row_offsets[i] = t.bad ? 0 : first_row[i];
    a.next_lengths[i] = a.lengths[i] + (t.bad ? 0 : a.new_tokens[i]);
  }
  if (start == 0) {
    a.row_offsets[a.batch] = t.bad ? 0 : (int32_t)t.rows;
    *a.next_used = used + (t.bad ? 0 : t.pages);
    if (t.bad && a.status) atomicOr(a.status, (int)GK_DEV_BAD_METADATA);
  }
  for (int64_t row = start; row < a.rows; row += step) {
    int32_t location = -1, position = -1, request = -1;
    if (!t.bad && row < t.rows) {
      // last request whose first row is <= row: requests without rows share the first row of the one behind them and
      // sort in front of it
      int lo = 0, hi = a.batch - 1;
      while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (first_row[mid] <= row) lo = mid; else hi = mid - 1;
      }
      const int64_t c = a.lengths[lo], j = row - first_row[lo], open = (a.page - c % a.page) % a.page;
      request = a.requests[lo];
      position = (int32_t)(c + j);
      int32_t* cells = a.table + (int64_t)request * a.table_stride;
      int64_t slot = -1;
      if (j < open) {
        const int64_t last = cells[c - 1];               // c > 0: a page is open
        if (last >= 0 && last % a.page == (c - 1) % a.page) slot = last + 1 + j;
        else if (a.status) atomicOr(a.status, (int)GK_DEV_BAD_TABLE);
      } else {
        const int64_t k = j - open, id = a.free_pages[used + first_page[lo] + k / a.page];
        if (id >= 0 && id <= (INT32_MAX - k % a.page) / a.page) slot = id * a.page + k % a.page;
        else if (a.status) atomicOr(a.status, (int)GK_DEV_BAD_SLOT);
      }
      if (slot >= 0 && slot <= INT32_MAX) {
        location = (int32_t)slot;
        cells[position] = location;
      }
    }
    a.locations[row] = location;
    a.positions[row] = position;
    a.row_requests[row] = request;
  }
}

template <int kItems>
__global__ void __launch_bounds__(kThreads) extend_kernel(const ExtendArgs a) {
  extern __shared__ int32_t shared_words[];
  wait_for_predecessor();
  int32_t* first_row = shared_words;
  int32_t* first_page = first_row + a.batch;
  const Totals t = scan_batch<kItems>(a, first_row, first_page, reinterpret_cast<unsigned*>(first_page + a.batch));
  expand_batch(a, t, first_row, first_page);
}

__global__ void __launch_bounds__(kThreads) extend_scan_kernel(const ExtendArgs a) {
  extern __shared__ int32_t shared_words[];
  wait_for_predecessor();
  const Totals t = scan_batch<4>(a, a.workspace, a.workspace + a.batch, reinterpret_cast<unsigned*>(shared_words));
  if (threadIdx.x == 0) {
    int64_t* verdict = reinterpret_cast<int64_t*>(a.workspace + 2 * (int64_t)a.batch);
    verdict[0] = t.rows;
    verdict[1] = t.pages;
    verdict[2] = t.bad;
  }
}

__global__ void __launch_bounds__(kThreads) extend_expand_kernel(const ExtendArgs a) {
  wait_for_predecessor();
  const int64_t* verdict = reinterpret_cast<const int64_t*>(a.workspace + 2 * (int64_t)a.batch);
  const Totals t{verdict[0], verdict[1], verdict[2] != 0};
  expand_batch(a, t, a.workspace, a.workspace + a.batch);
}

}  // namespace
}  // namespace gk

extern "C" int gk_extend_requests_workspace_bytes(int64_t batch, uint64_t* bytes_out) {
  if (!bytes_out || batch <= 0 || batch > gk::kMaxBatch) return GK_ERR_INVALID_ARGUMENT;
  *bytes_out = batch <= gk::kOneLaunchBatch ? 0 : (uint64_t)batch * 8 + 24;
  return GK_OK;
}

extern "C" int gk_extend_requests(int32_t* table, int64_t n_requests, int64_t context, int64_t table_stride,
                                  const int32_t* requests, const int64_t* lengths, const int32_t* new_tokens, int64_t batch,
                                  const int64_t* free_pages, int64_t n_free, const int64_t* used_pages, int64_t page_size,
                                  int64_t rows, void* workspace, int32_t* locations, int32_t* positions,
                                  int32_t* row_requests, int32_t* row_offsets, int64_t* next_lengths, int64_t* next_used,
                                  int32_t* status, gk_stream_t stream) {
  using namespace gk;
  if (!table || !requests || !lengths || !new_tokens || (!free_pages && n_free > 0) || !used_pages || !locations ||
      !positions || !row_requests || !row_offsets || !next_lengths || !next_used || batch <= 0 || n_requests <= 0 ||
      context <= 0 || context > INT32_MAX || table_stride < context || n_free < 0 || page_size <= 0 ||
      page_size > INT32_MAX || rows <= 0 || rows > INT32_MAX || (batch > kOneLaunchBatch && !workspace) ||
      (reinterpret_cast<uintptr_t>(workspace) & 7))
    return GK_ERR_INVALID_ARGUMENT;
  if (batch > kMaxBatch || n_requests > kMaxRequests) return GK_ERR_UNSUPPORTED;
  ExtendArgs a{table, n_requests, context, table_stride, requests, lengths, new_tokens, (int)batch, free_pages, n_free,
               used_pages, page_size, rows, locations, positions, row_requests, row_offsets, next_lengths, next_used,
               status, static_cast<int32_t*>(workspace)};
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  const size_t seen_bytes = (size_t)((n_requests + 31) / 32) * 4;
  const unsigned ctas = (unsigned)std::min<int64_t>(148, (std::max(rows, batch) + kThreads - 1) / kThreads);
  if (batch <= kOneLaunchBatch) {
    const size_t bytes = (size_t)batch * 8 + seen_bytes;
    const bool single = batch <= kThreads;
    static std::atomic<bool> configured[2][64];
    const int ready = opt_in_shared_memory(single ? extend_kernel<1> : extend_kernel<4>,
                                           kOneLaunchBatch * 8 + (int)(kMaxRequests / 8), configured[single]);
    if (ready != GK_OK) return ready;
    launch_after_predecessor(single ? extend_kernel<1> : extend_kernel<4>, dim3(ctas), dim3(kThreads), bytes, s, a);
    return check_launch();
  }
  launch_after_predecessor(extend_scan_kernel, dim3(1), dim3(kThreads), seen_bytes, s, a);
  const int rc = check_launch();
  if (rc != GK_OK) return rc;
  launch_after_predecessor(extend_expand_kernel, dim3(ctas), dim3(kThreads), 0, s, a);
  return check_launch();
}
