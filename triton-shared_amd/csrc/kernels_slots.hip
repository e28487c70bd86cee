// Block tables and slot maps of a batch from its requests' lengths.  With past = length - fresh of a request,
//   pages it has = ceil(past / page),  pages it needs = ceil(length / page)  (both at most the table's columns),
// the pages that are missing come off a stack of free ones in the order of the requests, and the rows of the step are the fresh tokens of
// one request after another:  row r of request b is at position past + r - starts[b], whose slot is table[b][position / page] * page + position % page.
#include <algorithm>
#include <climits>

#include "cache_ops.h"

namespace tts {

namespace {

constexpr int THREADS = 256;

struct Sums {
  int64_t rows, pages;
};

struct Request {
  int past, length;  // tokens
  int have, need;    // pages
};

__device__ __forceinline__ Request request_of(const SlotsParams &p, int b) {
  Request r;
  r.length = max(p.lengths[b], 0);
  r.past = r.length - min(max(p.fresh[b], 0), r.length);
  r.have = min(r.past == 0 ? 0 : (r.past - 1) / p.page + 1, p.columns);
  r.need = min(r.length == 0 ? 0 : (r.length - 1) / p.page + 1, p.columns);
  return r;
}

// the last of `n` that begin at `begins` (ascending) at or before `at`
__device__ __forceinline__ int last_begun(const int *begins, int n, int at) {
  int low = 0, high = n - 1;
  while (low < high) {
    const int mid = (low + high + 1) / 2;
    if (begins[mid] <= at) low = mid;
    else high = mid - 1;
  }
  return low;
}

// Every workgroup adds up all requests' rows and pages for itself (a few KB from L2, and no second launch), then takes its share of the
// rows and of the pages; a row finds its request by halving in LDS.
// What bounds it: a launch and a chain of loads (lengths, then the table or the stack).  64 requests of a token each 4.0 us, 211 with 3742 rows 5.0.
__global__ __launch_bounds__(THREADS) void page_slots_kernel(SlotsParams p) {
  extern __shared__ int begins[];  // of the requests' rows, and of their new pages
  __shared__ Sums waves[THREADS / 64];
  const int tid = threadIdx.x, lane = tid % 64, each = (p.requests + THREADS - 1) / THREADS;
  const int from = min(tid * each, p.requests), to = min(from + each, p.requests);
  Sums sum = {0, 0};
  for (int b = from; b < to; b++) {
    const Request r = request_of(p, b);
    sum.rows += r.length - r.past, sum.pages += r.need - r.have;
  }
  Sums upto = sum;  // with those of the lanes before
  for (int d = 1; d < 64; d *= 2) {
    const int64_t rows = __shfl_up(upto.rows, d), pages = __shfl_up(upto.pages, d);
    if (lane >= d) upto.rows += rows, upto.pages += pages;
  }
  if (lane == 63) waves[tid / 64] = upto;
  __syncthreads();
  Sums at = {upto.rows - sum.rows, upto.pages - sum.pages}, all = {0, 0};
  for (int w = 0; w < THREADS / 64; w++) {
    if (w < tid / 64) at.rows += waves[w].rows, at.pages += waves[w].pages;
    all.rows += waves[w].rows, all.pages += waves[w].pages;
  }
  int *first_row = begins, *first_page = begins + p.requests;
  for (int b = from; b < to; b++) {
    const Request r = request_of(p, b);
    // (what lies behind 2^31 rows has none)
    first_row[b] = (int)min(at.rows, (int64_t)INT_MAX), first_page[b] = (int)min(at.pages, (int64_t)INT_MAX);
    if (blockIdx.x == 0) p.starts[b] = first_row[b];
    at.rows += r.length - r.past, at.pages += r.need - r.have;
  }
  const int count = min(max(p.count[0], 0), p.stack);
  if (blockIdx.x == 0 && tid == 0) {
    p.starts[p.requests] = (int)min(all.rows, (int64_t)INT_MAX);
    p.left[0] = (int)max((int64_t)count - all.pages, (int64_t)0);
  }
  __syncthreads();
  const int64_t step = (int64_t)gridDim.x * THREADS, mine = (int64_t)blockIdx.x * THREADS + tid;
  for (int64_t row = mine; row < p.rows; row += step) {
    int slot = -1, position = -1, owner = -1;
    if (row < all.rows) {
      owner = last_begun(first_row, p.requests, (int)row);
      const Request r = request_of(p, owner);
      position = r.past + (int)row - first_row[owner];
      const int column = position / p.page;
      if (column < p.columns) {
        int page = -1;
        if (column < r.have) page = p.table[owner * p.ld_table + column];
        else {
          const int64_t from_top = (int64_t)first_page[owner] + (column - r.have);
          if (from_top < count) page = p.free[count - 1 - from_top];
        }
        const int64_t at_slot = (int64_t)page * p.page + position % p.page;
        if (page >= 0 && at_slot <= INT_MAX) slot = (int)at_slot;
      }
    }
    p.slots[row] = slot, p.positions[row] = position, p.owners[row] = owner;
  }
  const int64_t taken = min(all.pages, (int64_t)INT_MAX);
  for (int64_t i = mine; i < taken; i += step) {
    const int b = last_begun(first_page, p.requests, (int)i);
    const Request r = request_of(p, b);
    p.table[b * p.ld_table + r.have + ((int)i - first_page[b])] = i < count ? p.free[count - 1 - i] : -1;
  }
}

}  // namespace

hipError_t launch_slots(const SlotsParams &p, hipStream_t s) {
  const int64_t groups = std::max<int64_t>(1, std::min<int64_t>((p.rows + THREADS - 1) / THREADS, 1024));
  page_slots_kernel<<<dim3((unsigned)groups), THREADS, 2 * sizeof(int) * std::max(p.requests, 1), s>>>(p);
  return hipGetLastError();
}

}  // namespace tts
