// pages.cu -- the paged cache's book-keeping and page copies, on the device:
// nothing here waits for the host, so the calls can sit in a CUDA graph.
//
// Every choice is by number, never by arrival: free pages are taken lowest
// first, in the order of the rows that ask, so equal states give equal tables.
#include <stdexcept>
#include <string>
#include "paged.cuh"

namespace jb {
namespace {

constexpr int kPlanThreads = 1024;

void check_launch(const char* what) {
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess)
    throw std::runtime_error(std::string(what) + " launch: " + cudaGetErrorString(e));
}

__device__ __forceinline__ bool row_ok(const jb_page_cache& c, int32_t r) {
  return r >= 0 && uint32_t(r) < c.n_rows;
}
__device__ __forceinline__ bool page_ok(const jb_page_cache& c, int32_t p) {
  return p >= 0 && uint32_t(p) < c.n_pages;
}

// Sums of pages saturate here: far above any pool, and two of them fit an int.
constexpr int kManyPages = 0x3FFFFFFF;

// Inclusive prefix sum of one value a thread (0 to kManyPages, where sums
// saturate) over the block; *total gets the sum.
__device__ __forceinline__ int block_scan(int v, int* total) {
  __shared__ int sums[32];
  const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5;
  int x = v;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int y = __shfl_up_sync(0xFFFFFFFFu, x, d);
    if (lane >= d) x = min(x + y, kManyPages);
  }
  if (lane == 31) sums[wid] = x;
  __syncthreads();
  if (wid == 0) {
    int s = lane < int(blockDim.x >> 5) ? sums[lane] : 0;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const int y = __shfl_up_sync(0xFFFFFFFFu, s, d);
      if (lane >= d) s = min(s + y, kManyPages);
    }
    sums[lane] = s;
  }
  __syncthreads();
  const int before = wid ? sums[wid - 1] : 0;
  *total = sums[31];
  __syncthreads();
  return min(before + x, kManyPages);
}

// Scratch of a plan over n rows: owner[n_rows], need[n], upto[n], from[n]
// (fork: the page to copy), fill[n] (fork: its tokens), page[n_pages].
struct Plan {
  int32_t *owner, *have, *need, *upto, *from, *free_list;
  __host__ __device__ Plan(int32_t* s, const jb_page_cache& c, uint64_t n)
      : owner(s), have(s + c.n_rows), need(have + n), upto(need + n), from(upto + n),
        free_list(from + n) {}
};

// owner[row] = the first i that names the row.
__device__ void claim_rows(const jb_page_cache& c, const int32_t* rows, uint32_t n, int32_t* owner) {
  for (uint32_t r = threadIdx.x; r < c.n_rows; r += blockDim.x) owner[r] = 0x7FFFFFFF;
  __syncthreads();
  for (uint32_t i = threadIdx.x; i < n; i += blockDim.x)
    if (row_ok(c, rows[i])) atomicMin(owner + rows[i], int32_t(i));
  __syncthreads();
}

// The lowest `total` free pages, in order, into list; returns how many there are.
__device__ int lowest_free(const jb_page_cache& c, int total, int32_t* list) {
  int found = 0;
  for (uint64_t base = 0; base < c.n_pages && found < total; base += blockDim.x) {
    const uint64_t p = base + threadIdx.x;
    const int is = p < c.n_pages && c.refs[p] == 0;
    int sum;
    const int rank = found + block_scan(is, &sum) - 1;
    if (is && rank < total) list[rank] = int32_t(p);
    found += sum;
  }
  __syncthreads();
  return min(found, total);
}

// need[i] pages wanted by row i (0 for those refused), in order: upto[i] is
// their running sum.  Returns the total.
__device__ int sum_needs(uint32_t n, const int32_t* need, int32_t* upto) {
  int total = 0;
  for (uint32_t base = 0; base < n; base += blockDim.x) {
    const uint32_t i = base + threadIdx.x;
    const int v = i < n ? need[i] : 0;
    int sum;
    const int incl = block_scan(v, &sum);
    if (i < n) upto[i] = min(total + incl, kManyPages);
    total = min(total + sum, kManyPages);
  }
  __syncthreads();
  return total;
}

__global__ void __launch_bounds__(kPlanThreads)
extend_kernel(const jb_page_cache c, const int32_t* rows, const int32_t* tokens, uint32_t n,
              int32_t* scratch) {
  const Plan s(scratch, c, n);
  claim_rows(c, rows, n, s.owner);
  const int64_t ps = c.page_size;
  for (uint32_t i = threadIdx.x; i < n; i += blockDim.x) {
    const int32_t r = rows[i], more = tokens[i];
    int need = -1, have = 0;
    if (row_ok(c, r) && s.owner[r] == int32_t(i) && more >= 0) {
      const int64_t len = max(c.lengths[r], 0);
      have = int((len + ps - 1) / ps);
      const int64_t want = (len + more + ps - 1) / ps;
      if (want <= c.max_pages && len + more <= 0x7FFFFFFF) need = max(int(want) - have, 0);
    }
    if (need < 0) atomicOr(c.status, kPagesBadRow);
    s.have[i] = need < 0 ? -1 : have;
    s.need[i] = max(need, 0);
  }
  __syncthreads();
  const int total = min(sum_needs(n, s.need, s.upto), int(c.n_pages));
  const int n_free = lowest_free(c, total, s.free_list);
  const int lane = threadIdx.x & 31;
  for (uint32_t i = threadIdx.x >> 5; i < n; i += blockDim.x >> 5) {
    if (s.have[i] < 0) continue;
    const int need = s.need[i], upto = s.upto[i];
    if (need > 0 && upto > n_free) {
      if (lane == 0) atomicOr(c.status, kPagesExhausted);
      continue;
    }
    int32_t* row = c.table + rows[i] * c.table_stride + s.have[i];
    for (int j = lane; j < need; j += 32) {
      const int32_t p = s.free_list[upto - need + j];
      row[j] = p;
      c.refs[p] = 1;
    }
    if (lane == 0) c.lengths[rows[i]] = max(c.lengths[rows[i]], 0) + tokens[i];
  }
}

__global__ void __launch_bounds__(kPlanThreads)
fork_kernel(const jb_page_cache c, const int32_t* parents, const int32_t* children, uint32_t n,
            int32_t* scratch) {
  const Plan s(scratch, c, n);
  claim_rows(c, children, n, s.owner);
  const int32_t ps = int32_t(c.page_size);
  for (uint32_t i = threadIdx.x; i < n; i += blockDim.x) {
    const int32_t p = parents[i], ch = children[i];
    int32_t len = -1, from = -1;
    if (row_ok(c, p) && row_ok(c, ch) && s.owner[ch] == int32_t(i) && c.lengths[ch] == 0) {
      len = max(c.lengths[p], 0);
      if (uint32_t((int64_t(len) + ps - 1) / ps) > c.max_pages) {
        len = -1;
      } else if (len % ps) {
        from = c.table[p * c.table_stride + len / ps];
        if (!page_ok(c, from)) from = -1;
      }
    }
    if (len < 0) atomicOr(c.status, kPagesBadRow);
    s.have[i] = len;
    s.from[i] = from;
    s.need[i] = from >= 0;
  }
  __syncthreads();
  const int total = min(sum_needs(n, s.need, s.upto), int(c.n_pages));
  const int n_free = lowest_free(c, total, s.free_list);
  const int lane = threadIdx.x & 31;
  for (uint32_t i = threadIdx.x >> 5; i < n; i += blockDim.x >> 5) {
    const int32_t len = s.have[i];
    const bool given = len >= 0 && (s.need[i] == 0 || s.upto[i] <= n_free);
    int32_t page = -1;
    if (!given) {
      if (lane == 0 && len >= 0) atomicOr(c.status, kPagesExhausted);
    } else {
      const int32_t* src = c.table + parents[i] * c.table_stride;
      int32_t* dst = c.table + children[i] * c.table_stride;
      const int whole = len / ps;
      for (int j = lane; j < whole; j += 32) {
        const int32_t p = src[j];
        const bool ok = page_ok(c, p);
        dst[j] = ok ? p : -1;
        if (ok) atomicAdd(c.refs + p, 1);
      }
      if (s.need[i]) page = s.free_list[s.upto[i] - 1];
      if (lane == 0) {
        if (len % ps) dst[whole] = page;
        if (page >= 0) c.refs[page] = 1;
        c.lengths[children[i]] = len;
      }
    }
    // what the copies read: from[i] -> upto[i], need[i] tokens
    __syncwarp();
    if (lane == 0) {
      s.upto[i] = page;
      s.need[i] = page >= 0 ? len % ps : 0;
    }
  }
}

__global__ void __launch_bounds__(256)
free_kernel(const jb_page_cache c, const int32_t* rows, uint32_t n) {
  const uint32_t i = blockIdx.x;
  const int32_t r = rows[i];
  if (!row_ok(c, r)) {
    if (threadIdx.x == 0) atomicOr(c.status, kPagesBadRow);
    return;
  }
  int32_t* row = c.table + r * c.table_stride;
  for (uint32_t j = threadIdx.x; j < c.max_pages; j += blockDim.x) {
    // exchanged, so that a row named twice gives its pages back once
    if (row[j] < 0) continue;
    const int32_t p = atomicExch(row + j, -1);
    if (page_ok(c, p)) atomicSub(c.refs + p, 1);
  }
  if (threadIdx.x == 0) c.lengths[r] = 0;
}

__global__ void __launch_bounds__(kPlanThreads)
adopt_claim_kernel(const jb_page_cache c, const int32_t* rows, uint32_t n, int32_t* owner) {
  claim_rows(c, rows, n, owner);
}

__global__ void __launch_bounds__(128)
adopt_kernel(const jb_page_cache c, const int32_t* rows, const int32_t* pages, int64_t pages_stride,
             uint32_t m, const int32_t* lengths, const int32_t* owner) {
  const uint32_t i = blockIdx.x;
  const int32_t r = rows[i];
  const int64_t ps = c.page_size;
  const int64_t len = lengths ? int64_t(lengths[i]) : int64_t(m) * ps;
  const int64_t take = (len + ps - 1) / ps;
  const bool ok = row_ok(c, r) && owner[r] == int32_t(i) && c.lengths[r] == 0 && len >= 0 &&
                  take <= m && take <= c.max_pages && len <= 0x7FFFFFFF;
  __syncthreads();
  if (!ok) {
    if (threadIdx.x == 0) atomicOr(c.status, kPagesBadRow);
    return;
  }
  int32_t* row = c.table + r * c.table_stride;
  for (int64_t j = threadIdx.x; j < take; j += blockDim.x) {
    const int32_t p = pages[i * pages_stride + j];
    const bool is = page_ok(c, p);
    row[j] = is ? p : -1;
    if (is) atomicAdd(c.refs + p, 1);
    else if (p != -1) atomicOr(c.status, kPagesBadToken);
  }
  if (threadIdx.x == 0) c.lengths[r] = int32_t(len);
}

// moves[0]: how many; then the pages that move and, n_pages on, where to.
__global__ void __launch_bounds__(kPlanThreads)
compact_plan_kernel(const jb_page_cache c, int32_t* remap, int32_t* moves) {
  int n_live = 0;
  for (uint64_t base = 0; base < c.n_pages; base += blockDim.x) {
    const uint64_t p = base + threadIdx.x;
    int sum;
    block_scan(p < c.n_pages && c.refs[p] > 0, &sum);
    n_live += sum;
  }
  int32_t* src = moves + 1;
  int32_t* dst = src + c.n_pages;
  int holes = 0, movers = 0;
  for (uint64_t base = 0; base < c.n_pages; base += blockDim.x) {
    const uint64_t p = base + threadIdx.x;
    const bool in = p < c.n_pages;
    const bool live = in && c.refs[p] > 0;
    const int hole = in && !live && int64_t(p) < n_live, mover = live && int64_t(p) >= n_live;
    int sum;
    const int hr = block_scan(hole, &sum);
    if (hole) dst[holes + hr - 1] = int32_t(p);
    holes += sum;
    const int mr = block_scan(mover, &sum);
    if (mover) src[movers + mr - 1] = int32_t(p);
    movers += sum;
    if (in) remap[p] = live ? int32_t(p) : -1;
  }
  __syncthreads();
  for (int j = threadIdx.x; j < movers; j += blockDim.x) {
    remap[src[j]] = dst[j];
    c.refs[dst[j]] = c.refs[src[j]];
    c.refs[src[j]] = 0;
  }
  if (threadIdx.x == 0) moves[0] = movers;
}

__global__ void __launch_bounds__(256) remap_table_kernel(const jb_page_cache c, const int32_t* remap) {
  const uint64_t total = uint64_t(c.n_rows) * c.max_pages;
  for (uint64_t i = uint64_t(blockIdx.x) * blockDim.x + threadIdx.x; i < total;
       i += uint64_t(gridDim.x) * blockDim.x) {
    int32_t* e = c.table + int64_t(i / c.max_pages) * c.table_stride + i % c.max_pages;
    const int32_t p = *e;
    if (p >= 0) *e = page_ok(c, p) ? remap[p] : -1;
  }
}

// Copies of pages src[i] -> dst[i] in keys, values and every layer, tokens[i]
// tokens of each (null: all); n pairs, or *n_device.
__global__ void __launch_bounds__(256)
copy_pages_kernel(const jb_page_cache c, const int32_t* src, const int32_t* dst,
                  const int32_t* tokens, uint32_t n, const int32_t* n_device) {
  const uint32_t pairs = n_device ? uint32_t(max(*n_device, 0)) : n;
  const uint32_t planes = 2 * c.n_layers;
  const uint32_t chunks = c.head_dim / 8;  // 16 bytes each
  for (uint64_t item = blockIdx.x; item < uint64_t(pairs) * planes; item += gridDim.x) {
    const uint32_t i = uint32_t(item / planes), plane = uint32_t(item % planes);
    const int32_t from = src[i], to = dst[i];
    if (!page_ok(c, from) || !page_ok(c, to)) {
      if (threadIdx.x == 0 && !tokens) atomicOr(c.status, kPagesBadToken);
      continue;
    }
    uint16_t* base = static_cast<uint16_t*>(plane & 1 ? c.v : c.k) + (plane >> 1) * c.layer_stride;
    const uint16_t* s = base + from * c.page_stride;
    uint16_t* d = base + to * c.page_stride;
    const uint32_t nt = tokens ? uint32_t(tokens[i]) : c.page_size;
    for (uint32_t u = threadIdx.x; u < nt * c.n_kv_heads * chunks; u += blockDim.x) {
      const uint32_t th = u / chunks, e = u % chunks;
      const int64_t off = (th / c.n_kv_heads) * c.token_stride + (th % c.n_kv_heads) * c.head_stride + e * 8;
      *reinterpret_cast<uint4*>(d + off) = *reinterpret_cast<const uint4*>(s + off);
    }
  }
}

uint32_t copy_grid(uint64_t items) { return uint32_t(items < 148 * 8 ? (items ? items : 1) : 148 * 8); }

}  // namespace

size_t pages_plan_words(const jb_page_cache& c, uint64_t n) {
  return size_t(c.n_rows) + 4 * size_t(n) + 2 * size_t(c.n_pages) + 1;
}

void launch_extend(const jb_page_cache& c, const int32_t* rows, const int32_t* tokens, uint32_t n,
                   int32_t* scratch, cudaStream_t st) {
  if (n == 0) return;
  extend_kernel<<<1, kPlanThreads, 0, st>>>(c, rows, tokens, n, scratch);
  check_launch("extend");
}

void launch_fork(const jb_page_cache& c, const int32_t* parents, const int32_t* children, uint32_t n,
                 int32_t* scratch, cudaStream_t st) {
  if (n == 0) return;
  fork_kernel<<<1, kPlanThreads, 0, st>>>(c, parents, children, n, scratch);
  check_launch("fork");
  const Plan s(scratch, c, n);
  copy_pages_kernel<<<copy_grid(uint64_t(n) * 2 * c.n_layers), 256, 0, st>>>(c, s.from, s.upto, s.need, n,
                                                                            nullptr);
  check_launch("fork copy");
}

void launch_free(const jb_page_cache& c, const int32_t* rows, uint32_t n, cudaStream_t st) {
  if (n == 0) return;
  free_kernel<<<n, 256, 0, st>>>(c, rows, n);
  check_launch("free");
}

void launch_adopt(const jb_page_cache& c, const int32_t* rows, const int32_t* pages,
                  int64_t pages_stride, uint32_t m, const int32_t* lengths, uint32_t n,
                  int32_t* scratch, cudaStream_t st) {
  if (n == 0) return;
  adopt_claim_kernel<<<1, kPlanThreads, 0, st>>>(c, rows, n, scratch);
  check_launch("adopt");
  adopt_kernel<<<n, 128, 0, st>>>(c, rows, pages, pages_stride, m, lengths, scratch);
  check_launch("adopt");
}

void launch_compact(const jb_page_cache& c, int32_t* remap, int32_t* scratch, cudaStream_t st) {
  if (c.n_pages == 0) return;
  compact_plan_kernel<<<1, kPlanThreads, 0, st>>>(c, remap, scratch);
  check_launch("compact");
  remap_table_kernel<<<148 * 4, 256, 0, st>>>(c, remap);
  check_launch("compact table");
  copy_pages_kernel<<<copy_grid(uint64_t(c.n_pages) * 2 * c.n_layers), 256, 0, st>>>(
      c, scratch + 1, scratch + 1 + c.n_pages, nullptr, 0, scratch);
  check_launch("compact copy");
}

void launch_copy_pages(const jb_page_cache& c, const int32_t* src, const int32_t* dst, uint32_t n,
                       cudaStream_t st) {
  if (n == 0) return;
  copy_pages_kernel<<<copy_grid(uint64_t(n) * 2 * c.n_layers), 256, 0, st>>>(c, src, dst, nullptr, n,
                                                                            nullptr);
  check_launch("copy pages");
}

}  // namespace jb
