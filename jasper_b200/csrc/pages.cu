// pages.cu -- the paged cache's book-keeping and page copies, on the device:
// nothing here waits for the host, so the calls can sit in a CUDA graph.
//
// Every choice is by number, never by arrival: free pages are taken lowest
// first, in the order of the rows that ask, so equal states give equal tables.
#include <mutex>
#include <stdexcept>
#include <string>
#include "paged.cuh"

namespace jb {
namespace {

constexpr int kPlanThreads = 1024;
constexpr int kPlanBlocks = 8;           // one cluster; a pool of one block's pages takes one block
constexpr int kThreadPages = 16;         // a thread's pages, next to each other
constexpr uint32_t kBlockPages = kPlanThreads * kThreadPages;
constexpr uint32_t kRowsInBlock = 2048;  // rows of a call, and of the table, whose book-keeping
constexpr uint32_t kOwnersInBlock = 8192;  // a block keeps in its shared memory
constexpr size_t kPlanShared = 4 * kRowsInBlock * 4 + kOwnersInBlock * 4 + kBlockPages * 2;

__device__ __forceinline__ bool row_ok(const jb_page_cache& c, int32_t r) {
  return r >= 0 && uint32_t(r) < c.n_rows;
}
__device__ __forceinline__ bool page_ok(const jb_page_cache& c, int32_t p) {
  return p >= 0 && uint32_t(p) < c.n_pages;
}

// Pages of up to 2^31 tokens.
__device__ __forceinline__ uint32_t pages_for(uint32_t tokens, uint32_t page_size) {
  return (tokens + page_size - 1) / page_size;
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

// ── plans ────────────────────────────────────────────────────────────────
// extend, fork and compact decide over the whole pool at once, in one cluster
// of blocks: block r looks at the r-th part of the pages, the blocks' counts
// meet in distributed shared memory, and then every page knows its rank.  What
// a call names (rows, in order) every block works out for itself, in its own
// shared memory, or where that is too small in its own part of the scratch.
// Latency is what bounds them: a few dependent reads and two cluster barriers.
// One block that walked the pool 1024 pages at a time took 45 us for 65,536.
// A pool that one block sees in one turn takes one block, without barriers.

__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
template <int BLOCKS>
__device__ __forceinline__ void cluster_arrive() {
  if (BLOCKS > 1) asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
}
template <int BLOCKS>
__device__ __forceinline__ void cluster_wait() {
  if (BLOCKS > 1) asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
  else __syncthreads();
}

// Every block's `mine`, exchanged: *before gets the sum over the blocks below
// this one; returns the sum over all.  `box` is BLOCKS ints of shared memory
// of its own for each exchange of a kernel.  All threads call it, and have
// waited for the barrier that every block arrives at first: only then have all
// blocks started, and may be written to.
template <int BLOCKS>
__device__ __forceinline__ int exchange(int mine, int* box, int* before) {
  *before = 0;
  if (BLOCKS == 1) {
    __syncthreads();
    return mine;
  }
  const uint32_t rank = cluster_rank();
  if (threadIdx.x < BLOCKS) {
    uint32_t at;
    asm("mapa.shared::cluster.u32 %0, %1, %2;"
        : "=r"(at) : "r"(static_cast<uint32_t>(__cvta_generic_to_shared(box + rank))), "r"(threadIdx.x));
    asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(at), "r"(mine) : "memory");
  }
  cluster_arrive<BLOCKS>();
  cluster_wait<BLOCKS>();
  int all = 0;
#pragma unroll
  for (int i = 0; i < BLOCKS; i++) {
    if (i < int(rank)) *before = min(*before + box[i], kManyPages);
    all = min(all + box[i], kManyPages);
  }
  return all;
}

// The block's part of the pool, and the pages of a thread's turn in it.
struct PoolPart {
  uint32_t begin, end;
  __device__ __forceinline__ PoolPart(const jb_page_cache& c, uint32_t blocks) {
    const uint32_t each = (c.n_pages + blocks * kThreadPages - 1) / (blocks * kThreadPages) * kThreadPages;
    begin = min(cluster_rank() * each, c.n_pages);
    end = min(begin + each, c.n_pages);
  }
  __device__ __forceinline__ uint32_t turns() const { return (end - begin + kBlockPages - 1) / kBlockPages; }
  __device__ __forceinline__ uint32_t first(uint32_t turn) const {
    return begin + turn * kBlockPages + threadIdx.x * kThreadPages;
  }
};

// Which of the thread's pages from `first` on are free, as bits.
__device__ __forceinline__ uint32_t free_bits(const jb_page_cache& c, const PoolPart& part, uint32_t first) {
  uint32_t bits = 0;
  if (first + kThreadPages <= part.end && (reinterpret_cast<uintptr_t>(c.refs) & 15) == 0) {
    int4 v[kThreadPages / 4];
#pragma unroll
    for (int i = 0; i < kThreadPages / 4; i++) v[i] = reinterpret_cast<const int4*>(c.refs + first)[i];
#pragma unroll
    for (int i = 0; i < kThreadPages / 4; i++)
      bits |= ((v[i].x <= 0) | (v[i].y <= 0) << 1 | (v[i].z <= 0) << 2 | (v[i].w <= 0) << 3) << (4 * i);
  } else {
    for (uint32_t i = 0; i < kThreadPages && first + i < part.end; i++) bits |= (c.refs[first + i] <= 0) << i;
  }
  return bits;
}

// A call's rows as a block keeps them: the row, what it has, the pages that it
// and those before it want (saturating), and more.
struct Wants {
  int32_t *owner, *row, *have, *upto, *extra;
  uint16_t* free_list;
  __device__ Wants(const jb_page_cache& c, uint32_t n, unsigned char* shared, int32_t* scratch) {
    int32_t* mem = reinterpret_cast<int32_t*>(shared);
    scratch += size_t(cluster_rank()) * (size_t(c.n_rows) + 4 * size_t(n));
    owner = c.n_rows <= kOwnersInBlock ? mem + 4 * kRowsInBlock : scratch;
    free_list = reinterpret_cast<uint16_t*>(mem + 4 * kRowsInBlock + kOwnersInBlock);
    const bool fits = n <= kRowsInBlock;
    int32_t* lists = fits ? mem : scratch + c.n_rows;
    const size_t step = fits ? kRowsInBlock : n;
    row = lists;
    have = lists + step;
    upto = lists + 2 * step;
    extra = lists + 3 * step;
  }
  __device__ void clear(const jb_page_cache& c) {
    for (uint32_t r = threadIdx.x; r < c.n_rows; r += blockDim.x) owner[r] = 0x7FFFFFFF;
    __syncthreads();
  }
  // owner[row] = the first i that names the row
  __device__ void claim(uint32_t i, int32_t r, bool ok) {
    row[i] = r;
    if (ok) atomicMin(owner + r, int32_t(i));
  }
  // upto holds what each row wants, and then the running sum; returns the total
  __device__ int sum(uint32_t n) {
    int total = 0;
    for (uint32_t base = 0; base < n; base += blockDim.x) {
      const uint32_t i = base + threadIdx.x;
      const int v = i < n ? upto[i] : 0;
      int all;
      const int incl = block_scan(v, &all);
      if (i < n) upto[i] = min(total + incl, kManyPages);
      total = min(total + all, kManyPages);
    }
    __syncthreads();
    return total;
  }
  // the row that the rank-th new page goes to: the first with upto > rank
  __device__ uint32_t row_of(int rank, uint32_t n) const {
    uint32_t low = 0, high = n - 1;
    while (low < high) {
      const uint32_t mid = (low + high) / 2;
      if (upto[mid] > rank) high = mid;
      else low = mid + 1;
    }
    return low;
  }
};

// Finds the lowest free pages and calls give(row of the call, rank, page) for
// each rank below `total`; `bits0` are the thread's free pages of its first
// turn, `before` the free pages of the blocks below.  The pages go through a
// list (kBlockPages entries), so that each is a thread's of its own: a thread
// that gave its 16 away one by one took 4 us.  The row is searched for at
// kMarks ranks only, and stepped to between.
constexpr int kMarks = kPlanThreads;
template <typename F>
__device__ __forceinline__ void hand_out(const jb_page_cache& c, const PoolPart& part, uint32_t bits0, int before,
                                         int total, const Wants& w, uint32_t n_rows, F&& give) {
  __shared__ int marks[kMarks];
  for (uint32_t turn = 0; turn < part.turns() && before < total; turn++) {
    const uint32_t first = part.first(turn), base = part.begin + turn * kBlockPages;
    uint32_t bits = turn == 0 ? bits0 : free_bits(c, part, first);
    int all;
    const int n = __popc(bits);
    int at = block_scan(n, &all) - n;
    for (; bits; bits &= bits - 1) w.free_list[at++] = uint16_t(first - base + __ffs(bits) - 1);
    const int count = min(all, total - before);
    const int shift = max(0, 22 - __clz(count - 1 | 1));  // count <= kMarks << shift
    if (int(threadIdx.x) << shift < count) marks[threadIdx.x] = w.row_of(before + (int(threadIdx.x) << shift), n_rows);
    __syncthreads();
    for (int k = threadIdx.x; k < count; k += kPlanThreads) {
      int i = marks[k >> shift];
      while (w.upto[i] <= before + k) i++;
      give(uint32_t(i), before + k, int32_t(base + w.free_list[k]));
    }
    __syncthreads();
    before += all;
  }
}

// The thread's free pages of its first turn, and the block's count of all.
__device__ __forceinline__ int count_free(const jb_page_cache& c, const PoolPart& part, uint32_t bits0) {
  int n = __popc(bits0);
  for (uint32_t turn = 1; turn < part.turns(); turn++) n += __popc(free_bits(c, part, part.first(turn)));
  int all;
  block_scan(n, &all);
  return all;
}

template <int BLOCKS>
__global__ void __cluster_dims__(BLOCKS, 1, 1) __launch_bounds__(kPlanThreads)
extend_kernel(const jb_page_cache c, const int32_t* rows, const int32_t* tokens, uint32_t n, int32_t* scratch) {
  extern __shared__ __align__(16) unsigned char shared[];
  __shared__ int box[BLOCKS];
  follow();
  cluster_arrive<BLOCKS>();
  const PoolPart part(c, BLOCKS);
  const uint32_t bits = free_bits(c, part, part.first(0));
  Wants w(c, n, shared, scratch);
  // A turn of rows: what they name and have, read before anything waits.
  struct Turn {
    int32_t r = -1, more = -1, len = 0;
    __device__ Turn(const jb_page_cache& c, const int32_t* rows, const int32_t* tokens, uint32_t i, uint32_t n) {
      if (i >= n) return;
      r = rows[i];
      more = tokens[i];
      if (row_ok(c, r)) len = max(c.lengths[r], 0);
    }
  };
  const Turn first(c, rows, tokens, threadIdx.x, n);
  w.clear(c);
  for (uint32_t i = threadIdx.x; i < n; i += blockDim.x) {
    const Turn t = i == threadIdx.x ? first : Turn(c, rows, tokens, i, n);
    w.claim(i, t.r, row_ok(c, t.r));
    w.have[i] = t.len;
    w.extra[i] = t.more;
  }
  __syncthreads();
  const bool speaks = cluster_rank() == 0;  // one block sets status bits and lengths
  for (uint32_t i = threadIdx.x; i < n; i += blockDim.x) {
    const int32_t r = w.row[i], more = w.extra[i];
    const uint32_t len = uint32_t(w.have[i]), sum = len + uint32_t(max(more, 0));
    const uint32_t have = pages_for(len, c.page_size), pages = pages_for(sum, c.page_size);
    const bool ok = row_ok(c, r) && w.owner[r] == int32_t(i) && more >= 0 && sum <= 0x7FFFFFFFu && pages <= c.max_pages;
    if (!ok && speaks) atomicOr(c.status, kPagesBadRow);
    w.have[i] = ok ? int32_t(have) : -1;
    w.upto[i] = ok && pages > have ? int32_t(pages - have) : 0;
    w.extra[i] = ok ? int32_t(sum) : -1;  // the row's length behind the call
  }
  __syncthreads();
  const int total = w.sum(n);
  int before;
  cluster_wait<BLOCKS>();
  const int n_free = exchange<BLOCKS>(count_free(c, part, bits), box, &before);  // all lengths are read behind this
  hand_out(c, part, bits, before, min(total, n_free), w, n, [&](uint32_t i, int rank, int32_t page) {
    if (w.upto[i] > n_free) return;
    const int into = rank - (i ? w.upto[i - 1] : 0);
    c.table[w.row[i] * c.table_stride + w.have[i] + into] = page;
    c.refs[page] = 1;
  });
  if (!speaks) return;
  // A row that stays as it was is marked, so that an append to its last token
  // does not take the place of an old one.
  for (uint32_t i = threadIdx.x; i < n; i += blockDim.x) {
    const int32_t r = w.row[i];
    if (!row_ok(c, r) || w.owner[r] != int32_t(i)) continue;
    const bool ok = w.have[i] >= 0;
    const bool none = ok && pages_for(uint32_t(w.extra[i]), c.page_size) <= uint32_t(w.have[i]);
    const bool given = none || (ok && w.upto[i] <= n_free);
    if (given) c.lengths[r] = w.extra[i];
    else if (ok) atomicOr(c.status, kPagesExhausted);
    if (!c.marks) continue;
    if (!given) atomicOr(c.marks + r, kMarkRefused);
    else atomicAnd(c.marks + r, w.have[i] == 0 ? 0 : kMarkAdopted);  // an empty row begins anew
  }
}

// copies: from[n], to[n] (-1: none), tokens[n], length[n] (-1: pair refused);
// the copying kernel shares the whole pages
template <int BLOCKS>
__global__ void __cluster_dims__(BLOCKS, 1, 1) __launch_bounds__(kPlanThreads)
fork_kernel(const jb_page_cache c, const int32_t* parents, const int32_t* children, uint32_t n, int32_t* copies,
            int32_t* scratch) {
  extern __shared__ __align__(16) unsigned char shared[];
  __shared__ int box[BLOCKS];
  follow();
  cluster_arrive<BLOCKS>();
  const PoolPart part(c, BLOCKS);
  const uint32_t bits = free_bits(c, part, part.first(0));
  Wants w(c, n, shared, scratch);
  struct Turn {
    int32_t child = -1, len = -1, from = -1, mark = 0;  // len -1: no pair to fork
    __device__ Turn(const jb_page_cache& c, const int32_t* parents, const int32_t* children, uint32_t i, uint32_t n) {
      if (i >= n) return;
      const int32_t p = parents[i];
      child = children[i];
      const int32_t there = row_ok(c, child) ? c.lengths[child] : -1;
      const int32_t held = row_ok(c, p) ? max(c.lengths[p], 0) : -1;
      if (there != 0 || held < 0 || pages_for(uint32_t(held), c.page_size) > c.max_pages) return;
      len = held;
      if (c.marks) mark = c.marks[p];
      const uint32_t whole = uint32_t(len) / c.page_size;
      if (whole * c.page_size == uint32_t(len)) return;
      from = c.table[p * c.table_stride + whole];
      if (!page_ok(c, from)) from = -1;
    }
  };
  const Turn first(c, parents, children, threadIdx.x, n);
  w.clear(c);
  for (uint32_t i = threadIdx.x; i < n; i += blockDim.x) {
    const Turn t = i == threadIdx.x ? first : Turn(c, parents, children, i, n);
    w.claim(i, t.child, row_ok(c, t.child));
    w.have[i] = t.len;
    w.extra[i] = t.from;
  }
  __syncthreads();
  const bool speaks = cluster_rank() == 0;
  int32_t *from_of = copies, *to_of = copies + n, *tokens_of = to_of + n, *length_of = tokens_of + n;
  for (uint32_t i = threadIdx.x; i < n; i += blockDim.x) {
    if (w.have[i] >= 0 && w.owner[w.row[i]] != int32_t(i)) w.have[i] = w.extra[i] = -1;
    const int32_t len = w.have[i], from = w.extra[i];
    w.upto[i] = from >= 0;
    if (speaks) {
      if (len < 0) atomicOr(c.status, kPagesBadRow);
      from_of[i] = from;
      to_of[i] = -1;
      tokens_of[i] = from >= 0 ? int32_t(uint32_t(len) % c.page_size) : 0;
    }
  }
  __syncthreads();
  const int total = w.sum(n);
  int before;
  cluster_wait<BLOCKS>();
  const int n_free = exchange<BLOCKS>(count_free(c, part, bits), box, &before);  // rows are read, and copies set, behind this
  hand_out(c, part, bits, before, min(total, n_free), w, n, [&](uint32_t i, int, int32_t page) {
    c.table[w.row[i] * c.table_stride + uint32_t(w.have[i]) / c.page_size] = page;
    c.refs[page] = 1;
    to_of[i] = page;
  });
  if (!speaks) return;
  for (uint32_t i = threadIdx.x; i < n; i += blockDim.x) {
    const int32_t len = w.have[i];
    const bool given = len >= 0 && (w.extra[i] < 0 || w.upto[i] <= n_free);
    length_of[i] = given ? len : -1;
    if (given) {
      c.lengths[w.row[i]] = len;
      // A refused parent's last token is an old one in its child too.  Where
      // the parent ends as it was adopted, the child's last page is its own.
      // An empty parent may be another pair's child: its mark is not read.
      if (c.marks) {
        const int32_t mark = len == 0 ? 0 : i == threadIdx.x ? first.mark : c.marks[parents[i]];
        const int32_t adopted = mark & kMarkAdopted;
        c.marks[w.row[i]] = (mark & kMarkRefused) | (len > adopted ? adopted : 0);
      }
    } else if (len >= 0) {
      atomicOr(c.status, kPagesExhausted);
    }
  }
}

constexpr int kFreeThreads = 256;
__global__ void __launch_bounds__(kFreeThreads)
free_kernel(const jb_page_cache c, const int32_t* rows) {
  follow();
  const uint32_t i = blockIdx.x;
  const int32_t r = rows[i];
  if (!row_ok(c, r)) {
    if (threadIdx.x == 0) atomicOr(c.status, kPagesBadRow);
    return;
  }
  int32_t* row = c.table + r * c.table_stride;
  // four entries of a thread at once, for the latency of three dependent steps
  constexpr int kAtOnce = 4;
  for (uint64_t j0 = threadIdx.x; j0 < c.max_pages; j0 += kAtOnce * kFreeThreads) {
    int32_t p[kAtOnce];
#pragma unroll
    for (int k = 0; k < kAtOnce; k++) {
      const uint64_t j = j0 + k * kFreeThreads;
      p[k] = j < c.max_pages ? row[j] : -1;
    }
    // exchanged, so that a row named twice gives its pages back once
#pragma unroll
    for (int k = 0; k < kAtOnce; k++)
      if (p[k] >= 0) p[k] = atomicExch(row + j0 + k * kFreeThreads, -1);
#pragma unroll
    for (int k = 0; k < kAtOnce; k++)
      if (page_ok(c, p[k])) atomicSub(c.refs + p[k], 1);
  }
  if (threadIdx.x == 0) {
    c.lengths[r] = 0;
    if (c.marks) c.marks[r] = 0;
  }
}

// owner[row] = the first i that names the row
__global__ void __launch_bounds__(kPlanThreads)
adopt_claim_kernel(const jb_page_cache c, const int32_t* rows, uint32_t n, int32_t* owner) {
  follow();
  for (uint32_t r = threadIdx.x; r < c.n_rows; r += blockDim.x) owner[r] = 0x7FFFFFFF;
  __syncthreads();
  for (uint32_t i = threadIdx.x; i < n; i += blockDim.x)
    if (row_ok(c, rows[i])) atomicMin(owner + rows[i], int32_t(i));
}

__global__ void __launch_bounds__(128)
adopt_kernel(const jb_page_cache c, const int32_t* rows, const int32_t* pages, int64_t pages_stride,
             uint32_t m, const int32_t* lengths, const int32_t* owner) {
  follow();
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
  if (threadIdx.x == 0) {
    c.lengths[r] = int32_t(len);
    if (c.marks) c.marks[r] = len % ps ? int32_t(len) : 0;
  }
}

// moves[0]: how many; then the pages that move and, n_pages on, where to.
template <int BLOCKS>
__global__ void __cluster_dims__(BLOCKS, 1, 1) __launch_bounds__(kPlanThreads)
compact_plan_kernel(const jb_page_cache c, int32_t* remap, int32_t* moves) {
  __shared__ int live_box[BLOCKS], hole_box[BLOCKS], mover_box[BLOCKS];
  follow();
  cluster_arrive<BLOCKS>();
  const PoolPart part(c, BLOCKS);
  const uint32_t bits0 = free_bits(c, part, part.first(0));
  int unused;
  const int free_here = count_free(c, part, bits0);
  cluster_wait<BLOCKS>();
  const int n_live = exchange<BLOCKS>(int(part.end - part.begin) - free_here, live_box, &unused);
  // of the thread's pages from `first` on: holes, free and below n_live, and
  // movers, live and at or above it
  auto split = [&](uint32_t first, uint32_t bits, uint32_t* holes, uint32_t* movers) {
    const int inside = min(max(int(part.end) - int(first), 0), kThreadPages);
    const int below = min(max(n_live - int(first), 0), inside);
    *holes = bits & ((1u << below) - 1);
    *movers = ~bits & ((1u << inside) - 1) & ~((1u << below) - 1);
  };
  int n_holes = 0, n_movers = 0;
  for (uint32_t turn = 0; turn < part.turns(); turn++) {
    uint32_t holes, movers;
    split(part.first(turn), turn == 0 ? bits0 : free_bits(c, part, part.first(turn)), &holes, &movers);
    n_holes += __popc(holes);
    n_movers += __popc(movers);
  }
  int holes_here, movers_here, holes_before, movers_before;
  block_scan(n_holes, &holes_here);
  block_scan(n_movers, &movers_here);
  exchange<BLOCKS>(holes_here, hole_box, &holes_before);
  const int n_moves = exchange<BLOCKS>(movers_here, mover_box, &movers_before);
  int32_t* src = moves + 1;
  int32_t* dst = src + c.n_pages;
  for (uint32_t turn = 0; turn < part.turns(); turn++) {
    const uint32_t first = part.first(turn);
    const uint32_t bits = turn == 0 ? bits0 : free_bits(c, part, first);
    uint32_t holes, movers;
    split(first, bits, &holes, &movers);
    int all, at = holes_before + block_scan(__popc(holes), &all) - __popc(holes);
    holes_before += all;
    for (uint32_t m = holes; m; m &= m - 1) dst[at++] = int32_t(first + __ffs(m) - 1);
    at = movers_before + block_scan(__popc(movers), &all) - __popc(movers);
    movers_before += all;
    for (uint32_t m = movers; m; m &= m - 1) src[at++] = int32_t(first + __ffs(m) - 1);
    for (uint32_t i = 0; i < kThreadPages && first + i < part.end; i++)
      if (!(movers >> i & 1)) remap[first + i] = bits >> i & 1 ? -1 : int32_t(first + i);
  }
  if (cluster_rank() == 0 && threadIdx.x == 0) moves[0] = n_moves;
  cluster_arrive<BLOCKS>();
  cluster_wait<BLOCKS>();
  for (int j = cluster_rank() * kPlanThreads + threadIdx.x; j < n_moves; j += BLOCKS * kPlanThreads) {
    remap[src[j]] = dst[j];
    c.refs[dst[j]] = c.refs[src[j]];
    c.refs[src[j]] = 0;
  }
}

// ── copies ───────────────────────────────────────────────────────────────
// Pages src[i] -> dst[i] in keys, values and every layer, tokens[i] tokens of
// each (null: all); n pairs, or *n_device.  HBM bounds it: a warp takes some 4
// KB pieces of one page of one plane, eight 16-byte reads of each lane before
// the first write (301 pages of 1 MB: 101 us, 6.3 TB/s; with four reads and
// more warps 106).  On the way, with `remap` the rows' table is rewritten, and
// with `parents` the whole pages of forked rows are shared.
constexpr int kCopyThreads = 256, kCopyDepth = 8;

struct CopyArgs {
  jb_page_cache c;
  const int32_t *src, *dst, *tokens;
  uint32_t n;
  const int32_t* n_device;
  const int32_t* remap;
  const int32_t *parents, *children, *lengths;
  // a page's tokens lie as runs: `flat`, all in one run; `by_head`, a run for
  // each head; else a run for each token and head
  bool flat, by_head;
  uint32_t run;  // pieces of a plane's page that a warp takes one after the other
};

__global__ void __launch_bounds__(kCopyThreads, 3) copy_pages_kernel(const __grid_constant__ CopyArgs a) {
  const jb_page_cache& c = a.c;
  follow();
  if (a.remap) {
    const uint64_t total = uint64_t(c.n_rows) * c.max_pages;
    for (uint64_t i = uint64_t(blockIdx.x) * kCopyThreads + threadIdx.x; i < total; i += uint64_t(gridDim.x) * kCopyThreads) {
      int32_t* e = c.table + int64_t(i / c.max_pages) * c.table_stride + i % c.max_pages;
      const int32_t p = *e;
      if (p >= 0) *e = page_ok(c, p) ? a.remap[p] : -1;
    }
  }
  const uint32_t lane = threadIdx.x & 31;
  const uint64_t step = uint64_t(gridDim.x) * (kCopyThreads / 32);
  const uint64_t warp = uint64_t(blockIdx.x) * (kCopyThreads / 32) + threadIdx.x / 32;
  if (a.parents)
    for (uint64_t i = warp; i < a.n; i += step) {
      const int32_t len = a.lengths[i], whole = len / int32_t(c.page_size);
      if (len < 0) continue;
      const int32_t* from = c.table + a.parents[i] * c.table_stride;
      int32_t* to = c.table + a.children[i] * c.table_stride;
      for (int j = lane; j < whole; j += 32) {
        const int32_t p = from[j];
        const bool ok = page_ok(c, p);
        to[j] = ok ? p : -1;
        if (ok) atomicAdd(c.refs + p, 1);
      }
      if (lane == 0 && len % int32_t(c.page_size) && a.src[i] < 0) to[whole] = -1;
    }
  const uint32_t pairs = a.n_device ? min(uint32_t(max(*a.n_device, 0)), a.n) : a.n;
  const uint32_t planes = 2 * c.n_layers, row = c.head_dim / 8;  // 16-byte vectors of a head
  const uint32_t full = c.page_size * c.n_kv_heads * row;
  const uint32_t run = a.run * 32 * kCopyDepth, runs = (full + run - 1) / run;
  const uint32_t units = pairs * planes * runs;  // below 2^31: check_copies()
  for (uint32_t unit = uint32_t(warp); unit < units; unit += uint32_t(step)) {
    const uint32_t item = unit / runs, i = item / planes, plane = item - i * planes;
    const uint32_t begin = (unit - item * runs) * run;
    const int32_t from = a.src[i], to = a.dst[i];
    const uint32_t nt = a.tokens ? uint32_t(a.tokens[i]) : c.page_size;
    if (!page_ok(c, from) || !page_ok(c, to)) {
      if (lane == 0 && !a.tokens) atomicOr(c.status, kPagesBadToken);
      continue;
    }
    const uint32_t count = min(nt * c.n_kv_heads * row, begin + run);
    uint16_t* base = static_cast<uint16_t*>(plane & 1 ? c.v : c.k) + int64_t(plane >> 1) * c.layer_stride;
    const uint16_t* s = base + from * c.page_stride;
    uint16_t* d = base + to * c.page_stride;
    for (uint32_t v0 = begin + lane; v0 < count; v0 += 32 * kCopyDepth) {
      uint4 v[kCopyDepth];
      int64_t off[kCopyDepth];
#pragma unroll
      for (int k = 0; k < kCopyDepth; k++) {
        const uint32_t u = v0 + 32 * k;
        if (a.flat) {
          off[k] = int64_t(u) * 8;
        } else if (a.by_head) {
          const uint32_t h = u / (nt * row);
          off[k] = int64_t(h) * c.head_stride + int64_t(u - h * nt * row) * 8;
        } else {
          const uint32_t th = u / row, t = th / c.n_kv_heads;
          off[k] = int64_t(t) * c.token_stride + int64_t(th - t * c.n_kv_heads) * c.head_stride + int64_t(u - th * row) * 8;
        }
        if (u < count) v[k] = *reinterpret_cast<const uint4*>(s + off[k]);
      }
#pragma unroll
      for (int k = 0; k < kCopyDepth; k++)
        if (v0 + 32 * k < count) *reinterpret_cast<uint4*>(d + off[k]) = v[k];
    }
  }
}

void launch_copies(CopyArgs a, cudaStream_t st) {
  const jb_page_cache& c = a.c;
  const int64_t dim = c.head_dim, heads = c.n_kv_heads, ps = c.page_size;
  const bool token_rows = c.head_stride == dim && c.token_stride == heads * dim;  // a token's heads, then the next token
  a.by_head = c.token_stride == dim;
  a.flat = token_rows || (a.by_head && a.tokens == nullptr && c.head_stride == ps * dim);
  const uint64_t full = uint64_t(c.page_size) * c.n_kv_heads * (c.head_dim / 8);
  constexpr uint64_t kMost = 148 * 8;  // blocks: 8 an SM
  const uint64_t pieces = (full + 32 * kCopyDepth - 1) / (32 * kCopyDepth);
  uint64_t units = uint64_t(a.n) * 2 * c.n_layers * pieces;
  a.run = uint32_t(units / (kMost * (kCopyThreads / 32) * 2));  // two units at least for every warp
  a.run = a.run < 1 ? 1 : a.run > pieces ? uint32_t(pieces) : a.run;
  units = uint64_t(a.n) * 2 * c.n_layers * ((pieces + a.run - 1) / a.run);
  const uint64_t blocks = (units + kCopyThreads / 32 - 1) / (kCopyThreads / 32);
  launch("copy pages", copy_pages_kernel, dim3(uint32_t(blocks < kMost ? (blocks ? blocks : 1) : kMost)), kCopyThreads,
         0, st, 0, a);
}

// Launches a plan kernel; its shared memory is allowed once per device.
template <auto Kernel, int BLOCKS, typename... A>
void launch_plan_of(const char* what, cudaStream_t st, A... args) {
  static std::mutex m;
  static uint64_t ready = 0;
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (dev >= 64) throw std::runtime_error("device index out of range");
  {
    std::lock_guard<std::mutex> lock(m);
    if (e == cudaSuccess && !(ready >> dev & 1)) {
      e = cudaFuncSetAttribute(Kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, int(kPlanShared));
      if (e == cudaSuccess) ready |= uint64_t(1) << dev;
    }
  }
  if (e != cudaSuccess) {
    cudaGetLastError();
    throw std::runtime_error(std::string(what) + ": " + cudaGetErrorString(e));
  }
  launch(what, Kernel, dim3(BLOCKS), kPlanThreads, kPlanShared, st, 0, args...);
}
#define JB_LAUNCH_PLAN(kernel, what, c, ...)                                                    \
  do {                                                                                          \
    if ((c).n_pages <= kBlockPages) launch_plan_of<kernel<1>, 1>(what, __VA_ARGS__);            \
    else launch_plan_of<kernel<kPlanBlocks>, kPlanBlocks>(what, __VA_ARGS__);                   \
  } while (0)

}  // namespace

// What the copies count in 32 bits.
void check_copies(const jb_page_cache& c, uint64_t n) {
  if (uint64_t(c.page_size) * c.n_kv_heads * (c.head_dim / 8) > 0x7FFFFFFFull)
    throw std::invalid_argument("a page is too large");
  if (n * 2 * c.n_layers > (uint64_t(1) << 30)) throw std::invalid_argument("too many pages for one call");
}

size_t pages_plan_words(const jb_page_cache& c, uint64_t n) {
  const size_t lists = c.n_rows > kOwnersInBlock || n > kRowsInBlock ? kPlanBlocks * (size_t(c.n_rows) + 4 * size_t(n)) : 0;
  return lists + 4 * size_t(n) + 2 * size_t(c.n_pages) + 1;
}

void launch_extend(const jb_page_cache& c, const int32_t* rows, const int32_t* tokens, uint32_t n,
                   int32_t* scratch, cudaStream_t st) {
  if (n == 0) return;
  JB_LAUNCH_PLAN(extend_kernel, "extend", c, st, c, rows, tokens, n, scratch);
}

void launch_fork(const jb_page_cache& c, const int32_t* parents, const int32_t* children, uint32_t n,
                 int32_t* scratch, cudaStream_t st) {
  if (n == 0) return;
  JB_LAUNCH_PLAN(fork_kernel, "fork", c, st, c, parents, children, n, scratch, scratch + 4 * size_t(n));
  CopyArgs a{};
  a.c = c;
  a.n = n;
  a.src = scratch;
  a.dst = a.src + n;
  a.tokens = a.dst + n;
  a.lengths = a.tokens + n;
  a.parents = parents;
  a.children = children;
  launch_copies(a, st);
}

void launch_free(const jb_page_cache& c, const int32_t* rows, uint32_t n, cudaStream_t st) {
  if (n == 0) return;
  launch("free", free_kernel, dim3(n), kFreeThreads, 0, st, 0, c, rows);
}

void launch_adopt(const jb_page_cache& c, const int32_t* rows, const int32_t* pages,
                  int64_t pages_stride, uint32_t m, const int32_t* lengths, uint32_t n,
                  int32_t* scratch, cudaStream_t st) {
  if (n == 0) return;
  launch("adopt", adopt_claim_kernel, dim3(1), kPlanThreads, 0, st, 0, c, rows, n, scratch);
  launch("adopt", adopt_kernel, dim3(n), 128, 0, st, 0, c, rows, pages, pages_stride, m, lengths, scratch);
}

void launch_compact(const jb_page_cache& c, int32_t* remap, int32_t* scratch, cudaStream_t st) {
  if (c.n_pages == 0) return;
  JB_LAUNCH_PLAN(compact_plan_kernel, "compact", c, st, c, remap, scratch);
  CopyArgs a{};
  a.c = c;
  a.n = c.n_pages;
  a.n_device = scratch;
  a.src = scratch + 1;
  a.dst = a.src + c.n_pages;
  a.remap = remap;
  launch_copies(a, st);
}

void launch_copy_pages(const jb_page_cache& c, const int32_t* src, const int32_t* dst, uint32_t n,
                       cudaStream_t st) {
  if (n == 0) return;
  CopyArgs a{};
  a.c = c;
  a.n = n;
  a.src = src;
  a.dst = dst;
  launch_copies(a, st);
}

}  // namespace jb
