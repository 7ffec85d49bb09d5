// attend.cu -- attention of one new token of each row over the paged cache.
//
// out = sum_t p_t v_t, p = softmax(scale * q . k_t) over the tokens attended
// to, in one pass over keys and values with the running reference r and sum l
// of the softmax: weights are 2^(s - r), and a score far above r moves it and
// rescales what was gathered.
//
// What bounds it: every key and value is read once and used for a group of at
// most 16 query heads, 2 to 32 flops a byte, so HBM.  The rest is keeping
// enough bytes in flight and every SM equally long at work:
//
//  * A warp is a worker of its own.  All rows' tiles of 16 tokens, one row's
//    head after the other, form one line, and worker w of W takes the w-th of
//    W equal parts, whatever the rows' lengths.  A row's head that lies in one
//    part is finished there; one that spans several leaves a part result in
//    each, and a second kernel joins them in order (no atomics: equal inputs
//    give equal bits).
//  * The worker's tiles stream through its own ring of STAGES tiles in shared
//    memory by 16-byte cp.async, over the borders of rows, with no block-wide
//    barrier.  Tokens that are not attended to are not read: their rows are
//    filled with zeros, whatever the cache holds there.
//  * Products run on mma.sync m16n8k16 with tokens (then head elements) as the
//    16 rows and query heads as the 8 columns, S^T = K Q^T and O^T = V^T P^T,
//    so a group of 8 heads wastes nothing; movmatrix turns the weights from
//    accumulator to operand.  tcgen05 would take tiles of 64 or 128 tokens,
//    shared by warps, and the weights through tensor memory and back; the
//    tensor pipe is 15 % busy here, so it has nothing to give.
//  * A weight enters the second product as the sum of two 16-bit values (its
//    rounding, and the rounding of what that left), which carry it to 2^-17 of
//    itself in bfloat16, 2^-23 in float16.  The result is rounded to 2^-8 and
//    2^-11 of itself once, 500 times as much or more; one 16-bit value would
//    have cost as much as that rounding.  l sums the float32 weights.
//  * An infinite value times a weight's second half, or a weight that rounds to
//    zero, would be NaN, so a result that is not finite is looked at again: what
//    the values attended to hold in its place decides (settle()).
//  * Short rows take no part in this: warps, blocks or clusters of blocks have
//    a row's head each, and join in (distributed) shared memory.
//
// Measured: 64 rows of 1 to 8191 tokens, 8 heads of 128, bfloat16, 167 us, 6.4
// TB/s (0.99 of the measured copy rate); 400 k + 333 k tokens, float16, 446 us,
// 6.7 TB/s; one row of 1000 tokens 5.4 us in a table of its width, 9.3 in one of
// 16,000 tokens or more.
#include <cmath>
#include <mutex>
#include <stdexcept>
#include <string>
#include "paged.cuh"

namespace jb {
namespace {

constexpr uint32_t kFullMask = 0xFFFFFFFFu;
constexpr int kMaxListed = 1024;  // queries whose lengths a block keeps in shared memory
constexpr int TK = 16;            // tokens of a tile
// A weight is 2^(s - r): r is set kRefBelow below the largest score and stays
// until a score is kRefRoom above it.  In float16 weights reach 2^15, inside its
// range, and the largest is at least 2^6, so that a weight that float16 drops is
// below 2^-31 of the largest in the same worker's part: 2^18 of them, a part of a
// batch of 4 10^8 tokens, weigh less than half the result's rounding.  (12 below
// and room of 3 would drop 64 times less, for 1.4 % of the time of two long rows
// and 3 % of 1000 short ones.)  bfloat16 has float32's range, for weights and for
// values, and a sum of large values with weights above 1 would overflow: there r
// lies 8 above the largest score, weights are at most 1, and hundreds of tokens of
// equal weight with values near the end of the range still have a finite sum.

template <typename T>
struct Mma;
template <>
struct Mma<__half> {
  static constexpr uint32_t kExponent = 0x7C00;  // the bits of an infinity without its sign
  static constexpr float kRefBelow = 6.0f, kRefRoom = 15.0f;
  static __device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
  // (a, b) to 16 bits, and what that left, to 16 bits again
  static __device__ __forceinline__ void split(float a, float b, uint32_t& hi, uint32_t& lo) {
    const __half2 h = __floats2half2_rn(a, b);
    const float2 f = __half22float2(h);
    const __half2 l = __floats2half2_rn(a - f.x, b - f.y);
    hi = *reinterpret_cast<const uint32_t*>(&h);
    lo = *reinterpret_cast<const uint32_t*>(&l);
  }
  static __device__ __forceinline__ __half from(float v) { return __float2half_rn(v); }
};
template <>
struct Mma<__nv_bfloat16> {
  static constexpr uint32_t kExponent = 0x7F80;
  static constexpr float kRefBelow = -8.0f, kRefRoom = 0.0f;
  static __device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
  static __device__ __forceinline__ void split(float a, float b, uint32_t& hi, uint32_t& lo) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    const float2 f = __bfloat1622float2(h);
    const __nv_bfloat162 l = __floats2bfloat162_rn(a - f.x, b - f.y);
    hi = *reinterpret_cast<const uint32_t*>(&h);
    lo = *reinterpret_cast<const uint32_t*>(&l);
  }
  static __device__ __forceinline__ __nv_bfloat16 from(float v) { return __float2bfloat16_rn(v); }
};

__device__ __forceinline__ uint32_t smem_addr(const void* p) {
  return static_cast<uint32_t>(__cvta_generic_to_shared(p));
}
__device__ __forceinline__ void ldmatrix(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldmatrix_trans(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ uint32_t transposed(uint32_t v) {
  uint32_t r;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}
// 16 bytes to shared memory
__device__ __forceinline__ void copy16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
// the same, or 16 zeros
__device__ __forceinline__ void copy16(uint32_t dst, const void* src, bool real) {
  const int n = real ? 16 : 0;
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copies_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ float exp2_fast(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

// What a part's result adds to a sum, at a factor of 0 to 1: an infinity stays
// one, however small the factor is.
__device__ __forceinline__ float weighed(float x, float f) { return fabsf(x) == INFINITY ? x : x * f; }

// Where the part results of a call lie: worker w has slot 2w for a row's head
// that began before its part, slot 2w + 1 for one that goes on behind it.
struct Parts {
  float* o;        // [2 W][columns][DP]
  float2* rl;      // [2 W][columns]: reference and sum
  int4* spans;     // the rows' heads that lie in several parts: query, head
                   // tile, parts (0: none), first worker.  One entry for
                   // each row's head, or, if fewer, for each worker (in
                   // whose part at most one begins that goes on behind it)
  int64_t* prefix; // [n + 1] tiles before each query; null: blocks sum them
};

struct AttendParams {
  AttendArgs a;
  Parts parts;
  uint32_t group, head_tiles;  // query heads of a key-value head, and tiles of 8 NT of them
  uint32_t workers;
  bool by_worker;              // what parts.spans goes by
  uint32_t cluster;            // blocks to a row's head; 0: equal parts
  uint32_t share;              // with one block: rows' heads in it
  uint32_t warps_each;         // a block's warps to a row's head
  uint64_t row_heads;
  bool tiled_pages;            // pages are whole tiles: a tile lies in one page
};

// The tiles of TK tokens that query i reads.
struct Tiles {
  int32_t row, len, first, begin, end;
  uint32_t gap;  // where the row was adopted inside a page: from here on that page is not its own
};
__device__ __forceinline__ uint32_t gap_of(const jb_page_cache& c, int32_t row) {
  const int32_t adopted = c.marks && row >= 0 && uint32_t(row) < c.n_rows ? c.marks[row] & kMarkAdopted : 0;
  return adopted ? uint32_t(adopted) : 0xFFFFFFFFu;
}
__device__ __forceinline__ Tiles tiles_of(const AttendArgs& a, uint32_t i) {
  Tiles t;
  t.row = a.rows ? a.rows[i] : int32_t(i);
  int64_t len = 0;
  if (t.row >= 0 && uint32_t(t.row) < a.c.n_rows)
    len = min(int64_t(max(a.c.lengths[t.row], 0)), int64_t(a.c.max_pages) * a.c.page_size);
  t.len = int32_t(len);
  t.first = a.window && len > int64_t(a.window) ? int32_t(len - a.window) : 0;
  t.begin = t.first / TK;
  t.end = int32_t((len + TK - 1) / TK);
  t.gap = gap_of(a.c, t.row);
  return t;
}

// Inclusive sum over the block's THREADS threads of one value each.
template <int THREADS>
__device__ __forceinline__ int64_t block_sum_scan(int64_t v, int64_t* total) {
  __shared__ int64_t sums[THREADS / 32];
  const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int64_t y = __shfl_up_sync(kFullMask, v, d);
    if (lane >= d) v += y;
  }
  if (lane == 31) sums[wid] = v;
  __syncthreads();
  int64_t before = 0, all = 0;
#pragma unroll
  for (int i = 0; i < THREADS / 32; i++) {
    if (i < wid) before += sums[i];
    all += sums[i];
  }
  __syncthreads();
  *total = all;
  return v + before;
}

// The tiles before each query, for more queries than a block keeps itself.
__global__ void __launch_bounds__(1024) prefix_kernel(const AttendArgs a, int64_t* prefix) {
  follow();
  int64_t done = 0;
  for (uint64_t base = 0; base < a.n; base += 1024) {
    const uint64_t i = base + threadIdx.x;
    int64_t v = 0;
    if (i < a.n) {
      const Tiles t = tiles_of(a, uint32_t(i));
      v = max(t.end - t.begin, 0);
    }
    int64_t total;
    const int64_t upto = done + block_sum_scan<1024>(v, &total);
    if (i < a.n) prefix[i + 1] = upto;
    done += total;
  }
  if (threadIdx.x == 0) prefix[0] = 0;
}

// Warps of a block (one block an SM) and tiles of a warp's ring, for a padded
// head dim and columns: as many bytes in flight as shared memory holds, in as
// many warps as their registers allow.  Measured on 400 k + 333 k tokens of 8
// heads of 128: 12 warps with 2 tiles 447 us, 13 with 2 460, 8 with 3 467.
// 16 query heads to a key-value head (NT 2): 8 with 3 137 us, 12 with 2 141.
struct Ring {
  int warps, stages;
};
constexpr Ring ring_of(int DP, int NT) {
  return DP == 64    ? Ring{12, 4}
         : DP == 96  ? Ring{12, 2}
         : DP == 128 ? (NT == 1 ? Ring{12, 2} : Ring{8, 3})
                     : Ring{6, 2};
}

// Bytes from a row of a tile in shared memory to the next.  Eight consecutive
// rows at the same column must fall into different banks for ldmatrix: where
// rows are whole multiples of 128 bytes the 16-byte chunks are permuted by the
// row's last three bits, else an odd number of chunks lies between rows.
template <int DP>
struct TileLayout {
  static constexpr bool kPermuted = (DP * 2) % 128 == 0;
  static constexpr int kRowBytes = kPermuted ? DP * 2 : DP * 2 + 16;
  static __device__ __forceinline__ uint32_t at(int row, int chunk) {
    return row * kRowBytes + (kPermuted ? (chunk ^ (row & 7)) : chunk) * 16;
  }
  // at(row, chunk + 2 k), given at(row, chunk) in a tile on a multiple of
  // kRowBytes, for a chunk of 0 or 1
  static __device__ __forceinline__ uint32_t step(uint32_t addr, int k) {
    return kPermuted ? addr ^ (32 * k) : addr + 32 * k;
  }
};

// A place in the line of tiles: a query's head tile, and its tile.
struct Cursor {
  Tiles t;
  uint32_t i, vh;
  int32_t tile;
};

template <typename T, int DP, int NT, int WARPS, int STAGES>
struct Attend {
  using L = TileLayout<DP>;
  static constexpr int kThreads = WARPS * 32;
  static constexpr int kColumns = 8 * NT;
  static constexpr int kTileBytes = TK * L::kRowBytes;   // keys, then as much values
  static constexpr int kStageBytes = 2 * kTileBytes;
  static constexpr int kRingBytes = WARPS * STAGES * kStageBytes;
  static constexpr int shared_bytes() {
    return kRingBytes + WARPS * STAGES * 4 + kMaxListed * 12 + (kMaxListed + 1) * 8 + 8;
  }
  static constexpr int KS = DP / 16;                     // k steps of Q K, head tiles of 16 of P V
  static constexpr int kChunkLanes = DP <= 64 ? 8 : DP <= 128 ? 16 : 32;  // lanes a row of 16-byte chunks takes
  static constexpr int kRowsPerCopy = 32 / kChunkLanes;

  struct Lists {
    int32_t *row, *len;
    uint32_t* gap;
    int64_t* prefix;
  };

  const AttendParams& p;
  const Lists& lists;
  int lane;

  __device__ __forceinline__ Tiles load_tiles(uint32_t i) const {
    if (p.parts.prefix) return tiles_of(p.a, i);
    Tiles t;
    t.row = lists.row[i];
    t.len = lists.len[i];
    t.first = p.a.window && t.len > int64_t(p.a.window) ? int32_t(t.len - p.a.window) : 0;
    t.begin = t.first / TK;
    t.end = int32_t((int64_t(t.len) + TK - 1) / TK);
    t.gap = lists.gap[i];
    return t;
  }
  __device__ __forceinline__ uint32_t head_rows() const { return p.a.c.n_kv_heads * p.head_tiles; }

  __device__ __forceinline__ void next(Cursor& c) const {
    if (++c.tile < c.t.end) return;
    c.tile = c.t.begin;
    if (++c.vh < head_rows()) return;
    c.vh = 0;
    do {
      if (++c.i >= p.a.n) return;
      c.t = load_tiles(c.i);
    } while (c.t.end <= c.t.begin);
    c.tile = c.t.begin;
  }

  // Where a tile's tokens lie: the lane's token (lanes 16 on repeat lanes 0
  // on), or with pages of whole tiles the tile's first token for all lanes.
  struct Place {
    int32_t page;   // -1: not there
    uint32_t slot;
    bool seen;      // the lane's token is attended to, if its page is there
  };
  __device__ __forceinline__ Place place_of(const Cursor& c) const {
    Place x;
    const uint32_t t = uint32_t(c.tile) * TK + (lane & 15);
    x.seen = int32_t(t) >= c.t.first && int32_t(t) < c.t.len;
    if (x.seen && p.a.mask && t < p.a.mask_width) x.seen = p.a.mask[int64_t(c.i) * p.a.mask_stride + t];
    const uint32_t at = p.tiled_pages ? uint32_t(c.tile) * TK : min(t, uint32_t(c.t.len) - 1);
    const uint32_t pg = at / p.a.c.page_size;
    x.slot = at - pg * p.a.c.page_size;
    if (t >= c.t.gap && pg * p.a.c.page_size < c.t.gap) x.seen = false;
    x.page = p.a.c.table[c.t.row * p.a.c.table_stride + pg];
    return x;
  }

  __device__ __forceinline__ void load_tile(uint32_t stage, uint32_t* valid, const Cursor& c, const Place& x) const {
    const jb_page_cache& k = p.a.c;
    const bool there = uint32_t(x.page) < k.n_pages;
    const uint32_t mask = __ballot_sync(kFullMask, x.seen && there) & 0xFFFFu;
    if (lane == 0) *valid = mask;
    if (mask == 0) return;
    const int chunk = lane % kChunkLanes, row0 = lane / kChunkLanes;
    const bool inside = chunk < int(k.head_dim / 8);
    const int64_t base = int64_t(p.a.layer) * k.layer_stride + int64_t(c.vh / p.head_tiles) * k.head_stride + chunk * 8;
    const int64_t mine = there ? x.page * k.page_stride + x.slot * k.token_stride : 0;
    if (p.tiled_pages) {
      if (!inside) return;
      const T* from = static_cast<const T*>(k.k) + base + mine + row0 * k.token_stride;
      const int64_t to_v = static_cast<const T*>(k.v) - static_cast<const T*>(k.k);
      const int64_t step = kRowsPerCopy * k.token_stride;
      if (mask == 0xFFFFu) {
#pragma unroll
        for (int it = 0; it < TK / kRowsPerCopy; it++, from += step) {
          const uint32_t dst = stage + L::at(it * kRowsPerCopy + row0, chunk);
          copy16(dst, from);
          copy16(dst + kTileBytes, from + to_v);
        }
      } else {
#pragma unroll
        for (int it = 0; it < TK / kRowsPerCopy; it++, from += step) {
          const int row = it * kRowsPerCopy + row0;
          const bool real = (mask >> row) & 1;
          const uint32_t dst = stage + L::at(row, chunk);
          copy16(dst, real ? from : static_cast<const T*>(k.k), real);
          copy16(dst + kTileBytes, real ? from + to_v : static_cast<const T*>(k.v), real);
        }
      }
    } else {
#pragma unroll
      for (int it = 0; it < TK / kRowsPerCopy; it++) {
        const int row = it * kRowsPerCopy + row0;
        const int64_t off = __shfl_sync(kFullMask, mine, row) + base;
        if (!inside) continue;
        const bool real = (mask >> row) & 1;
        const uint32_t dst = stage + L::at(row, chunk);
        copy16(dst, static_cast<const T*>(k.k) + (real ? off : 0), real);
        copy16(dst + kTileBytes, static_cast<const T*>(k.v) + (real ? off : 0), real);
      }
    }
  }

  struct State {
    float o[NT][KS][4];
    float ref[NT][2], sum[NT][2];
    uint32_t q[NT][KS][2];
  };

  __device__ __forceinline__ uint32_t head_of(uint32_t vh, int column) const {
    return (vh / p.head_tiles) * p.group + (vh % p.head_tiles) * kColumns + column;
  }
  __device__ __forceinline__ bool head_real(uint32_t vh, int column) const {
    return (vh % p.head_tiles) * kColumns + column < p.group;
  }

  __device__ __forceinline__ void begin(State& s, uint32_t i, uint32_t vh) const {
#pragma unroll
    for (int n = 0; n < NT; n++) {
      const int column = 8 * n + lane / 4;
      const T* q = static_cast<const T*>(p.a.q.p) + int64_t(i) * p.a.q.token_stride +
                   int64_t(head_of(vh, column)) * p.a.q.head_stride;
      const bool real = head_real(vh, column);
#pragma unroll
      for (int k = 0; k < KS; k++)
#pragma unroll
        for (int j = 0; j < 2; j++) {
          const uint32_t d = 16 * k + 8 * j + 2 * (lane % 4);
          s.q[n][k][j] = real && d < p.a.c.head_dim ? *reinterpret_cast<const uint32_t*>(q + d) : 0u;
        }
#pragma unroll
      for (int k = 0; k < KS; k++)
#pragma unroll
        for (int j = 0; j < 4; j++) s.o[n][k][j] = 0.0f;
      s.ref[n][0] = s.ref[n][1] = -INFINITY;
      s.sum[n][0] = s.sum[n][1] = 0.0f;
    }
  }

  __device__ __forceinline__ void tile(State& s, uint32_t stage, uint32_t mask) const {
    // S^T: rows are tokens, columns are query heads
    float w[NT][4];
#pragma unroll
    for (int n = 0; n < NT; n++) w[n][0] = w[n][1] = w[n][2] = w[n][3] = 0.0f;
    const uint32_t keys = stage + L::at(lane & 15, lane >> 4);
#pragma unroll
    for (int k = 0; k < KS; k++) {
      uint32_t a[4];
      ldmatrix(a, L::step(keys, k));
#pragma unroll
      for (int n = 0; n < NT; n++) Mma<T>::mma(w[n], a, s.q[n][k][0], s.q[n][k][1]);
    }
    const float scale = p.a.scale * 1.4426950408889634f;  // log2(e)
    const bool seen0 = (mask >> (lane / 4)) & 1, seen1 = (mask >> (lane / 4 + 8)) & 1;
    bool far = false;
#pragma unroll
    for (int n = 0; n < NT; n++)
#pragma unroll
      for (int j = 0; j < 4; j++) {
        w[n][j] = (j < 2 ? seen0 : seen1) ? w[n][j] * scale : -INFINITY;
        far |= w[n][j] > s.ref[n][j & 1] + Mma<T>::kRefRoom;
      }
    if (__any_sync(kFullMask, far)) {
#pragma unroll
      for (int n = 0; n < NT; n++)
#pragma unroll
        for (int j = 0; j < 2; j++) {
          float top = fmaxf(w[n][j], w[n][j + 2]);
#pragma unroll
          for (int d = 4; d < 32; d <<= 1) top = fmaxf(top, __shfl_xor_sync(kFullMask, top, d));
          const float ref = fmaxf(s.ref[n][j], top - Mma<T>::kRefBelow);
          const float keep = s.ref[n][j] == -INFINITY ? 0.0f : exp2_fast(s.ref[n][j] - ref);
          s.ref[n][j] = ref;
          s.sum[n][j] *= keep;
#pragma unroll
          for (int k = 0; k < KS; k++) {
            s.o[n][k][j] *= keep;
            s.o[n][k][j + 2] *= keep;
          }
        }
    }
    // O^T += V^T P^T: rows are head elements
    uint32_t hi[NT][2], lo[NT][2];
#pragma unroll
    for (int n = 0; n < NT; n++) {
      const float r0 = s.ref[n][0] == -INFINITY ? 0.0f : s.ref[n][0];
      const float r1 = s.ref[n][1] == -INFINITY ? 0.0f : s.ref[n][1];
      const float a = exp2_fast(w[n][0] - r0), b = exp2_fast(w[n][1] - r1);
      const float c = exp2_fast(w[n][2] - r0), d = exp2_fast(w[n][3] - r1);
      s.sum[n][0] += a + c;
      s.sum[n][1] += b + d;
      Mma<T>::split(a, b, hi[n][0], lo[n][0]);
      Mma<T>::split(c, d, hi[n][1], lo[n][1]);
#pragma unroll
      for (int j = 0; j < 2; j++) {
        hi[n][j] = transposed(hi[n][j]);
        lo[n][j] = transposed(lo[n][j]);
      }
    }
    const uint32_t values = stage + kTileBytes + L::at((lane & 7) + ((lane >> 4) << 3), (lane >> 3) & 1);
#pragma unroll
    for (int k = 0; k < KS; k++) {
      uint32_t a[4];
      ldmatrix_trans(a, L::step(values, k));
#pragma unroll
      for (int n = 0; n < NT; n++) {
        Mma<T>::mma(s.o[n][k], a, hi[n][0], hi[n][1]);
        Mma<T>::mma(s.o[n][k], a, lo[n][0], lo[n][1]);
      }
    }
  }

  // Is a result of the warp's not finite?
  __device__ __forceinline__ bool odd(const State& s) const {
    float x[4] = {0.0f, 0.0f, 0.0f, 0.0f};  // NaN if one is infinite or NaN
#pragma unroll
    for (int n = 0; n < NT; n++)
#pragma unroll
      for (int k = 0; k < KS; k++)
#pragma unroll
        for (int j = 0; j < 4; j++) x[j] = fmaf(s.o[n][k][j], 0.0f, x[j]);
    return __any_sync(kFullMask, (x[0] + x[1]) + (x[2] + x[3]) != 0.0f);
  }

  // The columns whose sums are NaN, as bits: theirs stay NaN.
  __device__ __forceinline__ uint32_t nan_columns(const State& s) const {
    uint32_t bits = 0;
#pragma unroll
    for (int n = 0; n < NT; n++)
#pragma unroll
      for (int j = 0; j < 2; j++) bits |= uint32_t(isnan(s.sum[n][j])) << (8 * n + 2 * (lane % 4) + j);
    return __reduce_or_sync(kFullMask, bits);
  }

  // Behind finish(), where a result of query i's tiles `tile`, tile + step and so on
  // below `end` was odd(): elements whose values that are attended to are infinite
  // with one sign become that, however small the weights; with both, or with NaN,
  // NaN.  What is not finite for another reason stays.  The results are at o
  // (floats, `stride` to a column), or, if that is null, the call's output.  Calls
  // with finite values never get here: it is not inlined, and looks up again what
  // its callers would have to keep in registers.
  static __device__ __noinline__ void settle(const AttendParams& p, uint32_t i, uint32_t vh, int32_t tile, int32_t end,
                                             int32_t step, uint32_t nan_columns, float* o, int stride) {
    const Lists none{};
    const int lane = int(threadIdx.x & 31);
    const Attend self{p, none, lane};
    const jb_page_cache& k = p.a.c;
    Cursor c{tiles_of(p.a, i), i, vh, tile};
    const int chunk = lane % kChunkLanes, row0 = lane / kChunkLanes;
    const bool inside = chunk < int(k.head_dim / 8);
    const int64_t base = int64_t(p.a.layer) * k.layer_stride + int64_t(c.vh / p.head_tiles) * k.head_stride + chunk * 8;
    uint32_t bits = 0;  // +inf, -inf, NaN for each of the 8 elements of the chunk
    for (; c.tile < end; c.tile += step) {
      const Place x = self.place_of(c);
      const bool there = uint32_t(x.page) < k.n_pages;
      const uint32_t mask = __ballot_sync(kFullMask, x.seen && there) & 0xFFFFu;
      const uint32_t slot = x.slot + (p.tiled_pages ? lane & 15 : 0);
      const int64_t mine = there ? x.page * k.page_stride + slot * k.token_stride : 0;
      for (int row = row0; row < TK; row += kRowsPerCopy) {
        const int64_t off = __shfl_sync(kFullMask, mine, row) + base;
        if (!inside || !((mask >> row) & 1)) continue;
        const uint4 v = *reinterpret_cast<const uint4*>(static_cast<const T*>(k.v) + off);
        const uint32_t word[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int e = 0; e < 8; e++) {
          const uint32_t b = (word[e / 2] >> (16 * (e % 2))) & 0xFFFFu;
          if ((b & Mma<T>::kExponent) == Mma<T>::kExponent)
            bits |= ((b & 0x7FFFu) != Mma<T>::kExponent ? 4u : b >> 15 ? 2u : 1u) << (3 * e);
        }
      }
    }
#pragma unroll
    for (int d = kChunkLanes; d < 32; d <<= 1) bits |= __shfl_xor_sync(kFullMask, bits, d);
    // the lane's elements as finish() has them
    for (int d8 = 0; d8 < DP / 8; d8++) {
      const uint32_t b = (__shfl_sync(kFullMask, bits, d8) >> (3 * (lane / 4))) & 7;
      const int d = 8 * d8 + lane / 4;
      if (b == 0) continue;
      const float v = b == 1 ? INFINITY : b == 2 ? -INFINITY : NAN;
      for (int n = 0; n < NT; n++)
        for (int j = 0; j < 2; j++) {
          const int column = 8 * n + 2 * (lane % 4) + j;
          if (!self.head_real(c.vh, column) || ((nan_columns >> column) & 1)) continue;
          if (o)
            o[column * stride + d] = v;
          else
            static_cast<T*>(p.a.out.p)[int64_t(c.i) * p.a.out.token_stride +
                                       int64_t(self.head_of(c.vh, column)) * p.a.out.head_stride + d] = Mma<T>::from(v);
        }
    }
  }

  // The piece's end: the result, or a part of it (slot >= 0).
  __device__ __forceinline__ void finish(State& s, uint32_t i, uint32_t vh, int64_t slot) const {
#pragma unroll
    for (int n = 0; n < NT; n++)
#pragma unroll
      for (int j = 0; j < 2; j++) {
        float l = s.sum[n][j];
#pragma unroll
        for (int d = 4; d < 32; d <<= 1) l += __shfl_xor_sync(kFullMask, l, d);
        const int column = 8 * n + 2 * (lane % 4) + j;
        if (!head_real(vh, column)) continue;
        const uint32_t h = head_of(vh, column);
        if (slot >= 0) {
          float* o = p.parts.o + (slot * kColumns + column) * DP;
#pragma unroll
          for (int k = 0; k < KS; k++) {
            o[16 * k + lane / 4] = s.o[n][k][j];
            o[16 * k + lane / 4 + 8] = s.o[n][k][j + 2];
          }
          if (lane < 4) p.parts.rl[slot * kColumns + column] = make_float2(s.ref[n][j], l);
        } else {
          T* out = static_cast<T*>(p.a.out.p) + int64_t(i) * p.a.out.token_stride + int64_t(h) * p.a.out.head_stride;
          const float inv = l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll
          for (int k = 0; k < KS; k++) {
            const uint32_t d = 16 * k + lane / 4;
            if (d < p.a.c.head_dim) out[d] = Mma<T>::from(s.o[n][k][j] * inv);
            if (d + 8 < p.a.c.head_dim) out[d + 8] = Mma<T>::from(s.o[n][k][j + 2] * inv);
          }
          if (p.a.lse && lane < 4)
            p.a.lse[int64_t(i) * p.a.n_q_heads + h] =
                l == 0.0f ? -INFINITY : (s.ref[n][j] + log2f(l)) * 0.6931471805599453f;
        }
      }
  }

  // The last query whose tiles begin at or before `tile` (which is below the total).
  __device__ __forceinline__ uint32_t query_at(int64_t tile) const {
    const int64_t* pre = p.parts.prefix ? p.parts.prefix : lists.prefix;
    uint32_t low = 0, high = p.a.n;  // pre[low] <= tile < pre[high]
    while (high - low > 1) {         // 32 probes at a time
      const uint32_t step = (high - low + 31) / 32;
      const uint32_t probe = low + step * lane;
      const bool under = probe < high && pre[probe] <= tile;
      const int last = 31 - __clz(__ballot_sync(kFullMask, under));
      low += step * last;
      high = min(high, low + step);
    }
    return low;
  }

  __device__ __forceinline__ void work(uint32_t worker, unsigned char* ring, uint32_t* valid, int64_t total) const {
    // Parts of several tiles leave less to join, parts of one are done first.
    // Measured on one row, 8 heads of 128, 1 / 2 / 4 tiles: 10.7 / 11.8 / 13.2
    // us with 2000 tokens, 14.7 / 11.8 / 13.6 with 4000, 16.4 / 16.4 / 13.8
    // with 8000.
    const int64_t mean = total / (int64_t(p.a.n) * head_rows());
    const int64_t least = mean < 160 ? 1 : mean < 400 ? 2 : 4;
    const int64_t workers = min(int64_t(p.workers), (total + least - 1) / least);
    if (p.by_worker && lane == 0) p.parts.spans[worker] = make_int4(0, 0, 0, 0);
    if (worker >= workers) return;
    const int64_t each = total / workers, more = total % workers;
    const int64_t w0 = int64_t(worker) * each + min(int64_t(worker), more);
    int64_t left = each + (int64_t(worker) < more);
    const uint32_t heads = head_rows();
    Cursor c;
    c.i = query_at(w0 / heads);
    c.t = load_tiles(c.i);
    const int64_t* pre = p.parts.prefix ? p.parts.prefix : lists.prefix;
    const int64_t into = w0 - pre[c.i] * heads;
    const int32_t count = c.t.end - c.t.begin;
    c.vh = uint32_t(into / count);
    c.tile = c.t.begin + int32_t(into % count);

    Cursor ahead = c;       // the next tile to load
    int64_t to_load = left;
    Place place = place_of(ahead);
    const uint32_t stage0 = smem_addr(ring);
    int load_stage = 0;
    // loads the tile at `ahead`, and looks up the next one's pages
    auto load_next = [&] {
      if (to_load > 0) {
        load_tile(stage0 + load_stage * kStageBytes, valid + load_stage, ahead, place);
        if (--to_load > 0) {
          next(ahead);
          place = place_of(ahead);
        }
      }
      copies_commit();
      load_stage = load_stage + 1 == STAGES ? 0 : load_stage + 1;
    };
#pragma unroll
    for (int s = 0; s < STAGES - 1; s++) load_next();

    State s;
    begin(s, c.i, c.vh);
    int32_t piece = c.tile;  // the piece's first tile
    int stage = 0;
    for (;;) {
      copies_wait<STAGES - 2>();
      __syncwarp();
      load_next();
      const uint32_t mask = valid[stage];
      if (mask) tile(s, stage0 + stage * kStageBytes, mask);
      __syncwarp();
      stage = stage + 1 == STAGES ? 0 : stage + 1;
      left--;
      const bool ends = c.tile + 1 == c.t.end;
      if (ends || left == 0) {
        const bool whole = piece == c.t.begin;
        const int64_t slot_of = ends ? (whole ? -1 : 2 * int64_t(worker)) : whole ? 2 * int64_t(worker) + 1 : 2 * int64_t(worker);
        const bool odd_results = odd(s);
        finish(s, c.i, c.vh, slot_of);
        if (odd_results)
          settle(p, c.i, c.vh, piece, c.tile + 1, 1, nan_columns(s),
                 slot_of < 0 ? nullptr : p.parts.o + slot_of * kColumns * DP, DP);
        if (whole && lane == 0 && (!ends || !p.by_worker)) {
          int parts = 0;
          if (!ends) {  // the row's head goes on: in how many parts, this one included
            const int64_t last = pre[c.i] * heads + (int64_t(c.vh) + 1) * (c.t.end - c.t.begin) - 1;
            const int64_t border = more * (each + 1);
            const int64_t last_worker = last < border ? last / (each + 1) : more + (last - border) / each;
            parts = int(last_worker - worker + 1);
          }
          p.parts.spans[p.by_worker ? worker : c.i * heads + c.vh] =
              make_int4(int(c.i), int(c.vh), parts, int(worker));
        }
        if (left == 0) break;
        next(c);
        begin(s, c.i, c.vh);
        piece = c.tile;
      } else {
        c.tile++;
      }
    }
    copies_wait<0>();
  }
};

// Registers of a thread: 12 warps with 128 leave room on their SM for blocks of
// the kernel that follows, which are launched early (32 rows of 500 to 4000
// tokens, 8 heads of 128: 53.6 us, 55.7 with 166); 12 warps of 96 x 16 columns
// need their 168, fewer warps take what there is.
constexpr int registers_of(int DP, int NT) {
  return ring_of(DP, NT).warps < 12 ? 255 : DP == 96 && NT == 2 ? 168 : 128;
}

template <typename T, int DP, int NT, int WARPS, int STAGES>
__global__ void __maxnreg__(registers_of(DP, NT)) attend_kernel(const __grid_constant__ AttendParams p) {
  using A = Attend<T, DP, NT, WARPS, STAGES>;
  extern __shared__ __align__(1024) unsigned char smem[];
  uint32_t* valid = reinterpret_cast<uint32_t*>(smem + A::kRingBytes);
  int64_t* prefix = reinterpret_cast<int64_t*>(smem + ((A::kRingBytes + WARPS * STAGES * 4 + 7) & ~7));
  int32_t* row = reinterpret_cast<int32_t*>(prefix + kMaxListed + 1);
  int32_t* len = row + kMaxListed;
  uint32_t* gap = reinterpret_cast<uint32_t*>(len + kMaxListed);
  typename A::Lists lists{row, len, gap, prefix};
  const int wid = threadIdx.x >> 5;
  A self{p, lists, int(threadIdx.x & 31)};
  follow();
  if (p.a.c.head_dim < DP)  // columns that no copy writes
    for (int i = threadIdx.x; i < A::kRingBytes / 16; i += A::kThreads)
      reinterpret_cast<uint4*>(smem)[i] = make_uint4(0, 0, 0, 0);
  int64_t total = 0;
  if (p.parts.prefix) {
    total = p.parts.prefix[p.a.n];
  } else {
    for (uint32_t base = 0; base < p.a.n; base += A::kThreads) {
      const uint32_t i = base + threadIdx.x;
      int64_t v = 0;
      if (i < p.a.n) {
        const Tiles t = tiles_of(p.a, i);
        row[i] = t.row;
        len[i] = t.len;
        gap[i] = t.gap;
        v = max(t.end - t.begin, 0);
      }
      int64_t sum;
      const int64_t upto = total + block_sum_scan<A::kThreads>(v, &sum);
      if (i < p.a.n) prefix[i + 1] = upto;
      total += sum;
    }
    if (threadIdx.x == 0) prefix[0] = 0;
  }
  __syncthreads();
  // queries with nothing to attend to
  const int64_t* pre = p.parts.prefix ? p.parts.prefix : prefix;
  for (uint32_t i = blockIdx.x; i < p.a.n; i += gridDim.x) {
    if (pre[i + 1] != pre[i]) continue;
    for (uint32_t j = threadIdx.x; j < p.a.n_q_heads * p.a.c.head_dim; j += A::kThreads)
      static_cast<T*>(p.a.out.p)[int64_t(i) * p.a.out.token_stride +
                                 int64_t(j / p.a.c.head_dim) * p.a.out.head_stride + j % p.a.c.head_dim] =
          Mma<T>::from(0.0f);
    if (p.a.lse)
      for (uint32_t h = threadIdx.x; h < p.a.n_q_heads; h += A::kThreads)
        p.a.lse[int64_t(i) * p.a.n_q_heads + h] = -INFINITY;
    if (!p.by_worker)
      for (uint32_t h = threadIdx.x; h < self.head_rows(); h += A::kThreads)
        p.parts.spans[i * self.head_rows() + h] = make_int4(0, 0, 0, 0);
  }
  // neighbouring parts on different SMs, so that few tiles are spread over all
  self.work(wid * gridDim.x + blockIdx.x, smem + wid * STAGES * A::kStageBytes, valid + wid * STAGES,
            total * self.head_rows());
}

// The same for few rows of few tokens, where a call's latency is what counts:
// a cluster of 1, 2, 4 or 8 blocks, or some of one block's warps, take one row's
// head, a tile each in turn, and their results are joined through shared, and
// the blocks' through distributed shared memory, with no second kernel and no
// scratch.
constexpr int kCluster = 8;                // the largest
constexpr uint64_t kTokensOfBlock = 1500;  // of heads of 128, at most
constexpr uint64_t kMostShared = 300000;   // rows' heads: a grid has 65,535 blocks in y
// Fewer warps start, and are joined, sooner: 1000 tokens of 8 heads of 128
// took 6.4 us with 8 warps a block, 7.2 with 12, 6.7 with 4; 4000 tokens 9.4,
// 10.0 and 11.9.
constexpr Ring cluster_ring_of(int DP) { return DP == 256 ? Ring{6, 2} : Ring{8, 3}; }

template <typename T, int DP, int NT, int WARPS, int STAGES>
__global__ void __launch_bounds__(WARPS * 32) attend_cluster_kernel(const __grid_constant__ AttendParams p) {
  using A = Attend<T, DP, NT, WARPS, STAGES>;
  constexpr int C = A::kColumns;
  extern __shared__ __align__(1024) unsigned char smem[];
  __shared__ uint32_t valid[WARPS * STAGES];
  constexpr int OS = DP + 4;              // floats from a column of a warp's result to the next: no bank conflicts
  __shared__ float2 warp_rl[WARPS][C];    // a warp's references and sums
  __shared__ float warp_f[WARPS][C];      // what its result weighs in its group's
  __shared__ float2 group_rl[WARPS][C];
  __shared__ __align__(16) float block_o[C][DP];
  follow();
  const int wid = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const typename A::Lists none{};
  const A self{p, none, lane};
  // the warps of a row's head: `each` of a block's, in `blocks` blocks
  const int each = int(p.warps_each), group = wid / each, blocks = int(gridDim.x);
  const uint32_t rank = blockIdx.x;  // the grid is one cluster wide
  const uint32_t item = blockIdx.y * (WARPS / each) + group;
  const uint32_t heads = self.head_rows();
  const bool has = item < p.row_heads;
  Cursor c{};
  typename A::State s;
  if (has) {
    c.i = item / heads;
    c.vh = item % heads;
    self.begin(s, c.i, c.vh);
    c.t = tiles_of(p.a, c.i);
  }
  const int count = max(c.t.end - c.t.begin, 0);
  const int first = int(rank) * each + wid % each, step = blocks * each;
  unsigned char* ring = smem + wid * STAGES * A::kStageBytes;
  if (p.a.c.head_dim < DP) {  // columns that no copy writes
    for (int i = lane; i < STAGES * A::kStageBytes / 16; i += 32)
      reinterpret_cast<uint4*>(ring)[i] = make_uint4(0, 0, 0, 0);
    __syncwarp();
  }
  if (first < count) {
    const uint32_t stage0 = smem_addr(ring);
    uint32_t* mask_of = valid + wid * STAGES;
    int to_load = first, load_stage = 0;
    c.tile = c.t.begin + first;
    typename A::Place place = self.place_of(c);
    auto load_next = [&] {
      if (to_load < count) {
        self.load_tile(stage0 + load_stage * A::kStageBytes, mask_of + load_stage, c, place);
        to_load += step;
        if (to_load < count) {  // the next one's page is looked up ahead
          c.tile = c.t.begin + to_load;
          place = self.place_of(c);
        }
      }
      copies_commit();
      load_stage = load_stage + 1 == STAGES ? 0 : load_stage + 1;
    };
#pragma unroll
    for (int j = 0; j < STAGES - 1; j++) load_next();
    int stage = 0;
    for (int j = first; j < count; j += step) {
      __syncwarp();
      load_next();
      copies_wait<STAGES - 1>();
      __syncwarp();
      const uint32_t mask = mask_of[stage];
      if (mask) self.tile(s, stage0 + stage * A::kStageBytes, mask);
      stage = stage + 1 == STAGES ? 0 : stage + 1;
    }
    copies_wait<0>();
    __syncwarp();
  }
  const bool odd_results = first < count && self.odd(s);
  if (blocks == 1 && each == 1) {  // the warp has it all
    if (has) self.finish(s, c.i, c.vh, -1);
    if (odd_results) A::settle(p, c.i, c.vh, c.t.begin + first, c.t.end, step, self.nan_columns(s), nullptr, 0);
    return;
  }
  if (first < count) {
    // the ring is done with: it takes the warp's result
    float* o = reinterpret_cast<float*>(ring);
#pragma unroll
    for (int n = 0; n < NT; n++)
#pragma unroll
      for (int j = 0; j < 2; j++) {
        float l = s.sum[n][j];
#pragma unroll
        for (int d = 4; d < 32; d <<= 1) l += __shfl_xor_sync(kFullMask, l, d);
        const int column = 8 * n + 2 * (lane % 4) + j;
        if (lane < 4) warp_rl[wid][column] = make_float2(s.ref[n][j], l);
#pragma unroll
        for (int k = 0; k < A::KS; k++) {
          o[column * OS + 16 * k + lane / 4] = s.o[n][k][j];
          o[column * OS + 16 * k + lane / 4 + 8] = s.o[n][k][j + 2];
        }
      }
    if (odd_results) A::settle(p, c.i, c.vh, c.t.begin + first, c.t.end, step, self.nan_columns(s), o, OS);
  }
  __syncthreads();
  const int warp0 = group * each, t = int(threadIdx.x) - warp0 * 32;
  const int warps = min(each, max(0, count - int(rank) * each));  // those that had tiles
  const int columns = has ? min(C, int(p.group - (c.vh % p.head_tiles) * C)) : 0;
  if (t < each * C) {
    const int w = t / C, column = t % C;
    float ref = -INFINITY, l = 0.0f;
    for (int i = 0; i < warps; i++) ref = fmaxf(ref, warp_rl[warp0 + i][column].x);
    const float r = ref == -INFINITY ? 0.0f : ref;
    if (w < warps) warp_f[warp0 + w][column] = exp2_fast(warp_rl[warp0 + w][column].x - r);
    if (w == 0) {
      for (int i = 0; i < warps; i++) l += warp_rl[warp0 + i][column].y * exp2_fast(warp_rl[warp0 + i][column].x - r);
      group_rl[group][column] = make_float2(ref, l);
    }
  }
  __syncthreads();
  // four elements of a column at a time
  const int dim = int(p.a.c.head_dim);
  auto put = [&](int column, int d, float ref, float4 o, float l) {
    const uint32_t h = self.head_of(c.vh, column);
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    if (d < dim) {
      T* out = static_cast<T*>(p.a.out.p) + int64_t(c.i) * p.a.out.token_stride + int64_t(h) * p.a.out.head_stride + d;
      alignas(8) T v[4] = {Mma<T>::from(o.x * inv), Mma<T>::from(o.y * inv), Mma<T>::from(o.z * inv),
                           Mma<T>::from(o.w * inv)};
      *reinterpret_cast<uint2*>(out) = *reinterpret_cast<const uint2*>(v);
    }
    if (d == 0 && p.a.lse)
      p.a.lse[int64_t(c.i) * p.a.n_q_heads + h] = l == 0.0f ? -INFINITY : (ref + log2f(l)) * 0.6931471805599453f;
  };
  for (int e = 4 * t; e < columns * DP; e += 4 * each * 32) {
    const int column = e / DP, d = e % DP;
    float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    for (int w = warp0; w < warp0 + warps; w++) {
      const float f = warp_f[w][column];
      const float4 x = *reinterpret_cast<const float4*>(
          reinterpret_cast<const float*>(smem + w * STAGES * A::kStageBytes) + column * OS + d);
      o.x += weighed(x.x, f);
      o.y += weighed(x.y, f);
      o.z += weighed(x.z, f);
      o.w += weighed(x.w, f);
    }
    if (blocks == 1) put(column, d, group_rl[group][column].x, o, group_rl[group][column].y);
    else *reinterpret_cast<float4*>(&block_o[column][d]) = o;
  }
  if (blocks == 1) return;
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
  auto remote = [&](const void* at, int block) {
    uint32_t a;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem_addr(at)), "r"(block));
    return a;
  };
  for (int e = 4 * (int(rank) * WARPS * 32 + int(threadIdx.x)); e < columns * DP; e += 4 * step * 32) {
    const int column = e / DP, d = e % DP;
    float2 rl[kCluster];
    float4 part[kCluster];
    float ref = -INFINITY;
#pragma unroll
    for (int b = 0; b < kCluster; b++) {
      rl[b] = make_float2(-INFINITY, 0.0f);
      part[b] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
      if (b >= blocks) continue;
      asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];"
                   : "=f"(rl[b].x), "=f"(rl[b].y) : "r"(remote(&group_rl[0][column], b)) : "memory");
      asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
                   : "=f"(part[b].x), "=f"(part[b].y), "=f"(part[b].z), "=f"(part[b].w)
                   : "r"(remote(&block_o[column][d], b)) : "memory");
      ref = fmaxf(ref, rl[b].x);
    }
    const float r = ref == -INFINITY ? 0.0f : ref;
    float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    float l = 0.0f;
#pragma unroll
    for (int b = 0; b < kCluster; b++) {
      const float f = exp2_fast(rl[b].x - r);
      o.x += weighed(part[b].x, f);
      o.y += weighed(part[b].y, f);
      o.z += weighed(part[b].z, f);
      o.w += weighed(part[b].w, f);
      l += rl[b].y * f;
    }
    put(column, d, ref, o, l);
  }
  // no block leaves while another may read its shared memory
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

// Joins the parts of a row's head (a span), for one query head (blockIdx.y):
// out = sum_i o_i 2^(r_i - r) / sum_i l_i 2^(r_i - r), r the largest
// reference.  What it takes is the latency of its dependent reads, so a warp
// reads the references, sums and outputs of several parts at once.  With
// few parts to a span (SHARED 1) a warp takes each, else a block of SHARED
// warps, every SHARED-th part each.
constexpr int kJoinSpans = 8;  // spans of a block with SHARED 1
constexpr int join_warps(int shared) { return shared == 1 ? kJoinSpans : shared; }

template <typename T, int DP, int NT, int SHARED>
__global__ void __launch_bounds__(join_warps(SHARED) * 32) join_kernel(const __grid_constant__ AttendParams p, uint32_t spans) {
  constexpr int kColumns = 8 * NT, N = DP / 32, B = SHARED == 16 ? 8 : 4;
  __shared__ float share[SHARED == 1 ? 1 : SHARED][SHARED == 1 ? 1 : DP];
  __shared__ float2 share_rl[SHARED];
  const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5;
  const uint32_t item = SHARED == 1 ? blockIdx.x * kJoinSpans + wid : blockIdx.x;
  follow();
  if (item >= spans) return;
  const int4 span = p.parts.spans[item];
  const int column = blockIdx.y;
  const uint32_t vh = uint32_t(span.y);
  if (span.z == 0 || (vh % p.head_tiles) * kColumns + column >= p.group) return;
  // part 0 is the first worker's last piece, part j > 0 the next workers' first
  auto slot = [&](int j) { return (2 * (int64_t(span.w) + j) + (j == 0)) * kColumns + column; };
  float o[N], l = 0.0f, ref = -INFINITY;
#pragma unroll
  for (int k = 0; k < N; k++) o[k] = 0.0f;
  for (int j0 = SHARED == 1 ? 0 : wid; j0 < span.z; j0 += SHARED * B) {
    float2 rl[B];
    float part[B][N];
    float top = ref;
#pragma unroll
    for (int b = 0; b < B; b++) {
      const int64_t at = slot(min(j0 + SHARED * b, span.z - 1));
      rl[b] = p.parts.rl[at];
#pragma unroll
      for (int k = 0; k < N; k++) part[b][k] = p.parts.o[at * DP + lane + 32 * k];
    }
#pragma unroll
    for (int b = 0; b < B; b++) {
      if (j0 + SHARED * b >= span.z) rl[b].x = -INFINITY;  // read twice: weighs once
      top = fmaxf(top, rl[b].x);
    }
    const float r = top == -INFINITY ? 0.0f : top;  // parts without a score weigh nothing, unless they are NaN
    const float keep = exp2_fast(ref - r);
    l *= keep;
#pragma unroll
    for (int k = 0; k < N; k++) o[k] = weighed(o[k], keep);
#pragma unroll
    for (int b = 0; b < B; b++) {
      const float f = exp2_fast(rl[b].x - r);
      l += rl[b].y * f;
#pragma unroll
      for (int k = 0; k < N; k++) o[k] += weighed(part[b][k], f);
    }
    ref = top;
  }
  const uint32_t h = (vh / p.head_tiles) * p.group + (vh % p.head_tiles) * kColumns + column;
  T* out = static_cast<T*>(p.a.out.p) + int64_t(span.x) * p.a.out.token_stride + int64_t(h) * p.a.out.head_stride;
  float* lse = p.a.lse ? p.a.lse + int64_t(span.x) * p.a.n_q_heads + h : nullptr;
  if constexpr (SHARED == 1) {
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll
    for (int k = 0; k < N; k++)
      if (lane + 32 * k < p.a.c.head_dim) out[lane + 32 * k] = Mma<T>::from(o[k] * inv);
    if (lse && lane == 0) *lse = l == 0.0f ? -INFINITY : (ref + log2f(l)) * 0.6931471805599453f;
  } else {
#pragma unroll
    for (int k = 0; k < N; k++) share[wid][lane + 32 * k] = o[k];
    if (lane == 0) share_rl[wid] = make_float2(ref, l);
    __syncthreads();
    float top = -INFINITY;
#pragma unroll
    for (int i = 0; i < SHARED; i++) top = fmaxf(top, share_rl[i].x);
    const float r = top == -INFINITY ? 0.0f : top;
    for (uint32_t d = threadIdx.x; d < p.a.c.head_dim; d += SHARED * 32) {
      float v = 0.0f;
      l = 0.0f;
#pragma unroll
      for (int i = 0; i < SHARED; i++) {
        const float f = exp2_fast(share_rl[i].x - r);
        v += weighed(share[i][d], f);
        l += share_rl[i].y * f;
      }
      out[d] = Mma<T>::from(l == 0.0f ? 0.0f : v / l);
      if (lse && d == 0) *lse = l == 0.0f ? -INFINITY : (top + log2f(l)) * 0.6931471805599453f;
    }
  }
}

void check_cuda(cudaError_t e, const char* what) {
  if (e != cudaSuccess) {
    cudaGetLastError();
    throw std::runtime_error(std::string(what) + ": " + cudaGetErrorString(e));
  }
}

int sm_count() {
  constexpr int kMaxDevices = 64;
  static std::mutex m;
  static int counts[kMaxDevices] = {};
  int dev = 0;
  check_cuda(cudaGetDevice(&dev), "get device");
  std::lock_guard<std::mutex> lock(m);
  if (dev >= kMaxDevices) throw std::runtime_error("device index out of range");
  if (counts[dev] == 0) check_cuda(cudaDeviceGetAttribute(&counts[dev], cudaDevAttrMultiProcessorCount, dev), "SM count");
  return counts[dev];
}

// Padded head dim, columns and workers of a call.
struct Shape {
  int dp, nt, warps;
  uint32_t group, head_tiles, workers;
  uint64_t row_heads;
  uint32_t cluster, share;
};
Shape shape_of(const AttendArgs& a) {
  Shape s;
  const uint32_t d = a.c.head_dim;
  s.dp = d <= 64 ? 64 : d <= 96 ? 96 : d <= 128 ? 128 : 256;
  s.group = a.n_q_heads / a.c.n_kv_heads;
  s.nt = s.group <= 8 ? 1 : 2;
  s.head_tiles = (s.group + 8 * s.nt - 1) / (8 * s.nt);
  s.warps = ring_of(s.dp, s.nt).warps;
  s.workers = uint32_t(sm_count() * s.warps);
  s.row_heads = uint64_t(a.n) * a.c.n_kv_heads * s.head_tiles;
  // For 148 SMs: clusters as large as all run at once (15 of 8 blocks take 7 us,
  // 16 take 13; 33 and 36 of 4, 7.8 and 13.4), where rows are short enough that
  // unequal lengths cost less than the second kernel.  How long they are is
  // known here by the table's width or the window only: in a wide table short
  // rows take the equal parts too (20 rows of 50 tokens, 8 heads: 4.5 us in a
  // table of 64 tokens, 10.7 in one of 16,000).  Clusters / equal parts, heads
  // of 128: one row of 1000 tokens and 8 heads 6.4 / 10.0 us, of 8000 14.0 /
  // 14.0; 32 rows' heads of 4000 tokens 18 / 21, of 1000 to 4000 14 / 15; 64 of
  // 4000 28 / 31, of 1000 to 4000 26 / 24.
  const uint64_t wide = uint64_t(a.c.max_pages) * a.c.page_size;
  const uint64_t longest = a.window && a.window < wide ? a.window : wide;
  s.cluster = s.row_heads <= 15 ? 8 : s.row_heads <= 32 ? 4 : s.row_heads <= 74 ? 2 : 1;
  s.share = s.row_heads <= 148 ? 1 : s.row_heads <= 296 ? 2 : s.row_heads <= 592 ? 4 : 8;
  if (s.row_heads > kMostShared || longest * s.dp * s.share > kTokensOfBlock * 128 * s.cluster) s.cluster = 0;
  return s;
}

size_t aligned(size_t n) { return (n + 255) & ~size_t(255); }

// Sets the kernel's shared memory once per device.
template <typename K>
void allow_shared(K kernel, int bytes, uint64_t& ready, std::mutex& m) {
  int dev = 0;
  check_cuda(cudaGetDevice(&dev), "get device");
  std::lock_guard<std::mutex> lock(m);
  if (ready >> dev & 1) return;
  check_cuda(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes),
             "attend shared memory");
  ready |= uint64_t(1) << dev;
}

template <typename T, int DP, int NT>
void launch_typed(const AttendParams& p, cudaStream_t st) {
  constexpr int kWarps = ring_of(DP, NT).warps, kStages = ring_of(DP, NT).stages;
  using A = Attend<T, DP, NT, kWarps, kStages>;
  auto kernel = attend_kernel<T, DP, NT, kWarps, kStages>;
  static std::mutex m;
  static uint64_t ready = 0, cluster_ready = 0;  // devices where the kernels have their shared memory
  const uint64_t row_heads = uint64_t(p.a.n) * p.a.c.n_kv_heads * p.head_tiles;
  if (p.cluster) {
    constexpr Ring ring = cluster_ring_of(DP);
    using C = Attend<T, DP, NT, ring.warps, ring.stages>;
    auto cluster_kernel = attend_cluster_kernel<T, DP, NT, ring.warps, ring.stages>;
    allow_shared(cluster_kernel, C::kRingBytes, cluster_ready, m);
    AttendParams q = p;
    q.warps_each = p.share > uint32_t(ring.warps) ? 1 : ring.warps / p.share;
    const uint32_t groups = ring.warps / q.warps_each;
    launch("attend", cluster_kernel, dim3(p.cluster, uint32_t((row_heads + groups - 1) / groups)), C::kThreads,
           C::kRingBytes, st, p.cluster, q);
    return;
  }
  allow_shared(kernel, A::shared_bytes(), ready, m);
  if (p.parts.prefix) {
    launch("attend prefix", prefix_kernel, dim3(1), 1024, 0, st, 0, p.a, p.parts.prefix);
  }
  launch("attend", kernel, dim3(p.workers / kWarps), A::kThreads, A::shared_bytes(), st, 0, p);
  // rows of one tile are never split
  if (uint64_t(p.a.c.max_pages) * p.a.c.page_size <= TK) return;
  const uint32_t spans = p.by_worker ? p.workers : uint32_t(row_heads);
  const uint32_t parts = p.workers / spans;  // about as many to a span
  const int shared = parts >= 48 ? 16 : parts >= 6 ? 4 : 1;
  auto join = shared == 16  ? join_kernel<T, DP, NT, 16>
              : shared == 4 ? join_kernel<T, DP, NT, 4>
                            : join_kernel<T, DP, NT, 1>;
  launch("attend join", join,
         dim3(shared == 1 ? (spans + kJoinSpans - 1) / kJoinSpans : spans, p.group < 8 * NT ? p.group : 8 * NT),
         join_warps(shared) * 32, 0, st, 0, p, spans);
}

template <typename T>
void launch_any(const AttendParams& p, int dp, int nt, cudaStream_t st) {
  if (nt == 1) {
    if (dp == 64) launch_typed<T, 64, 1>(p, st);
    else if (dp == 96) launch_typed<T, 96, 1>(p, st);
    else if (dp == 128) launch_typed<T, 128, 1>(p, st);
    else launch_typed<T, 256, 1>(p, st);
  } else {
    if (dp == 64) launch_typed<T, 64, 2>(p, st);
    else if (dp == 96) launch_typed<T, 96, 2>(p, st);
    else if (dp == 128) launch_typed<T, 128, 2>(p, st);
    else launch_typed<T, 256, 2>(p, st);
  }
}

}  // namespace

size_t attend_scratch_bytes(const AttendArgs& a) {
  if (a.n == 0 || a.n_q_heads == 0) return 0;
  const Shape s = shape_of(a);
  if (s.cluster) return 0;
  const size_t slots = size_t(2) * s.workers * 8 * s.nt;
  return aligned(slots * s.dp * sizeof(float)) + aligned(slots * sizeof(float2)) +
         aligned(s.workers * sizeof(int4)) + (a.n > uint32_t(kMaxListed) ? (size_t(a.n) + 1) * sizeof(int64_t) : 0);
}

void launch_attend(const AttendArgs& a, void* scratch, cudaStream_t st) {
  if (a.n == 0 || a.n_q_heads == 0) return;
  const Shape s = shape_of(a);
  AttendParams p{};
  p.a = a;
  p.group = s.group;
  p.head_tiles = s.head_tiles;
  p.workers = s.workers;
  if (double(s.row_heads) * double(a.c.max_pages) * a.c.page_size > 4e18)
    throw std::invalid_argument("rows, heads and tokens are too many for one call");
  p.by_worker = s.row_heads > s.workers;
  p.cluster = s.cluster;
  p.share = s.share;
  p.row_heads = s.row_heads;
  p.tiled_pages = a.c.page_size % TK == 0;
  const size_t slots = size_t(2) * s.workers * 8 * s.nt;
  unsigned char* at = static_cast<unsigned char*>(scratch);
  p.parts.o = reinterpret_cast<float*>(at);
  at += aligned(slots * s.dp * sizeof(float));
  p.parts.rl = reinterpret_cast<float2*>(at);
  at += aligned(slots * sizeof(float2));
  p.parts.spans = reinterpret_cast<int4*>(at);
  at += aligned(s.workers * sizeof(int4));
  if (a.n > uint32_t(kMaxListed)) p.parts.prefix = reinterpret_cast<int64_t*>(at);
  if (a.c.dtype == JB_F16) launch_any<__half>(p, s.dp, s.nt, st);
  else launch_any<__nv_bfloat16>(p, s.dp, s.nt, st);
}

}  // namespace jb
