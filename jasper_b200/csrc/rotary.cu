// rotary.cu -- rotary positions, and new keys and values into the cache's
// pages, in one kernel.
//
// A head's pair (a, b) of pair index i at position p becomes
//     s (a cos t - b sin t),  s (b cos t + a sin t),   t = p theta_i,
// and the gradient is the same turn backwards.  theta_i comes as a fraction
// of a turn in 64-bit fixed point: p * freq wraps at whole turns, so the top
// 32 bits of the product are the reduced angle, exact for that theta and every
// int64 position; only then does it become a float32 (error 2^-26 of a turn, to
// which theta's rounding adds up to 2^-65 of a turn a position).
//
// HBM bounds prompts, latency single tokens.  A block takes a few tokens: it
// computes their cosines and sines once (half a head of pairs each, shared by
// all heads) into shared memory while its first heads are on their way, then
// streams the tokens' heads through registers, two 16-byte vectors of a pair's
// two sides at a time.  A thread keeps its place in the head, so nothing is
// divided on the way.  One pair of vectors a thread in flight and 1536 threads
// an SM beat more of them in fewer threads: 8192 tokens of 40 heads of 128 in
// bfloat16 took 31 us so, 34 and 48 with two and four in flight.
#include <stdexcept>
#include <string>
#include "paged.cuh"

namespace jb {
namespace {

constexpr int kMaxThreads = 256;  // a block has as many whole heads' units as fit
constexpr int kMaxTokens = 16;    // per block
constexpr int kBlocks = 6;        // of 256 threads an SM, by registers

template <typename T>
struct Elem;
template <>
struct Elem<__half> {
  static __device__ __forceinline__ float to(__half v) { return __half2float(v); }
  static __device__ __forceinline__ __half from(float v) { return __float2half_rn(v); }
};
template <>
struct Elem<__nv_bfloat16> {
  static __device__ __forceinline__ float to(__nv_bfloat16 v) { return __bfloat162float(v); }
  static __device__ __forceinline__ __nv_bfloat16 from(float v) { return __float2bfloat16_rn(v); }
};
template <>
struct Elem<float> {
  static __device__ __forceinline__ float to(float v) { return v; }
  static __device__ __forceinline__ float from(float v) { return v; }
};

template <typename T, int VEC>
struct alignas(sizeof(T) * VEC) Vec {
  T v[VEC];
};

struct RotaryParams {
  HeadsView q, q_out, k, v;  // q alone for jb_rotary
  uint32_t n_q, n_kv, dim, tokens_per_block;
  uint32_t units;      // of a head: pairs of vectors
  bool stream;         // results are more than L2 keeps: write them through
  uint64_t n_tokens;
  Positions pos;
  RotaryArgs r;
  // append only
  jb_page_cache c;
  const int32_t* rows;
  const int32_t* index;
  int64_t layer_offset;
};

template <typename T, int VEC, bool APPEND>
__global__ void __launch_bounds__(kMaxThreads, kBlocks) rotary_kernel(const __grid_constant__ RotaryParams a) {
  extern __shared__ float2 cs[];  // [tokens][VEC][rot / 2 / VEC]: neighbouring threads read neighbours
  __shared__ int64_t place[kMaxTokens];
  using V = Vec<T, VEC>;
  follow();
  const uint32_t half = a.r.rot / 2, pair_units = half / VEC;
  const uint64_t t0 = uint64_t(blockIdx.x) * a.tokens_per_block;
  const uint32_t nt = uint32_t(min(uint64_t(a.tokens_per_block), a.n_tokens - t0));
  const uint32_t heads = a.n_q + (APPEND ? 2 * a.n_kv : 0);
  const uint32_t e = threadIdx.x % a.units, stride = blockDim.x / a.units;
  const bool turn = e < pair_units;
  // the unit's two vectors in its head
  const uint32_t o0 = turn ? (a.r.interleaved ? 2 * VEC * e : VEC * e) : a.r.rot + 2 * VEC * (e - pair_units);
  const uint32_t o1 = turn && !a.r.interleaved ? o0 + half : o0 + VEC;
  const bool two = o1 < a.dim;

  // heads of the block's tokens, one after the other
  struct Head {
    uint32_t tok, h;
  };
  auto from = [&](const Head& x) {
    const uint64_t t = t0 + x.tok;
    uint32_t h = x.h;
    const HeadsView* v = &a.q;
    if (APPEND && h >= a.n_q) {
      h -= a.n_q;
      v = &a.k;
      if (h >= a.n_kv) {
        h -= a.n_kv;
        v = &a.v;
      }
    }
    return static_cast<const T*>(v->p) + t * v->token_stride + h * v->head_stride;
  };
  auto advance = [&](Head& x) {
    x.h += stride;
    while (x.h >= heads) {
      x.h -= heads;
      x.tok++;
    }
  };
  Head at{0, threadIdx.x / a.units};
  while (at.h >= heads) {
    at.h -= heads;
    at.tok++;
  }
  V x0, x1;
  auto load = [&] {
    const T* src = from(at);
    x0 = *reinterpret_cast<const V*>(src + o0);
    if (two) x1 = *reinterpret_cast<const V*>(src + o1);
  };
  auto store = [&](T* dst, const V& v) {
    if constexpr (sizeof(V) == 16) {
      if (a.stream) {
        __stcs(reinterpret_cast<uint4*>(dst), *reinterpret_cast<const uint4*>(&v));
        return;
      }
    }
    *reinterpret_cast<V*>(dst) = v;
  };
  if (at.tok < nt) load();

  if (APPEND && threadIdx.x < nt) {
    // the token's place in its page, -1 where there is none
    const uint64_t t = t0 + threadIdx.x;
    const int32_t row = a.rows[t];
    int64_t to = -1;
    if (row >= 0 && uint32_t(row) < a.c.n_rows) {
      // a row that was refused room has no new last token
      const int32_t mark = a.c.marks ? a.c.marks[row] : 0;
      const int64_t i = a.index ? int64_t(a.index[t]) : mark < 0 ? int64_t(-1) : int64_t(a.c.lengths[row]) - 1;
      const uint32_t adopted = uint32_t(mark & kMarkAdopted);
      // the rest of the page in which it was adopted is not the row's
      const bool others = adopted % a.c.page_size && i >= int64_t(adopted) &&
                          uint32_t(i) / a.c.page_size == adopted / a.c.page_size;
      if (i >= 0 && !others && uint32_t(i) / a.c.page_size < a.c.max_pages) {
        const uint32_t pg = uint32_t(i) / a.c.page_size, slot = uint32_t(i) % a.c.page_size;
        const int32_t page = a.c.table[row * a.c.table_stride + pg];
        if (page >= 0 && uint32_t(page) < a.c.n_pages)
          to = a.layer_offset + page * a.c.page_stride + slot * a.c.token_stride;
      }
    }
    place[threadIdx.x] = to;
    if (to < 0) atomicOr(a.c.status, kPagesBadToken);
  }
  for (uint32_t j = threadIdx.x; j < nt * half; j += blockDim.x) {
    const uint32_t tok = j / half, i = j - tok * half;
    const uint64_t t = t0 + tok;
    int64_t p;
    if (!APPEND || a.pos.p32 || a.pos.p64) {
      p = a.pos.at(t);
    } else if (a.index) {
      p = a.index[t];
    } else {
      const int32_t row = a.rows[t];
      p = row >= 0 && uint32_t(row) < a.c.n_rows ? a.c.lengths[row] - 1 : 0;
    }
    const uint64_t phase = uint64_t(p) * uint64_t(a.r.freq[i]);
    float sn, cn;
    sincospif(float(int32_t(phase >> 32)) * 0x1p-31f, &sn, &cn);
    cs[tok * half + (i % VEC) * pair_units + i / VEC] = make_float2(cn * a.r.scale, (a.r.inverse ? -sn : sn) * a.r.scale);
  }
  __syncthreads();

  for (; at.tok < nt; advance(at)) {
    if (at.tok || at.h >= stride) load();  // the first is there
    const uint64_t t = t0 + at.tok;
    T* dst;
    bool turned = turn;
    if (!APPEND || at.h < a.n_q) {
      dst = static_cast<T*>(a.q_out.p) + t * a.q_out.token_stride + at.h * a.q_out.head_stride;
    } else {
      if (place[at.tok] < 0) continue;
      const bool is_k = at.h - a.n_q < a.n_kv;
      const uint32_t h = at.h - a.n_q - (is_k ? 0 : a.n_kv);
      dst = static_cast<T*>(is_k ? a.c.k : a.c.v) + place[at.tok] + h * a.c.head_stride;
      turned = turn && is_k;
    }
    if (turned) {
      const float2* c = cs + at.tok * half + e;
      if (a.r.interleaved) {
#pragma unroll
        for (int i = 0; i < VEC; i++) {  // pair i: elements 2i, 2i + 1 of the two vectors
          const float2 w = c[i * pair_units];
          T& ra = 2 * i < VEC ? x0.v[(2 * i) % VEC] : x1.v[(2 * i) % VEC];
          T& rb = 2 * i + 1 < VEC ? x0.v[(2 * i + 1) % VEC] : x1.v[(2 * i + 1) % VEC];
          const float fa = Elem<T>::to(ra), fb = Elem<T>::to(rb);
          ra = Elem<T>::from(fa * w.x - fb * w.y);
          rb = Elem<T>::from(fb * w.x + fa * w.y);
        }
      } else {
#pragma unroll
        for (int i = 0; i < VEC; i++) {
          const float2 w = c[i * pair_units];
          const float fa = Elem<T>::to(x0.v[i]), fb = Elem<T>::to(x1.v[i]);
          x0.v[i] = Elem<T>::from(fa * w.x - fb * w.y);
          x1.v[i] = Elem<T>::from(fb * w.x + fa * w.y);
        }
      }
    }
    store(dst + o0, x0);
    if (two) store(dst + o1, x1);
  }
}

// Elements per vector: the most, up to 16 bytes, that every address and
// section length is a multiple of.
struct Widest {
  uint64_t bits = 0;
  void ptr(const void* p, size_t size) { bits |= reinterpret_cast<uintptr_t>(p) / size; }
  void count(int64_t n) { bits |= uint64_t(n); }
  void view(const HeadsView& v, size_t size) {
    ptr(v.p, size);
    count(v.token_stride);
    count(v.head_stride);
  }
  int vec(size_t size) const {
    int n = int(16 / size);
    while (n > 1 && bits % n) n /= 2;
    return n;
  }
};

template <typename T, bool APPEND>
void launch_typed(RotaryParams a, cudaStream_t st) {
  if (a.n_tokens == 0) return;
  Widest w;
  w.view(a.q, sizeof(T));
  w.view(a.q_out, sizeof(T));
  if (APPEND) {
    w.view(a.k, sizeof(T));
    w.view(a.v, sizeof(T));
  }
  w.count(a.r.rot / 2);
  w.count(a.dim);
  const uint32_t heads = a.n_q + (APPEND ? 2 * a.n_kv : 0);
  if (heads == 0) return;
  const int vec = w.vec(sizeof(T));
  a.units = a.r.rot / 2 / vec + (a.dim - a.r.rot + 2 * vec - 1) / (2 * vec);
  // Many tokens go two to a block, few get a block each, for their latency.
  // Two tokens of many heads stay longer in 128 threads than in 256 and hide
  // more (40 heads of 128: 28.9 and 29.8 us for 8192 tokens); of few heads
  // they would take more turns (12 heads of 80: 7.3 and 6.2 us for 4099).
  const bool many = a.n_tokens >= 1024;
  a.tokens_per_block = many ? 2 : 1;
  const bool half_block = many && a.units <= kMaxThreads / 2 && 2 * uint64_t(a.units) * heads >= 2 * kMaxThreads;
  const uint32_t most = half_block ? kMaxThreads / 2 : kMaxThreads;
  const uint32_t threads = most / a.units * a.units;
  a.stream = a.n_tokens * heads * a.dim * sizeof(T) > (uint64_t(32) << 20);
  const uint64_t blocks = (a.n_tokens + a.tokens_per_block - 1) / a.tokens_per_block;
  if (blocks > 0x7FFFFFFFull) throw std::invalid_argument("too many tokens");
  const size_t smem = size_t(a.tokens_per_block) * (a.r.rot / 2) * sizeof(float2);
  const dim3 grid(static_cast<uint32_t>(blocks));
  if (vec == 8) {
    if constexpr (sizeof(T) == 2) launch("rotary", rotary_kernel<T, 8, APPEND>, grid, threads, smem, st, 0, a);
  } else if (vec == 4) {
    launch("rotary", rotary_kernel<T, 4, APPEND>, grid, threads, smem, st, 0, a);
  } else if (vec == 2) {
    launch("rotary", rotary_kernel<T, 2, APPEND>, grid, threads, smem, st, 0, a);
  } else {
    launch("rotary", rotary_kernel<T, 1, APPEND>, grid, threads, smem, st, 0, a);
  }
}

template <bool APPEND>
void launch_any(const RotaryParams& a, int dtype, cudaStream_t st) {
  if (dtype == JB_F16) return launch_typed<__half, APPEND>(a, st);
  if (dtype == JB_BF16) return launch_typed<__nv_bfloat16, APPEND>(a, st);
  if constexpr (!APPEND)
    if (dtype == JB_F32) return launch_typed<float, false>(a, st);
  throw std::invalid_argument("dtype must be JB_F16, JB_BF16 or (jb_rotary) JB_F32");
}

}  // namespace

void launch_rotary(HeadsView x, HeadsView y, int dtype, uint64_t n_tokens, uint32_t n_heads,
                   uint32_t dim, Positions pos, const RotaryArgs& r, cudaStream_t st) {
  RotaryParams p{};
  p.q = x;
  p.q_out = y;
  p.n_q = n_heads;
  p.dim = dim;
  p.n_tokens = n_tokens;
  p.pos = pos;
  p.r = r;
  launch_any<false>(p, dtype, st);
}

void launch_append(const AppendArgs& a, cudaStream_t st) {
  RotaryParams p{};
  p.q = a.q;
  p.q_out = a.q_out;
  p.k = a.k;
  p.v = a.v;
  p.n_q = a.n_q_heads;
  p.n_kv = a.c.n_kv_heads;
  p.dim = a.c.head_dim;
  p.n_tokens = a.n_tokens;
  p.pos = a.pos;
  p.r = a.rotary;
  p.c = a.c;
  p.rows = a.rows;
  p.index = a.index;
  p.layer_offset = int64_t(a.layer) * a.c.layer_stride;
  launch_any<true>(p, a.c.dtype, st);
}

}  // namespace jb
