// rotary.cu -- rotary positions, and new keys and values into the cache's
// pages, in one kernel.
//
// A head's pair (a, b) of pair index i at position p becomes
//     s (a cos t - b sin t),  s (b cos t + a sin t),   t = p theta_i,
// and the gradient is the same turn backwards.  theta_i comes as a fraction
// of a turn in 64-bit fixed point: p * freq wraps at whole turns, so the top
// 32 bits of the product are the reduced angle, exact for every int64
// position; only then does it become a float32 (error 2^-25 of a turn).
//
// A block takes a few tokens: it first computes their cosines and sines once
// (half a head of pairs each, shared by all heads) into shared memory, then
// streams the tokens' heads through registers, two vectors of a pair's two
// sides at a time.
#include <stdexcept>
#include <string>
#include "paged.cuh"

namespace jb {
namespace {

constexpr int kThreads = 256;
constexpr int kMaxTokens = 16;  // per block

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
__global__ void __launch_bounds__(kThreads) rotary_kernel(const RotaryParams a) {
  extern __shared__ float2 cs[];  // [tokens][rot / 2]
  __shared__ int64_t place[kMaxTokens];
  const uint32_t half = a.r.rot / 2;
  const uint64_t t0 = uint64_t(blockIdx.x) * a.tokens_per_block;
  const uint32_t nt = uint32_t(min(uint64_t(a.tokens_per_block), a.n_tokens - t0));

  if (APPEND && threadIdx.x < nt) {
    // the token's place in its page, -1 where there is none
    const uint64_t t = t0 + threadIdx.x;
    const int32_t row = a.rows[t];
    int64_t at = -1;
    if (row >= 0 && uint32_t(row) < a.c.n_rows) {
      const int64_t i = a.index ? int64_t(a.index[t]) : int64_t(a.c.lengths[row]) - 1;
      if (i >= 0 && uint64_t(i) / a.c.page_size < a.c.max_pages) {
        const uint32_t pg = uint32_t(i) / a.c.page_size, slot = uint32_t(i) % a.c.page_size;
        const int32_t page = a.c.table[row * a.c.table_stride + pg];
        if (page >= 0 && uint32_t(page) < a.c.n_pages)
          at = a.layer_offset + page * a.c.page_stride + slot * a.c.token_stride;
      }
    }
    place[threadIdx.x] = at;
    if (at < 0) atomicOr(a.c.status, kPagesBadToken);
  }
  for (uint32_t j = threadIdx.x; j < nt * half; j += kThreads) {
    const uint32_t tok = j / half, i = j % half;
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
    cs[j] = make_float2(cn * a.r.scale, (a.r.inverse ? -sn : sn) * a.r.scale);
  }
  __syncthreads();

  const uint32_t pair_units = half / VEC;
  const uint32_t units = pair_units + (a.dim - a.r.rot + 2 * VEC - 1) / (2 * VEC);
  const uint32_t heads = a.n_q + (APPEND ? 2 * a.n_kv : 0);
  using V = Vec<T, VEC>;
  for (uint32_t u = threadIdx.x; u < nt * heads * units; u += kThreads) {
    const uint32_t hu = u / units, e = u % units;
    const uint32_t tok = hu / heads;
    uint32_t h = hu % heads;
    const uint64_t t = t0 + tok;
    const T* src;
    T* dst;
    bool turn = e < pair_units, plain_head = false;
    if (h < a.n_q) {
      src = static_cast<const T*>(a.q.p) + t * a.q.token_stride + h * a.q.head_stride;
      dst = static_cast<T*>(a.q_out.p) + t * a.q_out.token_stride + h * a.q_out.head_stride;
    } else {
      if (place[tok] < 0) continue;
      h -= a.n_q;
      const bool is_k = h < a.n_kv;
      if (!is_k) h -= a.n_kv;
      const HeadsView& s = is_k ? a.k : a.v;
      src = static_cast<const T*>(s.p) + t * s.token_stride + h * s.head_stride;
      dst = static_cast<T*>(is_k ? a.c.k : a.c.v) + place[tok] + h * a.c.head_stride;
      plain_head = !is_k;
    }
    uint32_t o0, o1;  // the unit's two vectors
    if (turn) {
      o0 = a.r.interleaved ? 2 * VEC * e : VEC * e;
      o1 = a.r.interleaved ? o0 + VEC : o0 + half;
    } else {
      o0 = a.r.rot + 2 * VEC * (e - pair_units);
      o1 = o0 + VEC;
    }
    const bool two = o1 < a.dim;
    V x0 = *reinterpret_cast<const V*>(src + o0), x1;
    if (two) x1 = *reinterpret_cast<const V*>(src + o1);
    if (turn && !plain_head) {
      const float2* c = cs + tok * half + VEC * e;
      if (a.r.interleaved) {
#pragma unroll
        for (int i = 0; i < VEC; i++) {  // pair i: elements 2i, 2i + 1 of the two vectors
          const float2 w = c[i];
          T& ra = 2 * i < VEC ? x0.v[(2 * i) % VEC] : x1.v[(2 * i) % VEC];
          T& rb = 2 * i + 1 < VEC ? x0.v[(2 * i + 1) % VEC] : x1.v[(2 * i + 1) % VEC];
          const float fa = Elem<T>::to(ra), fb = Elem<T>::to(rb);
          ra = Elem<T>::from(fa * w.x - fb * w.y);
          rb = Elem<T>::from(fb * w.x + fa * w.y);
        }
      } else {
#pragma unroll
        for (int i = 0; i < VEC; i++) {
          const float2 w = c[i];
          const float fa = Elem<T>::to(x0.v[i]), fb = Elem<T>::to(x1.v[i]);
          x0.v[i] = Elem<T>::from(fa * w.x - fb * w.y);
          x1.v[i] = Elem<T>::from(fb * w.x + fa * w.y);
        }
      }
    }
    *reinterpret_cast<V*>(dst + o0) = x0;
    if (two) *reinterpret_cast<V*>(dst + o1) = x1;
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
  a.tokens_per_block = 1;
  const uint64_t blocks = (a.n_tokens + a.tokens_per_block - 1) / a.tokens_per_block;
  if (blocks > 0x7FFFFFFFull) throw std::invalid_argument("too many tokens");
  const size_t smem = size_t(a.tokens_per_block) * (a.r.rot / 2) * sizeof(float2);
  switch (vec) {
    case 8:
      if constexpr (sizeof(T) == 2)
        rotary_kernel<T, 8, APPEND><<<uint32_t(blocks), kThreads, smem, st>>>(a);
      break;
    case 4: rotary_kernel<T, 4, APPEND><<<uint32_t(blocks), kThreads, smem, st>>>(a); break;
    case 2: rotary_kernel<T, 2, APPEND><<<uint32_t(blocks), kThreads, smem, st>>>(a); break;
    default: rotary_kernel<T, 1, APPEND><<<uint32_t(blocks), kThreads, smem, st>>>(a); break;
  }
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess)
    throw std::runtime_error(std::string("rotary launch: ") + cudaGetErrorString(e));
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
