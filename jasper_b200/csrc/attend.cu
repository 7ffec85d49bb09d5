// attend.cu -- attention of one new token of each row over the paged cache.
//
// out = sum_t p_t v_t, p = softmax(scale * q . k_t) over the tokens attended
// to, in one pass with the running maximum m and sum l of the softmax: a
// score above m rescales what was gathered by exp(m_old - m_new).
//
// One warp per (row, query head): each lane holds head_dim / 32 of the
// query's and the output's elements.
#include <cmath>
#include <stdexcept>
#include <string>
#include "paged.cuh"

namespace jb {
namespace {

constexpr int kMaxPerLane = 8;  // head_dim up to 256

template <typename T>
__device__ __forceinline__ float to_float(T v);
template <>
__device__ __forceinline__ float to_float<__half>(__half v) { return __half2float(v); }
template <>
__device__ __forceinline__ float to_float<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T>
__device__ __forceinline__ T from_float(float v);
template <>
__device__ __forceinline__ __half from_float<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

template <typename T>
__global__ void __launch_bounds__(32) attend_warp_kernel(const AttendArgs a) {
  const jb_page_cache& c = a.c;
  const uint32_t i = blockIdx.x / a.n_q_heads, hq = blockIdx.x % a.n_q_heads;
  const uint32_t h = hq / (a.n_q_heads / c.n_kv_heads);
  const int lane = threadIdx.x;
  const int32_t row = a.rows ? a.rows[i] : int32_t(i);
  int64_t len = 0;
  if (row >= 0 && uint32_t(row) < c.n_rows)
    len = min(int64_t(max(c.lengths[row], 0)), int64_t(c.max_pages) * c.page_size);
  const int64_t first = a.window && len > int64_t(a.window) ? len - a.window : 0;
  const T* q = static_cast<const T*>(a.q.p) + i * a.q.token_stride + hq * a.q.head_stride;
  const T* k = static_cast<const T*>(c.k) + int64_t(a.layer) * c.layer_stride + h * c.head_stride;
  const T* v = static_cast<const T*>(c.v) + int64_t(a.layer) * c.layer_stride + h * c.head_stride;
  float qf[kMaxPerLane], o[kMaxPerLane];
#pragma unroll
  for (int j = 0; j < kMaxPerLane; j++) {
    const uint32_t d = lane + 32 * j;
    qf[j] = d < c.head_dim ? to_float(q[d]) * a.scale : 0.0f;
    o[j] = 0.0f;
  }
  float m = -INFINITY, l = 0.0f;
  for (int64_t t = first; t < len; t++) {
    if (a.mask && t < a.mask_width && !a.mask[i * a.mask_stride + t]) continue;
    const int32_t page = c.table[row * c.table_stride + t / c.page_size];
    if (page < 0 || uint32_t(page) >= c.n_pages) continue;
    const int64_t off = page * c.page_stride + (t % c.page_size) * c.token_stride;
    float s = 0.0f;
#pragma unroll
    for (int j = 0; j < kMaxPerLane; j++) {
      const uint32_t d = lane + 32 * j;
      if (d < c.head_dim) s += qf[j] * to_float(k[off + d]);
    }
#pragma unroll
    for (int w = 16; w; w >>= 1) s += __shfl_xor_sync(0xFFFFFFFFu, s, w);
    const float mn = fmaxf(m, s);
    const float keep = m == -INFINITY ? 0.0f : expf(m - mn);
    const float p = mn == -INFINITY ? 0.0f : expf(s - mn);
    m = mn;
    l = l * keep + p;
#pragma unroll
    for (int j = 0; j < kMaxPerLane; j++) {
      const uint32_t d = lane + 32 * j;
      if (d < c.head_dim) o[j] = o[j] * keep + p * to_float(v[off + d]);
    }
  }
  T* out = static_cast<T*>(a.out.p) + i * a.out.token_stride + hq * a.out.head_stride;
  const float inv = l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll
  for (int j = 0; j < kMaxPerLane; j++) {
    const uint32_t d = lane + 32 * j;
    if (d < c.head_dim) out[d] = from_float<T>(o[j] * inv);
  }
  if (a.lse && lane == 0) a.lse[uint64_t(i) * a.n_q_heads + hq] = l == 0.0f ? -INFINITY : m + logf(l);
}

}  // namespace

size_t attend_scratch_bytes(const AttendArgs&) { return 0; }

void launch_attend(const AttendArgs& a, void*, cudaStream_t st) {
  if (a.n == 0 || a.n_q_heads == 0) return;
  const uint64_t blocks = uint64_t(a.n) * a.n_q_heads;
  if (blocks > 0x7FFFFFFFull) throw std::invalid_argument("too many query heads");
  if (a.c.dtype == JB_F16) attend_warp_kernel<__half><<<uint32_t(blocks), 32, 0, st>>>(a);
  else attend_warp_kernel<__nv_bfloat16><<<uint32_t(blocks), 32, 0, st>>>(a);
  const cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess)
    throw std::runtime_error(std::string("attend launch: ") + cudaGetErrorString(e));
}

}  // namespace jb
