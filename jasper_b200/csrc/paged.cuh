// paged.cuh -- the paged key-value cache: what its kernels see of it, and
// their launchers (rotary.cu, pages.cu, attend.cu).  The reference has no
// counterpart: it ends where the search's answer does.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <cstddef>
#include <cstdint>
#include <stdexcept>
#include <string>
#include "../../include/jasper_b200.h"

namespace jb {

// A decode step is a chain of kernels of a few microseconds, so each is launched
// while the one before it still runs (programmatic dependent launch), and
// begins with follow(): it lets the next one start, and waits until all that
// came before has ended and can be read.  Every thread of every kernel here
// calls it before it touches global memory or returns, so that no kernel ends
// before its predecessors.  In a stream, 8 heads of one row of 1000 tokens: 8.2
// -> 6.5 us a call; rotary positions of 4099 x 12 x 80 float32: 8.2 -> 6.3.
__device__ __forceinline__ void follow() {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
}

// Launches a kernel that begins with follow(); cluster > 0: in clusters of so
// many blocks (a kernel's own cluster size otherwise).
template <typename... P, typename... A>
void launch(const char* what, void (*kernel)(P...), dim3 grid, uint32_t threads, size_t shared, cudaStream_t st,
            uint32_t cluster, const A&... args) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = shared;
  cfg.stream = st;
  cudaLaunchAttribute attrs[2]{};
  attrs[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attrs[0].val.programmaticStreamSerializationAllowed = 1;
  attrs[1].id = cudaLaunchAttributeClusterDimension;
  attrs[1].val.clusterDim.x = cluster;
  attrs[1].val.clusterDim.y = attrs[1].val.clusterDim.z = 1;
  cfg.attrs = attrs;
  cfg.numAttrs = cluster ? 2 : 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, args...);
  if (e != cudaSuccess) {
    cudaGetLastError();
    throw std::runtime_error(std::string(what) + " launch: " + cudaGetErrorString(e));
  }
}

// Bits of a cache's status word (jb_page_cache::status).
constexpr int kPagesExhausted = JB_PAGES_EXHAUSTED;
constexpr int kPagesBadRow = JB_PAGES_BAD_ROW;
constexpr int kPagesBadToken = JB_PAGES_BAD_TOKEN;

// Bits of a row's mark (jb_page_cache::marks): its last extend was refused; and
// the length at which it was adopted, if that is inside a page.  What follows in
// that page is not the row's.
constexpr int32_t kMarkRefused = INT32_MIN, kMarkAdopted = INT32_MAX;

// Rotary positions as the kernels take them: freq[i] is pair i's turn for one
// position in units of 2^-64 of a turn, so position * freq wraps at whole
// turns and its top bits are the angle, reduced exactly for every int64
// position.
struct RotaryArgs {
  const int64_t* freq = nullptr;  // null: no rotation
  uint32_t rot = 0;               // rotated elements of a head (even)
  float scale = 1.0f;             // factor on the rotated elements
  bool interleaved = false;       // pairs (2i, 2i+1) instead of (i, i + rot/2)
  bool inverse = false;           // turn backwards (the gradient)
};

// Positions as int32 or int64, whichever pointer is not null.
struct Positions {
  const int32_t* p32 = nullptr;
  const int64_t* p64 = nullptr;
  __device__ __forceinline__ int64_t at(uint64_t i) const { return p64 ? p64[i] : int64_t(p32[i]); }
};

// [tokens][heads][dim] elements at any token and head stride, dim contiguous.
struct HeadsView {
  void* p = nullptr;
  int64_t token_stride = 0, head_stride = 0;
};

void launch_rotary(HeadsView x, HeadsView y, int dtype, uint64_t n_tokens, uint32_t n_heads,
                   uint32_t dim, Positions pos, const RotaryArgs& r, cudaStream_t st);

struct AppendArgs {
  jb_page_cache c;
  uint32_t layer;
  uint64_t n_tokens;
  HeadsView q, q_out, k, v;
  uint32_t n_q_heads;
  const int32_t* rows;
  const int32_t* index;  // null: the row's last token
  Positions pos;         // both null: the token's index
  RotaryArgs rotary;
};
void launch_append(const AppendArgs& a, cudaStream_t st);

// Throws if the copies of n pages cannot be counted in 32 bits; before a call
// that copies pages changes anything.
void check_copies(const jb_page_cache& c, uint64_t n);
// The page operations' scratch, in int32 words.
size_t pages_plan_words(const jb_page_cache& c, uint64_t n);
void launch_extend(const jb_page_cache& c, const int32_t* rows, const int32_t* tokens, uint32_t n,
                   int32_t* scratch, cudaStream_t st);
void launch_fork(const jb_page_cache& c, const int32_t* parents, const int32_t* children,
                 uint32_t n, int32_t* scratch, cudaStream_t st);
void launch_free(const jb_page_cache& c, const int32_t* rows, uint32_t n, cudaStream_t st);
void launch_adopt(const jb_page_cache& c, const int32_t* rows, const int32_t* pages,
                  int64_t pages_stride, uint32_t m, const int32_t* lengths, uint32_t n,
                  int32_t* scratch, cudaStream_t st);
void launch_compact(const jb_page_cache& c, int32_t* remap, int32_t* scratch, cudaStream_t st);
void launch_copy_pages(const jb_page_cache& c, const int32_t* src, const int32_t* dst, uint32_t n,
                       cudaStream_t st);

struct AttendArgs {
  jb_page_cache c;
  uint32_t layer;
  uint32_t n;            // queries: one new token of each of n rows
  uint32_t n_q_heads;
  HeadsView q, out;
  const int32_t* rows;   // null: query i is row i
  const uint8_t* mask;   // [n][mask_stride] truth values of the first mask_width tokens, or null
  int64_t mask_stride;
  uint32_t mask_width;
  float* lse;            // [n][n_q_heads], or null
  float scale;
  uint32_t window;       // the last `window` tokens only; 0: all
};
// Scratch of one call, in bytes (0: none).
size_t attend_scratch_bytes(const AttendArgs& a);
void launch_attend(const AttendArgs& a, void* scratch, cudaStream_t st);

}  // namespace jb
