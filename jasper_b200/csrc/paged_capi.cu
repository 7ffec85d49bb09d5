// paged_capi.cu -- extern "C" entry points of the paged key-value cache
// (include/jasper_b200.h): argument checks, the cache's device, per-call
// scratch from the library's stream-ordered pool.
#include <cmath>
#include <functional>
#include <stdexcept>
#include <string>
#include "paged.cuh"

namespace jb {
int capi_guarded(const std::function<void()>& f);
void capi_pool_alloc(void** p, size_t bytes, cudaStream_t st);
}  // namespace jb

namespace {

void require(bool ok, const char* message) {
  if (!ok) throw std::invalid_argument(message);
}

// Runs with the cache's device current, restoring the caller's afterwards.
struct OnDevice {
  int prev = -1;
  explicit OnDevice(int dev) {
    int cur = -1;
    cudaError_t e = cudaGetDevice(&cur);
    if (e == cudaSuccess && cur != dev) {
      e = cudaSetDevice(dev);
      if (e == cudaSuccess) prev = cur;
    }
    if (e != cudaSuccess) {
      cudaGetLastError();
      throw std::runtime_error(std::string("set device: ") + cudaGetErrorString(e));
    }
  }
  ~OnDevice() {
    if (prev >= 0) cudaSetDevice(prev);
  }
};

// Scratch from the pool, freed in stream order.
struct Scratch {
  void* p = nullptr;
  cudaStream_t st;
  Scratch(size_t bytes, cudaStream_t s) : st(s) {
    if (bytes) jb::capi_pool_alloc(&p, bytes, s);
  }
  ~Scratch() {
    if (p && cudaFreeAsync(p, st) != cudaSuccess) cudaGetLastError();
  }
};

bool aligned16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

const jb_page_cache& checked(const jb_page_cache* c) {
  require(c != nullptr, "cache is null");
  require(c->dtype == JB_F16 || c->dtype == JB_BF16, "the cache's dtype must be JB_F16 or JB_BF16");
  require(c->head_dim > 0 && c->head_dim % 8 == 0 && c->head_dim <= 256,
          "head_dim must be a multiple of 8, at most 256");
  require(c->page_size > 0 && c->page_size <= (1u << 20), "page_size must be 1 to 2^20");
  require(c->n_kv_heads > 0 && c->n_kv_heads <= 65536, "n_kv_heads must be 1 to 65536");
  require(c->n_pages < (1u << 29), "n_pages must be below 2^29");
  require(c->n_rows < (1u << 30) && c->max_pages < (1u << 30), "n_rows and max_pages must be below 2^30");
  require(c->table && c->lengths && c->refs && c->status, "null pointer in the cache");
  require((c->k && c->v) || c->n_pages == 0 || c->n_layers == 0, "null pointer in the cache");
  require(aligned16(c->k) && aligned16(c->v), "keys and values must be 16-byte aligned");
  require(c->layer_stride % 8 == 0 && c->page_stride % 8 == 0 && c->token_stride % 8 == 0 &&
              c->head_stride % 8 == 0,
          "the cache's strides must be multiples of 16 bytes");
  require(c->n_rows <= 1 || c->table_stride >= int64_t(c->max_pages), "table_stride < max_pages");
  return *c;
}

jb::RotaryArgs rotary_args(const int64_t* freq, uint32_t rot_dim, uint32_t head_dim, float scale,
                           int32_t interleaved, bool inverse) {
  jb::RotaryArgs r;
  if (freq == nullptr) return r;
  require(rot_dim % 2 == 0 && rot_dim <= head_dim, "rot_dim must be even and at most head_dim");
  r.freq = freq;
  r.rot = rot_dim;
  r.scale = scale;
  r.interleaved = interleaved != 0;
  r.inverse = inverse;
  return r;
}

jb::Positions positions_of(const void* p, int32_t is64) {
  jb::Positions pos;
  if (is64) pos.p64 = static_cast<const int64_t*>(p);
  else pos.p32 = static_cast<const int32_t*>(p);
  return pos;
}

jb::HeadsView view_of(const void* p, int64_t ts, int64_t hs) {
  jb::HeadsView v;
  v.p = const_cast<void*>(p);
  v.token_stride = ts;
  v.head_stride = hs;
  return v;
}

}  // namespace

extern "C" {

int jb_rotary(const void* x, int64_t x_token_stride, int64_t x_head_stride, void* y,
              int64_t y_token_stride, int64_t y_head_stride, int32_t dtype, uint64_t n_tokens,
              uint32_t n_heads, uint32_t head_dim, uint32_t rot_dim, const void* positions,
              int32_t positions_64, const int64_t* freq, float scale, int32_t interleaved,
              int32_t inverse, void* stream) {
  return jb::capi_guarded([&] {
    require(dtype == JB_F16 || dtype == JB_BF16 || dtype == JB_F32, "dtype must be JB_F16, JB_BF16 or JB_F32");
    require(head_dim > 0 && head_dim <= 512, "head_dim must be 1 to 512");
    require(n_heads <= 65536, "n_heads must be at most 65536");
    if (n_tokens == 0 || n_heads == 0) return;
    require(x && y && positions && freq, "null pointer argument");
    jb::launch_rotary(view_of(x, x_token_stride, x_head_stride), view_of(y, y_token_stride, y_head_stride),
                      dtype, n_tokens, n_heads, head_dim, positions_of(positions, positions_64),
                      rotary_args(freq, rot_dim, head_dim, scale, interleaved, inverse != 0),
                      static_cast<cudaStream_t>(stream));
  });
}

int jb_kv_append(const jb_page_cache* cache, uint32_t layer, uint64_t n_tokens, const void* q,
                 int64_t q_token_stride, int64_t q_head_stride, void* q_out,
                 int64_t q_out_token_stride, int64_t q_out_head_stride, uint32_t n_q_heads,
                 const void* k, int64_t k_token_stride, int64_t k_head_stride, const void* v,
                 int64_t v_token_stride, int64_t v_head_stride, const int32_t* rows,
                 const int32_t* index, const void* positions, int32_t positions_64,
                 const int64_t* freq, uint32_t rot_dim, float scale, int32_t interleaved,
                 void* stream) {
  return jb::capi_guarded([&] {
    jb::AppendArgs a{};
    a.c = checked(cache);
    require(layer < a.c.n_layers, "layer out of range");
    require(n_q_heads <= 65536, "n_q_heads must be at most 65536");
    if (n_tokens == 0) return;
    require(k && v && rows, "null pointer argument");
    require(!q || (q_out && freq), "q needs q_out and freq");
    require(index || a.c.marks, "without index the cache's marks are needed");
    a.layer = layer;
    a.n_tokens = n_tokens;
    if (q) {
      a.q = view_of(q, q_token_stride, q_head_stride);
      a.q_out = view_of(q_out, q_out_token_stride, q_out_head_stride);
      a.n_q_heads = n_q_heads;
    }
    a.k = view_of(k, k_token_stride, k_head_stride);
    a.v = view_of(v, v_token_stride, v_head_stride);
    a.rows = rows;
    a.index = index;
    a.pos = positions_of(positions, positions_64);
    a.rotary = rotary_args(freq, rot_dim, a.c.head_dim, scale, interleaved, false);
    OnDevice on(a.c.device);
    jb::launch_append(a, static_cast<cudaStream_t>(stream));
  });
}

int jb_pages_extend(const jb_page_cache* cache, const int32_t* rows, const int32_t* tokens,
                    uint32_t n, void* stream) {
  return jb::capi_guarded([&] {
    const jb_page_cache& c = checked(cache);
    if (n == 0) return;
    require(rows && tokens, "null pointer argument");
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    OnDevice on(c.device);
    Scratch s(jb::pages_plan_words(c, n) * sizeof(int32_t), st);
    jb::launch_extend(c, rows, tokens, n, static_cast<int32_t*>(s.p), st);
  });
}

int jb_pages_fork(const jb_page_cache* cache, const int32_t* parents, const int32_t* children,
                  uint32_t n, void* stream) {
  return jb::capi_guarded([&] {
    const jb_page_cache& c = checked(cache);
    if (n == 0) return;
    require(parents && children, "null pointer argument");
    jb::check_copies(c, n);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    OnDevice on(c.device);
    Scratch s(jb::pages_plan_words(c, n) * sizeof(int32_t), st);
    jb::launch_fork(c, parents, children, n, static_cast<int32_t*>(s.p), st);
  });
}

int jb_pages_free(const jb_page_cache* cache, const int32_t* rows, uint32_t n, void* stream) {
  return jb::capi_guarded([&] {
    const jb_page_cache& c = checked(cache);
    if (n == 0) return;
    require(rows != nullptr, "null pointer argument");
    require(n < (1u << 30), "too many rows");
    OnDevice on(c.device);
    jb::launch_free(c, rows, n, static_cast<cudaStream_t>(stream));
  });
}

int jb_pages_adopt(const jb_page_cache* cache, const int32_t* rows, const int32_t* pages,
                   int64_t pages_stride, uint32_t m, const int32_t* lengths, uint32_t n,
                   void* stream) {
  return jb::capi_guarded([&] {
    const jb_page_cache& c = checked(cache);
    if (n == 0) return;
    require(rows && (pages || m == 0), "null pointer argument");
    require(n < (1u << 30), "too many rows");
    require(m <= c.max_pages, "more pages than a row of the table holds");
    require(!lengths || c.marks, "with lengths the cache's marks are needed");
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    OnDevice on(c.device);
    Scratch s(size_t(c.n_rows) * sizeof(int32_t), st);
    jb::launch_adopt(c, rows, pages, pages_stride, m, lengths, n, static_cast<int32_t*>(s.p), st);
  });
}

int jb_pages_compact(const jb_page_cache* cache, int32_t* remap, void* stream) {
  return jb::capi_guarded([&] {
    const jb_page_cache& c = checked(cache);
    if (c.n_pages == 0) return;
    require(remap != nullptr, "null pointer argument");
    jb::check_copies(c, c.n_pages);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    OnDevice on(c.device);
    Scratch s(jb::pages_plan_words(c, 0) * sizeof(int32_t), st);
    jb::launch_compact(c, remap, static_cast<int32_t*>(s.p), st);
  });
}

int jb_pages_copy(const jb_page_cache* cache, const int32_t* src, const int32_t* dst, uint32_t n,
                  void* stream) {
  return jb::capi_guarded([&] {
    const jb_page_cache& c = checked(cache);
    if (n == 0) return;
    require(src && dst, "null pointer argument");
    jb::check_copies(c, n);
    OnDevice on(c.device);
    jb::launch_copy_pages(c, src, dst, n, static_cast<cudaStream_t>(stream));
  });
}

int jb_paged_attention(const jb_page_cache* cache, uint32_t layer, const void* q,
                       int64_t q_row_stride, int64_t q_head_stride, void* out,
                       int64_t out_row_stride, int64_t out_head_stride, uint32_t n,
                       uint32_t n_q_heads, const int32_t* rows, const uint8_t* mask,
                       int64_t mask_stride, uint32_t mask_width, uint32_t window, float scale,
                       float* lse, void* stream) {
  return jb::capi_guarded([&] {
    jb::AttendArgs a{};
    a.c = checked(cache);
    require(layer < a.c.n_layers, "layer out of range");
    require(n_q_heads % a.c.n_kv_heads == 0, "n_q_heads must be a multiple of n_kv_heads");
    require(n_q_heads <= 65536 && n < (1u << 30), "too many query heads or rows");
    require(std::isfinite(scale), "scale must be finite");
    if (n == 0 || n_q_heads == 0) return;
    require(q && out, "null pointer argument");
    require(aligned16(q) && aligned16(out) && q_row_stride % 8 == 0 && q_head_stride % 8 == 0 &&
                out_row_stride % 8 == 0 && out_head_stride % 8 == 0,
            "q and out must be 16-byte aligned, at strides that are multiples of 16 bytes");
    require(uint64_t(a.c.max_pages) * a.c.page_size <= 0x7FFFFFFFull,
            "max_pages * page_size must be below 2^31");
    a.layer = layer;
    a.n = n;
    a.n_q_heads = n_q_heads;
    a.q = view_of(q, q_row_stride, q_head_stride);
    a.out = view_of(out, out_row_stride, out_head_stride);
    a.rows = rows;
    a.mask = mask;
    a.mask_stride = mask_stride;
    a.mask_width = mask ? mask_width : 0;
    a.window = window;
    a.scale = scale;
    a.lse = lse;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    OnDevice on(a.c.device);
    Scratch s(jb::attend_scratch_bytes(a), st);
    jb::launch_attend(a, s.p, st);
  });
}

}  // extern "C"
