// Storage of the 3-bit KV cache shared by its kernels: the cache and pool
// structures, the record layout (described in ft_kv3.cu) and the layout maps.
#pragma once

#include <algorithm>
#include <vector>

#include "ft_internal.cuh"

struct ft_kv3 {
  int device = 0;
  int64_t batch = 0, kv_heads = 0, cap = 0;  // cap: slots per row, multiple of 32
  int64_t head = 0, len = 0;                   // ring start slot, live positions
  uint32_t* blocks = nullptr;  // [row][cap/32] block records
  ft::Workspace part;  // split partials
  int mode = 0;                // 0: the reference's min/max scheme, 1: mode T
  float* signs = nullptr;      // mode T: the 128 rotation signs (device)
  ft::Workspace rot;           // mode T: the rotated queries
  ft::Workspace scores;        // decode with weights: every position's score
  ft::Workspace tree;          // tree decode: split partials
  std::vector<void*> retired;  // outgrown buffers (see ensure_ws)
};

// The page pool of the paged cache: page P holds 32 positions of every kv
// head, record (P, h) at (P * kv_heads + h) * 3584 bytes -- the ring's record,
// so the same kernels serve both.  The pool is storage only: which pages a
// sequence owns, and in which order, is the caller's block table.
struct ft_kvp {
  int device = 0;
  int64_t n_pages = 0, kv_heads = 0;
  uint32_t* blocks = nullptr;
  int mode = 0;
  float* signs = nullptr;
  ft::Workspace part, rot, scores, tree;
  std::vector<void*> retired;
};

namespace ft {

constexpr int kD = 128;                  // head dim = quantisation group
constexpr int kRec = 48;                 // bytes of codes per vector
constexpr int kBlk = 32;                 // slots per block
constexpr int kBlkWords = kBlk * kRec / 4;  // 384
constexpr int kBlkBytes = kBlk * kRec;   // 1536 (both K and V)
constexpr int kMmBlkBytes = kBlk * 8;    // 256
constexpr int kRecBytes = 2 * kBlkBytes + 2 * kMmBlkBytes;  // 3584: K | V | K min/max | V min/max
constexpr int kRecWords = kRecBytes / 4;
constexpr int kRecV = kBlkWords, kRecKmm = 2 * kBlkWords, kRecVmm = 2 * kBlkWords + 2 * kBlk;

__device__ __forceinline__ float load_act(const void* p, int64_t i, int bf16) {
  return bf16 ? __uint_as_float((uint32_t) static_cast<const uint16_t*>(p)[i] << 16)
              : static_cast<const float*>(p)[i];
}

// ---- layout maps (word indices within a 384-word block) ----
// triple base word and quad of K code (slot s, dim d) / V code (slot s, dim d)
__device__ __forceinline__ int k_triple(int s, int d) {
  return (4 * (s & 7) + ((d >> 2) & 3)) * 12 + 3 * (s >> 3);
}
__device__ __forceinline__ int k_quad(int d) { return d >> 4; }
__device__ __forceinline__ int k_elem(int s, int d) { return d & 3; }
__device__ __forceinline__ int v_triple(int s, int d) {
  return (4 * (d & 7) + (s & 3)) * 12 + 3 * (d >> 5);
}
__device__ __forceinline__ int v_quad(int s, int d) {
  return 2 * (2 * ((d >> 4) & 1) + ((d >> 3) & 1)) + ((s >> 2) & 1);
}
__device__ __forceinline__ int v_elem(int s) { return s >> 3; }
__device__ __forceinline__ int mm_index(int s) { return (s & 7) * 4 + (s >> 3); }

__device__ __forceinline__ uint32_t triple_get(const uint32_t* t, int Q, int b) {
  if (Q < 6) return (t[Q >> 1] >> (8 * b + 3 * (Q & 1))) & 7u;
  return ((t[Q - 6] >> (8 * b + 6)) & 3u) | (((t[2] >> (8 * b + Q)) & 1u) << 2);
}
// writes code c at (Q, b) of a shared-memory triple; concurrent writers touch
// disjoint bits
__device__ __forceinline__ void triple_put(uint32_t* t, int Q, int b, uint32_t c) {
  if (Q < 6) {
    const int sh = 8 * b + 3 * (Q & 1);
    atomicAnd(&t[Q >> 1], ~(7u << sh));
    atomicOr(&t[Q >> 1], c << sh);
  } else {
    atomicAnd(&t[Q - 6], ~(3u << (8 * b + 6)));
    atomicOr(&t[Q - 6], (c & 3u) << (8 * b + 6));
    atomicAnd(&t[2], ~(1u << (8 * b + Q)));
    atomicOr(&t[2], (c >> 2) << (8 * b + Q));
  }
}
__device__ __forceinline__ uint32_t k_code(const uint32_t* blk, int s, int d) {
  return triple_get(blk + k_triple(s, d), k_quad(d), k_elem(s, d));
}
__device__ __forceinline__ uint32_t v_code(const uint32_t* blk, int s, int d) {
  return triple_get(blk + v_triple(s, d), v_quad(s, d), v_elem(s));
}

// A page index read from a caller's block table, checked: out-of-range
// entries are recorded in the error word (site `code`) and replaced by -1.
__device__ __forceinline__ int64_t checked_page(const int32_t* table, int64_t idx,
                                                int64_t n_pages, int* err, int code) {
  const int32_t pg = table[idx];
  if (pg < 0 || pg >= n_pages) {
    if (err) atomicCAS(err, 0, code);
    return -1;
  }
  return pg;
}

class DeviceScope {
 public:
  explicit DeviceScope(int dev) : dev_(dev) {
    cudaGetDevice(&prev_);
    if (prev_ != dev) cudaSetDevice(dev);
  }
  ~DeviceScope() {
    if (prev_ >= 0 && prev_ != dev_) cudaSetDevice(prev_);
  }

 private:
  int dev_ = 0, prev_ = -1;
};

// Grows a workspace outside stream capture (a capture may only reuse it).  A buffer
// that a capture has used is kept in `retired` until the cache is destroyed, since the
// graph still uses it, and the next one is at least twice as large, so that the kept
// ones add up to less than the last.  Any other is freed first (cudaFree waits for the
// work in flight), and the next has an eighth to spare, or what is needed where that
// does not fit.
inline int ensure_ws(Workspace& w, size_t need, cudaStream_t s, const char* what,
                     std::vector<void*>& retired) {
  cudaStreamCaptureStatus cs = cudaStreamCaptureStatusNone;
  if (s) cudaStreamIsCapturing(s, &cs);
  if (w.bytes >= need) {
    if (cs != cudaStreamCaptureStatusNone) w.captured = true;
    return FT_OK;
  }
  FT_CHECK(cs == cudaStreamCaptureStatusNone, FT_ERR_UNSUPPORTED,
           "the %s buffer must grow but the stream is being captured", what);
  size_t size = w.bytes ? need + need / 8 : need;
  if (w.captured) {
    size = std::max(size, 2 * w.bytes);
    try {
      retired.push_back(w.ptr);
    } catch (...) {  // no exception crosses the C boundary
      return fail(FT_ERR_OOM, "out of host memory");
    }
  } else if (w.ptr) {
    FT_CUDA(cudaFree(w.ptr));
  }
  w = Workspace{};
  cudaError_t e = cudaMalloc(&w.ptr, size);
  if (e == cudaErrorMemoryAllocation && size > need) {
    cudaGetLastError();
    size = need;
    e = cudaMalloc(&w.ptr, size);
  }
  if (e != cudaSuccess) {
    w.ptr = nullptr;
    cudaGetLastError();
    return fail(e == cudaErrorMemoryAllocation ? FT_ERR_OOM : FT_ERR_GPU,
                "the %s buffer of %zu bytes: %s", what, size, cudaGetErrorString(e));
  }
  w.bytes = size;
  return FT_OK;
}

// A new ring of at least `need` slots whose head lies in its first block
// (ft_kv3.cu); synchronises the stream, and fails while it is captured.
int kv3_grow(ft_kv3* c, int64_t need, cudaStream_t s);

}  // namespace ft
