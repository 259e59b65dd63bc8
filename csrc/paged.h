// The paged key/value cache shared by its write / read kernels (csrc/paged.cu) and its attention kernels.
//
// A pool holds `pages` pages of `page` tokens (a power of two): keys and values [pages, Hk, page, D], bf16 or e4m3
// bytes; e4m3 pools carry one E8M0 scale byte per (token, key head), [pages, Hk, page], value = e4m3 * 2^(byte - 127).
// Token t of sequence b sits in page table[b, t / page], slot t % page.
#pragma once
#include <c10/cuda/CUDAException.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

#include <mutex>

#include "common.cuh"

namespace ng {

struct PagedPool {
  void* k;
  void* v;
  uint8_t* ksf;  // null: bf16 pool
  uint8_t* vsf;
  const int* table;
  int64_t ld_table;
  int width;       // table columns
  int pages;
  int Hk, D;
  int page_shift;  // log2(page)
};

// Scale exponents are kept in [kScaleLo, kScaleHi]: the ratio of two scales and of their products with probabilities
// then stays inside fp32's normal range (values beyond 448 * 2^63 saturate, values below 2^-71 round to zero).
constexpr int kScaleLo = -62, kScaleHi = 63;

__device__ __forceinline__ float exp2i(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }  // |e| <= 126

// two e4m3 bytes (the low half of w) -> f16x2, exact
__device__ __forceinline__ uint32_t e4m3x2_f16x2(uint32_t w) {
  uint32_t r;
  asm("{\n\t.reg .b16 lo;\n\tcvt.u16.u32 lo, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, lo;\n\t}\n" : "=r"(r) : "r"(w));
  return r;
}
// four e4m3 bytes times a power of two -> two bf16x2, exact (e4m3 has 4 significant bits)
__device__ __forceinline__ uint2 e4m3x4_bf16x4(uint32_t w, float f) {
  uint32_t a, b;
  asm("{\n\t.reg .b16 lo, hi;\n\tmov.b32 {lo, hi}, %2;\n\t"
      "cvt.rn.f16x2.e4m3x2 %0, lo;\n\tcvt.rn.f16x2.e4m3x2 %1, hi;\n\t}\n"
      : "=r"(a), "=r"(b)
      : "r"(w));
  const float2 x = __half22float2(*reinterpret_cast<__half2*>(&a)), y = __half22float2(*reinterpret_cast<__half2*>(&b));
  return make_uint2(pack_bf16(x.x * f, x.y * f), pack_bf16(y.x * f, y.y * f));
}

// 16 bytes to shared memory, zeros where not live
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool live) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(live ? 16 : 0) : "memory");
}

// First row of (page, head) in units of tokens; 64-bit, a pool may hold more than 2^31 elements.
__device__ __forceinline__ int64_t paged_row(const PagedPool& p, int pg, int head, int slot) {
  return ((((int64_t)pg * p.Hk + head) << p.page_shift) + slot);
}

// Page of token t of sequence b, or -1 (status word: kErrPage) when the table does not lead to a page of the pool.
__device__ __forceinline__ int paged_page(const PagedPool& p, int b, int t, int* err) {
  const int i = t >> p.page_shift;
  if (i >= 0 && i < p.width) {
    const int pg = __ldg(p.table + (int64_t)b * p.ld_table + i);
    if (pg >= 0 && pg < p.pages) return pg;
  }
  raise_error(err, kErrPage);
  return -1;
}

// Sequence of packed row r: the b with cu[b] <= r < cu[b + 1], or -1 past the last sequence.
__device__ __forceinline__ int row_sequence(const int* cu, int B, int r) {
  int lo = 0, hi = B;  // first b in [0, B] with cu[b + 1] > r
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (__ldg(cu + mid + 1) > r)
      hi = mid;
    else
      lo = mid + 1;
  }
  return lo < B && __ldg(cu + lo) <= r ? lo : -1;
}

// Attention of packed new rows over the pool (csrc/paged_rows.cu, csrc/paged_tiles.cu).
struct PagedAttnArgs {
  PagedPool p;
  const __nv_bfloat16* q;  // [T, H * D], row stride ldq
  int64_t ldq;
  __nv_bfloat16* o;  // [T, H * D]
  float* lse;        // [T, H]
  const int* total;
  const int* cu;
  int B, T, H, causal;
  int max_new, max_total;  // what the launch is sized for: no more than q's rows, no more than the table can hold
  int bound_new, bound_total;  // the caller's bounds
  float scale_log2;  // softmax scale * log2(e)
  int* err;
  // work split over the keys: split i of a sequence takes keys [i split_len, (i + 1) split_len)
  int splits, split_len, row_tiles;
  float* part;  // splits > 1: [splits][T * H][D] unnormalised outputs, then [splits][T * H][2] (maximum, sum)
};

constexpr int kSMs = 148;
constexpr int kMaxTokens = INT32_MAX - 8192;  // of a sequence: positions a tile past the end stay inside an int

// Sets the status word where sequence b is beyond the caller's bounds, or beyond what its row of the table holds; what
// follows works on rows and tokens cut down to the launch's. Once a sequence and launch.
__device__ __forceinline__ void paged_check(const PagedAttnArgs& a, int b) {
  const int n = min(__ldg(a.cu + b + 1), a.T) - max(0, __ldg(a.cu + b)), total = __ldg(a.total + b);
  if (n > a.bound_new || total > a.bound_total)
    raise_error(a.err, kErrBound);
  else if (n > 0 && total > a.max_total)
    raise_error(a.err, kErrPage);
}

// Allows a kernel `bytes` of dynamic shared memory, once a device: the attribute belongs to the function on the current
// device. `done` is the kernel's own.
struct SmemAllowed {
  std::once_flag device[64];
};
template <typename K>
inline void allow_smem(K* kernel, int bytes, SmemAllowed& done) {
  int dev = 0;
  C10_CUDA_CHECK(cudaGetDevice(&dev));
  auto set = [&] { C10_CUDA_CHECK(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes)); };
  if (dev < 64)
    std::call_once(done.device[dev], set);
  else
    set();
}

void paged_rows_launch(PagedAttnArgs a, cudaStream_t st);
void paged_tiles_launch(PagedAttnArgs a, cudaStream_t st);
void paged_merge_launch(const PagedAttnArgs& a, cudaStream_t st);

__device__ __forceinline__ int paged_used_splits(const PagedAttnArgs& a, int total) {
  total = max(0, min(total, a.max_total));
  return max(1, (total + a.split_len - 1) / a.split_len);
}

// A row, or a part of it, that saw no key has m = -inf and l = 0. A NaN score moves no maximum (fmaxf drops it) but
// makes the sum NaN, so m alone does not tell: the sum decides, here and in every merge.
__device__ __forceinline__ bool paged_saw_nothing(float m, float l) { return m == -INFINITY && l == 0.f; }

// log-sum-exp (natural) of a row from its maximum (log2 units) and its sum relative to it; NaN where the sum is
__device__ __forceinline__ float paged_lse(float m, float l) {
  return l == 0.f ? -INFINITY : (m + log2f(l)) * 0.69314718055994531f;
}
// what the unnormalised output is multiplied by
__device__ __forceinline__ float paged_inv(float l) { return l == 0.f ? 0.f : 1.f / l; }

}  // namespace ng
