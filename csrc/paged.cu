// Paged key/value cache (layout: csrc/paged.h): write with or without quantisation to e4m3, read back, and attention
// of a chunk of new tokens over it, for sm_100a.
//
// Packed rows: row r of sequence b (cu[b] <= r < cu[b + 1]) is token pos[b] + r - cu[b]. Rows past cu[B] are not
// touched by a write and read back as zeros. A table entry that leads outside the pool raises kErrPage; its token is
// skipped (write) or zero (read).
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/extension.h>

#include <cmath>

#include "common.cuh"
#include "msg.h"
#include "paged.h"
#include "status.h"

namespace ng {

using bf16 = __nv_bfloat16;

namespace {

// e = ceil(log2(amax / 448)) inside the cache's range, 0 for an all-zero row
__device__ __forceinline__ int cache_scale_exp(float amax) {
  return max(kScaleLo, min(kScaleHi, mx_scale_exp(amax)));
}

struct CopyArgs {
  PagedPool p;
  bf16* k;  // packed rows [T, Hk * D]
  bf16* v;
  int64_t ldk, ldv;
  const int* pos;
  const int* cu;
  int B, T, rows;  // rows of a CTA
  int* err;
};

__device__ __forceinline__ float amax8(const uint4& u) {
  float m = 0.f;
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) m = fmaxf(m, fmaxf(fabsf(bf16_bits_lo(w[i])), fabsf(bf16_bits_hi(w[i]))));
  return m;
}

constexpr int kCopyRows = 16;  // packed rows of a CTA, at most

// Where the CTA's rows sit in the pool: at[i] = (page, slot) of row r0 + i, page -1 for none.
__device__ __forceinline__ void find_rows(const CopyArgs& a, int64_t r0, int2 (&at)[kCopyRows]) {
  if (threadIdx.x < a.rows) {
    const int64_t r = r0 + threadIdx.x;
    int b = -1, t = 0, pg = -1;
    if (r < a.T) b = row_sequence(a.cu, a.B, (int)r);
    if (b >= 0) {
      t = __ldg(a.pos + b) + (int)r - __ldg(a.cu + b);
      pg = paged_page(a.p, b, t, a.err);
    }
    at[threadIdx.x] = make_int2(pg, t & ((1 << a.p.page_shift) - 1));
  }
  __syncthreads();
}

// A group of D / 8 lanes per (row, head), 8 elements of K and of V a lane; two units of a group in flight. Bound by
// bytes: the rows' pages are looked up once a CTA, while the first data loads are already on their way. 67,500 tokens
// of 8 heads of 128 to e4m3: 89 us, 4.7 TB/s (a lookup per row and head, one unit a group: 104 us; four units in
// flight: 90).
template <int D, bool Q8>
__global__ void __launch_bounds__(256) cache_write_kernel(const CopyArgs a) {
  constexpr int L = D / 8, GR = 256 / L;  // groups of the CTA
  __shared__ int2 at[kCopyRows];
  const int64_t r0 = (int64_t)blockIdx.x * a.rows;
  const int l = threadIdx.x % L, units = a.rows * a.p.Hk;
  const int rounds = (units + 2 * GR - 1) / (2 * GR);
  for (int k = 0; k < rounds; ++k) {
    uint4 kv[2][2];
    int i[2], h[2];
    bool live[2];
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      const int u = (k * 2 + x) * GR + threadIdx.x / L;
      i[x] = u / a.p.Hk;
      h[x] = u - i[x] * a.p.Hk;
      live[x] = u < units && r0 + i[x] < a.T;
      if (live[x]) {
        kv[x][0] = __ldcs(reinterpret_cast<const uint4*>(a.k + (r0 + i[x]) * a.ldk + h[x] * D + l * 8));
        kv[x][1] = __ldcs(reinterpret_cast<const uint4*>(a.v + (r0 + i[x]) * a.ldv + h[x] * D + l * 8));
      } else {
        kv[x][0] = kv[x][1] = make_uint4(0, 0, 0, 0);
      }
    }
    if (k == 0) find_rows(a, r0, at);
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      const int2 w = live[x] ? at[i[x]] : make_int2(-1, 0);
      const int64_t row = w.x >= 0 ? paged_row(a.p, w.x, h[x], w.y) : 0;
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        void* pool = c ? a.p.v : a.p.k;
        const uint4 u = kv[x][c];
        if (!Q8) {
          if (w.x >= 0) *reinterpret_cast<uint4*>(static_cast<bf16*>(pool) + row * D + l * 8) = u;
          continue;
        }
        float m = amax8(u);
#pragma unroll
        for (int o = 1; o < L; o <<= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
        if (w.x < 0) continue;
        const int e = cache_scale_exp(m);
        const float inv = ldexpf(1.f, -e);
        *reinterpret_cast<uint2*>(static_cast<uint8_t*>(pool) + row * D + l * 8) =
            make_uint2(e4m3x4(bf16_bits_lo(u.x) * inv, bf16_bits_hi(u.x) * inv, bf16_bits_lo(u.y) * inv,
                              bf16_bits_hi(u.y) * inv),
                       e4m3x4(bf16_bits_lo(u.z) * inv, bf16_bits_hi(u.z) * inv, bf16_bits_lo(u.w) * inv,
                              bf16_bits_hi(u.w) * inv));
        if (l == 0) (c ? a.p.vsf : a.p.ksf)[row] = (uint8_t)(e + 127);
      }
    }
  }
}

// The inverse: the loads of four units a group are issued before the first is converted and stored. 70,000 tokens of
// 8 heads of 128 out of e4m3 pages: 84 us, 5.2 TB/s (one unit at a time, a lookup for each: 110 us).
template <int D, bool Q8>
__global__ void __launch_bounds__(256) cache_read_kernel(const CopyArgs a) {
  constexpr int L = D / 8, GR = 256 / L;
  __shared__ int2 at[kCopyRows];
  const int64_t r0 = (int64_t)blockIdx.x * a.rows;
  const int l = threadIdx.x % L, units = a.rows * a.p.Hk;
  find_rows(a, r0, at);
  const int rounds = (units + 4 * GR - 1) / (4 * GR);
  for (int k = 0; k < rounds; ++k) {
    uint4 kv[4][2];
    uint8_t sf[4][2];
    int i[4], h[4];
    bool live[4];
#pragma unroll
    for (int x = 0; x < 4; ++x) {  // all loads of four units first
      const int u = (k * 4 + x) * GR + threadIdx.x / L;
      i[x] = u / a.p.Hk;
      h[x] = u - i[x] * a.p.Hk;
      live[x] = u < units && r0 + i[x] < a.T;
      const int2 w = live[x] ? at[i[x]] : make_int2(-1, 0);
      const int64_t row = w.x >= 0 ? paged_row(a.p, w.x, h[x], w.y) : 0;
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const void* pool = c ? a.p.v : a.p.k;
        kv[x][c] = make_uint4(0, 0, 0, 0);
        sf[x][c] = 127;
        if (w.x < 0) continue;
        if (Q8) {
          const uint2 u2 = __ldcs(reinterpret_cast<const uint2*>(static_cast<const uint8_t*>(pool) + row * D + l * 8));
          kv[x][c].x = u2.x, kv[x][c].y = u2.y;
          sf[x][c] = (c ? a.p.vsf : a.p.ksf)[row];
        } else {
          kv[x][c] = __ldcs(reinterpret_cast<const uint4*>(static_cast<const bf16*>(pool) + row * D + l * 8));
        }
      }
    }
#pragma unroll
    for (int x = 0; x < 4; ++x) {
      if (!live[x]) continue;
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        uint4 u = kv[x][c];
        if (Q8) {
          const float s = ldexpf(1.f, (int)sf[x][c] - 127);
          const uint2 lo = e4m3x4_bf16x4(u.x, s), hi = e4m3x4_bf16x4(u.y, s);
          u = make_uint4(lo.x, lo.y, hi.x, hi.y);
        }
        __stcs(reinterpret_cast<uint4*>((c ? a.v : a.k) + (r0 + i[x]) * (c ? a.ldv : a.ldk) + h[x] * D + l * 8), u);
      }
    }
  }
}

// Joins the splits of a (row, query head) of the row kernel, a warp each: o = sum_i 2^(m_i - M) o_i / sum_i 2^(m_i -
// M) l_i, in the order of the splits.
template <int D>
__global__ void __launch_bounds__(256) paged_merge_kernel(const PagedAttnArgs a) {
  constexpr int E = D / 32;
  const int64_t units = (int64_t)a.T * a.H, at = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  if (at >= units) return;
  const int b = row_sequence(a.cu, a.B, (int)(at / a.H));
  if (b < 0) return;
  const int used = paged_used_splits(a, __ldg(a.total + b));
  if (used == 1) return;  // written by its only split
  const float2* ml = reinterpret_cast<const float2*>(a.part + a.splits * units * D);
  float m = -INFINITY;
  for (int i = lane; i < used; i += 32) m = fmaxf(m, ml[i * units + at].x);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  float l = 0.f, acc[E];
#pragma unroll
  for (int e = 0; e < E; ++e) acc[e] = 0.f;
#pragma unroll 4
  for (int i = 0; i < used; ++i) {
    const float2 x = ml[i * units + at];
    if (paged_saw_nothing(x.x, x.y)) continue;
    const float w = ex2_ftz(x.x - m);
    l += x.y * w;
    const float* src = a.part + (i * units + at) * D + lane * E;
#pragma unroll
    for (int e = 0; e < E; ++e) acc[e] += src[e] * w;
  }
  const float inv = paged_inv(l);
#pragma unroll
  for (int e = 0; e < E; e += 2)
    *reinterpret_cast<uint32_t*>(a.o + at * D + lane * E + e) = pack_bf16(acc[e] * inv, acc[e + 1] * inv);
  if (lane == 0) a.lse[at] = paged_lse(m, l);
}

// ------------------------------------------------------------------------------------------------------- torch glue
// Rows of a key head (new tokens times its query heads) up to which the row kernel runs; above, the tile kernel. It
// reads the cache once per 16 rows where the tile kernel reads it once, but pays no 128-row tiles and splits the keys
// further. Both measured, us, 8 key heads of 128 (row / tile kernel):
//   bf16   16 rows: 1 x 8192 keys 26 / 50, 64 x 8192 346 / 402;   32 rows: 1 x 8192 28 / 52, 8 x 512 16 / 21,
//          8 x 8192 91 / 82, 64 x 8192 478 / 404: 32 rows pay while the key heads of all sequences leave SMs idle
//   e4m3   32 rows: 1 x 8192 28 / 65, 8 x 8192 85 / 159, 64 x 8192 456 / 1009; 64 rows: 38 / 67, 128 / 159, 884 / 1015
//          (the tile kernel converts the tiles); 96 rows: tile kernel 69, 165, 1025, where another 200 for each 16 rows
//          of the row kernel would pass it at 64 x 8192
// Heads of 64: bf16, 16 rows: 1 x 8192 19 / 50, 64 x 8192 192 / 386; 32 rows: 8 x 8192 56 / 73; e4m3, 64 rows: 28 / 58,
// 85 / 116, 566 / 693.
inline int64_t rows_max(bool q8, int64_t heads) { return q8 ? 64 : heads < kSMs / 2 ? 32 : 16; }

bool opt(const c10::optional<at::Tensor>& t) { return t.has_value() && t->defined(); }

void check_i32(const at::Tensor& t, const char* name, int64_t n, const at::Device& dev) {
  TORCH_CHECK(t.device() == dev && t.scalar_type() == at::kInt && t.dim() == 1 && t.size(0) == n && t.is_contiguous(),
              msg("paged: ", name, " must be a contiguous int32 [", n, "] on the cache's device"));
}

PagedPool pool_of(const at::Tensor& k, const at::Tensor& v, const c10::optional<at::Tensor>& ksf,
                  const c10::optional<at::Tensor>& vsf, const at::Tensor& table) {
  TORCH_CHECK(k.is_cuda() && k.dim() == 4 && k.is_contiguous() && v.is_contiguous() && v.sizes() == k.sizes() &&
                  v.device() == k.device() && v.scalar_type() == k.scalar_type(),
              "paged: k and v must be contiguous [pages, heads, page, dim] pools of one type on one device");
  const bool q8 = k.scalar_type() == at::kByte;
  TORCH_CHECK(q8 || k.scalar_type() == at::kBFloat16, "paged: the pool must be bf16 or uint8 (e4m3 bytes)");
  TORCH_CHECK(q8 == opt(ksf) && q8 == opt(vsf), "paged: e4m3 pools need both scale pools, bf16 pools none");
  if (q8)
    for (const at::Tensor& s : {*ksf, *vsf}) {
      TORCH_CHECK(s.device() == k.device() && s.scalar_type() == at::kByte && s.is_contiguous() && s.dim() == 3 &&
                      s.size(0) == k.size(0) && s.size(1) == k.size(1) && s.size(2) == k.size(2),
                  "paged: scales must be a contiguous uint8 [pages, heads, page]");
      TORCH_CHECK(reinterpret_cast<uintptr_t>(s.data_ptr()) % 4 == 0,  // four tokens a copy in csrc/paged_rows.cu
                  "paged: scale pools must be 4-byte aligned");
    }
  const int64_t page = k.size(2), D = k.size(3);
  TORCH_CHECK(D == 64 || D == 128, msg("paged: head dim must be 64 or 128, got ", D));
  TORCH_CHECK(page >= 8 && page <= 1024 && (page & (page - 1)) == 0,
              msg("paged: the page size must be a power of two from 8 to 1024, got ", page));
  TORCH_CHECK(k.size(0) <= INT32_MAX && k.size(1) >= 1 && k.size(1) <= 65535, "paged: too many pages or heads");
  TORCH_CHECK(reinterpret_cast<uintptr_t>(k.data_ptr()) % 16 == 0 &&
                  reinterpret_cast<uintptr_t>(v.data_ptr()) % 16 == 0,
              "paged: pools must be 16-byte aligned");
  TORCH_CHECK(table.device() == k.device() && table.scalar_type() == at::kInt && table.dim() == 2 &&
                  (table.size(1) <= 1 || table.stride(1) == 1),
              "paged: table must be int32 [sequences, pages a sequence] with last stride 1 on the cache's device");
  PagedPool p{};
  p.k = k.data_ptr();
  p.v = v.data_ptr();
  p.ksf = q8 ? ksf->data_ptr<uint8_t>() : nullptr;
  p.vsf = q8 ? vsf->data_ptr<uint8_t>() : nullptr;
  p.table = table.data_ptr<int>();
  p.ld_table = table.stride(0);
  p.width = (int)table.size(1);
  p.pages = (int)k.size(0);
  p.Hk = (int)k.size(1);
  p.D = (int)D;
  while ((1 << p.page_shift) < page) ++p.page_shift;
  return p;
}

// packed rows [T, cols] bf16, last stride 1, rows 16-byte aligned
void check_packed(const at::Tensor& t, const char* name, int64_t T, int64_t cols, const at::Device& dev) {
  TORCH_CHECK(t.device() == dev && t.scalar_type() == at::kBFloat16 && t.dim() == 2 && t.size(0) == T &&
                  t.size(1) == cols && (T == 0 || t.stride(1) == 1),
              msg("paged: ", name, " must be bf16 [", T, ", ", cols,
                  "] with last stride 1 on the cache's device, got sizes ", msg_sizes(t.sizes())));
  TORCH_CHECK(T == 0 || (reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0 && (T == 1 || t.stride(0) % 8 == 0)),
              msg("paged: the rows of ", name, " must be 16-byte aligned"));
  TORCH_CHECK(T <= INT32_MAX, "paged: too many rows");
}

template <bool WRITE>
void copy_launch(CopyArgs a) {
  const auto st = at::cuda::getCurrentCUDAStream();
  // rows of a CTA: kCopyRows, fewer where that would leave SMs without work
  a.rows = (int)std::max<int64_t>(1, std::min<int64_t>(kCopyRows, (int64_t)a.T / (4 * kSMs)));
  const int64_t grid = ((int64_t)a.T + a.rows - 1) / a.rows;
  TORCH_CHECK(grid <= INT32_MAX, "paged: too many rows");
  const bool q8 = a.p.ksf != nullptr;
#define NG_COPY(D, Q)                                        \
  if (WRITE)                                                 \
    cache_write_kernel<D, Q><<<(int)grid, 256, 0, st>>>(a);  \
  else                                                       \
    cache_read_kernel<D, Q><<<(int)grid, 256, 0, st>>>(a)
  if (a.p.D == 128) {
    if (q8) {
      NG_COPY(128, true);
    } else {
      NG_COPY(128, false);
    }
  } else {
    if (q8) {
      NG_COPY(64, true);
    } else {
      NG_COPY(64, false);
    }
  }
#undef NG_COPY
  NG_LAUNCH_CHECK();
}

}  // namespace

void paged_merge_launch(const PagedAttnArgs& a, cudaStream_t st) {
  const int grid = (int)(((int64_t)a.T * a.H + 7) / 8);
  if (a.p.D == 128)
    paged_merge_kernel<128><<<grid, 256, 0, st>>>(a);
  else
    paged_merge_kernel<64><<<grid, 256, 0, st>>>(a);
  NG_LAUNCH_CHECK();
}

void cache_write(const at::Tensor& pk, const at::Tensor& pv, const c10::optional<at::Tensor>& ksf,
                 const c10::optional<at::Tensor>& vsf, const at::Tensor& k, const at::Tensor& v,
                 const at::Tensor& table, const at::Tensor& pos, const at::Tensor& cu) {
  const at::cuda::OptionalCUDAGuard guard(pk.device());
  CopyArgs a{};
  a.p = pool_of(pk, pv, ksf, vsf, table);
  const int64_t B = table.size(0), T = k.size(0), cols = (int64_t)a.p.Hk * a.p.D;
  check_packed(k, "k", T, cols, pk.device());
  check_packed(v, "v", T, cols, pk.device());
  check_i32(pos, "pos", B, pk.device());
  check_i32(cu, "cu", B + 1, pk.device());
  if (T == 0 || B == 0) return;
  a.k = reinterpret_cast<bf16*>(k.data_ptr());
  a.v = reinterpret_cast<bf16*>(v.data_ptr());
  a.ldk = k.stride(0);
  a.ldv = v.stride(0);
  a.pos = pos.data_ptr<int>();
  a.cu = cu.data_ptr<int>();
  a.B = (int)B;
  a.T = (int)T;
  a.err = status_word();
  copy_launch<true>(a);
}

std::vector<at::Tensor> cache_read(const at::Tensor& pk, const at::Tensor& pv, const c10::optional<at::Tensor>& ksf,
                                   const c10::optional<at::Tensor>& vsf, const at::Tensor& table,
                                   const at::Tensor& pos, const at::Tensor& cu, int64_t rows) {
  const at::cuda::OptionalCUDAGuard guard(pk.device());
  CopyArgs a{};
  a.p = pool_of(pk, pv, ksf, vsf, table);
  const int64_t B = table.size(0), cols = (int64_t)a.p.Hk * a.p.D;
  check_i32(pos, "pos", B, pk.device());
  check_i32(cu, "cu", B + 1, pk.device());
  TORCH_CHECK(rows >= 0 && rows <= INT32_MAX, "paged: rows out of range");
  const auto opts = pk.options().dtype(at::kBFloat16);
  at::Tensor k = at::empty({rows, cols}, opts), v = at::empty({rows, cols}, opts);
  if (rows == 0) return {k, v};
  a.k = reinterpret_cast<bf16*>(k.data_ptr());
  a.v = reinterpret_cast<bf16*>(v.data_ptr());
  a.ldk = a.ldv = cols;
  a.pos = pos.data_ptr<int>();
  a.cu = cu.data_ptr<int>();
  a.B = (int)B;
  a.T = (int)rows;
  a.err = status_word();
  copy_launch<false>(a);
  return {k, v};
}

// (o [T, H * D] bf16, lse [T, H] fp32)
std::vector<at::Tensor> paged_attn(const at::Tensor& q, const at::Tensor& pk, const at::Tensor& pv,
                                   const c10::optional<at::Tensor>& ksf, const c10::optional<at::Tensor>& vsf,
                                   const at::Tensor& table, const at::Tensor& total, const at::Tensor& cu,
                                   int64_t max_new, int64_t max_total, double scale, bool causal) {
  const at::cuda::OptionalCUDAGuard guard(pk.device());
  PagedAttnArgs a{};
  a.p = pool_of(pk, pv, ksf, vsf, table);
  const int64_t B = table.size(0), T = q.size(0), D = a.p.D;
  TORCH_CHECK(q.dim() == 2 && q.size(1) > 0 && q.size(1) % (a.p.Hk * D) == 0,
              msg("paged: q must be [rows, heads * ", D, "] with a multiple of ", a.p.Hk, " heads, got ",
                  msg_sizes(q.sizes())));
  check_packed(q, "q", T, q.size(1), pk.device());
  check_i32(total, "total", B, pk.device());
  check_i32(cu, "cu", B + 1, pk.device());
  // as the kernels hold it: a scale that rounds to 0 would make NaN of a masked score, -inf
  const float scale_log2 = (float)(scale * 1.4426950408889634);
  TORCH_CHECK(scale_log2 > 0 && std::isfinite(scale_log2), "paged: scale must be positive, in fp32's range");
  TORCH_CHECK(max_new >= 0 && max_total >= 0 && max_new <= INT32_MAX && max_total <= INT32_MAX,
              "paged: max_new / max_total out of range");
  const int64_t H = q.size(1) / D;
  TORCH_CHECK(T * H <= INT32_MAX - 256, "paged: too many rows");
  at::Tensor o = at::empty({T, H * D}, q.options()), lse = at::empty({T, H}, q.options().dtype(at::kFloat));
  if (T == 0) return {o, lse};
  if (B == 0 || max_new == 0) {  // no row belongs to a sequence, or none may: every row is padding
    o.zero_();
    lse.fill_(-INFINITY);
    if (B == 0) return {o, lse};
  }
  a.q = reinterpret_cast<const bf16*>(q.data_ptr());
  a.ldq = q.stride(0);
  a.o = reinterpret_cast<bf16*>(o.data_ptr());
  a.lse = lse.data_ptr<float>();
  a.total = total.data_ptr<int>();
  a.cu = cu.data_ptr<int>();
  a.B = (int)B;
  a.T = (int)T;
  a.H = (int)H;
  a.bound_new = (int)max_new;
  // Row tiles, their first rows in 32 bits, are counted for rows that exist; one at least, which sets the status word
  // where a sequence has rows in spite of max_new = 0.
  max_new = std::max<int64_t>(1, std::min(max_new, T));
  a.max_new = (int)max_new;
  a.bound_total = (int)max_total;
  // a bound is often loose (a captured graph's, "any length"): splits and their workspace go by what the table holds
  const int64_t held = std::min<int64_t>(max_total, (int64_t)a.p.width << a.p.page_shift);
  TORCH_CHECK(held <= kMaxTokens, "paged: max_total and the table allow a sequence of too many tokens");
  a.max_total = (int)held;
  a.causal = causal;
  a.scale_log2 = scale_log2;
  a.err = status_word();
  const auto st = at::cuda::getCurrentCUDAStream();
  if (max_new * (H / a.p.Hk) <= rows_max(a.p.ksf != nullptr, B * a.p.Hk))
    paged_rows_launch(a, st);
  else
    paged_tiles_launch(a, st);
  return {o, lse};
}

}  // namespace ng
