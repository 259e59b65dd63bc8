// RMSNorm with the residual's addition in front of it, for sm_100a: forward with a bf16 or an MXFP8 output, and the
// gradient.
//
//   s = res + x               rounded once to the residual stream's type (bf16 or fp32)
//   rstd = 1 / sqrt(mean(s^2) + eps),  h = w s rstd      from the unrounded fp32 sum
//   MXFP8: per 32 columns e = ceil(log2(amax / 448)), q = e4m3(h 2^-e); h is rounded once, not through bf16
// Backward with xn = s rstd, dxn = dh w:
//   dx = rstd (dxn - xn mean(dxn xn)) + ds  (the gradient of x and of res),   dw += sum_rows dh xn
#include <ATen/cuda/CUDAContext.h>
#include <c10/cuda/CUDAGuard.h>
#include <torch/extension.h>

#include "common.cuh"
#include "msg.h"
#include "reduce.h"
#include "status.h"

namespace ng {

using bf16 = __nv_bfloat16;

namespace {

constexpr int kMaxWidth = 16384;

__device__ __forceinline__ void load8(const bf16* p, float (&f)[8]) {
  const uint4 u = *reinterpret_cast<const uint4*>(p);
  f[0] = bf16_bits_lo(u.x), f[1] = bf16_bits_hi(u.x), f[2] = bf16_bits_lo(u.y), f[3] = bf16_bits_hi(u.y);
  f[4] = bf16_bits_lo(u.z), f[5] = bf16_bits_hi(u.z), f[6] = bf16_bits_lo(u.w), f[7] = bf16_bits_hi(u.w);
}
__device__ __forceinline__ void load8(const float* p, float (&f)[8]) {
  const float4 a = reinterpret_cast<const float4*>(p)[0], b = reinterpret_cast<const float4*>(p)[1];
  f[0] = a.x, f[1] = a.y, f[2] = a.z, f[3] = a.w, f[4] = b.x, f[5] = b.y, f[6] = b.z, f[7] = b.w;
}
__device__ __forceinline__ void store8(bf16* p, const float (&f)[8]) {
  *reinterpret_cast<uint4*>(p) =
      make_uint4(pack_bf16(f[0], f[1]), pack_bf16(f[2], f[3]), pack_bf16(f[4], f[5]), pack_bf16(f[6], f[7]));
}
__device__ __forceinline__ void store8(float* p, const float (&f)[8]) {
  reinterpret_cast<float4*>(p)[0] = make_float4(f[0], f[1], f[2], f[3]);
  reinterpret_cast<float4*>(p)[1] = make_float4(f[4], f[5], f[6], f[7]);
}

// 8 columns as they are stored
template <typename R>
struct Raw;
template <>
struct Raw<bf16> {
  uint4 u;
  __device__ __forceinline__ void load(const bf16* p) { u = *reinterpret_cast<const uint4*>(p); }
  __device__ __forceinline__ void get(float (&f)[8]) const {
    f[0] = bf16_bits_lo(u.x), f[1] = bf16_bits_hi(u.x), f[2] = bf16_bits_lo(u.y), f[3] = bf16_bits_hi(u.y);
    f[4] = bf16_bits_lo(u.z), f[5] = bf16_bits_hi(u.z), f[6] = bf16_bits_lo(u.w), f[7] = bf16_bits_hi(u.w);
  }
};
template <>
struct Raw<float> {
  float f_[8];
  __device__ __forceinline__ void load(const float* p) { load8(p, f_); }
  __device__ __forceinline__ void get(float (&f)[8]) const {
#pragma unroll
    for (int j = 0; j < 8; ++j) f[j] = f_[j];
  }
};

// Sum of v over the block (blockDim.x a multiple of 32, at most 1024), in every thread.
__device__ __forceinline__ float block_sum(float v, float* red) {
  v = warp_sum(v);
  const int nw = blockDim.x >> 5;
  if (nw == 1) return v;
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  float t = 0.f;
  for (int i = 0; i < nw; ++i) t += red[i];
  return t;
}

struct AddRmsArgs {
  const bf16* x;
  const void* res;
  const float* w;
  bf16* h;
  uint8_t* q;
  uint8_t* sf;
  void* s;
  float* rstd;
  int64_t ldx, ldr;
  int M, C;
  float eps;
};

// One CTA per row, VPT vectors of 8 columns a thread, held in registers between the sum and the output: one read of x
// and of the stream, one write of each output. Bound by bytes where rows are many (20480 x 2048 to MXFP8: 56 us a
// call, 5.3 TB/s; 4099 x 5120 with an fp32 stream: 43 us, 5.9 TB/s), by the launch and the call where they are few
// (16 x 2048: 10 us a call). One vector a thread up to 4096 columns: the most loads in flight a row and the fewest
// registers.
template <typename R, bool MXO, int VPT>
__global__ void __launch_bounds__(512) add_rms_fwd_kernel(const AddRmsArgs a) {
  __shared__ float red[32];
  const int64_t row = blockIdx.x;
  const int nv = a.C >> 3;
  if (MXO && row >= a.M) {  // padding rows of the scale blocks hold scale 1
    for (int v = threadIdx.x; v < nv; v += blockDim.x)
      if ((v & 3) == 0) a.sf[mx_sf_offset((int)row, v >> 2, a.C / 128)] = 127;
    return;
  }
  float f[VPT][8];
  float ss = 0.f;
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    const int v = threadIdx.x + i * blockDim.x;
    if (v < nv) {
      float xf[8];
      load8(a.x + row * a.ldx + v * 8, xf);
      load8(static_cast<const R*>(a.res) + row * a.ldr + v * 8, f[i]);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        f[i][j] += xf[j];
        ss += f[i][j] * f[i][j];
      }
      store8(static_cast<R*>(a.s) + row * a.C + v * 8, f[i]);
    }
  }
  const float r = rsqrtf(block_sum(ss, red) / (float)a.C + a.eps);
  if (threadIdx.x == 0) a.rstd[row] = r;
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    const int v = threadIdx.x + i * blockDim.x;
    const bool live = v < nv;
    float am = 0.f;
    if (live) {
      float wf[8];
      load8(a.w + v * 8, wf);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        f[i][j] = f[i][j] * r * wf[j];
        am = fmaxf(am, fabsf(f[i][j]));
      }
      if (!MXO) store8(a.h + row * a.C + v * 8, f[i]);
    }
    if (MXO) {  // a 32-column block is the vectors of four adjacent lanes
      am = fmaxf(am, __shfl_xor_sync(0xffffffffu, am, 1));
      am = fmaxf(am, __shfl_xor_sync(0xffffffffu, am, 2));
      if (live) {
        const int e = mx_scale_exp(am);
        const float inv = ldexpf(1.f, -e);
        const float(&g)[8] = f[i];
        *reinterpret_cast<uint2*>(a.q + row * a.C + v * 8) =
            make_uint2(e4m3x4(g[0] * inv, g[1] * inv, g[2] * inv, g[3] * inv),
                       e4m3x4(g[4] * inv, g[5] * inv, g[6] * inv, g[7] * inv));
        if ((v & 3) == 0) a.sf[mx_sf_offset((int)row, v >> 2, a.C / 128)] = (uint8_t)(e + 127);
      }
    }
  }
}

struct AddRmsBwdArgs {
  const bf16* dh;
  const void* ds;  // null: no gradient of the stream
  const void* s;
  const float* rstd;
  const float* w;
  void* dx;
  float* part;  // [CTAs][C], null: no weight gradient
  int64_t lddh, ldds, lds;
  int M, C, rows_per_cta;
};

// A CTA walks its rows; a thread owns VPT vectors of 8 columns for all of them, so the weight gradient's partial sums
// stay in registers and every byte is read once. Bound by bytes and the latency of a row's reduction: the stream's
// gradient is loaded before the reduction, which takes one barrier (its partial sums alternate between two buffers),
// and eight CTAs a SM hide it. 32768 x 1024 in bf16: 62 us a call, about 10 of them the column sums of the partials
// (269 MB, 41 us at the copy's rate). Eight CTAs of 128 threads fit a SM at 64 registers: left to itself the compiler
// takes 73, six CTAs fit, the grid becomes two waves and the call 85 us. Two or four rows a step, with more
// registers, took 72 us for the kernel alone.
template <typename R, int VPT>
__global__ void __launch_bounds__(512, VPT == 1 && sizeof(R) == 2 ? 2 : 0) add_rms_bwd_kernel(const AddRmsBwdArgs a) {
  __shared__ float red[2][16];
  const int nv = a.C >> 3, warp = threadIdx.x >> 5, nw = blockDim.x >> 5;
  const int64_t r0 = (int64_t)blockIdx.x * a.rows_per_cta, r1 = min((int64_t)a.M, r0 + a.rows_per_cta);
  float dw[VPT][8], wf[VPT][8];
#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    const int v = threadIdx.x + i * blockDim.x;
#pragma unroll
    for (int j = 0; j < 8; ++j) dw[i][j] = wf[i][j] = 0.f;
    if (v < nv) load8(a.w + v * 8, wf[i]);
  }
  int buf = 0;
  for (int64_t row = r0; row < r1; ++row, buf ^= 1) {
    float g[VPT][8], xn[VPT][8];
    Raw<R> ds[VPT];
    const float rs = a.rstd[row];
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int v = threadIdx.x + i * blockDim.x;
      if (v < nv) {
        load8(a.dh + row * a.lddh + v * 8, g[i]);
        load8(static_cast<const R*>(a.s) + row * a.lds + v * 8, xn[i]);
        if (a.ds != nullptr) ds[i].load(static_cast<const R*>(a.ds) + row * a.ldds + v * 8);
      } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) g[i][j] = xn[i][j] = 0.f;
      }
    }
    float acc = 0.f;
#pragma unroll
    for (int i = 0; i < VPT; ++i)
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        xn[i][j] *= rs;
        dw[i][j] += g[i][j] * xn[i][j];
        g[i][j] *= wf[i][j];
        acc += g[i][j] * xn[i][j];
      }
    acc = warp_sum(acc);
    if (nw > 1) {
      if ((threadIdx.x & 31) == 0) red[buf][warp] = acc;
      __syncthreads();
      acc = 0.f;
      for (int k = 0; k < nw; ++k) acc += red[buf][k];
    }
    const float cm = acc / (float)a.C;
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int v = threadIdx.x + i * blockDim.x;
      if (v < nv) {
        float o[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) o[j] = 0.f;
        if (a.ds != nullptr) ds[i].get(o);
#pragma unroll
        for (int j = 0; j < 8; ++j) o[j] += rs * (g[i][j] - xn[i][j] * cm);
        store8(static_cast<R*>(a.dx) + row * a.C + v * 8, o);
      }
    }
  }
  if (a.part != nullptr) {
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int v = threadIdx.x + i * blockDim.x;
      if (v < nv) store8(a.part + (int64_t)blockIdx.x * a.C + v * 8, dw[i]);
    }
  }
}

// A [M, C] operand: last stride 1, rows 16-byte aligned.
void check_mat(const at::Tensor& t, const char* name, int64_t M, int64_t C, const at::Device& dev) {
  TORCH_CHECK(t.device() == dev, msg("add_rms: ", name, " must be on the first operand's device"));
  TORCH_CHECK(t.dim() == 2 && t.size(0) == M && t.size(1) == C,
              msg("add_rms: ", name, " must be [", M, ", ", C, "], got ", msg_sizes(t.sizes())));
  TORCH_CHECK(t.stride(1) == 1 || M == 0, msg("add_rms: ", name, " needs last stride 1"));
  const int64_t es = t.element_size();
  TORCH_CHECK(M == 0 || (reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0 && (M == 1 || t.stride(0) * es % 16 == 0)),
              msg("add_rms: the rows of ", name, " must be 16-byte aligned"));
}

void check_common(const at::Tensor& x, const at::Tensor& w) {
  TORCH_CHECK(x.is_cuda() && x.dim() == 2, "add_rms: a CUDA matrix expected");
  const int64_t M = x.size(0), C = x.size(1);
  TORCH_CHECK(C > 0 && C % 8 == 0 && C <= kMaxWidth,
              msg("add_rms: the width must be a multiple of 8 up to ", kMaxWidth, ", got ", C));
  TORCH_CHECK(M <= INT32_MAX - 256, "add_rms: too many rows");
  TORCH_CHECK(w.device() == x.device() && w.scalar_type() == at::kFloat && w.dim() == 1 && w.size(0) == C &&
                  w.is_contiguous() && reinterpret_cast<uintptr_t>(w.data_ptr()) % 16 == 0,
              msg("add_rms: w must be a contiguous, 16-byte aligned fp32 [", C, "] on x's device"));
}

bool stream_fp32(const at::Tensor& t, const char* name) {
  TORCH_CHECK(t.scalar_type() == at::kBFloat16 || t.scalar_type() == at::kFloat,
              msg("add_rms: ", name, " must be bf16 or fp32"));
  return t.scalar_type() == at::kFloat;
}

}  // namespace

// (h, s, rstd), or with mx (q, sf, s, rstd).
std::vector<at::Tensor> add_rms_fwd(const at::Tensor& x, const at::Tensor& res, const at::Tensor& w, double eps,
                                    bool mx) {
  check_common(x, w);
  const int64_t M = x.size(0), C = x.size(1);
  TORCH_CHECK(x.scalar_type() == at::kBFloat16, "add_rms: x must be bf16");
  check_mat(x, "x", M, C, x.device());
  check_mat(res, "res", M, C, x.device());
  const bool f32 = stream_fp32(res, "res");
  TORCH_CHECK(!mx || C % 128 == 0,
              msg("add_rms: the MXFP8 output needs a width that is a multiple of 128, got ", C));
  const at::cuda::CUDAGuard guard(x.device());
  const auto o8 = x.options().dtype(at::kByte);
  const int64_t pad = (M + 255) / 256 * 256;
  at::Tensor h = mx ? at::empty({M, C}, o8) : at::empty({M, C}, x.options());
  at::Tensor sf = mx ? at::empty({pad / 128, C / 128, 512}, o8) : at::Tensor();
  at::Tensor s = at::empty({M, C}, res.options());
  at::Tensor rstd = at::empty({M}, w.options());
  if (M > 0) {
    AddRmsArgs a{};
    a.x = reinterpret_cast<const bf16*>(x.data_ptr());
    a.res = res.data_ptr();
    a.w = w.data_ptr<float>();
    if (mx) {
      a.q = h.data_ptr<uint8_t>();
      a.sf = sf.data_ptr<uint8_t>();
    } else {
      a.h = reinterpret_cast<bf16*>(h.data_ptr());
    }
    a.s = s.data_ptr();
    a.rstd = rstd.data_ptr<float>();
    a.ldx = x.stride(0);
    a.ldr = res.stride(0);
    a.M = (int)M;
    a.C = (int)C;
    a.eps = (float)eps;
    const int nv = (int)C / 8, vpt = nv > 1024 ? 4 : nv > 512 ? 2 : 1;
    const int threads = ((nv + vpt - 1) / vpt + 31) / 32 * 32;
    const int grid = (int)(mx ? pad : M);
    const auto st = at::cuda::getCurrentCUDAStream();
#define NG_ADD_RMS(R, MXO, V) add_rms_fwd_kernel<R, MXO, V><<<grid, threads, 0, st>>>(a)
#define NG_ADD_RMS_V(R, MXO) \
  if (vpt == 1)              \
    NG_ADD_RMS(R, MXO, 1);   \
  else if (vpt == 2)         \
    NG_ADD_RMS(R, MXO, 2);   \
  else                       \
    NG_ADD_RMS(R, MXO, 4)
    if (f32) {
      if (mx) {
        NG_ADD_RMS_V(float, true);
      } else {
        NG_ADD_RMS_V(float, false);
      }
    } else {
      if (mx) {
        NG_ADD_RMS_V(bf16, true);
      } else {
        NG_ADD_RMS_V(bf16, false);
      }
    }
#undef NG_ADD_RMS_V
#undef NG_ADD_RMS
    NG_LAUNCH_CHECK();
  }
  if (mx) return {h, sf, s, rstd};
  return {h, s, rstd};
}

// dx (the stream's type); dw [C] fp32 is added to when given.
at::Tensor add_rms_bwd(const at::Tensor& dh, const c10::optional<at::Tensor>& ds, const at::Tensor& s,
                       const at::Tensor& rstd, const at::Tensor& w, const c10::optional<at::Tensor>& dw) {
  check_common(dh, w);
  const int64_t M = dh.size(0), C = dh.size(1);
  TORCH_CHECK(dh.scalar_type() == at::kBFloat16, "add_rms: dh must be bf16");
  check_mat(dh, "dh", M, C, dh.device());
  check_mat(s, "s", M, C, dh.device());
  const bool f32 = stream_fp32(s, "s");
  const bool has_ds = ds.has_value() && ds->defined(), has_dw = dw.has_value() && dw->defined();
  if (has_ds) {
    check_mat(*ds, "ds", M, C, dh.device());
    TORCH_CHECK(ds->scalar_type() == s.scalar_type(), "add_rms: ds must have the type of s");
  }
  TORCH_CHECK(rstd.device() == dh.device() && rstd.scalar_type() == at::kFloat && rstd.dim() == 1 &&
                  rstd.size(0) == M && rstd.is_contiguous(),
              msg("add_rms: rstd must be a contiguous fp32 [", M, "]"));
  if (has_dw)
    TORCH_CHECK(dw->device() == dh.device() && dw->scalar_type() == at::kFloat && dw->dim() == 1 &&
                    dw->size(0) == C && dw->is_contiguous(),
                msg("add_rms: dw_acc must be a contiguous fp32 [", C, "]"));
  const at::cuda::CUDAGuard guard(dh.device());
  at::Tensor dx = at::empty({M, C}, s.options());
  if (M == 0) return dx;
  const int nv = (int)C / 8, vpt = nv > 1024 ? 4 : nv > 512 ? 2 : 1;
  const int threads = ((nv + vpt - 1) / vpt + 31) / 32 * 32;
  const int rows = (int)std::max<int64_t>(1, (M + 1183) / 1184);  // eight CTAs a SM
  const int grid = (int)((M + rows - 1) / rows);
  at::Tensor part = has_dw ? at::empty({grid, C}, w.options()) : at::Tensor();
  AddRmsBwdArgs a{};
  a.dh = reinterpret_cast<const bf16*>(dh.data_ptr());
  a.ds = has_ds ? ds->data_ptr() : nullptr;
  a.s = s.data_ptr();
  a.rstd = rstd.data_ptr<float>();
  a.w = w.data_ptr<float>();
  a.dx = dx.data_ptr();
  a.part = has_dw ? part.data_ptr<float>() : nullptr;
  a.lddh = dh.stride(0);
  a.ldds = has_ds ? ds->stride(0) : 0;
  a.lds = s.stride(0);
  a.M = (int)M;
  a.C = (int)C;
  a.rows_per_cta = rows;
  const auto st = at::cuda::getCurrentCUDAStream();
#define NG_ADD_RMS_BWD(R)                                           \
  if (vpt == 1)                                                     \
    add_rms_bwd_kernel<R, 1><<<grid, threads, 0, st>>>(a);       \
  else if (vpt == 2)                                                \
    add_rms_bwd_kernel<R, 2><<<grid, threads, 0, st>>>(a);       \
  else                                                              \
    add_rms_bwd_kernel<R, 4><<<grid, threads, 0, st>>>(a)
  if (f32) {
    NG_ADD_RMS_BWD(float);
  } else {
    NG_ADD_RMS_BWD(bf16);
  }
#undef NG_ADD_RMS_BWD
  NG_LAUNCH_CHECK();
  if (has_dw) colsum_launch(part.data_ptr<float>(), false, grid, (int)C, C, dw->data_ptr<float>(), true, st);
  return dx;
}

}  // namespace ng
