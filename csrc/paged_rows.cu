// Attention of a few new tokens (16 rows a key head and tile) over the paged cache, for sm_100a: one decoding
// step, or the few tokens of a draft.
//
// Every byte of the cache is read once and meets at most 16 query rows, so the kernel is bound by the cache's bytes:
// its products run on warp-level mma.sync m16n8k16 (16 rows are what that shape holds; a 128-row tcgen05 tile would be
// seven eighths padding and its shared-memory and TMEM round trips only add latency), and the design is about bytes in
// flight. A CTA of 4 warps takes (sequence, key head, 16-row tile, split of the keys). Each warp walks its own key
// tiles of KT keys through a private ring of ST cp.async stages (8 KiB a stage: 2 CTAs a SM keep up to 128 KiB in
// flight; no CTA barrier in the loop), with its own running maximum and sum in fp32. The four warps, then the splits,
// are merged by their maxima in a fixed order (csrc/paged.cu, paged_merge_kernel).
//
// e4m3 pools: an e4m3 value is exact in f16, so the products run in f16 on the stored bytes, unscaled. The row of Q
// is brought to [2^14, 2^15) by a power of two first (exact but for values 2^-29 below the row's largest). The key's
// scale multiplies the fp32 score; the value's, 2^e, enters the exponent: w = 2^(s + e - M), o = sum w v8, l = sum w
// 2^-e, with M the running maximum of s + e, less 15: weights reach 2^15. P is rounded to f16 (bf16 pools: bf16, the
// type of V) for its product; the row sum keeps the unrounded fp32 values. One token can lie far above the others in
// s + e and still add nothing to a column (a zero value, whose scale is 1, or a single loud channel), so weights of
// any size must keep their bits: where a tile has weights below 2^-16 (the least that f16 rounds as finely as bf16),
// what the rounding left of them is multiplied again, 2^40 up, into accumulators that are scaled along.
//
// One step of 64 sequences of up to 16384 tokens, 8 key heads of 128, e4m3 (1.34 GB): 300 us a call, 9 of them the
// merge, 4.5 TB/s of the copy's 6.6 (290 without the look for small weights; where scores spread so far that every
// tile has some, a step takes up to 1.5 times as long). Two CTAs, 8 warps, a SM issue 0.55 instructions a cycle and
// scheduler, the ALU pipe is 54 % busy: conversions and the softmax of padded rows, with too few warps to cover their
// chain, not the loads (three CTAs a SM with two stages: the same time). 8 captions of 320 tokens: 8 us a call, all
// latency.
#include <ATen/cuda/CUDAContext.h>
#include <torch/extension.h>

#include "common.cuh"
#include "paged.h"
#include "status.h"

namespace ng {

using bf16 = __nv_bfloat16;

namespace {

constexpr int kWarps = 4, kStages = 3, kRows = 16;
// e4m3 pools: the largest weight, 2^kTop; the least that f16 rounds to 2^-9 of it; and what the remainders of smaller
// ones, at most 2^-25, are lifted by, at most twice (to 2^-96 of weights up to 2^15; the accumulators then stay below
// 512 keys * 448 * 2^15 * 2^80 < 2^113)
constexpr float kTop = 15.f, kLeastWeight = 0x1p-16f, kLift = 0x1p40f;
constexpr int kLifts = 2;
constexpr int kStageBytes = 8192;  // K and V of one warp's tile

template <int D, bool Q8>
struct Tile {
  static constexpr int RB = D * (Q8 ? 1 : 2);            // bytes of a cached row
  static constexpr int KT = kStageBytes / 2 / RB;        // keys of a tile
  static constexpr int CH = RB / 16;                     // 16-byte chunks of a row
  static constexpr int SF = Q8 ? 2 * KT : 0;             // scale bytes of a tile
  static constexpr int SMEM = kWarps * kStages * (kStageBytes + SF);
  // shared-memory offset of chunk c of row r: eight consecutive rows fall into different banks for every c
  __device__ static __forceinline__ int off(int r, int c) {
    if (CH >= 8) return r * RB + ((c ^ (r & 7)) << 4);
    return r * RB + ((c ^ ((r >> 1) & 3)) << 4);
  }
};

__device__ __forceinline__ void cp4(uint32_t dst, const void* src, bool live) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(live ? 4 : 0) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr));
}
__device__ __forceinline__ void ldsm4t(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr));
}
template <bool HALF>
__device__ __forceinline__ void mma16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if (HALF)
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t pack_half(float lo, float hi) {
  __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<uint32_t*>(&h);
}
__device__ __forceinline__ __half2 as_half2(uint32_t w) { return *reinterpret_cast<__half2*>(&w); }

// e4m3 pools: O += P V for the 16 keys of step kt of the tile's values at shared-memory address v
template <int D>
__device__ __forceinline__ void add_pv8(float (&o)[D / 8][4], const uint32_t (&p)[4], uint32_t v, int kt, int lane) {
  // matrices: keys 0-7 | 8-15 | 0-7 | 8-15 with columns 0-15 | 0-15 | 16-31 | 16-31; a register holds two columns of
  // two keys, sorted by column before the conversion
#pragma unroll
  for (int d = 0; d < D / 32; ++d) {
    uint32_t r[4];
    ldsm4t(r, v + Tile<D, true>::off(kt * 16 + (lane & 15), d * 2 + (lane >> 4)));
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const uint32_t u0 = __byte_perm(r[h * 2], 0, 0x3120), u1 = __byte_perm(r[h * 2 + 1], 0, 0x3120);
      mma16<true>(o[d * 4 + h * 2], p, e4m3x2_f16x2(u0), e4m3x2_f16x2(u1));
      mma16<true>(o[d * 4 + h * 2 + 1], p, e4m3x2_f16x2(u0 >> 16), e4m3x2_f16x2(u1 >> 16));
    }
  }
}

__device__ __forceinline__ float quad_max(float v) {
  v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 1));
  return fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 2));
}
__device__ __forceinline__ float quad_sum(float v) {
  v += __shfl_xor_sync(0xffffffffu, v, 1);
  return v + __shfl_xor_sync(0xffffffffu, v, 2);
}

}  // namespace

template <int D, bool Q8>
__global__ void __launch_bounds__(kWarps * 32, 2) paged_rows_kernel(const PagedAttnArgs a) {
  using T = Tile<D, Q8>;
  constexpr int KT = T::KT, NT = KT / 8, DT = D / 8;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ float s_m[kWarps][kRows], s_l[kWarps][kRows];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  // block -> (sequence, key head, row tile, split); splits are adjacent
  int id = blockIdx.x;
  const int split = id % a.splits;
  id /= a.splits;
  const int rt = id % a.row_tiles;
  id /= a.row_tiles;
  const int hk = id % a.p.Hk, b = id / a.p.Hk;
  const int G = a.H / a.p.Hk;
  const int row0 = max(0, __ldg(a.cu + b));
  const int n = max(0, min(__ldg(a.cu + b + 1), a.T) - row0);
  if (threadIdx.x == 0 && split == 0 && rt == 0 && hk == 0) paged_check(a, b);
  const int total = max(0, min(__ldg(a.total + b), a.max_total));
  const int R = min(kRows, n * G - rt * kRows);  // rows of this tile; row r: token (rt * 16 + r) / G, head hk G + rest
  if (R <= 0) return;
  const int used = paged_used_splits(a, total);
  if (split >= used) return;
  const int k0 = split * a.split_len, k1 = min(total, k0 + a.split_len);

  const int t4 = lane & 3, rq = lane >> 2;
  // rows rq and rq + 8 of the tile: last visible key, packed row and head
  int last[2];
  int64_t qoff[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int r = rt * kRows + rq + 8 * i;
    const bool live = rq + 8 * i < R;
    const int tok = live ? r / G : 0;
    last[i] = live ? (a.causal ? total - n + tok : total - 1) : -1;
    qoff[i] = live ? (int64_t)(row0 + tok) * a.ldq + (hk * G + r - tok * G) * D : -1;
  }
  // ---- Q fragments. e4m3: column order within 16 is 4 t, 4 t + 1 | 4 t + 2, 4 t + 3, as the keys' bytes come out
  uint32_t qf[D / 16][4];
  float sc[2] = {a.scale_log2, a.scale_log2};
#pragma unroll
  for (int s = 0; s < D / 16; ++s)
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      uint2 u = make_uint2(0u, 0u);
      if (qoff[i] >= 0) {
        const bf16* q = a.q + qoff[i] + s * 16;
        if (Q8) {
          u = *reinterpret_cast<const uint2*>(q + t4 * 4);
        } else {
          u.x = *reinterpret_cast<const uint32_t*>(q + t4 * 2);
          u.y = *reinterpret_cast<const uint32_t*>(q + t4 * 2 + 8);
        }
      }
      qf[s][i] = u.x;
      qf[s][i + 2] = u.y;
    }
  if (Q8) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      float m = 0.f;
#pragma unroll
      for (int s = 0; s < D / 16; ++s)
#pragma unroll
        for (int j = i; j < 4; j += 2)
          m = fmaxf(m, fmaxf(fabsf(bf16_bits_lo(qf[s][j])), fabsf(bf16_bits_hi(qf[s][j]))));
      m = quad_max(m);
      const int e = max(-100, min(126, (int)(__float_as_uint(m) >> 23) - 127 - 14));
      const float up = exp2i(-e);
      sc[i] = a.scale_log2 * exp2i(e);
#pragma unroll
      for (int s = 0; s < D / 16; ++s)
#pragma unroll
        for (int j = i; j < 4; j += 2)
          qf[s][j] = pack_half(bf16_bits_lo(qf[s][j]) * up, bf16_bits_hi(qf[s][j]) * up);
    }
  }

  uint8_t* ring = smem + warp * kStages * (kStageBytes + T::SF);
  const uint32_t ring_u = smem_u32(ring);
  const int ntile = (k1 - k0 + KT - 1) / KT;
  const int mine = ntile > warp ? (ntile - warp + kWarps - 1) / kWarps : 0;
  // ---- loads of the warp's i-th tile into stage i % kStages; slots past the split's keys are zero-filled
  auto load = [&](int i) {
    const int key0 = k0 + (warp + i * kWarps) * KT;
    const uint32_t st = ring_u + (i % kStages) * (kStageBytes + T::SF);
    int64_t base[KT > 32 ? 2 : 1];
#pragma unroll
    for (int j = 0; j < (KT > 32 ? 2 : 1); ++j) {
      const int r = lane + 32 * j, key = key0 + r;
      base[j] = -1;
      if (r < KT && key < k1) {
        const int pg = paged_page(a.p, b, key, a.err);
        if (pg >= 0) base[j] = paged_row(a.p, pg, hk, key & ((1 << a.p.page_shift) - 1));
      }
    }
    constexpr int PER = KT * T::CH / 32;  // 16-byte chunks of K (and of V) a lane
#pragma unroll
    for (int c = 0; c < PER; ++c) {
      const int ch = c * 32 + lane, r = ch / T::CH, col = ch % T::CH;
      const int64_t row = __shfl_sync(0xffffffffu, base[KT > 32 ? (c * 32 / T::CH) / 32 : 0], r & 31);
      const bool live = row >= 0;
      const int64_t src = (live ? row : 0) * T::RB + col * 16;
      const uint32_t dst = st + T::off(r, col);
      cp_async16(dst, static_cast<const uint8_t*>(a.p.k) + src, live);
      cp_async16(dst + kStageBytes / 2, static_cast<const uint8_t*>(a.p.v) + src, live);
    }
    if (Q8) {  // scale bytes, four tokens a copy (pages are multiples of eight tokens)
      const int r = (lane * 4) % KT;
      const int64_t row = __shfl_sync(0xffffffffu, base[0], r & 31);
      const int64_t row2 = KT > 32 ? __shfl_sync(0xffffffffu, base[KT > 32 ? 1 : 0], r & 31) : -1;
      const int64_t row_ = r < 32 ? row : row2;
      const bool live = row_ >= 0;
      if (lane < KT / 2)
        cp4(st + kStageBytes + (lane * 4 < KT ? 0 : KT) + r, (lane * 4 < KT ? a.p.ksf : a.p.vsf) + (live ? row_ : 0),
            live);
    }
  };

  float o[DT][4];
#pragma unroll
  for (int i = 0; i < DT; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) o[i][j] = 0.f;
  float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};

#pragma unroll
  for (int i = 0; i < kStages - 1; ++i) {
    if (i < mine) load(i);
    cp_commit();
  }
  for (int i = 0; i < mine; ++i) {
    cp_wait<kStages - 2>();
    __syncwarp();  // tile i has landed for every lane, and every lane has left tile i - 1's stage
    if (i + kStages - 1 < mine) load(i + kStages - 1);
    cp_commit();
    const int key0 = k0 + (warp + i * kWarps) * KT;
    const uint32_t st = ring_u + (i % kStages) * (kStageBytes + T::SF);
    const uint8_t* sf = ring + (i % kStages) * (kStageBytes + T::SF) + kStageBytes;
    // ---- S = Q K^T
    float s[NT][4];
#pragma unroll
    for (int j = 0; j < NT; ++j) s[j][0] = s[j][1] = s[j][2] = s[j][3] = 0.f;
#pragma unroll
    for (int kt = 0; kt < KT / 16; ++kt) {
      if (Q8) {
        // matrices: keys 0-7 | 0-7 | 8-15 | 8-15 with columns 0-15 | 16-31 | 0-15 | 16-31 of a 32-column step
#pragma unroll
        for (int d = 0; d < D / 32; ++d) {
          uint32_t r[4];
          ldsm4(r, st + T::off(kt * 16 + (lane & 7) + ((lane >> 4) << 3), d * 2 + ((lane >> 3) & 1)));
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            mma16<true>(s[kt * 2], qf[d * 2 + h], e4m3x2_f16x2(r[h]), e4m3x2_f16x2(r[h] >> 16));
            mma16<true>(s[kt * 2 + 1], qf[d * 2 + h], e4m3x2_f16x2(r[2 + h]), e4m3x2_f16x2(r[2 + h] >> 16));
          }
        }
      } else {
        // matrices: keys 0-7 | 0-7 | 8-15 | 8-15 with columns 0-7 | 8-15 | 0-7 | 8-15 of a 16-column step
#pragma unroll
        for (int d = 0; d < D / 16; ++d) {
          uint32_t r[4];
          ldsm4(r, st + T::off(kt * 16 + (lane & 7) + ((lane >> 4) << 3), d * 2 + ((lane >> 3) & 1)));
          mma16<false>(s[kt * 2], qf[d], r[0], r[1]);
          mma16<false>(s[kt * 2 + 1], qf[d], r[2], r[3]);
        }
      }
    }
    // ---- scores in log2 units (e4m3: plus the value's exponent), mask, running maximum
    float mt[2] = {-INFINITY, -INFINITY};
    float un[NT][2];  // 2^-e of the values' scales
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      float ks[2] = {1.f, 1.f}, ve[2] = {0.f, 0.f};
      if (Q8) {
        const uint32_t kb = *reinterpret_cast<const uint16_t*>(sf + j * 8 + t4 * 2);
        const uint32_t vb = *reinterpret_cast<const uint16_t*>(sf + KT + j * 8 + t4 * 2);
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          const uint32_t vv = (vb >> (8 * c)) & 0xFFu;
          ks[c] = __uint_as_float(((kb >> (8 * c)) & 0xFFu) << 23);
          ve[c] = (float)((int)vv - 127);
          un[j][c] = __uint_as_float(min(254u, 254u - vv) << 23);
        }
      }
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const int key = key0 + j * 8 + t4 * 2 + (c & 1);
        const float x = Q8 ? s[j][c] * (sc[c >> 1] * ks[c & 1]) + ve[c & 1] : s[j][c] * sc[c >> 1];
        s[j][c] = key <= last[c >> 1] && key < k1 ? x : -INFINITY;
        mt[c >> 1] = fmaxf(mt[c >> 1], s[j][c]);
      }
    }
    float ms[2];
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const float mq = quad_max(mt[r]);
      // less kTop, but where rounding or an infinity would let a weight pass 2^kTop
      const float mn = fmaxf(m[r], Q8 && mq - (mq - kTop) <= kTop ? mq - kTop : mq);
      ms[r] = mn == -INFINITY ? 0.f : mn;  // no visible key yet: weights 2^(-inf) = 0
      const float c = ex2_ftz(m[r] - ms[r]);
      m[r] = mn;
      l[r] *= c;
#pragma unroll
      for (int d = 0; d < DT; ++d) {
        o[d][2 * r] *= c;
        o[d][2 * r + 1] *= c;
      }
    }
    // ---- P and O += P V
    const uint32_t vst = st + kStageBytes / 2;
    uint32_t pf[KT / 16][4];
#pragma unroll
    for (int kt = 0; kt < KT / 16; ++kt) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        float(&x)[4] = s[kt * 2 + h];
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          x[c] = ex2_ftz(x[c] - ms[c >> 1]);
          l[c >> 1] += Q8 ? x[c] * un[kt * 2 + h][c & 1] : x[c];
        }
        pf[kt][h * 2] = Q8 ? pack_half(x[0], x[1]) : pack_bf16(x[0], x[1]);
        pf[kt][h * 2 + 1] = Q8 ? pack_half(x[2], x[3]) : pack_bf16(x[2], x[3]);
      }
      if (Q8) {
        add_pv8<D>(o, pf[kt], vst, kt, lane);
      } else {
        // matrices: keys 0-7 | 8-15 | 0-7 | 8-15 with columns 0-7 | 0-7 | 8-15 | 8-15
#pragma unroll
        for (int d = 0; d < D / 16; ++d) {
          uint32_t r[4];
          ldsm4t(r, vst + T::off(kt * 16 + (lane & 15), d * 2 + (lane >> 4)));
          mma16<false>(o[d * 2], pf[kt], r[0], r[1]);
          mma16<false>(o[d * 2 + 1], pf[kt], r[2], r[3]);
        }
      }
    }
    if (Q8) {  // weights that f16 cut short (masked keys, weight 0, look like them at first)
      bool low = false;
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        __half2 least = as_half2(pf[0][r]);
#pragma unroll
        for (int i = 1; i < KT / 8; ++i) least = __hmin2(least, as_half2(pf[i >> 1][(i & 1) * 2 + r]));
        low |= last[r] >= 0 && !__hbge2(least, __float2half2_rn(kLeastWeight));
      }
      float lifted = 1.f;
      if (__any_sync(0xffffffffu, low)) {
#pragma unroll 1
        for (int i = 0; i < kLifts; ++i) {
          bool rest = false;
#pragma unroll
          for (int j = 0; j < NT; ++j)
#pragma unroll
            for (int c = 0; c < 4; ++c) {  // the remainder, exact
              float& x = s[j][c];
              x = fabsf(x) < kLeastWeight ? x - __half2float(__float2half_rn(x)) : 0.f;
              rest |= x != 0.f;
              x *= kLift;
            }
          if (!__any_sync(0xffffffffu, rest)) break;
          lifted *= kLift;
#pragma unroll
          for (int d = 0; d < DT; ++d)
#pragma unroll
            for (int c = 0; c < 4; ++c) o[d][c] *= kLift;
#pragma unroll
          for (int kt = 0; kt < KT / 16; ++kt) {
            const float(&x)[4] = s[kt * 2], (&y)[4] = s[kt * 2 + 1];
            const uint32_t pr[4] = {pack_half(x[0], x[1]), pack_half(x[2], x[3]), pack_half(y[0], y[1]),
                                    pack_half(y[2], y[3])};
            add_pv8<D>(o, pr, vst, kt, lane);
          }
        }
        const float down = 1.f / lifted;
#pragma unroll
        for (int d = 0; d < DT; ++d)
#pragma unroll
          for (int c = 0; c < 4; ++c) o[d][c] *= down;
      }
    }
  }
  cp_wait<0>();

  // ---- the four warps meet: common maximum, scaled sums
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    l[r] = quad_sum(l[r]);
    if (t4 == 0) {
      s_m[warp][rq + 8 * r] = m[r];
      s_l[warp][rq + 8 * r] = l[r];
    }
  }
  __syncthreads();  // also: no warp reads its ring any more
  float* so = reinterpret_cast<float*>(smem);  // [kWarps][kRows][D + 4]
  constexpr int LD = D + 4;
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    float mc = -INFINITY;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) mc = fmaxf(mc, s_m[w][rq + 8 * r]);
    const float c = mc == -INFINITY ? 0.f : ex2_ftz(m[r] - mc);
    float* dst = so + (warp * kRows + rq + 8 * r) * LD;
#pragma unroll
    for (int d = 0; d < DT; ++d) {
      if (Q8) {  // tile pairs hold columns 4 t + {0, 2} and 4 t + {1, 3} of 16
        if ((d & 1) == 0)
          *reinterpret_cast<float4*>(dst + (d >> 1) * 16 + t4 * 4) =
              make_float4(o[d][2 * r] * c, o[d + 1][2 * r] * c, o[d][2 * r + 1] * c, o[d + 1][2 * r + 1] * c);
      } else {
        *reinterpret_cast<float2*>(dst + d * 8 + t4 * 2) = make_float2(o[d][2 * r] * c, o[d][2 * r + 1] * c);
      }
    }
  }
  __syncthreads();
  const bool one = used == 1;
  for (int i = threadIdx.x; i < R * (D / 4); i += kWarps * 32) {
    const int r = i / (D / 4), c = (i % (D / 4)) * 4;
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
    float mc = -INFINITY, lc = 0.f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) mc = fmaxf(mc, s_m[w][r]);
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const float4 x = *reinterpret_cast<const float4*>(so + (w * kRows + r) * LD + c);
      v.x += x.x, v.y += x.y, v.z += x.z, v.w += x.w;
      lc += mc == -INFINITY ? s_l[w][r] : s_l[w][r] * ex2_ftz(s_m[w][r] - mc);
    }
    const int tok = (rt * kRows + r) / G;
    const int64_t at = (int64_t)(row0 + tok) * a.H + hk * G + rt * kRows + r - tok * G;  // (packed row, head)
    if (one) {
      const float inv = paged_inv(lc);
      *reinterpret_cast<uint2*>(a.o + at * D + c) =
          make_uint2(pack_bf16(v.x * inv, v.y * inv), pack_bf16(v.z * inv, v.w * inv));
      if (c == 0) a.lse[at] = paged_lse(mc, lc);
    } else {
      const int64_t units = (int64_t)a.T * a.H;
      *reinterpret_cast<float4*>(a.part + (split * units + at) * D + c) = v;
      if (c == 0)
        *reinterpret_cast<float2*>(a.part + a.splits * units * D + (split * units + at) * 2) = make_float2(mc, lc);
    }
  }
}

template <int D, bool Q8>
static void launch_rows(const PagedAttnArgs& a, cudaStream_t st) {
  const int smem = std::max(Tile<D, Q8>::SMEM, kWarps * kRows * (D + 4) * 4);
  static SmemAllowed allowed;
  allow_smem(paged_rows_kernel<D, Q8>, smem, allowed);
  const int64_t grid = (int64_t)a.B * a.p.Hk * a.row_tiles * a.splits;
  paged_rows_kernel<D, Q8><<<(int)grid, kWarps * 32, smem, st>>>(a);
  NG_LAUNCH_CHECK();
}

void paged_rows_launch(PagedAttnArgs a, cudaStream_t st) {
  const int G = a.H / a.p.Hk;
  a.row_tiles = (a.max_new * G + kRows - 1) / kRows;
  const int64_t tiles = (int64_t)a.B * a.p.Hk * a.row_tiles;
  // Keys of a split: enough splits for four CTAs a SM, none shorter than 512 keys (the merge costs a launch), none
  // longer than 2048 (sequences differ in length: short CTAs even the load out).
  const int64_t want = (tiles * a.max_total + 4 * kSMs - 1) / (4 * kSMs);
  a.split_len = (int)std::min<int64_t>(2048, std::max<int64_t>(512, (want + 63) / 64 * 64));
  a.splits = std::max(1, (a.max_total + a.split_len - 1) / a.split_len);
  TORCH_CHECK(tiles * a.splits <= INT32_MAX && tiles <= INT32_MAX, "paged: too many rows");
  at::Tensor part;
  if (a.splits > 1) {
    part = at::empty({(int64_t)a.splits * a.T * a.H * (a.p.D + 2)},
                     at::TensorOptions().device(at::kCUDA).dtype(at::kFloat));
    a.part = part.data_ptr<float>();
  }
  const bool q8 = a.p.ksf != nullptr;
  if (a.p.D == 128)
    q8 ? launch_rows<128, true>(a, st) : launch_rows<128, false>(a, st);
  else
    q8 ? launch_rows<64, true>(a, st) : launch_rows<64, false>(a, st);
  if (a.splits > 1) paged_merge_launch(a, st);
}

}  // namespace ng
