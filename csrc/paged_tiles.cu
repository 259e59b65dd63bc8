// Attention of a chunk of new tokens over the paged cache on the 5th-generation tensor cores (tcgen05 + TMEM), for
// sm_100a.
//
// An item is (sequence, key head, 256 rows). Rows are (token, query head of the group) pairs, token by token, so the G
// query heads of a key head share every K / V tile it reads; two 128-row tiles A and B ping-pong on the tensor core.
// One persistent CTA per SM: the items' key tiles, laid end to end, are dealt out in equal shares (causal rows and
// ragged sequences differ by far more than a wave could even out), so an item may be cut between CTAs; its pieces are
// then merged by their maxima in a fixed order (paged_tiles_merge_kernel). Per 128-key tile j of a piece:
//   MMA warp      S_X(j) = Q_X K_j^T into TMEM;  O_X += P_X(j) V_j with P_X read from TMEM
//   softmax warps (a thread per row, a warpgroup per tile) S_X(j) -> registers, mask, running maximum and sum in fp32,
//                 P_X(j) over S_X(j)'s own columns (two 16-bit values a column), O_X rescaled only when a maximum
//                 moved by more than 2^8 (P stays below 2^8; the result does not depend on which maximum scales it)
//   load warps    bf16 pool: TMA boxes, one per page and 64 columns; e4m3 pool: 16-byte loads, scaled to bf16 (exact)
//                 into the swizzled tile by all four warps
// The softmax is the longest link of the chain S -> P -> O, so it must never wait: a tile is worked off in halves of
// 64 keys with an S buffer each, and S of half u + 1 is on its way while the softmax works on half u. Order of issue,
// per half u: PV(u - 2) S(u), by a warp for A and one for B; the products of one warp run in order, so S(u) finds P(u
// - 2) in its buffer read.
//
// e4m3 pools: a stored value times its scale is exact in bf16 (4 significant bits, scales within 2^+-63), so the load
// warps hand over bf16 tiles and all else is the bf16 path. (Scales kept out of the tiles and applied to the scores,
// as the row kernel does, cost three shared-memory words per key and row: 1.5 times the time, bound by shared-memory
// reads.)
//
// 4 prompts of up to 1000 new tokens over 8192, 16 / 8 heads of 128 in bf16 (124 GFLOP): 147 us and 17 us for the
// merge of the cut items; the products alone are 2648 cycles a tile pair (isolated), a pair takes about 3700, two
// halves of softmax at 1500 being the longer half of the chain (the exponentials alone are 1024). The roles' code
// competes for the instruction cache (tensor pipe 39 %, special functions 39 %, issue slots 34 % of the launch): one
// copy of each role's loop took captions from 150 to 97 us and e4m3 chunks from 1790 to 1200. e4m3 tiles are bound by
// their conversion (four warps, 1.6 to 2.6 thousand cycles an operand).
//
// Slots past the keys a CTA may see are zero in V's tile (whatever the pool holds there); in K's tile they are masked.
// TMEM: S_A [0, 64) and [64, 128), S_B [128, 192) and [192, 256), O_A [256, 256 + D), O_B [256 + D, 256 + 2 D).
#include <ATen/cuda/CUDAContext.h>
#include <torch/extension.h>

#include "common.cuh"
#include "gemm.h"
#include "paged.h"
#include "status.h"

namespace ng {

using bf16 = __nv_bfloat16;

namespace {

constexpr int kTileRows = 128, kKeys = 128, kHalf = 64;
// warps: 0-3 K / V, 4-7 softmax A, 8-11 softmax B, 12-13 MMA issue, 14 (e4m3) or 1-3 (bf16) Q, 15 pieces
constexpr int kThreads = 512;
constexpr float kRescaleLog2 = 8.f;
constexpr int kAtom = 128 * 128;  // bytes of a [128 rows][64 x 16-bit] swizzled atom

template <int D>
struct Lay {
  static constexpr int TB = (D / 64) * kAtom;   // a Q, K or V tile
  static constexpr int QB = D == 64 ? 2 : 1;    // Q buffers (the next piece's Q loads under this one's products)
  static constexpr int Q = 0;                   // [QB][A, B]
  static constexpr int K = Q + QB * 2 * TB;     // [2 stages]
  static constexpr int V = K + 2 * TB;          // [2 stages]
  static constexpr int BAR = V + 2 * TB;        // barriers, TMEM address, abort flag, the pieces' ring
  static constexpr int TAB = BAR + 1024;        // running costs of the entries
  static constexpr int SMEM = TAB + (2048 + 4) * 4 + 1024;
};

// byte offset of 16-byte chunk c of row r in a tile of 64-column atoms with the 128-byte swizzle
__device__ __forceinline__ int tile_off(int r, int c) {
  return (c >> 3) * kAtom + r * 128 + (((c & 7) ^ (r & 7)) << 4);
}

__device__ __forceinline__ void cp_async_wait_all() { asm volatile("cp.async.wait_all;" ::: "memory"); }

// D[tmem] (+)= A B^T with descriptors given as halves (the upper half a constant): A from shared memory, or from TMEM.
__device__ __forceinline__ void umma_ss(uint32_t d, uint32_t a_lo, uint32_t b_lo, uint32_t hi, uint32_t idesc,
                                        uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p, e;\n\t.reg .b64 da, db;\n\t"
      "elect.sync _|e, 0xffffffff;\n\tsetp.ne.b32 p, %5, 0;\n\t"
      "mov.b64 da, {%1, %3};\n\tmov.b64 db, {%2, %3};\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %4, p;\n\t}\n" ::"r"(d),
      "r"(a_lo), "r"(b_lo), "r"(hi), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void umma_ts(uint32_t d, uint32_t a_tmem, uint32_t b_lo, uint32_t hi, uint32_t idesc,
                                        uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p, e;\n\t.reg .b64 db;\n\t"
      "elect.sync _|e, 0xffffffff;\n\tsetp.ne.b32 p, %5, 0;\n\t"
      "mov.b64 db, {%2, %3};\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], db, %4, p;\n\t}\n" ::"r"(d),
      "r"(a_tmem), "r"(b_lo), "r"(hi), "r"(idesc), "r"(accumulate)
      : "memory");
}

// Arrives once on `bar` when every product issued so far has completed (a converged warp calls it).
__device__ __forceinline__ void umma_commit_elect(uint64_t* bar) {
  asm volatile(
      "{\n\t.reg .pred e;\n\telect.sync _|e, 0xffffffff;\n\t"
      "@e tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}\n" ::"r"(smem_u32(bar))
      : "memory");
}

// Bounded wait that ignores the abort flag: for what is still in flight when a CTA gives up.
__device__ __forceinline__ void mbar_drain(uint64_t* bar, uint32_t parity) {
  const uint64_t t0 = globaltimer_ns();
  while (!mbar_try_wait(bar, parity))
    if (globaltimer_ns() - t0 > NG_WAIT_BUDGET_NS) return;
}

template <int N>
__device__ __forceinline__ void regs_more() {
  asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N));
}
template <int N>
__device__ __forceinline__ void regs_less() {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N));
}

// Registers a thread of each warpgroup; together the launch's 512 x 128.
template <bool Q8>
constexpr int kRegsKV = Q8 ? 128 : 112;
template <bool Q8>
constexpr int kRegsRest = Q8 ? 96 : 112;
template <bool Q8>
constexpr int kRegsSoftmax = 144;
static_assert(kRegsKV<true> + kRegsRest<true> + 2 * kRegsSoftmax<true> <= 512, "more registers than the launch has");
static_assert(kRegsKV<false> + kRegsRest<false> + 2 * kRegsSoftmax<false> <= 512, "more registers than the launch has");

// ------------------------------------------------------------------------------------------------ work distribution
constexpr int kMaxEntries = 2048;  // (sequence, row tile) pairs whose running costs fit the table
constexpr int kCutTiles = 8;       // items of fewer key tiles are never cut
constexpr int kMargin = 2;         // nor is any cut closer than this many tiles to its ends
constexpr int kItemCost = 3;       // an item's Q load, pipeline fill and output, in key tiles

struct TileArgs {
  PagedAttnArgs a;
  int entries, balanced;  // balanced: entries <= kMaxEntries, shares from the table; else items are dealt in turn
  float* part;            // [2 * CTAs][256][D] unnormalised outputs, then [2 * CTAs][256][2] (maximum, sum)
  int* cuts;              // [CTAs][8]: start of the share, then a Cut where that start is an item's first cut
};

// An item that is cut: its pieces are the end piece of CTA c - 1 and the first pieces of the CTAs c .. last.
struct Cut {
  int row0, r0, rows, hk, last;  // rows 0: nothing cut here
};

// (sequence, row tile) pair e: rows [r0, r0 + rows) of the sequence's n * G, keys [0, kend) visible to any of them.
struct Entry {
  int b, r0, row0, n, total, rows, kend, tiles, halves_a;
};

__device__ __forceinline__ Entry entry_of(const PagedAttnArgs& a, int e) {
  Entry w;
  const int G = a.H / a.p.Hk;
  w.b = e / a.row_tiles;
  w.r0 = (e - w.b * a.row_tiles) * 2 * kTileRows;
  w.row0 = max(0, __ldg(a.cu + w.b));
  w.n = max(0, min(__ldg(a.cu + w.b + 1), a.T) - w.row0);
  w.total = max(0, min(__ldg(a.total + w.b), a.max_total));
  w.rows = max(0, min(2 * kTileRows, w.n * G - w.r0));
  auto seen = [&](int r) { return a.causal ? max(0, min(w.total, w.total - w.n + r / G + 1)) : w.total; };
  w.kend = w.rows > 0 ? seen(w.r0 + w.rows - 1) : 0;
  w.tiles = (w.kend + kKeys - 1) / kKeys;
  w.halves_a = w.rows > 0 ? (seen(w.r0 + min(w.rows, kTileRows) - 1) + kHalf - 1) / kHalf : 0;
  return w;
}

// Running costs of the entries in `tab` [entries + 1]: tiles + kItemCost per key head, 0 for an entry without rows.
// All threads of the block.
__device__ __forceinline__ void cost_table(const TileArgs& t, int* tab, int* warp_sums) {
  const int per = (t.entries + blockDim.x - 1) / blockDim.x, e0 = min(t.entries, (int)threadIdx.x * per);
  const int e1 = min(t.entries, e0 + per), lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int sum = 0;
  for (int e = e0; e < e1; ++e) {
    const Entry w = entry_of(t.a, e);
    tab[e + 1] = w.rows > 0 ? (w.tiles + kItemCost) * t.a.p.Hk : 0;
    sum += tab[e + 1];
  }
  int inc = sum;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int v = __shfl_up_sync(0xffffffffu, inc, o);
    if (lane >= o) inc += v;
  }
  if (lane == 31) warp_sums[warp] = inc;
  __syncthreads();
  int run = inc - sum;
  for (int i = 0; i < warp; ++i) run += warp_sums[i];
  if (threadIdx.x == 0) tab[0] = 0;
  for (int e = e0; e < e1; ++e) {
    run += tab[e + 1];
    tab[e + 1] = run;
  }
  __syncthreads();
}

struct Place {
  int e, cost, item, off;  // entry, cost of its items, start of the item, offset (the key tile) inside it
};

__device__ __forceinline__ Place place_of(const TileArgs& t, const int* tab, int u) {
  int lo = 0, hi = t.entries;  // the last e with tab[e] <= u and a cost
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (tab[mid + 1] > u)
      hi = mid;
    else
      lo = mid + 1;
  }
  Place p;
  p.e = lo;
  p.cost = lo < t.entries ? (tab[lo + 1] - tab[lo]) / t.a.p.Hk : 1;
  p.off = (u - tab[lo]) % p.cost;
  p.item = u - p.off;
  return p;
}

// Start of CTA c's share: its even share, moved to an item's start or end where a cut would be too short.
__device__ __forceinline__ int share_start(const TileArgs& t, const int* tab, int c, int ctas) {
  const int all = tab[t.entries];
  if (c >= ctas) return all;
  const int u = all / ctas * c + all % ctas * c / ctas;
  if (u >= all) return all;
  const Place p = place_of(t, tab, u);
  const int tiles = p.cost - kItemCost;
  if (p.off == 0 || (tiles < kCutTiles && p.off <= tiles / 2) || p.off < kMargin) return p.item;
  if (tiles < kCutTiles || p.off > tiles - kMargin) return p.item + p.cost;
  return u;
}

// A piece of an item: key tiles [j0, j1); tile A sees the half tiles below ja.
struct __align__(16) Piece {
  int b, hk, r0, row0, rows, kend;
  int first;  // causal: the row of token i sees keys up to first + i
  int j0, j1, ja, whole, valid;
};

// The pieces of this CTA, one after the other, into a ring in shared memory: one thread runs this.
constexpr int kRing = 4;

struct Pieces {
  const TileArgs& t;
  const int* tab;
  int u, end;
  __device__ Pieces(const TileArgs& t_, const int* tab_) : t(t_), tab(tab_) {
    u = t.balanced ? share_start(t, tab, blockIdx.x, gridDim.x) : blockIdx.x;
    end = t.balanced ? share_start(t, tab, blockIdx.x + 1, gridDim.x) : t.entries * t.a.p.Hk;
  }
  __device__ __forceinline__ Piece next() {
    Piece s;
    s.valid = 0;
    while (u < end && !s.valid) {
      Entry w;
      if (t.balanced) {
        const Place p = place_of(t, tab, u);
        w = entry_of(t.a, p.e);
        s.hk = (p.item - tab[p.e]) / p.cost;
        s.j0 = p.off;
        const int stop = min(p.item + p.cost, end);
        s.j1 = min(w.tiles, stop - p.item);
        u = stop;
      } else {
        w = entry_of(t.a, u / t.a.p.Hk);
        s.hk = u % t.a.p.Hk;
        s.j0 = 0;
        s.j1 = w.tiles;
        u += gridDim.x;
      }
      s.valid = w.rows > 0;
      s.b = w.b, s.r0 = w.r0, s.row0 = w.row0, s.rows = w.rows, s.kend = w.kend;
      s.first = t.a.causal ? w.total - w.n : w.total;
      s.ja = w.halves_a;
      s.whole = s.j0 == 0 && s.j1 == w.tiles;
    }
    return s;
  }
};

}  // namespace

template <int D, bool Q8>
__global__ void __launch_bounds__(kThreads, 1)
    paged_tiles_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV,
                       const __grid_constant__ TileArgs t) {
  using L = Lay<D>;
  constexpr uint32_t C_S = 0, C_O = 256;
  constexpr int kQWarps = Q8 ? 1 : 3;
  const PagedAttnArgs& a = t.a;
  const int G = a.H / a.p.Hk;

  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + L::BAR);
  uint64_t* q_full = bars + 2;     // [QB] Q ready (the Q warps)
  uint64_t* q_empty = bars + 4;    // [QB] the piece's S products completed
  uint64_t* k_full = bars + 6;     // [2]
  uint64_t* k_empty = bars + 8;    // [2]
  uint64_t* v_full = bars + 10;    // [2]
  uint64_t* v_empty = bars + 12;   // [2]
  uint64_t* s_full = bars + 14;    // [A0, A1, B0, B1] S product of that half completed
  uint64_t* p_full = bars + 18;    // [A0, A1, B0, B1] P written, O rescaled (4 warps)
  uint64_t* pv_done = bars + 22;   // [A0, A1, B0, B1] P V product completed
  uint64_t* o_empty = bars + 26;   // [A, B] O read (4 warps)
  uint64_t* tail = bars + 28;      // the boxes of an item's last V tile landed
  uint64_t* drain = bars + 29;     // [A, B]
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 31);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  uint64_t* d_full = bars + 32;    // [kRing] a piece's description is in its slot
  uint64_t* d_empty = bars + 36;   // [kRing] every role has read it
  Piece* ring = reinterpret_cast<Piece*>(smem + L::BAR + 512);
  int* warp_sums = reinterpret_cast<int*>(ring + kRing);  // [16]
  int* tab = reinterpret_cast<int*>(smem + L::TAB);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int i = 0; i < 2; ++i) {
      mbar_init(&q_full[i], kQWarps);
      mbar_init(&q_empty[i], 2);
      mbar_init(&k_full[i], Q8 ? 4 : 1);
      mbar_init(&v_full[i], Q8 ? 4 : 1);
      mbar_init(&k_empty[i], 2);
      mbar_init(&v_empty[i], 2);
      mbar_init(&drain[i], 1);
      mbar_init(&o_empty[i], 4);
    }
    for (int i = 0; i < 4; ++i) {
      mbar_init(&s_full[i], 1);
      mbar_init(&p_full[i], 4);
      mbar_init(&pv_done[i], 1);
    }
    for (int i = 0; i < kRing; ++i) {
      mbar_init(&d_full[i], 1);
      mbar_init(&d_empty[i], (Q8 ? 4 : 1) + kQWarps + 2 + 8);  // K / V, Q, MMA and softmax warps
    }
    mbar_init(tail, 1);
    *abort_flag = 0;
    fence_barrier_init();
  }
  if (warp == 12) {
    tmem_alloc(tmem_slot, 512);
    tmem_relinquish();
  }
  for (int b = blockIdx.x * kThreads + threadIdx.x; b < a.B; b += gridDim.x * kThreads) paged_check(a, b);
  if (t.balanced) cost_table(t, tab, warp_sums);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  Piece s;
  uint32_t taken = 0;
  auto wait_all = [&](uint64_t* bar, uint32_t parity, int code) -> bool {  // a warp's lanes together
    return __all_sync(0xffffffffu, mbar_wait(bar, parity, abort_flag, a.err, code));
  };
  auto take = [&]() -> bool {  // the next piece
    const uint32_t k = taken % kRing, ph = (taken / kRing) & 1;
    if (!wait_all(&d_full[k], ph, kErrWaitFull)) return false;
    s = ring[k];
    __syncwarp();
    if (lane == 0) mbar_arrive(&d_empty[k]);
    ++taken;
    return s.valid != 0;
  };

  // Q of every piece: by warp 14, or by the three warps that K / V tiles by TMA leave idle. Called in one place of
  // either instantiation.
  auto load_q = [&](int qw) {
    constexpr int CQ = D / 8;
    for (uint32_t k = 0; take();) {
      if (s.j0 >= s.j1) continue;
      const uint32_t qb = k % L::QB, ph = ((k / L::QB) & 1) ^ 1;
      if (!wait_all(&q_empty[qb], ph, kErrWaitEmpty)) break;
      ++k;
      uint8_t* q = smem + L::Q + qb * 2 * L::TB;
      const int rows = s.rows > kTileRows ? 2 * kTileRows : kTileRows;
      // row -> (token, head): r0 once, the rest by a product (exact: local < 2^17, half a step from any integer)
      const int tok0 = s.r0 / G, rem0 = s.r0 - tok0 * G, c = lane % CQ;
      const float inv_g = 1.f / (float)G;
#pragma unroll 4
      for (int row = qw * (32 / CQ) + lane / CQ; row < rows; row += kQWarps * (32 / CQ)) {
        const int local = rem0 + row, t1 = (int)(((float)local + 0.5f) * inv_g);
        const bool live = row < s.rows;
        const bf16* src =
            a.q + (live ? (int64_t)(s.row0 + tok0 + t1) * a.ldq + (s.hk * G + local - t1 * G) * D + c * 8 : 0);
        cp_async16(smem_u32(q + (row >> 7) * L::TB + tile_off(row & 127, c)), src, live);
      }
      cp_async_wait_all();
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(&q_full[qb]);
    }
  };

  if (warp < 4) {
    // ------------------------------------------------------------------------------------------------ K / V tiles
    regs_less<kRegsKV<Q8>>();
    if (Q8) {
      // A thread loads 16-byte pieces of rows warp * 32 + i * (32 / CH) + lane / CH; the row addresses come from the
      // lane that looked its page up. A tile's pieces stay in registers until its buffer is free; the next tile's
      // loads are issued right behind the stores.
      constexpr int CH = D / 16, RI = 32 / CH;  // 16-byte pieces of a row, rows a warp instruction covers
      int64_t base = -1;                        // pool row of key warp * 32 + lane of the tile whose loads run
      int j = 0;
      auto next_piece = [&]() -> bool {  // the next piece with key tiles
        while (take())
          if (s.j0 < s.j1) {
            j = s.j0;
            return true;
          }
        return false;
      };
      auto rows_at = [&]() {
        const int key = j * kKeys + warp * 32 + lane;
        base = -1;
        if (key < s.kend) {
          const int pg = paged_page(a.p, s.b, key, a.err);
          if (pg >= 0) base = paged_row(a.p, pg, s.hk, key & ((1 << a.p.page_shift) - 1));
        }
      };
      uint4 rk[CH], rv[CH];
      uint32_t sk = 0, sv = 0;
      auto fetch = [&](uint4(&r)[CH], const void* pool) {
#pragma unroll
        for (int i = 0; i < CH; ++i) {
          const int64_t row = __shfl_sync(0xffffffffu, base, i * RI + lane / CH);
          r[i] = make_uint4(0u, 0u, 0u, 0u);
          if (row >= 0)
            r[i] = __ldg(
                reinterpret_cast<const uint4*>(static_cast<const uint8_t*>(pool) + row * D + (lane % CH) * 16));
        }
      };
      auto put = [&](const uint4(&r)[CH], uint32_t scale, uint8_t* dst) {
        const int c = lane % CH;
        // lanes of the upper half of a row store their second chunk first: no two lanes of a store share a bank
        const int first = c >= CH / 2 ? 1 : 0;
#pragma unroll
        for (int i = 0; i < CH; ++i) {
          const int row = warp * 32 + i * RI + lane / CH;
          const float f = exp2i((int)__shfl_sync(0xffffffffu, scale, i * RI + lane / CH) - 127);
          const uint2 x0 = e4m3x4_bf16x4(r[i].x, f), x1 = e4m3x4_bf16x4(r[i].y, f);
          const uint2 x2 = e4m3x4_bf16x4(r[i].z, f), x3 = e4m3x4_bf16x4(r[i].w, f);
          const uint4 lo = make_uint4(x0.x, x0.y, x1.x, x1.y), hi = make_uint4(x2.x, x2.y, x3.x, x3.y);
          *reinterpret_cast<uint4*>(dst + tile_off(row, 2 * c + first)) = first ? hi : lo;
          *reinterpret_cast<uint4*>(dst + tile_off(row, 2 * c + 1 - first)) = first ? lo : hi;
        }
      };
      auto scale_of = [&](const uint8_t* sf) -> uint32_t { return base >= 0 ? __ldg(sf + base) : 127u; };
      bool have = next_piece();
      if (have) {
        rows_at();
        fetch(rk, a.p.k);
        sk = scale_of(a.p.ksf);
        fetch(rv, a.p.v);
        sv = scale_of(a.p.vsf);
      }
      for (uint32_t g = 0; have; ++g) {
        const int st = g & 1;
        const uint32_t ph = ((g >> 1) & 1) ^ 1;
        if (!wait_all(&k_empty[st], ph, kErrWaitEmpty)) break;
        put(rk, sk, smem + L::K + st * L::TB);
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&k_full[st]);
        const bool early = j + 1 < s.j1;  // K of the piece's next tile is asked for before V of this one is stored
        if (early) {
          ++j;
          rows_at();
          fetch(rk, a.p.k);
          sk = scale_of(a.p.ksf);
        }
        if (!wait_all(&v_empty[st], ph, kErrWaitEmpty)) break;
        put(rv, sv, smem + L::V + st * L::TB);
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&v_full[st]);
        // the next piece is taken only now: every tile of the earlier ones is in place, so no role waits for this one
        if (!early) {
          have = next_piece();
          if (have) {
            rows_at();
            fetch(rk, a.p.k);
            sk = scale_of(a.p.ksf);
          }
        }
        if (have) {
          fetch(rv, a.p.v);
          sv = scale_of(a.p.vsf);
        }
      }
    } else if (warp > 0) {
      load_q(warp - 1);
    } else {
      // One box per page (or per 128 keys of a longer page) and 64 columns, a lane each.
      const int boxes = max(1, kKeys >> a.p.page_shift);
      const int box_rows = min(kKeys, 1 << a.p.page_shift);
      const int i = lane / (D / 64), half = lane % (D / 64), dst = half * kAtom + i * box_rows * 128;
      uint32_t g = 0, tails = 0;
      bool ok = true;
      while (ok && take()) {
        for (int j = s.j0; ok && j < s.j1; ++j, ++g) {
          const int st = g & 1;
          const uint32_t ph = ((g >> 1) & 1) ^ 1;
          const int key0 = j * kKeys, key = key0 + i * box_rows, nv = s.kend - key0;
          int pg = -1;
          if (i < boxes && key < s.kend) pg = paged_page(a.p, s.b, key, a.err);
          const bool live = pg >= 0;
          const uint32_t bytes = __popc(__ballot_sync(0xffffffffu, live)) * box_rows * 128;
          const int z = live ? pg * a.p.Hk + s.hk : 0, y = key & ((1 << a.p.page_shift) - 1);
          ok = wait_all(&k_empty[st], ph, kErrWaitEmpty);
          if (!ok) break;
          if (lane == 0) mbar_arrive_expect_tx(&k_full[st], bytes);
          __syncwarp();
          if (live) tma_load_3d(&tmK, &k_full[st], smem + L::K + st * L::TB + dst, half * 64, y, z);
          ok = wait_all(&v_empty[st], ph, kErrWaitEmpty);
          if (!ok) {
            mbar_drain(&k_full[st], ph ^ 1);
            break;
          }
          uint64_t* vb = nv < kKeys ? tail : &v_full[st];
          if (lane == 0) mbar_arrive_expect_tx(vb, bytes);
          __syncwarp();
          if (live) tma_load_3d(&tmV, vb, smem + L::V + st * L::TB + dst, half * 64, y, z);
          if (nv < kKeys) {  // an item's last tile: zero V's rows past the visible keys, then hand it over
            const uint32_t tp = tails++ & 1;
            ok = wait_all(tail, tp, kErrWaitFull);
            if (!ok) {
              mbar_drain(&k_full[st], ph ^ 1);
              mbar_drain(tail, tp);
              break;
            }
            for (int c = lane; c < (kKeys - nv) * (D / 8); c += 32) {
              const int r = nv + c / (D / 8);
              *reinterpret_cast<uint4*>(smem + L::V + st * L::TB + tile_off(r, c % (D / 8))) = make_uint4(0, 0, 0, 0);
            }
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(&v_full[st]);
          }
        }
      }
      if (*abort_flag)  // no box may land in shared memory that this CTA no longer owns
        for (uint32_t i2 = g > 2 ? g - 2 : 0; i2 < g; ++i2) {
          mbar_drain(&k_full[i2 & 1], (i2 >> 1) & 1);
          mbar_drain(&v_full[i2 & 1], (i2 >> 1) & 1);
        }
    }
  } else if (warp >= 12) {
    regs_less<kRegsRest<Q8>>();
    if (warp == 15) {
      // ----------------------------------------------------------------------------------------------------- pieces
      if (lane == 0) {
        Pieces pieces(t, tab);
        for (uint32_t k = 0;; ++k) {
          const Piece p = pieces.next();
          if (!mbar_wait(&d_empty[k % kRing], ((k / kRing) & 1) ^ 1, abort_flag, a.err, kErrWaitEmpty)) break;
          ring[k % kRing] = p;
          mbar_arrive(&d_full[k % kRing]);
          if (!p.valid) break;
        }
        if (t.cuts != nullptr) {  // for the merge
          const int c = blockIdx.x, ctas = gridDim.x, u = share_start(t, tab, c, ctas);
          int* out = t.cuts + c * 8;
          Cut cut = {0, 0, 0, 0, c};
          if (u < tab[t.entries]) {
            const Place p = place_of(t, tab, u);
            if (p.off > 0 && share_start(t, tab, c - 1, ctas) <= p.item) {
              const Entry w = entry_of(a, p.e);
              cut = {w.row0, w.r0, w.rows, (p.item - tab[p.e]) / p.cost, c};
              while (cut.last + 1 < ctas && share_start(t, tab, cut.last + 1, ctas) < p.item + p.cost) ++cut.last;
            }
          }
          out[0] = u, out[1] = cut.row0, out[2] = cut.r0, out[3] = cut.rows, out[4] = cut.hk, out[5] = cut.last;
          out[6] = share_start(t, tab, c + 1, ctas);
        }
      }
    } else if (warp == 14) {
      if (Q8) load_q(0);
    } else {
      // ------------------------------------------------------------------------------------------------- MMA issue
      constexpr uint32_t idesc_s = idesc_bf16_f32(kTileRows, kHalf, 0, 0);
      constexpr uint32_t idesc_o = idesc_bf16_f32(kTileRows, D, 0, 1);
      // A warp per row tile, so that one's bookkeeping runs under the other's products: descriptors are a constant
      // upper half and a lower half that only takes additions of constants, or the issue itself bounds the kernel
      // (recomputed descriptors: 6600 cycles a tile pair, three times the products' own time).
      constexpr uint32_t hi = (uint32_t)(1024 >> 4) | (1u << 14) | (2u << 29);  // stride 1024, version 1, 128 B swizzle
      constexpr uint32_t lbo = (uint32_t)(kAtom >> 4) << 16;                    // between V's 64-column atoms
      const uint32_t q_lo = (smem_u32(smem + L::Q) >> 4) | (1u << 16), k_lo = (smem_u32(smem + L::K) >> 4) | (1u << 16);
      const uint32_t v_lo = (smem_u32(smem + L::V) >> 4) | lbo;
      const int X = warp - 12;
      const uint32_t q_x = q_lo + X * (L::TB >> 4), s_x = tmem + C_S + X * kKeys, o_x = tmem + C_O + X * D;
      uint32_t g = 0, q = 0;      // key tiles of this CTA before the piece (ring position), pieces
      uint32_t pp = 0;            // phase bits of p_full, per half
      uint32_t outs = 0;          // outputs finished
      bool ok = true;
      while (ok && take()) {
        const int n = s.j1 - s.j0;
        if (n <= 0) continue;
        const bool live_b = s.rows > kTileRows;
        const int all = min(2 * n, (s.kend - s.j0 * kKeys + kHalf - 1) / kHalf);  // halves of the piece
        const int mine = X == 1 ? (live_b ? all : 0) : (live_b ? max(0, min(all, s.ja - 2 * s.j0)) : all);
        const uint32_t qb = q % L::QB, qd = q_x + qb * 2 * (L::TB >> 4);
        ok = wait_all(&q_full[qb], (q / L::QB) & 1, kErrWaitFull);
        ++q;
#pragma unroll 1
        for (int u = 0; ok && u < all + 2; ++u) {
          const uint32_t h = u & 1, hs = s_x + h * kHalf;
          const bool ends = h == 1;
          // O += P V of half u - 2
          if (u >= 2) {
            const int v = u - 2;
            const uint32_t gg = g + (v >> 1), st = gg & 1;
            if (v < mine) {
              if (h == 0) ok = wait_all(&v_full[st], (gg >> 1) & 1, kErrWaitFull);
              ok = ok && wait_all(&p_full[X * 2 + h], (pp >> h) & 1, kErrWaitFull);
              pp ^= 1u << h;
              // the piece's first product overwrites O: the previous piece's output has been read
              if (v == 0 && outs > 0) ok = ok && wait_all(&o_empty[X], (outs - 1) & 1, kErrWaitAccEmpty);
              if (!ok) break;
              tc_fence_after();
              const uint32_t vd = v_lo + st * (L::TB >> 4) + h * (kHalf * 128 >> 4);
#pragma unroll
              for (int k = 0; k < kHalf / 16; ++k)
                umma_ts(o_x, hs + k * 8, vd + k * (2048 >> 4), hi, idesc_o, (k != 0 || v != 0) ? 1u : 0u);
              umma_commit_elect(&pv_done[X * 2 + h]);
              if (v + 1 == mine) ++outs;
            } else if (ends || v + 1 == all) {  // a tile this one does not see is released once it is there
              if (mine <= (v & ~1)) ok = wait_all(&v_full[st], (gg >> 1) & 1, kErrWaitFull);
            }
            if (ends || v + 1 == all) umma_commit_elect(&v_empty[st]);
          }
          // S of half u (its buffer: P V of half u - 2, issued before, has read P there)
          if (u < all) {
            const uint32_t gg = g + (u >> 1), st = gg & 1;
            if (h == 0) ok = ok && wait_all(&k_full[st], (gg >> 1) & 1, kErrWaitFull);
            if (!ok) break;
            if (u < mine) {
              const uint32_t kd = k_lo + st * (L::TB >> 4) + h * (kHalf * 128 >> 4);
#pragma unroll
              for (int k = 0; k < D / 16; ++k) {
                const uint32_t off = (k >> 2) * (kAtom >> 4) + (k & 3) * (32 >> 4);
                umma_ss(hs, qd + off, kd + off, hi, idesc_s, k != 0 ? 1u : 0u);
              }
              umma_commit_elect(&s_full[X * 2 + h]);
            }
            if (ends || u + 1 == all) umma_commit_elect(&k_empty[st]);
            if (u + 1 == all) umma_commit_elect(&q_empty[qb]);
          }
        }
        g += n;
      }
      if (!ok || *abort_flag) {  // products in flight finish before TMEM is released
        umma_commit_elect(&drain[X]);
        mbar_drain(&drain[X], 0);
      }
    }
  } else {
    // ---------------------------------------------------------------------------------------------------- softmax
    regs_more<kRegsSoftmax<Q8>>();
    const int X = (warp - 4) >> 2, quarter = warp & 3;
    const int row = quarter * 32 + lane;
    const uint32_t trow = tmem + ((uint32_t)(quarter * 32) << 16);
    uint32_t used = 0;  // parity of the halves worked off in buffer 0 and 1
    bool ok = true;
    while (ok && take()) {
      const int n = s.j1 - s.j0;
      if (X == 1 && s.rows <= kTileRows) continue;
      const int r = s.r0 + X * kTileRows + row;
      const bool live = X * kTileRows + row < s.rows;
      const int tok = live ? r / G : 0;
      // last visible key (dead rows: every key, so that they never ask for a mask)
      const int last = live && a.causal ? min(s.kend - 1, s.first + tok) : s.kend - 1;
      const int all = n > 0 ? min(2 * n, (s.kend - s.j0 * kKeys + kHalf - 1) / kHalf) : 0;
      const int nx = X == 0 && s.rows > kTileRows ? max(0, min(all, s.ja - 2 * s.j0)) : all;
      const float scale = a.scale_log2;
      float m = -INFINITY, l = 0.f;
#pragma unroll 1
      for (int u = 0; u < nx; ++u) {
        const uint32_t h = u & 1;
        if (!wait_all(&s_full[X * 2 + h], (used >> h) & 1, kErrWaitAccFull)) {
          ok = false;
          break;
        }
        used ^= 1u << h;
        tc_fence_after();
        const uint32_t ts = trow + C_S + X * kKeys + h * kHalf;
        const int lim = last - s.j0 * kKeys - u * kHalf;  // columns up to lim are visible
        const bool full = __all_sync(0xffffffffu, lim >= kHalf - 1);
        // Two rolled passes of 32 columns, read from TMEM again for the second: the roles' loops share a small
        // instruction cache, and 64 unrolled columns held in registers ran slower.
        float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll 1
        for (int c = 0; c < kHalf; c += 32) {
          uint32_t sc[32];
          tmem_ld32(ts + c, sc);
          tmem_wait_ld();
          if (!full) {
#pragma unroll
            for (int k = 0; k < 32; ++k)
              if (c + k > lim) sc[k] = 0xFF800000u;
          }
#pragma unroll
          for (int k = 0; k < 32; k += 8)
#pragma unroll
            for (int i = 0; i < 4; ++i)
              mx[i] = fmax3(mx[i], __uint_as_float(sc[k + 2 * i]), __uint_as_float(sc[k + 2 * i + 1]));
        }
        const float mt = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])), mn = mt * scale;
        // the first visible keys set the maximum (m = -inf before); later it moves by more than kRescaleLog2 only
        const bool move = mn > m + kRescaleLog2 || (m == -INFINITY && mn > m);
        const float corr = move ? ex2_ftz(m - mn) : 1.f;
        if (move) m = mn;
        const bool rescale = u > 0 && __any_sync(0xffffffffu, move);
        const float ms = m == -INFINITY ? 0.f : m;  // no visible key yet: weights 2^(-inf) = 0
        const float2 sc2 = make_float2(scale, scale), nm2 = make_float2(-ms, -ms);
        float2 acc0 = make_float2(0.f, 0.f), acc1 = make_float2(0.f, 0.f);
#pragma unroll 1
        for (int c = 0; c < kHalf; c += 32) {
          uint32_t sc[32], p[16];
          tmem_ld32(ts + c, sc);
          tmem_wait_ld();
          if (!full) {
#pragma unroll
            for (int k = 0; k < 32; ++k)
              if (c + k > lim) sc[k] = 0xFF800000u;
          }
#pragma unroll
          for (int k = 0; k < 32; k += 4) {
            const float2 v0 = make_float2(__uint_as_float(sc[k]), __uint_as_float(sc[k + 1]));
            const float2 v1 = make_float2(__uint_as_float(sc[k + 2]), __uint_as_float(sc[k + 3]));
            float2 x0 = ffma2(v0, sc2, nm2), x1 = ffma2(v1, sc2, nm2);
            x0 = make_float2(ex2_ftz(x0.x), ex2_ftz(x0.y));
            x1 = make_float2(ex2_ftz(x1.x), ex2_ftz(x1.y));
            acc0 = fadd2(acc0, x0);
            acc1 = fadd2(acc1, x1);
            p[k / 2] = pack_bf16(x0.x, x0.y);
            p[k / 2 + 1] = pack_bf16(x1.x, x1.y);
          }
          tmem_st16(ts + c / 2, p);
        }
        if (rescale) {  // O holds the halves before this one: once their last product has completed, move it
          if (!wait_all(&pv_done[X * 2 + (h ^ 1)], ((used >> (h ^ 1)) & 1) ^ 1, kErrWaitAccFull)) {
            ok = false;
            break;
          }
          tc_fence_after();
#pragma unroll 1
          for (int c = 0; c < D / 16; ++c) {  // rolled: rare, and the code of the roles competes for instruction cache
            uint32_t o[16];
            tmem_ld16(trow + C_O + X * D + c * 16, o);
            tmem_wait_ld();
#pragma unroll
            for (int k = 0; k < 16; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) * corr);
            tmem_st16(trow + C_O + X * D + c * 16, o);
          }
        }
        l = l * corr + (acc0.x + acc0.y) + (acc1.x + acc1.y);
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_full[X * 2 + h]);
      }
      if (!ok) break;
      if (nx > 0) {
        const uint32_t h = (nx - 1) & 1;
        ok = wait_all(&pv_done[X * 2 + h], ((used >> h) & 1) ^ 1, kErrWaitAccFull);
        if (!ok) break;
        tc_fence_after();
      }
      const int64_t at = (int64_t)(s.row0 + tok) * a.H + s.hk * G + r - tok * G;  // (packed row, head)
      const float inv = paged_inv(l);
      const int slot = 2 * blockIdx.x + (s.j0 > 0 ? 0 : 1);
      const int64_t prow = (int64_t)slot * 2 * kTileRows + X * kTileRows + row;
#pragma unroll 1
      for (int c = 0; c < D / 32; ++c) {
        uint32_t o[32];
        __syncwarp();
        if (nx > 0) {
          tmem_ld32(trow + C_O + X * D + c * 32, o);
          tmem_wait_ld();
        }
        if (l == 0.f) {  // nothing seen
#pragma unroll
          for (int k = 0; k < 32; ++k) o[k] = 0u;
        }
        if (live && s.whole) {
          uint4* dst = reinterpret_cast<uint4*>(a.o + at * D + c * 32);
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            float f[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) f[i] = __uint_as_float(o[8 * k + i]) * inv;
            dst[k] = make_uint4(pack_bf16(f[0], f[1]), pack_bf16(f[2], f[3]), pack_bf16(f[4], f[5]),
                                pack_bf16(f[6], f[7]));
          }
        } else if (live) {
          uint4* dst = reinterpret_cast<uint4*>(t.part + prow * D + c * 32);
#pragma unroll
          for (int k = 0; k < 8; ++k) dst[k] = make_uint4(o[4 * k], o[4 * k + 1], o[4 * k + 2], o[4 * k + 3]);
        }
      }
      tc_fence_before();
      __syncwarp();
      if (nx > 0 && lane == 0) mbar_arrive(&o_empty[X]);
      if (live) {
        if (s.whole)
          a.lse[at] = paged_lse(m, l);
        else
          *reinterpret_cast<float2*>(t.part + (int64_t)gridDim.x * 4 * kTileRows * D + prow * 2) = make_float2(m, l);
      }
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 12) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// Merges the pieces of the item cut by the start of CTA c = blockIdx.x + 1's share (Cut), in the order of the CTAs.
// blockIdx.y: 16 of its rows, a warp per row in turn.
template <int D>
__global__ void __launch_bounds__(256) paged_tiles_merge_kernel(const __grid_constant__ TileArgs t, int ctas) {
  constexpr int E = D / 32;
  const PagedAttnArgs& a = t.a;
  const int c = blockIdx.x + 1, warp = threadIdx.x >> 5, lane = threadIdx.x & 31, G = a.H / a.p.Hk;
  const int* cut = t.cuts + c * 8;
  const int row0 = cut[1], r0 = cut[2], rows = cut[3], hk = cut[4], last = cut[5];
  const float2* ml = reinterpret_cast<const float2*>(t.part + (int64_t)ctas * 4 * kTileRows * D);
  for (int i = warp; i < 16; i += 8) {
    const int row = blockIdx.y * 16 + i;
    if (row >= rows) break;
    float m = -INFINITY;
    for (int k = c - 1; k <= last; ++k) {
      if (k >= c && t.cuts[k * 8] >= t.cuts[k * 8 + 6]) continue;  // an empty share
      m = fmaxf(m, ml[(int64_t)(k < c ? 2 * k + 1 : 2 * k) * 2 * kTileRows + row].x);
    }
    float l = 0.f, acc[E];
#pragma unroll
    for (int e = 0; e < E; ++e) acc[e] = 0.f;
    for (int k = c - 1; k <= last; ++k) {
      if (k >= c && t.cuts[k * 8] >= t.cuts[k * 8 + 6]) continue;
      const int64_t at = (int64_t)(k < c ? 2 * k + 1 : 2 * k) * 2 * kTileRows + row;
      const float2 x = ml[at];
      if (paged_saw_nothing(x.x, x.y)) continue;
      const float f = ex2_ftz(x.x - m);
      l += x.y * f;
#pragma unroll
      for (int e = 0; e < E; ++e) acc[e] += t.part[at * D + lane * E + e] * f;
    }
    const float inv = paged_inv(l);
    const int r = r0 + row, tok = r / G;
    const int64_t at = (int64_t)(row0 + tok) * a.H + hk * G + r - tok * G;
#pragma unroll
    for (int e = 0; e < E; e += 2)
      *reinterpret_cast<uint32_t*>(a.o + at * D + lane * E + e) = pack_bf16(acc[e] * inv, acc[e + 1] * inv);
    if (lane == 0) a.lse[at] = paged_lse(m, l);
  }
}

template <int D, bool Q8>
static void launch_tiles(const TileArgs& t, int grid, cudaStream_t st) {
  static SmemAllowed allowed;
  allow_smem(paged_tiles_kernel<D, Q8>, Lay<D>::SMEM, allowed);
  const PagedPool& p = t.a.p;
  CUtensorMap mk{}, mv{};
  if (!Q8) {
    const int64_t page = 1ll << p.page_shift, z = (int64_t)p.pages * p.Hk;
    const int box = (int)std::min<int64_t>(kKeys, page);
    mk = make_tmap_bf16(p.k, D, page, z, D, page * D, 64, box);
    mv = make_tmap_bf16(p.v, D, page, z, D, page * D, 64, box);
  }
  paged_tiles_kernel<D, Q8><<<grid, kThreads, Lay<D>::SMEM, st>>>(mk, mv, t);
  NG_LAUNCH_CHECK();
}

void paged_tiles_launch(PagedAttnArgs a, cudaStream_t st) {
  const int G = a.H / a.p.Hk;
  a.row_tiles = (int)(((int64_t)a.max_new * G + 2 * kTileRows - 1) / (2 * kTileRows));
  TileArgs t{};
  const int64_t entries = (int64_t)a.B * a.row_tiles, tiles = ((int64_t)a.max_total + kKeys - 1) / kKeys;
  const int64_t most = entries * a.p.Hk * (tiles + kItemCost);  // bound of the whole cost
  TORCH_CHECK(entries * a.p.Hk <= INT32_MAX / 2, "paged: too many rows");
  t.entries = (int)entries;
  t.balanced = entries <= kMaxEntries && most <= INT32_MAX;
  // a CTA per SM, fewer where a share would fall below four key tiles
  const int grid = (int)std::max<int64_t>(1, std::min<int64_t>(kSMs, t.balanced ? most / 4 : entries * a.p.Hk));
  const bool cuts = t.balanced && tiles >= kCutTiles && grid > 1;
  at::Tensor part;
  if (cuts) {
    const int64_t floats = (int64_t)grid * 4 * kTileRows * (a.p.D + 2);
    part = at::empty({floats + grid * 8}, at::TensorOptions().device(at::kCUDA).dtype(at::kFloat));
    t.part = part.data_ptr<float>();
    t.cuts = reinterpret_cast<int*>(t.part + floats);
  }
  t.a = a;
  const bool q8 = a.p.ksf != nullptr;
  if (a.p.D == 128)
    q8 ? launch_tiles<128, true>(t, grid, st) : launch_tiles<128, false>(t, grid, st);
  else
    q8 ? launch_tiles<64, true>(t, grid, st) : launch_tiles<64, false>(t, grid, st);
  if (cuts) {
    const dim3 mg(grid - 1, 2 * kTileRows / 16);
    if (a.p.D == 128)
      paged_tiles_merge_kernel<128><<<mg, 256, 0, st>>>(t, grid);
    else
      paged_tiles_merge_kernel<64><<<mg, 256, 0, st>>>(t, grid);
    NG_LAUNCH_CHECK();
  }
}

}  // namespace ng
