// Gated projection and its gradients (sm_100a, tcgen05), bf16 or fp16:
//
//   g = x Wg^T, u = x Wu^T, h = act(g) * u
//   dg = dh * u * act'(g), du = dh * act(g);  dx = dg Wg + du Wu;  dWg = dg^T x, dWu = du^T x
//
// One persistent GEMM in three forms (products of matrix tiles, f32 accumulators in tensor memory, operands through a
// ring of shared-memory stages filled by tiled copies):
//   forward  an accumulator holds the same columns of g and u side by side (Wg's and Wu's rows are the two halves of the
//            tile's second operand; in a CTA pair each CTA loads one of them), so act(g) * u needs no exchange; x is read
//            once for both.  With gradients to come, g and u are stored too, in f32: rounded to the type they made the
//            gradients' error 1.8 times that of their own rounding, where the rounding of dg and du alone makes it 1.4 times
//            (4 M F bytes more to write and to read: 3 % of a 4096 x 3584 x 18944 step; computing them again: 4 M F K operations).
//   dx       the K loop runs over dg Wg, then du Wu, in one accumulator; the weights are read as they lie ([F, K]: the
//            second operand with its columns contiguous)
//   dW       both operands lie with their columns contiguous ([M, F] and [M, K]); nothing is transposed in memory
// Tiles of 256 x 256 by CTA pairs, of 128 x 256 or of 128 x 128 by single CTAs; what is left after whole rounds of tiles may be
// split along the sum, the parts added by a kernel behind (glu_plan).
#include <algorithm>
#include <cstring>

#include <cuda_fp16.h>

#include "common.cuh"
#include "kernels.h"
#include "pair.cuh"

namespace {
using namespace dfl;

enum { kForward = 0, kDx = 1, kDw = 2 };

constexpr int BM = 128, BK = 64;
constexpr int kEpiWarps = 8, kThreads = 64 + 32 * kEpiWarps;  // copies, products, then the results: two warps to a lane quarter
// CG: CTAs per tile (2: a pair).  A tile is 128 CG rows and BN accumulator columns; each CTA loads 128 rows of the first operand
// and BN / CG rows (or columns) of the second per stage.
template <int CG, int BN>
struct Cfg {
  static constexpr int kA = BM * BK * 2, kCols = BN / CG, kB = kCols * BK * 2, kStage = kA + kB;
  static constexpr int kStages = kStage > 32768 ? 4 : 6;
  static constexpr int kBarOff = kStages * kStage;
  static constexpr int kRowsOff = (kBarOff + (2 * kStages + 4) * 8 + 16 + 15) / 16 * 16;  // 32 x 33 16-bit values per epilogue warp
  static constexpr int kSmem = kRowsOff + kEpiWarps * 32 * 33 * 2 + 1024;
  static_assert(kSmem <= 232448, "shared memory budget");
};
constexpr int kChunk = 64 * BK * 2;  // 64 columns of an operand whose columns are contiguous
constexpr int kGroupM = 16;  // tile raster: 16 M blocks per group, for L2 reuse

struct GluParams {
  CUtensorMap a[2], b[2];
  void* d[2];        // outputs (forward: h; dW: one for each problem)
  float* g;          // forward: the kept projections
  float* u;
  long long ldd, lds;
  int M, N, K;       // of one problem: rows and columns of the output, length of the sums (of each segment)
  int num_m, num_n, tiles;  // tiles of one problem
  // Items: `whole` tiles, then the rest of them in `splits` parts each, whose sums go to ws [tile of the rest][part][row][column].
  int whole, splits, items;
  float* ws;
  int act;
};

template <bool F16>
DFL_DEVICE uint32_t pack2(float lo, float hi) {
  if constexpr (F16) {
    __half2 v = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<uint32_t*>(&v);
  } else {
    return pack_bf16x2(lo, hi);
  }
}
template <bool F16>
DFL_DEVICE float2 unpack2(uint32_t v) {
  if constexpr (F16) return __half22float2(*reinterpret_cast<__half2*>(&v));
  else return unpack_bf16x2(v);
}
template <bool F16>
DFL_DEVICE float load1(const void* p, long long i) {
  const uint16_t v = __ldcg(reinterpret_cast<const uint16_t*>(p) + i);
  if constexpr (F16) return __half2float(__ushort_as_half(v));
  else return __bfloat162float(__ushort_as_bfloat16(v));
}
template <bool F16>
DFL_DEVICE void store1(void* p, long long i, float v) {
  if constexpr (F16) reinterpret_cast<__half*>(p)[i] = __float2half_rn(v);
  else reinterpret_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(v);
}

// act(x) = x s(x), and its derivative s + x s'(x).  SiLU: s = 1 / (1 + e^-x).  GELU, tanh form:
// 0.5 (1 + tanh z) = 1 / (1 + e^-2z), z = sqrt(2 / pi) (x + 0.044715 x^3), which keeps the relative accuracy where
// the result is small.  Exact GELU: s = Phi(x) = erfc(-x / sqrt 2) / 2, s' = e^(-x^2 / 2) / sqrt(2 pi); with z = |x|,
// Phi(-z) = e^(-z^2 / 2) t p(t), t = 1 / (1 + 0.3 z), p of degree 7 fitted to least relative error over 0 <= z <= 14
// (1.5e-7; 4e-6 at z = 13, where the rounding of z^2 counts).  erfcf took 28 us where this takes 24 (1000 x 1024 x 2816, g and u kept).
DFL_DEVICE float sigmoid(float x) { return __fdividef(1.f, 1.f + __expf(-x)); }  // (2^126 < e^-x gives 0, as it should)
DFL_DEVICE float gelu_arg(float x) { return 1.5957691216057308f * x * (1.f + 0.044715f * x * x); }
DFL_DEVICE float2 normal(float x) {  // (Phi(x), e^(-x^2 / 2))
  const float z = fabsf(x), t = __fdividef(1.f, 1.f + 0.3f * z), e = __expf(-0.5f * z * z);
  float p = 0.035675063729286194f;
  p = fmaf(p, t, -0.15720424056053162f);
  p = fmaf(p, t, 0.20635543763637543f);
  p = fmaf(p, t, -0.05368535965681076f);
  p = fmaf(p, t, 0.12856251001358032f);
  p = fmaf(p, t, 0.09991323202848434f);
  p = fmaf(p, t, 0.12075399607419968f);
  p = fmaf(p, t, 0.11962929368019104f);
  const float low = e * t * p;
  return make_float2(x > 0.f ? 1.f - low : low, e);
}
template <int ACT>
DFL_DEVICE float act_of(float x) {
  if constexpr (ACT == kGluSilu) return x * sigmoid(x);
  if constexpr (ACT == kGluGelu) return x * sigmoid(gelu_arg(x));
  return x * normal(x).x;
}
template <int ACT>
DFL_DEVICE float2 act_grad(float x) {  // (act, act')
  if constexpr (ACT == kGluSilu) {
    const float s = sigmoid(x);
    return make_float2(x * s, s * (1.f + x * (1.f - s)));
  }
  if constexpr (ACT == kGluGelu) {
    const float s = sigmoid(gelu_arg(x));
    return make_float2(x * s, s * (1.f + x * (1.f - s) * 1.5957691216057308f * (1.f + 3.f * 0.044715f * x * x)));
  }
  const float2 n = normal(x);
  return make_float2(x * n.x, n.x + x * 0.3989422804014327f * n.y);
}

// K blocks [kb0, kb1) of split item `split`; a block is (segment, offset) in the two-segment sums of dx.
template <int MODE>
DFL_DEVICE int k_blocks(const GluParams& p) { return (p.K + BK - 1) / BK * (MODE == kDx ? 2 : 1); }

struct Tile {
  int which, mb, nb, kb0, kb1;
  int part;  // of the rest's sums, -1: the whole sum
};
template <int MODE>
DFL_DEVICE Tile tile_of(const GluParams& p, int t) {
  Tile r;
  const int n = k_blocks<MODE>(p);
  r.part = -1, r.kb0 = 0, r.kb1 = n;
  if (t >= p.whole && p.splits > 1) {
    r.part = t - p.whole;
    const int s = r.part % p.splits, per = (n + p.splits - 1) / p.splits;
    t = p.whole + r.part / p.splits;
    r.kb0 = min(n, s * per), r.kb1 = min(n, r.kb0 + per);
  }
  r.which = t / p.tiles;
  t -= r.which * p.tiles;
  const int group = t / (kGroupM * p.num_n), first = group * kGroupM, gm = min(kGroupM, p.num_m - first);
  t -= group * kGroupM * p.num_n;
  r.mb = first + t % gm, r.nb = t / gm;
  return r;
}

// A whole 32-byte sector at once: a row a lane, stores of 16 bytes would write every sector twice.
DFL_DEVICE void st_sector(void* p, uint32_t a, uint32_t b, uint32_t c, uint32_t d, uint32_t e, uint32_t f, uint32_t g, uint32_t h) {
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(a), "r"(b), "r"(c), "r"(d), "r"(e), "r"(f), "r"(g), "r"(h)
               : "memory");
}

// 32 columns of the rows of a warp (lane: row): whole 16-byte pieces where every row allows it, else through shared memory, so that
// the lanes write along a row (a row each would cost a line per lane and value).
template <bool F16>
DFL_DEVICE void store_cols(void* base, long long row0, int rows, long long ld, int col, const float (&v)[32], int cols, bool wide,
                           uint16_t (*stage)[33]) {
  const int lane = threadIdx.x % 32;
  uint32_t w[16];
#pragma unroll
  for (int q = 0; q < 16; ++q) w[q] = pack2<F16>(v[2 * q], v[2 * q + 1]);
  if (wide && cols >= 32) {
    uint16_t* d = reinterpret_cast<uint16_t*>(base) + (row0 + lane) * ld + col;
    if (lane >= rows) return;
    if (ld % 16 == 0 && (reinterpret_cast<uintptr_t>(base) & 31) == 0) {
#pragma unroll
      for (int q = 0; q < 2; ++q)
        st_sector(d + 16 * q, w[8 * q], w[8 * q + 1], w[8 * q + 2], w[8 * q + 3], w[8 * q + 4], w[8 * q + 5], w[8 * q + 6], w[8 * q + 7]);
    } else {
#pragma unroll
      for (int q = 0; q < 4; ++q) reinterpret_cast<uint4*>(d)[q] = make_uint4(w[4 * q], w[4 * q + 1], w[4 * q + 2], w[4 * q + 3]);
    }
    return;
  }
  __syncwarp();
#pragma unroll
  for (int q = 0; q < 16; ++q) stage[lane][2 * q] = (uint16_t)w[q], stage[lane][2 * q + 1] = (uint16_t)(w[q] >> 16);
  __syncwarp();
  uint16_t* d = reinterpret_cast<uint16_t*>(base) + row0 * ld + col + lane;
  if (lane < cols)
    for (int r = 0; r < rows; ++r) d[r * ld] = stage[r][lane];
}

DFL_DEVICE void keep_cols(float* d, const float (&v)[32], int cols) {  // (rows are 32-byte aligned)
  if (cols >= 32) {
#pragma unroll
    for (int q = 0; q < 4; ++q)
      st_sector(d + 8 * q, __float_as_uint(v[8 * q]), __float_as_uint(v[8 * q + 1]), __float_as_uint(v[8 * q + 2]),
                __float_as_uint(v[8 * q + 3]), __float_as_uint(v[8 * q + 4]), __float_as_uint(v[8 * q + 5]),
                __float_as_uint(v[8 * q + 6]), __float_as_uint(v[8 * q + 7]));
  } else {
#pragma unroll
    for (int j = 0; j < 32; ++j)
      if (j < cols) d[j] = v[j];
  }
}

template <int CG>
DFL_DEVICE void load_tile(uint8_t* dst, const CUtensorMap* map, uint64_t* bar, int c0, int c1) {
  if constexpr (CG == 2) tma_load_2d_pair(dst, map, bar, c0, c1);
  else tma_load_2d(dst, map, bar, c0, c1);
}

template <int MODE, int CG, int BN, bool F16>
__global__ void __launch_bounds__(kThreads, 1) glu_kernel(const __grid_constant__ GluParams p, int* err) {
  using C = Cfg<CG, BN>;
  constexpr int STAGES = C::kStages;
  constexpr uint32_t kTmemCols = 2 * BN;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* full_bar = reinterpret_cast<uint64_t*>(smem + C::kBarOff);
  uint64_t* empty_bar = full_bar + STAGES;
  uint64_t* tfull_bar = empty_bar + STAGES;
  uint64_t* tempty_bar = tfull_bar + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(tempty_bar + 2);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const uint32_t rank = CG == 2 ? cluster_rank() : 0u;
  const int first = blockIdx.x / CG, step = gridDim.x / CG;
  const int items = p.items;

  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(&full_bar[s], 1);   // CTA 0's producer posts the bytes of all
      mbar_init(&empty_bar[s], 1);  // the issuing thread's commit, to every CTA of the tile
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(&tfull_bar[a], 1);
      mbar_init(&tempty_bar[a], 32 * kEpiWarps * CG);  // (CTA 0's copy is the one used)
    }
    *abort_flag = 0;
    fence_barrier_init();
    fence_proxy_async_shared();
    prefetch_tmap(&p.a[0]);
    prefetch_tmap(&p.b[0]);
  }
  if (warp == 1) {
    if constexpr (CG == 2) {
      asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)),
                   "r"(kTmemCols));
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;");
    } else {
      tmem_alloc(tmem_slot, kTmemCols);
      tmem_relinquish();
    }
  }
  tc_fence_before();
  __syncthreads();
  if constexpr (CG == 2) cluster_sync();  // both CTAs' barriers exist before any remote traffic
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  griddep_wait();  // (launched while the kernel before it ends)

  if (warp == 0) {
    if (lane == 0) {
      int stage = 0;
      uint32_t phase = 0, issued_par = 0;  // a bit per stage: parity of its last copy
      int issued = 0;
      bool ok = true;
      for (int t = first; t < items && ok; t += step) {
        const Tile it = tile_of<MODE>(p, t);
        for (int kb = it.kb0; kb < it.kb1; ++kb) {
          if (!mbar_wait(&empty_bar[stage], phase ^ 1u, err, kKidGlu, 10 + stage, abort_flag)) {
            ok = false;
            break;
          }
          uint8_t* sa = smem + stage * C::kStage;
          uint8_t* sb = sa + C::kA;
          uint64_t* bar = &full_bar[stage];
          if (rank == 0) mbar_arrive_expect_tx(bar, CG * C::kStage);
          const int m0 = it.mb * BM * CG + (int)rank * BM;
          if constexpr (MODE == kForward) {
            load_tile<CG>(sa, &p.a[0], bar, kb * BK, m0);
            const int n0 = it.nb * (BN / 2);
            if constexpr (CG == 2) {  // rank 0: rows of Wg, rank 1: of Wu
              load_tile<CG>(sb, &p.b[rank], bar, kb * BK, n0);
            } else {
              load_tile<CG>(sb, &p.b[0], bar, kb * BK, n0);
              load_tile<CG>(sb + C::kB / 2, &p.b[1], bar, kb * BK, n0);
            }
          } else if constexpr (MODE == kDx) {
            const int half = (p.K + BK - 1) / BK, seg = kb >= half, k0 = (kb - seg * half) * BK;
            load_tile<CG>(sa, &p.a[seg], bar, k0, m0);
#pragma unroll
            for (int c = 0; c < C::kCols / 64; ++c)
              load_tile<CG>(sb + c * kChunk, &p.b[seg], bar, it.nb * BN + (int)rank * C::kCols + 64 * c, k0);
          } else {
            load_tile<CG>(sa, &p.a[it.which], bar, m0, kb * BK);
            load_tile<CG>(sa + kChunk, &p.a[it.which], bar, m0 + 64, kb * BK);
#pragma unroll
            for (int c = 0; c < C::kCols / 64; ++c)
              load_tile<CG>(sb + c * kChunk, &p.b[0], bar, it.nb * BN + (int)rank * C::kCols + 64 * c, kb * BK);
          }
          issued |= 1 << stage;
          issued_par = (issued_par & ~(1u << stage)) | (phase << stage);
          if (++stage == STAGES) {
            stage = 0;
            phase ^= 1u;
          }
        }
      }
      if (!ok && rank == 0)  // given up: the copies in flight must land before the CTAs exit
        for (int s = 0; s < STAGES; ++s)
          if ((issued >> s) & 1) mbar_wait(&full_bar[s], (issued_par >> s) & 1u, nullptr, 0, 0, nullptr, 200000000LL);
    }
  } else if (warp == 1) {
    if (lane == 0 && rank == 0) {
      constexpr bool a_mn = MODE == kDw, b_mn = MODE != kForward;
      constexpr uint32_t kF16Bits = F16 ? (1u << 7) | (1u << 10) : 0u;  // clears the two bf16 format bits
      constexpr uint32_t idesc = make_idesc_bf16_f32(BM * CG, BN, a_mn, b_mn) & ~kF16Bits;
      // K-major: rows of 64 K values, 16 of them 32 bytes apart.  MN-major: chunks of 64 columns, 64 rows of K each;
      // 16 rows are 2048 bytes.
      auto desc = [](uint32_t addr, int k, bool mn) {
        return mn ? make_sdesc_sw128(addr + k * 2048, kChunk, 1024) : make_sdesc_sw128(addr + k * 32, 16, 1024);
      };
      int stage = 0, acc = 0;
      uint32_t phase = 0, acc_phase = 0;
      bool ok = true;
      for (int t = first; t < items && ok; t += step) {
        const Tile it = tile_of<MODE>(p, t);
        if (!mbar_wait(&tempty_bar[acc], acc_phase ^ 1u, err, kKidGlu, 20 + acc, abort_flag)) break;
        tc_fence_after();
        const uint32_t d_tmem = tmem_base + acc * BN;
        for (int kb = it.kb0; kb < it.kb1; ++kb) {
          if (!mbar_wait(&full_bar[stage], phase, err, kKidGlu, 30 + stage, abort_flag)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const uint32_t a_addr = smem_u32(smem + stage * C::kStage), b_addr = a_addr + C::kA;
#pragma unroll
          for (int k = 0; k < BK / 16; ++k) {
            const uint32_t more = (kb > it.kb0 || k > 0) ? 1u : 0u;
            if constexpr (CG == 2) umma_f16_pair(d_tmem, desc(a_addr, k, a_mn), desc(b_addr, k, b_mn), idesc, more);
            else umma_f16_ss(d_tmem, desc(a_addr, k, a_mn), desc(b_addr, k, b_mn), idesc, more);
          }
          if constexpr (CG == 2) umma_commit_pair(&empty_bar[stage]);
          else umma_commit(&empty_bar[stage]);
          if (++stage == STAGES) {
            stage = 0;
            phase ^= 1u;
          }
        }
        if (!ok) break;
        if constexpr (CG == 2) umma_commit_pair(&tfull_bar[acc]);
        else umma_commit(&tfull_bar[acc]);
        acc ^= 1;
        if (acc == 0) acc_phase ^= 1u;
      }
    }
  } else {
    const int sub = warp & 3;  // the tensor-memory lane quarter that this warp may read
    const int half = (warp - 2) / 4;  // of the tile's columns
    uint16_t(*stage_rows)[33] = reinterpret_cast<uint16_t(*)[33]>(smem + C::kRowsOff) + 32 * (warp - 2);
    int acc = 0;
    uint32_t acc_phase = 0;
    for (int t = first; t < items; t += step) {
      const Tile it = tile_of<MODE>(p, t);
      if (!mbar_wait_warp(&tfull_bar[acc], acc_phase, err, kKidGlu, 40 + acc, abort_flag)) break;
      tc_fence_after();
      const int row = it.mb * BM * CG + (int)rank * BM + sub * 32 + lane;
      const uint32_t tbase = tmem_base + ((uint32_t)(sub * 32) << 16) + acc * BN;
      auto release = [&]() {
        tc_fence_before();
        if (CG == 1 || rank == 0) mbar_arrive(&tempty_bar[acc]);
        else mbar_arrive_cta0(&tempty_bar[acc]);
      };
      const int row0 = row - lane, rows = min(32, p.M - row0);  // the warp's
      if (it.part >= 0) {  // sums of a part: the whole tile, whatever lies outside
        float* part = p.ws + (long long)it.part * (BM * CG * BN) + ((int)rank * BM + sub * 32 + lane) * BN;
#pragma unroll 1
        for (int c = half * (BN / 2); c < (half + 1) * (BN / 2); c += 32) {
          uint32_t r[32];
          tmem_ld_32x32b_x32(tbase + c, r);
          tmem_wait_ld();
          if (c + 32 == (half + 1) * (BN / 2)) release();
#pragma unroll
          for (int q = 0; q < 4; ++q)
            st_sector(part + c + 8 * q, r[8 * q], r[8 * q + 1], r[8 * q + 2], r[8 * q + 3], r[8 * q + 4], r[8 * q + 5], r[8 * q + 6], r[8 * q + 7]);
        }
      } else if constexpr (MODE == kForward) {
        const bool wide = p.ldd % 8 == 0 && (reinterpret_cast<uintptr_t>(p.d[0]) & 15) == 0;
#pragma unroll 1
        for (int c = half * (BN / 4); c < (half + 1) * (BN / 4); c += 32) {
          uint32_t gr[32], ur[32];
          tmem_ld_32x32b_x32(tbase + c, gr);
          tmem_ld_32x32b_x32(tbase + BN / 2 + c, ur);
          tmem_wait_ld();
          if (c + 32 == (half + 1) * (BN / 4)) release();
          const int col = it.nb * (BN / 2) + c, cols = p.N - col;
          if (rows <= 0 || cols <= 0) continue;
          float g[32], u[32];
#pragma unroll
          for (int j = 0; j < 32; ++j) g[j] = __uint_as_float(gr[j]), u[j] = __uint_as_float(ur[j]);
          if (p.g) {
            if (lane < rows) {
              keep_cols(p.g + row * p.lds + col, g, cols);
              keep_cols(p.u + row * p.lds + col, u, cols);
            }
          }
          if (p.act == kGluSilu) {
#pragma unroll
            for (int j = 0; j < 32; ++j) u[j] *= act_of<kGluSilu>(g[j]);
          } else if (p.act == kGluGelu) {
#pragma unroll
            for (int j = 0; j < 32; ++j) u[j] *= act_of<kGluGelu>(g[j]);
          } else {
#pragma unroll
            for (int j = 0; j < 32; ++j) u[j] *= act_of<kGluGeluErf>(g[j]);
          }
          store_cols<F16>(p.d[0], row0, rows, p.ldd, col, u, cols, wide, stage_rows);
        }
      } else {
#pragma unroll 1
        for (int c = half * (BN / 2); c < (half + 1) * (BN / 2); c += 32) {
          uint32_t r[32];
          tmem_ld_32x32b_x32(tbase + c, r);
          tmem_wait_ld();
          if (c + 32 == (half + 1) * (BN / 2)) release();
          const int col = it.nb * BN + c, cols = p.N - col;
          if (rows <= 0 || cols <= 0) continue;
          float v[32];
#pragma unroll
          for (int j = 0; j < 32; ++j) v[j] = __uint_as_float(r[j]);
          store_cols<F16>(p.d[it.which], row0, rows, p.ldd, col, v, cols, true, stage_rows);
        }
      }
      acc ^= 1;
      if (acc == 0) acc_phase ^= 1u;
    }
  }

  tc_fence_before();
  __syncthreads();
  if constexpr (CG == 2) cluster_sync();  // no remote arrive or load is in flight towards a CTA that leaves
  tc_fence_after();
  if (warp == 1) {
    if constexpr (CG == 2)
      asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(kTmemCols));
    else
      tmem_dealloc(tmem_base, kTmemCols);
  }
}

// ---------------------------------------------------------------------------
// Few rows: bound by reading both weights once (4 F K bytes).  A CTA of 8 warps owns 16 output columns; its warps take 128-wide
// pieces of K in turn and multiply on the warp-level m16n8k16 instruction, the weights' rows as the 16-row operand
// straight from global memory (both operands in the same permuted K order, so that a lane loads 16 contiguous bytes).  The
// warps' sums are added in their order.
// ---------------------------------------------------------------------------
constexpr int kRowsMax = 32;

template <bool F16>
DFL_DEVICE void mma16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  if constexpr (F16)
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
  else
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// (launched while the kernel before ends: what that writes is read past L1)
DFL_DEVICE uint4 ld_once(const uint16_t* p) { return __ldcg(reinterpret_cast<const uint4*>(p)); }

// NB: groups of 8 rows.
template <int NB, bool F16>
__global__ void __launch_bounds__(256, NB == 4 ? 1 : 2) glu_rows_kernel(GluArgs a) {
  constexpr int U = NB == 4 ? 2 : 4;  // pieces of 32 K values in flight
  __shared__ float red[8][2][16][8 * NB + 1];
  griddep_wait();
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, quad = lane / 4, t = lane % 4;
  const int n0 = blockIdx.x * 16, r0 = min(n0 + quad, a.F - 1), r1 = min(n0 + quad + 8, a.F - 1);
  const uint16_t* w[4] = {reinterpret_cast<const uint16_t*>(a.wg) + r0 * a.ldwg, reinterpret_cast<const uint16_t*>(a.wg) + r1 * a.ldwg,
                          reinterpret_cast<const uint16_t*>(a.wu) + r0 * a.ldwu, reinterpret_cast<const uint16_t*>(a.wu) + r1 * a.ldwu};
  const uint16_t* x = reinterpret_cast<const uint16_t*>(a.x);
  float c[2][NB][4];
#pragma unroll
  for (int s = 0; s < 2; ++s)
#pragma unroll
    for (int g = 0; g < NB; ++g) c[s][g][0] = c[s][g][1] = c[s][g][2] = c[s][g][3] = 0.f;
  const uint4 zero = make_uint4(0u, 0u, 0u, 0u);
  for (int k0 = warp * 32 * U; k0 < a.K; k0 += 8 * 32 * U) {
    uint4 v[U][4], b[U][NB];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int k = k0 + 32 * u + 8 * t;  // K is a multiple of 8: a lane's piece is inside or outside
#pragma unroll
      for (int i = 0; i < 4; ++i) v[u][i] = k < a.K ? ld_once(w[i] + k) : zero;
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int k = k0 + 32 * u + 8 * t;
#pragma unroll
      for (int g = 0; g < NB; ++g)
        b[u][g] = k < a.K && 8 * g + quad < a.M ? __ldcg(reinterpret_cast<const uint4*>(x + (8 * g + quad) * a.ldx + k)) : zero;
    }
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int g = 0; g < NB; ++g)
#pragma unroll
        for (int s = 0; s < 2; ++s) {
          mma16816<F16>(c[s][g], v[u][2 * s].x, v[u][2 * s + 1].x, v[u][2 * s].y, v[u][2 * s + 1].y, b[u][g].x, b[u][g].y);
          mma16816<F16>(c[s][g], v[u][2 * s].z, v[u][2 * s + 1].z, v[u][2 * s].w, v[u][2 * s + 1].w, b[u][g].z, b[u][g].w);
        }
  }
  // c[s][g][2 i + e]: column quad + 8 i of the gate (s = 0) or the other projection, row 8 g + 2 t + e
#pragma unroll
  for (int s = 0; s < 2; ++s)
#pragma unroll
    for (int g = 0; g < NB; ++g)
#pragma unroll
      for (int i = 0; i < 4; ++i) red[warp][s][quad + 8 * (i / 2)][8 * g + 2 * t + i % 2] = c[s][g][i];
  __syncthreads();
  const int n = threadIdx.x % 16, col = n0 + n;
  if (col >= a.F) return;
  for (int m = threadIdx.x / 16; m < a.M; m += 16) {
    float g = 0.f, u = 0.f;
#pragma unroll
    for (int k = 0; k < 8; ++k) g += red[k][0][n][m], u += red[k][1][n][m];
    if (a.g) a.g[m * a.lds + col] = g, a.u[m * a.lds + col] = u;
    const float v = a.act == kGluSilu ? act_of<kGluSilu>(g) : a.act == kGluGelu ? act_of<kGluGelu>(g) : act_of<kGluGeluErf>(g);
    store1<F16>(a.h, m * a.ldh + col, v * u);
  }
}

template <bool F16>
int launch_rows(const GluArgs* a, cudaStream_t stream) {
  const auto kern = a->M <= 8 ? glu_rows_kernel<1, F16> : a->M <= 16 ? glu_rows_kernel<2, F16> : glu_rows_kernel<4, F16>;
  return (int)dfl_host::launch_early(kern, (unsigned)((a->F + 15) / 16), 256, 0, stream, *a);
}

// The rest's tiles from their parts, added in order: a thread takes 4 columns of a row.  (A block stays within a tile.)
template <int MODE, int ROWS, int BN, bool F16>
__global__ void __launch_bounds__(256) glu_join_kernel(const __grid_constant__ GluParams p) {
  griddep_wait();
  constexpr int kCols = MODE == kForward ? BN / 2 : BN, kQuads = kCols / 4, kBlocks = ROWS * kQuads / 256;
  constexpr int kTile = ROWS * BN;
  const int t = blockIdx.x / kBlocks, i = blockIdx.x % kBlocks * 256 + threadIdx.x, r = i / kQuads, q = i % kQuads * 4;
  const Tile it = tile_of<MODE>(p, p.whole + t * p.splits);
  const int row = it.mb * ROWS + r, col = it.nb * kCols + q;
  if (row >= p.M || col >= p.N) return;
  const float* from = p.ws + (long long)t * p.splits * kTile + r * BN + q;
  float v[2][4] = {};
#pragma unroll 4
  for (int s = 0; s < p.splits; ++s)
#pragma unroll
    for (int h = 0; h < (MODE == kForward ? 2 : 1); ++h) {
      const float4 x = __ldcg(reinterpret_cast<const float4*>(from + (long long)s * kTile + h * kCols));
      v[h][0] += x.x, v[h][1] += x.y, v[h][2] += x.z, v[h][3] += x.w;
    }
  if constexpr (MODE == kForward) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if (col + e >= p.N) break;
      const float g = v[0][e], u = v[1][e];
      if (p.g) p.g[row * p.lds + col + e] = g, p.u[row * p.lds + col + e] = u;
      const float a = p.act == kGluSilu ? act_of<kGluSilu>(g) : p.act == kGluGelu ? act_of<kGluGelu>(g) : act_of<kGluGeluErf>(g);
      store1<F16>(p.d[0], row * p.ldd + col + e, a * u);
    }
  } else {  // (N and the rows' pitch are multiples of 8)
    *reinterpret_cast<uint2*>(reinterpret_cast<uint16_t*>(p.d[it.which]) + row * p.ldd + col) =
        make_uint2(pack2<F16>(v[0][0], v[0][1]), pack2<F16>(v[0][2], v[0][3]));
  }
}

// dg, du: 8 columns a thread.  Bound by its bytes (14 M F): 4096 x 18944 169 us, 6.4 TB/s.
template <bool F16, int ACT>
__global__ void __launch_bounds__(256) glu_grad_kernel(GluGradArgs a) {
  griddep_wait();
  const int per_row = (a.F + 7) / 8;
  const long long n = a.M * per_row;
  const bool wide = a.lddh % 8 == 0 && (reinterpret_cast<uintptr_t>(a.dh) & 15) == 0;
  for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < n; i += (long long)gridDim.x * 256) {
    const long long row = i / per_row;
    const int col = (int)(i - row * per_row) * 8, cols = min(8, a.F - col);
    const long long at = row * a.lds + col;
    // (the rows of g, u, dg and du are padded to whole pieces)
    float g[8], u[8], d[8];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const float4 x = __ldcg(reinterpret_cast<const float4*>(a.g + at) + h), y = __ldcg(reinterpret_cast<const float4*>(a.u + at) + h);
      g[4 * h] = x.x, g[4 * h + 1] = x.y, g[4 * h + 2] = x.z, g[4 * h + 3] = x.w;
      u[4 * h] = y.x, u[4 * h + 1] = y.y, u[4 * h + 2] = y.z, u[4 * h + 3] = y.w;
    }
    if (wide && cols == 8) {
      const uint4 dv = __ldcg(reinterpret_cast<const uint4*>(reinterpret_cast<const uint16_t*>(a.dh) + row * a.lddh + col));
      const uint32_t w[4] = {dv.x, dv.y, dv.z, dv.w};
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float2 f = unpack2<F16>(w[e]);
        d[2 * e] = f.x, d[2 * e + 1] = f.y;
      }
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) d[e] = e < cols ? load1<F16>(a.dh, row * a.lddh + col + e) : 0.f;
    }
    uint32_t og[4], ou[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float2 x = act_grad<ACT>(g[2 * e]), y = act_grad<ACT>(g[2 * e + 1]);
      og[e] = pack2<F16>(d[2 * e] * u[2 * e] * x.y, d[2 * e + 1] * u[2 * e + 1] * y.y);
      ou[e] = pack2<F16>(d[2 * e] * x.x, d[2 * e + 1] * y.x);
    }
    *reinterpret_cast<uint4*>(reinterpret_cast<uint16_t*>(a.dg) + at) = make_uint4(og[0], og[1], og[2], og[3]);
    *reinterpret_cast<uint4*>(reinterpret_cast<uint16_t*>(a.du) + at) = make_uint4(ou[0], ou[1], ou[2], ou[3]);
  }
}

bool al16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// How a product is laid out.  Per K block an SM needs (cycles): a pair's 256 x 256 tile 560 (its products: 524), a 128 x 256 tile
// 750 and a 128 x 128 tile 512 (both bound by the copies: 48 and 32 KB); a tile's results 2500, or 1250, beside the next
// tile's products.  What is left after whole rounds is split along the sum where that is shorter: every part of a tile costs
// its sums' way through L2, the join a launch.
struct Plan {
  int cg, bn, whole, splits;
};
template <int MODE>
Plan glu_plan(long long rows, long long cols, int problems, int blocks, int sms) {
  struct Shape {
    int cg, bn;
    double block;
  };
  constexpr Shape shapes[3] = {{2, 256, 560.}, {1, 256, 750.}, {1, 128, 512.}};
  Plan best{};
  double least = 0.;
  for (const Shape& s : shapes) {
    const int width = MODE == kForward ? s.bn / 2 : s.bn;
    const long long tiles = (rows + 128 * s.cg - 1) / (128 * s.cg) * ((cols + width - 1) / width) * problems, slots = sms / s.cg;
    const long long rounds = tiles / slots, rest = tiles % slots;
    const auto take = [&](long long whole, int splits, double cost) {
      if (best.cg == 0 || cost < least) best = Plan{s.cg, s.bn, (int)whole, splits}, least = cost;
    };
    const double results = s.bn * 10., whole = std::max(blocks * s.block, results);
    take(tiles, 1, (rounds + (rest > 0)) * whole + results);
    if (rest == 0) continue;
    for (int n = 2; n <= slots / rest && blocks / n >= 4 && n <= 32; ++n)
      if ((n - 1) * ((blocks + n - 1) / n) < blocks)  // (every part holds something)
        take(rounds * slots, n, rounds * whole + (blocks + n - 1) / n * s.block + results + 6000. + rest * n * 128. * s.cg * s.bn * 8 / 2600.);
  }
  return best;
}

template <int MODE>
int setup(GluParams& p, const Plan& plan, int problems) {
  const long long width = MODE == kForward ? plan.bn / 2 : plan.bn, m = ((long long)p.M + 128 * plan.cg - 1) / (128 * plan.cg),
                  n = (p.N + width - 1) / width;
  if (m * n * problems > (1 << 28)) return -9;
  p.num_m = (int)m, p.num_n = (int)n, p.tiles = (int)(m * n);
  p.whole = plan.whole, p.splits = plan.splits;
  p.items = p.whole + (p.tiles * problems - p.whole) * p.splits;
  return 0;
}
long long ws_floats(const Plan& plan, long long items) {
  return plan.splits > 1 ? (items - plan.whole) * 128ll * plan.cg * plan.bn : 0;
}

template <int MODE, int CG, int BN, bool F16>
int launch_glu(const GluParams& p, int sms, int dev, int* err, cudaStream_t stream) {
  auto kern = glu_kernel<MODE, CG, BN, F16>;
  constexpr int smem = Cfg<CG, BN>::kSmem;
  static bool attr[16] = {false};
  if (!attr[dev & 15]) {
    const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return (int)e;
    attr[dev & 15] = true;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(CG * std::min(p.items, sms / CG)), 1, 1);
  cfg.blockDim = dim3(kThreads, 1, 1);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  at[1].id = cudaLaunchAttributeClusterDimension;
  at[1].val.clusterDim.x = CG;
  at[1].val.clusterDim.y = at[1].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = CG == 2 ? 2 : 1;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, kern, p, err);
  if (e != cudaSuccess || p.splits == 1) return (int)e;
  const int rest = (p.items - p.whole) / p.splits;
  constexpr int rows = BM * CG, blocks = rows * (MODE == kForward ? BN / 8 : BN / 4) / 256;
  return (int)dfl_host::launch_early(glu_join_kernel<MODE, rows, BN, F16>, (unsigned)(rest * blocks), 256, 0, stream, p);
}

template <int MODE>
int launch_mode(const GluParams& p, const Plan& plan, int f16, int sms, int dev, int* err, cudaStream_t stream) {
  if (p.splits > 1 && !p.ws) return -10;
  if (plan.cg == 2) return f16 ? launch_glu<MODE, 2, 256, true>(p, sms, dev, err, stream) : launch_glu<MODE, 2, 256, false>(p, sms, dev, err, stream);
  if (plan.bn == 256) return f16 ? launch_glu<MODE, 1, 256, true>(p, sms, dev, err, stream) : launch_glu<MODE, 1, 256, false>(p, sms, dev, err, stream);
  return f16 ? launch_glu<MODE, 1, 128, true>(p, sms, dev, err, stream) : launch_glu<MODE, 1, 128, false>(p, sms, dev, err, stream);
}

int blocks_of(int K) { return (K + BK - 1) / BK; }
Plan plan_forward(int M, int K, int F, int sms) { return glu_plan<kForward>(M, F, 1, blocks_of(K), sms); }
Plan plan_dx(int M, int K, int F, int sms) { return glu_plan<kDx>(M, K, 1, 2 * blocks_of(F), sms); }
Plan plan_dw(int M, int K, int F, int problems, int sms) { return glu_plan<kDw>(F, K, problems, blocks_of(M), sms); }

}  // namespace

// Floats that a call's parts take; what: 0 forward, 1 dx, 2 dW of both weights, 3 of one.
extern "C" long long dfl_glu_ws(int what, int M, int K, int F) {
  int dev = 0;
  cudaGetDevice(&dev);
  const int sms = dfl_host::num_sms(dev);
  if (what == 0 && M <= kRowsMax) return 0;
  const Plan plan = what == 0 ? plan_forward(M, K, F, sms) : what == 1 ? plan_dx(M, K, F, sms) : plan_dw(M, K, F, what == 2 ? 2 : 1, sms);
  GluParams p{};
  p.M = what >= 2 ? F : M, p.N = what == 0 ? F : K;
  const int rc = what == 0 ? setup<kForward>(p, plan, 1) : what == 1 ? setup<kDx>(p, plan, 1) : setup<kDw>(p, plan, what == 2 ? 2 : 1);
  return rc ? 0 : ws_floats(plan, p.items);
}

extern "C" int dfl_glu(const GluArgs* a, cudaStream_t stream) {
  if (a->M <= 0 || a->F <= 0 || a->K <= 0 || a->K % 8 || a->act < 0 || a->act > kGluGeluErf) return -2;
  if (!al16(a->x) || !al16(a->wg) || !al16(a->wu) || (a->ldx | a->ldwg | a->ldwu) % 8) return -3;
  auto al32 = [](const void* q) { return (reinterpret_cast<uintptr_t>(q) & 31) == 0; };
  if (a->g && (!a->u || !al32(a->g) || !al32(a->u) || a->lds % 8 || a->lds < a->F)) return -4;
  if (a->M <= kRowsMax) return a->f16 ? launch_rows<true>(a, stream) : launch_rows<false>(a, stream);
  int dev = 0;
  cudaGetDevice(&dev);
  const int sms = dfl_host::num_sms(dev);
  const Plan plan = plan_forward(a->M, a->K, a->F, sms);
  GluParams p;
  std::memset(&p, 0, sizeof(p));
  int rc = dfl_host::make_tmap_2d_bf16(&p.a[0], a->x, a->K, a->M, a->ldx, BK, BM, true);
  if (rc) return 1000 + rc;
  rc = dfl_host::make_tmap_2d_bf16(&p.b[0], a->wg, a->K, a->F, a->ldwg, BK, plan.bn / 2, true);
  if (rc) return 2000 + rc;
  rc = dfl_host::make_tmap_2d_bf16(&p.b[1], a->wu, a->K, a->F, a->ldwu, BK, plan.bn / 2, true);
  if (rc) return 3000 + rc;
  p.d[0] = a->h, p.ldd = a->ldh;
  p.g = a->g, p.u = a->u, p.lds = a->lds;
  p.M = a->M, p.N = a->F, p.K = a->K, p.act = a->act;
  rc = setup<kForward>(p, plan, 1);
  if (rc) return rc;
  if (ws_floats(plan, p.items) > a->ws_floats || (reinterpret_cast<uintptr_t>(a->ws) & 31)) return -10;
  p.ws = a->ws;
  return launch_mode<kForward>(p, plan, a->f16, sms, dev, a->err, stream);
}

extern "C" int dfl_glu_grad(const GluGradArgs* a, cudaStream_t stream) {
  if (a->M <= 0 || a->F <= 0 || a->act < 0 || a->act > kGluGeluErf) return -2;
  if (!al16(a->g) || !al16(a->u) || !al16(a->dg) || !al16(a->du) || a->lds % 8 || a->lds < a->F) return -4;
  const long long n = a->M * ((a->F + 7) / 8), blocks = (n + 255) / 256;
  const unsigned grid = (unsigned)std::min<long long>(blocks, 148 * 16);
  auto kern = a->f16 ? (a->act == kGluSilu ? glu_grad_kernel<true, kGluSilu> : a->act == kGluGelu ? glu_grad_kernel<true, kGluGelu>
                                                                                             : glu_grad_kernel<true, kGluGeluErf>)
                     : (a->act == kGluSilu ? glu_grad_kernel<false, kGluSilu> : a->act == kGluGelu ? glu_grad_kernel<false, kGluGelu>
                                                                                              : glu_grad_kernel<false, kGluGeluErf>);
  return (int)dfl_host::launch_early(kern, grid, 256, 0, stream, *a);
}

static int check_gemm(const GluGemmArgs* a) {
  if (a->M <= 0 || a->F <= 0 || a->K <= 0 || a->K % 8) return -2;
  if (!al16(a->dg) || !al16(a->du) || a->lds % 8 || a->lds < a->F) return -4;
  return 0;
}

extern "C" int dfl_glu_dx(const GluGemmArgs* a, cudaStream_t stream) {
  int rc = check_gemm(a);
  if (rc) return rc;
  if (!al16(a->wg) || !al16(a->wu) || !al16(a->dx) || (a->ldwg | a->ldwu) % 8) return -3;
  int dev = 0;
  cudaGetDevice(&dev);
  const int sms = dfl_host::num_sms(dev);
  const Plan plan = plan_dx(a->M, a->K, a->F, sms);
  GluParams p;
  std::memset(&p, 0, sizeof(p));
  for (int i = 0; i < 2; ++i) {
    rc = dfl_host::make_tmap_2d_bf16(&p.a[i], i ? a->du : a->dg, a->F, a->M, a->lds, BK, BM, true);
    if (rc) return 1000 + rc;
    rc = dfl_host::make_tmap_2d_bf16(&p.b[i], i ? a->wu : a->wg, a->K, a->F, i ? a->ldwu : a->ldwg, 64, BK, true);
    if (rc) return 2000 + rc;
  }
  p.d[0] = a->dx, p.ldd = a->K;
  p.M = a->M, p.N = a->K, p.K = a->F;
  rc = setup<kDx>(p, plan, 1);
  if (rc) return rc;
  if (ws_floats(plan, p.items) > a->ws_floats || (reinterpret_cast<uintptr_t>(a->ws) & 31)) return -10;
  p.ws = a->ws;
  return launch_mode<kDx>(p, plan, a->f16, sms, dev, a->err, stream);
}

extern "C" int dfl_glu_dw(const GluGemmArgs* a, cudaStream_t stream) {
  int rc = check_gemm(a);
  if (rc) return rc;
  if (!al16(a->x) || a->ldx % 8 || !al16(a->dwg) || !al16(a->dwu) || (!a->dwg && !a->dwu)) return -3;
  int dev = 0;
  cudaGetDevice(&dev);
  const int problems = a->dwg && a->dwu ? 2 : 1, sms = dfl_host::num_sms(dev);
  const Plan plan = plan_dw(a->M, a->K, a->F, problems, sms);
  GluParams p;
  std::memset(&p, 0, sizeof(p));
  int n = 0;
  for (int i = 0; i < 2; ++i) {
    void* d = i ? a->dwu : a->dwg;
    if (!d) continue;
    rc = dfl_host::make_tmap_2d_bf16(&p.a[n], i ? a->du : a->dg, a->F, a->M, a->lds, 64, BK, true);
    if (rc) return 1000 + rc;
    p.d[n++] = d;
  }
  rc = dfl_host::make_tmap_2d_bf16(&p.b[0], a->x, a->K, a->M, a->ldx, 64, BK, true);
  if (rc) return 2000 + rc;
  p.ldd = a->K;
  p.M = a->F, p.N = a->K, p.K = a->M;
  rc = setup<kDw>(p, plan, problems);
  if (rc) return rc;
  if (ws_floats(plan, p.items) > a->ws_floats || (reinterpret_cast<uintptr_t>(a->ws) & 31)) return -10;
  p.ws = a->ws;
  return launch_mode<kDw>(p, plan, a->f16, sms, dev, a->err, stream);
}
