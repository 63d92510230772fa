// Gated projection and its gradients (sm_100a, tcgen05), bf16 or fp16:
//
//   g = x Wg^T, u = x Wu^T, h = act(g) * u
//   dg = dh * u * act'(g), du = dh * act(g);  dx = dg Wg + du Wu;  dWg = dg^T x, dWu = du^T x
//
// One persistent GEMM in three forms (products of matrix tiles, f32 accumulators in tensor memory, operands through a
// ring of shared-memory stages filled by tiled copies):
//   forward  an accumulator holds the same columns of g and u side by side (Wg's and Wu's rows are the two halves of the
//            tile's second operand; in a CTA pair each CTA loads one of them), so act(g) * u needs no exchange; x is read
//            once for both.  With gradients to come, g and u are stored too, rounded to the type (at most 2^-8 of each
//            value in bf16; the gradients are rounded to it anyway: the alternative, computing them again, costs another
//            4 M F K operations).
//   dx       the K loop runs over dg Wg, then du Wu, in one accumulator; the weights are read as they lie ([F, K]: the
//            second operand with its columns contiguous)
//   dW       both operands lie with their columns contiguous ([M, F] and [M, K]); nothing is transposed in memory
// Tiles of 256 x 256 by CTA pairs, or 128 x 128 by single CTAs where those fill the SMs better (glu_plan).
#include <algorithm>
#include <cstring>

#include <cuda_fp16.h>

#include "common.cuh"
#include "kernels.h"
#include "pair.cuh"

namespace {
using namespace dfl;

enum { kForward = 0, kDx = 1, kDw = 2 };

constexpr int BM = 128, BK = 64, STAGES = 6, kThreads = 192;
constexpr int kOpBytes = 128 * BK * 2;  // each CTA loads 128 rows (or columns) of both operands per stage
constexpr int kStageBytes = 2 * kOpBytes;
constexpr int kBarOff = STAGES * kStageBytes;
constexpr int kSmem = kBarOff + (2 * STAGES + 4) * 8 + 16 + 1024;
static_assert(kSmem <= 232448, "shared memory budget");
constexpr int kGroupM = 16;  // tile raster: 16 M blocks per group, for L2 reuse

struct GluParams {
  CUtensorMap a[2], b[2];
  void* d[2];        // outputs (forward: h; dW: one for each problem)
  void* g;           // forward: the kept projections
  void* u;
  long long ldd, lds;
  float* ws;         // dx: partial sums [splits][M][N]
  int M, N, K;       // of one problem: rows and columns of the output, length of the sums (of each segment)
  int num_m, num_n, tiles, splits;
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
  if constexpr (F16) return __half2float(reinterpret_cast<const __half*>(p)[i]);
  else return __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(p)[i]);
}
template <bool F16>
DFL_DEVICE void store1(void* p, long long i, float v) {
  if constexpr (F16) reinterpret_cast<__half*>(p)[i] = __float2half_rn(v);
  else reinterpret_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(v);
}

// act(x) = x s(x), and its derivative s + x s'(x).  SiLU: s = 1 / (1 + e^-x).  GELU, tanh form:
// 0.5 (1 + tanh z) = 1 / (1 + e^-2z), z = sqrt(2 / pi) (x + 0.044715 x^3), which keeps the relative accuracy where
// the result is small.  Exact GELU: s = erfc(-x / sqrt 2) / 2, s' = e^(-x^2 / 2) / sqrt(2 pi).
DFL_DEVICE float sigmoid(float x) { return __fdividef(1.f, 1.f + __expf(-x)); }  // (2^126 < e^-x gives 0, as it should)
DFL_DEVICE float gelu_arg(float x) { return 1.5957691216057308f * x * (1.f + 0.044715f * x * x); }
template <int ACT>
DFL_DEVICE float act_of(float x) {
  if constexpr (ACT == kGluSilu) return x * sigmoid(x);
  if constexpr (ACT == kGluGelu) return x * sigmoid(gelu_arg(x));
  return 0.5f * x * erfcf(-0.7071067811865476f * x);
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
  const float s = 0.5f * erfcf(-0.7071067811865476f * x);
  return make_float2(x * s, s + x * 0.3989422804014327f * __expf(-0.5f * x * x));
}

// K blocks [kb0, kb1) of split item `split`; a block is (segment, offset) in the two-segment sums of dx.
template <int MODE>
DFL_DEVICE int k_blocks(const GluParams& p) { return (p.K + BK - 1) / BK * (MODE == kDx ? 2 : 1); }

struct Tile {
  int which, mb, nb, split, kb0, kb1;
};
template <int MODE>
DFL_DEVICE Tile tile_of(const GluParams& p, int t) {
  Tile r;
  r.split = t % p.splits;
  t /= p.splits;
  r.which = t / p.tiles;
  t -= r.which * p.tiles;
  const int group = t / (kGroupM * p.num_n), first = group * kGroupM, gm = min(kGroupM, p.num_m - first);
  t -= group * kGroupM * p.num_n;
  r.mb = first + t % gm, r.nb = t / gm;
  const int n = k_blocks<MODE>(p), per = (n + p.splits - 1) / p.splits;
  r.kb0 = min(n, r.split * per), r.kb1 = min(n, r.kb0 + per);
  return r;
}

// 32 columns of a row: whole 16-byte pieces where the row allows it.
template <bool F16>
DFL_DEVICE void store_cols(void* base, long long at, const float (&v)[32], int cols, bool wide) {
  if (wide && cols >= 32) {
    uint4* d = reinterpret_cast<uint4*>(reinterpret_cast<uint16_t*>(base) + at);
#pragma unroll
    for (int q = 0; q < 4; ++q)
      d[q] = make_uint4(pack2<F16>(v[8 * q], v[8 * q + 1]), pack2<F16>(v[8 * q + 2], v[8 * q + 3]),
                        pack2<F16>(v[8 * q + 4], v[8 * q + 5]), pack2<F16>(v[8 * q + 6], v[8 * q + 7]));
  } else {
#pragma unroll
    for (int j = 0; j < 32; ++j)
      if (j < cols) store1<F16>(base, at + j, v[j]);
  }
}

template <int CG>
DFL_DEVICE void load_tile(uint8_t* dst, const CUtensorMap* map, uint64_t* bar, int c0, int c1) {
  if constexpr (CG == 2) tma_load_2d_pair(dst, map, bar, c0, c1);
  else tma_load_2d(dst, map, bar, c0, c1);
}

// CG: CTAs per tile (2: a pair).  A tile is 128 CG rows and 128 CG accumulator columns.
template <int MODE, int CG, bool F16>
__global__ void __launch_bounds__(kThreads, 1) glu_kernel(const __grid_constant__ GluParams p, int* err) {
  constexpr int BN = 128 * CG;
  constexpr uint32_t kTmemCols = 2 * BN;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* full_bar = reinterpret_cast<uint64_t*>(smem + kBarOff);
  uint64_t* empty_bar = full_bar + STAGES;
  uint64_t* tfull_bar = empty_bar + STAGES;
  uint64_t* tempty_bar = tfull_bar + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(tempty_bar + 2);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const uint32_t rank = CG == 2 ? cluster_rank() : 0u;
  const int first = blockIdx.x / CG, step = gridDim.x / CG;
  const int items = p.tiles * (MODE == kDw ? (p.d[1] ? 2 : 1) : 1) * p.splits;

  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(&full_bar[s], 1);   // CTA 0's producer posts the bytes of all
      mbar_init(&empty_bar[s], 1);  // the issuing thread's commit, to every CTA of the tile
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(&tfull_bar[a], 1);
      mbar_init(&tempty_bar[a], 128 * CG);  // (CTA 0's copy is the one used)
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
          uint8_t* sa = smem + stage * kStageBytes;
          uint8_t* sb = sa + kOpBytes;
          uint64_t* bar = &full_bar[stage];
          if (rank == 0) mbar_arrive_expect_tx(bar, CG * kStageBytes);
          const int m0 = it.mb * BM * CG + (int)rank * BM;
          if constexpr (MODE == kForward) {
            load_tile<CG>(sa, &p.a[0], bar, kb * BK, m0);
            const int n0 = it.nb * (BN / 2);
            if constexpr (CG == 2) {  // rank 0: rows of Wg, rank 1: of Wu
              load_tile<CG>(sb, &p.b[rank], bar, kb * BK, n0);
            } else {
              load_tile<CG>(sb, &p.b[0], bar, kb * BK, n0);
              load_tile<CG>(sb + kOpBytes / 2, &p.b[1], bar, kb * BK, n0);
            }
          } else if constexpr (MODE == kDx) {
            const int half = (p.K + BK - 1) / BK, seg = kb >= half, k0 = (kb - seg * half) * BK;
            const int n0 = it.nb * BN + (int)rank * 128;
            load_tile<CG>(sa, &p.a[seg], bar, k0, m0);
            load_tile<CG>(sb, &p.b[seg], bar, n0, k0);
            load_tile<CG>(sb + kOpBytes / 2, &p.b[seg], bar, n0 + 64, k0);
          } else {
            const int n0 = it.nb * BN + (int)rank * 128;
            load_tile<CG>(sa, &p.a[it.which], bar, m0, kb * BK);
            load_tile<CG>(sa + kOpBytes / 2, &p.a[it.which], bar, m0 + 64, kb * BK);
            load_tile<CG>(sb, &p.b[0], bar, n0, kb * BK);
            load_tile<CG>(sb + kOpBytes / 2, &p.b[0], bar, n0 + 64, kb * BK);
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
      // 16 rows are 2048 bytes, the next chunk is kOpBytes / 2 away.
      auto desc = [](uint32_t addr, int k, bool mn) {
        return mn ? make_sdesc_sw128(addr + k * 2048, kOpBytes / 2, 1024) : make_sdesc_sw128(addr + k * 32, 16, 1024);
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
          const uint32_t a_addr = smem_u32(smem + stage * kStageBytes), b_addr = a_addr + kOpBytes;
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
      if constexpr (MODE == kForward) {
        const bool wide = p.ldd % 8 == 0 && (reinterpret_cast<uintptr_t>(p.d[0]) & 15) == 0;
#pragma unroll 1
        for (int c = 0; c < BN / 2; c += 32) {
          uint32_t gr[32], ur[32];
          tmem_ld_32x32b_x32(tbase + c, gr);
          tmem_ld_32x32b_x32(tbase + BN / 2 + c, ur);
          tmem_wait_ld();
          if (c + 32 == BN / 2) release();
          const int col = it.nb * (BN / 2) + c, cols = p.N - col;
          if (row >= p.M || cols <= 0) continue;
          float g[32], u[32];
#pragma unroll
          for (int j = 0; j < 32; ++j) g[j] = __uint_as_float(gr[j]), u[j] = __uint_as_float(ur[j]);
          if (p.g) {
            store_cols<F16>(p.g, row * p.lds + col, g, cols, true);
            store_cols<F16>(p.u, row * p.lds + col, u, cols, true);
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
          store_cols<F16>(p.d[0], row * p.ldd + col, u, cols, wide);
        }
      } else {
        const bool none = it.kb0 >= it.kb1;  // (a sum over nothing)
#pragma unroll 1
        for (int c = 0; c < BN; c += 32) {
          uint32_t r[32];
          tmem_ld_32x32b_x32(tbase + c, r);
          tmem_wait_ld();
          if (c + 32 == BN) release();
          const int col = it.nb * BN + c, cols = p.N - col;
          if (row >= p.M || cols <= 0) continue;
          float v[32];
#pragma unroll
          for (int j = 0; j < 32; ++j) v[j] = none ? 0.f : __uint_as_float(r[j]);
          if (MODE == kDx && p.splits > 1) {  // N is a multiple of 8
            float4* d = reinterpret_cast<float4*>(p.ws + ((long long)it.split * p.M + row) * p.N + col);
#pragma unroll
            for (int q = 0; q < 8; ++q)
              if (4 * q < cols) d[q] = make_float4(v[4 * q], v[4 * q + 1], v[4 * q + 2], v[4 * q + 3]);
          } else {
            store_cols<F16>(p.d[it.which], row * p.ldd + col, v, cols, true);
          }
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

// dx from its partial sums, added in order.
template <bool F16>
__global__ void __launch_bounds__(256) glu_join_kernel(const float* ws, void* dx, long long n, int splits) {
  griddep_wait();
  for (long long i = ((long long)blockIdx.x * 256 + threadIdx.x) * 4; i < n; i += (long long)gridDim.x * 1024) {
    float4 s = __ldcg(reinterpret_cast<const float4*>(ws + i));
    for (int k = 1; k < splits; ++k) {
      const float4 v = __ldcg(reinterpret_cast<const float4*>(ws + k * n + i));
      s.x += v.x, s.y += v.y, s.z += v.z, s.w += v.w;
    }
    *reinterpret_cast<uint2*>(reinterpret_cast<uint16_t*>(dx) + i) = make_uint2(pack2<F16>(s.x, s.y), pack2<F16>(s.z, s.w));
  }
}

// dg, du: 8 columns a thread.  Bound by its bytes (10 M F).
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
    const uint4 gv = __ldcg(reinterpret_cast<const uint4*>(reinterpret_cast<const uint16_t*>(a.g) + at));
    const uint4 uv = __ldcg(reinterpret_cast<const uint4*>(reinterpret_cast<const uint16_t*>(a.u) + at));
    float d[8];
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
    const uint32_t gw[4] = {gv.x, gv.y, gv.z, gv.w}, uw[4] = {uv.x, uv.y, uv.z, uv.w};
    uint32_t og[4], ou[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float2 g = unpack2<F16>(gw[e]), u = unpack2<F16>(uw[e]);
      const float2 x = act_grad<ACT>(g.x), y = act_grad<ACT>(g.y);
      og[e] = pack2<F16>(d[2 * e] * u.x * x.y, d[2 * e + 1] * u.y * y.y);
      ou[e] = pack2<F16>(d[2 * e] * x.x, d[2 * e + 1] * y.x);
    }
    *reinterpret_cast<uint4*>(reinterpret_cast<uint16_t*>(a.dg) + at) = make_uint4(og[0], og[1], og[2], og[3]);
    *reinterpret_cast<uint4*>(reinterpret_cast<uint16_t*>(a.du) + at) = make_uint4(ou[0], ou[1], ou[2], ou[3]);
  }
}

bool al16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// CTAs per tile: pairs take 256 x 256 in the time (per K block) that a single CTA needs for about 1.6 tiles of 128 x 128;
// whichever needs fewer rounds' time.
int glu_ctas(long long rows, long long cols, int problems, int sms) {
  auto tiles = [&](int n) { return ((rows + n - 1) / n) * ((cols + n - 1) / n) * problems; };
  const long long pairs = (tiles(256) + sms / 2 - 1) / (sms / 2), singles = (tiles(128) + sms - 1) / sms;
  return pairs * 16 <= singles * 10 ? 2 : 1;
}

template <int MODE, int CG, bool F16>
int launch_glu(const GluParams& p, int problems, int sms, int dev, int* err, cudaStream_t stream) {
  auto kern = glu_kernel<MODE, CG, F16>;
  static bool attr[16] = {false};
  if (!attr[dev & 15]) {
    const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem);
    if (e != cudaSuccess) return (int)e;
    attr[dev & 15] = true;
  }
  const long long items = (long long)p.tiles * problems * p.splits, slots = sms / CG;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(CG * std::min(items, slots)), 1, 1);
  cfg.blockDim = dim3(kThreads, 1, 1);
  cfg.dynamicSmemBytes = kSmem;
  cfg.stream = stream;
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  at[1].id = cudaLaunchAttributeClusterDimension;
  at[1].val.clusterDim.x = CG;
  at[1].val.clusterDim.y = at[1].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = CG == 2 ? 2 : 1;
  return (int)cudaLaunchKernelEx(&cfg, kern, p, err);
}

template <int MODE>
int launch_mode(const GluParams& p, int cg, int f16, int problems, int sms, int dev, int* err, cudaStream_t stream) {
  if (cg == 2)
    return f16 ? launch_glu<MODE, 2, true>(p, problems, sms, dev, err, stream)
               : launch_glu<MODE, 2, false>(p, problems, sms, dev, err, stream);
  return f16 ? launch_glu<MODE, 1, true>(p, problems, sms, dev, err, stream)
             : launch_glu<MODE, 1, false>(p, problems, sms, dev, err, stream);
}

int tiles_of(GluParams& p, int cg, int cols) {
  const long long m = ((long long)p.M + 128 * cg - 1) / (128 * cg), n = ((long long)p.N + cols - 1) / cols;
  if (m * n > (1 << 28)) return -9;
  p.num_m = (int)m, p.num_n = (int)n, p.tiles = (int)(m * n);
  return 0;
}

}  // namespace

extern "C" int dfl_glu(const GluArgs* a, cudaStream_t stream) {
  if (a->M <= 0 || a->F <= 0 || a->K <= 0 || a->K % 8 || a->act < 0 || a->act > kGluGeluErf) return -2;
  if (!al16(a->x) || !al16(a->wg) || !al16(a->wu) || (a->ldx | a->ldwg | a->ldwu) % 8) return -3;
  if (a->g && (!a->u || !al16(a->g) || !al16(a->u) || a->lds % 8 || a->lds < a->F)) return -4;
  int dev = 0;
  cudaGetDevice(&dev);
  const int sms = dfl_host::num_sms(dev), cg = glu_ctas(a->M, 2ll * a->F, 1, sms);
  GluParams p;
  std::memset(&p, 0, sizeof(p));
  int rc = dfl_host::make_tmap_2d_bf16(&p.a[0], a->x, a->K, a->M, a->ldx, BK, BM, true);
  if (rc) return 1000 + rc;
  rc = dfl_host::make_tmap_2d_bf16(&p.b[0], a->wg, a->K, a->F, a->ldwg, BK, 64 * cg, true);
  if (rc) return 2000 + rc;
  rc = dfl_host::make_tmap_2d_bf16(&p.b[1], a->wu, a->K, a->F, a->ldwu, BK, 64 * cg, true);
  if (rc) return 3000 + rc;
  p.d[0] = a->h, p.ldd = a->ldh;
  p.g = a->g, p.u = a->u, p.lds = a->lds;
  p.M = a->M, p.N = a->F, p.K = a->K, p.splits = 1, p.act = a->act;
  rc = tiles_of(p, cg, 64 * cg);
  return rc ? rc : launch_mode<kForward>(p, cg, a->f16, 1, sms, dev, a->err, stream);
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

extern "C" long long dfl_glu_dx_ws(int M, int K, int F) { return 0; }

extern "C" int dfl_glu_dx(const GluGemmArgs* a, cudaStream_t stream) {
  int rc = check_gemm(a);
  if (rc) return rc;
  if (!al16(a->wg) || !al16(a->wu) || !al16(a->dx) || (a->ldwg | a->ldwu) % 8) return -3;
  int dev = 0;
  cudaGetDevice(&dev);
  const int sms = dfl_host::num_sms(dev), cg = glu_ctas(a->M, a->K, 1, sms);
  GluParams p;
  std::memset(&p, 0, sizeof(p));
  for (int i = 0; i < 2; ++i) {
    rc = dfl_host::make_tmap_2d_bf16(&p.a[i], i ? a->du : a->dg, a->F, a->M, a->lds, BK, BM, true);
    if (rc) return 1000 + rc;
    rc = dfl_host::make_tmap_2d_bf16(&p.b[i], i ? a->wu : a->wg, a->K, a->F, i ? a->ldwu : a->ldwg, 64, BK, true);
    if (rc) return 2000 + rc;
  }
  p.d[0] = a->dx, p.ldd = a->K;
  p.M = a->M, p.N = a->K, p.K = a->F, p.splits = 1;
  rc = tiles_of(p, cg, 128 * cg);
  return rc ? rc : launch_mode<kDx>(p, cg, a->f16, 1, sms, dev, a->err, stream);
}

extern "C" int dfl_glu_dw(const GluGemmArgs* a, cudaStream_t stream) {
  int rc = check_gemm(a);
  if (rc) return rc;
  if (!al16(a->x) || a->ldx % 8 || !al16(a->dwg) || !al16(a->dwu) || (!a->dwg && !a->dwu)) return -3;
  int dev = 0;
  cudaGetDevice(&dev);
  const int problems = a->dwg && a->dwu ? 2 : 1, sms = dfl_host::num_sms(dev), cg = glu_ctas(a->F, a->K, problems, sms);
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
  p.M = a->F, p.N = a->K, p.K = a->M, p.splits = 1;
  rc = tiles_of(p, cg, 128 * cg);
  return rc ? rc : launch_mode<kDw>(p, cg, a->f16, problems, sms, dev, a->err, stream);
}
