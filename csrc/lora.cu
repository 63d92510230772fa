// Low-rank adapters of many requests beside a shared projection (sm_100a).
//
//   y = epi(x W^T + b + s_i (x A_i^T) B_i^T),   i = adapter of the row, -1 for none
//
// Two launches.  lora_shrink_kernel reads x once: for each 128-row tile it finds the adapters
// its rows use, computes x A_j^T for all of them on the tensor cores (up to 128 accumulator columns a
// pass), and stores T_j = s_j x A_j^T rounded to bf16, zero in the rows of other adapters.  The GEMM (gemm.cu,
// gemm2.cu) then runs x W^T and goes on over the tile's list with T_j B_j^T in the same f32 accumulator, so
// the adapters cost it ceil(rank / 64) K blocks per adapter a tile holds, and its epilogue is unchanged.
//
// Up to 32 rows (single tokens of a batch) take two kernels of their own, lora_rows_t_kernel and
// lora_rows_kernel below: there the weight's bytes are all that counts.
//
// The shrink is bound by reading x (2 M K bytes): a cluster of up to eight CTAs shares a tile, each
// taking a range of K, so that few tiles still occupy many SMs; the f32 partial sums are added through
// distributed shared memory in a fixed order.  Where a tile's adapters take several passes, several such clusters share them.
#include <algorithm>

#include "common.cuh"
#include "kernels.h"

namespace {
using namespace dfl;

constexpr int kBM = 128, kBK = 64, kMaxStages = 12;
constexpr int kXBytes = kBM * kBK * 2;         // 16 KB
constexpr int kThreads = 192;
constexpr int kMaxAdapters = 1024;
// Shared memory: a region for the stages (x tile, adapter rows), later for the partial sums; then
// barriers, TMEM slot, abort flag, adapter bitmap, list (count, ids: at most 256) and the list position of every row.
// With no more tiles than SMs one CTA per SM takes a large region (a K block arrives about 1.4 us after it was
// asked for, so the depth sets the rate: 5120 x 4096 rank 32 takes 15 us with 64 KB in flight); else two share an SM.
constexpr int kRegionTwo = 96 * 1024, kRegionOne = 208 * 1024;
constexpr int kMisc = (2 * kMaxStages + 1) * 8;
constexpr int kBitmap = (kMisc + 8 + 15) / 16 * 16;
constexpr int kList = kBitmap + kMaxAdapters / 8;
constexpr int kSlot = kList + 257 * 4;
constexpr int kTail = (kSlot + kBM * 2 + 15) / 16 * 16 + 1024;
static_assert(kRegionTwo + kTail <= 113 * 1024, "two CTAs per SM");
static_assert(kRegionOne + kTail <= 232448, "one CTA per SM");
static_assert((kBM + 7) * (128 + 4) * 4 <= kRegionTwo, "partial sums reuse the stages");

struct ShrinkParams {
  const int* ids;
  int rows_per_id;
  const float* scale;
  int n_adapters, rank, cap, tile_rows;
  int per_pass;  // adapters per pass: at most 128 accumulator columns
  int tiles, slices;
  int region, stages;  // stages of kXBytes + per_pass * rank * 128 bytes
  __nv_bfloat16* t;
  int* list;
  int* sem;
  int sem_count;
  int M, K;
};

DFL_DEVICE uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
DFL_DEVICE uint32_t cluster_size() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(r));
  return r;
}
DFL_DEVICE void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
DFL_DEVICE void st_cluster4(float* p, uint32_t rank, const uint32_t* v) {  // 16 bytes into CTA `rank` of the cluster
  uint32_t a;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem_u32(p)), "r"(rank));
  asm volatile("st.shared::cluster.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(a), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3])
               : "memory");
}
DFL_DEVICE void mbar_expect_tx(uint64_t* bar, uint32_t bytes) {
  asm volatile("mbarrier.expect_tx.relaxed.cta.shared::cta.b64 [%0], %1;" ::"r"(smem_u32(bar)), "r"(bytes) : "memory");
}

__global__ void __launch_bounds__(kThreads, 2)
    lora_shrink_kernel(const __grid_constant__ CUtensorMap tx, const __grid_constant__ CUtensorMap ta, ShrinkParams p,
                       int* err) {
  // (launched while the kernel before it ends: what that may write is not read through the read-only path)
  griddep_wait();
  griddep_launch();  // the GEMM may start on x W^T; it waits for this kernel before its first adapter block
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* full_bar = reinterpret_cast<uint64_t*>(smem + p.region);
  uint64_t* empty_bar = full_bar + kMaxStages;
  uint64_t* done_bar = empty_bar + kMaxStages;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + p.region + kMisc);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  uint32_t* bitmap = reinterpret_cast<uint32_t*>(smem + p.region + kBitmap);
  int* list = reinterpret_cast<int*>(smem + p.region + kList);
  int16_t* slot = reinterpret_cast<int16_t*>(smem + p.region + kSlot);
  float* part = reinterpret_cast<float*>(smem);

  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const uint32_t rank = cluster_rank(), ranks = cluster_size();
  const int tile = blockIdx.x / ranks % p.tiles;  // 128-row tile
  const int slice = blockIdx.x / ranks / p.tiles; // of the tile's passes: every p.slices-th
  const int per_group = p.tile_rows / kBM;        // 128-row tiles per M tile of the GEMM
  const int group = tile / per_group;
  const long long row0 = (long long)tile * kBM, grow0 = (long long)group * p.tile_rows;

  if (blockIdx.x == 0)
    for (int i = threadIdx.x; i < p.sem_count; i += kThreads) p.sem[i] = 0;
  if (threadIdx.x < kMaxAdapters / 32) bitmap[threadIdx.x] = 0u;
  if (threadIdx.x == 0) {
    for (int s = 0; s < kMaxStages; ++s) mbar_init(&full_bar[s], 1), mbar_init(&empty_bar[s], 1);
    mbar_init(done_bar, 1);
    *abort_flag = 0;
    fence_barrier_init();
    fence_proxy_async_shared();
    prefetch_tmap(&tx);
    prefetch_tmap(&ta);
  }
  if (warp == 1) {
    tmem_alloc(tmem_slot, 128);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;

  // this CTA's K blocks; the first x tiles are on their way while the adapters are looked up
  const int stages = p.stages, stage_bytes = kXBytes + p.per_pass * p.rank * kBK * 2;
  const int num_k = (p.K + kBK - 1) / kBK, per = (num_k + (int)ranks - 1) / (int)ranks;
  const int kb0 = min(num_k, (int)rank * per), kb1 = min(num_k, kb0 + per);
  const int early = min(stages, kb1 - kb0);
  if (warp == 0 && lane == 0)
    for (int i = 0; i < early; ++i) {
      mbar_expect_tx(&full_bar[i], kXBytes);
      tma_load_2d(smem + i * stage_bytes, &tx, &full_bar[i], (kb0 + i) * kBK, (int)row0);
    }

  // the adapters used by the rows of the GEMM's M tile, ascending
  auto id_of = [&](long long r) { return p.ids[p.rows_per_id > 0 ? r / p.rows_per_id : r]; };
  for (int r = threadIdx.x; r < p.tile_rows; r += kThreads) {
    if (grow0 + r >= p.M) continue;
    const int id = id_of(grow0 + r);
    if (id >= 0 && id < p.n_adapters) atomicOr(&bitmap[id / 32], 1u << (id % 32));
    else if (id != -1) record_error(err, kErrBounds, kKidLora, 10, (int)(grow0 + r));
  }
  __syncthreads();
  if (warp == 0) {
    const uint32_t w = bitmap[lane];
    int at = __popc(w);
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, at, o);
      if (lane >= o) at += v;
    }
    if (lane == 31) list[0] = at;
    at -= __popc(w);
    for (uint32_t v = w; v; v &= v - 1) list[1 + at++] = lane * 32 + __ffs(v) - 1;
  }
  __syncthreads();
  const int count = min(list[0], p.cap);  // (cap holds whatever the rows of a tile can name)
  for (int r = threadIdx.x; r < kBM; r += kThreads) {
    int s = -1;
    if (row0 + r < p.M) {
      const int id = id_of(row0 + r);
      for (int j = 0; j < count; ++j)
        if (list[1 + j] == id) s = j;
    }
    slot[r] = (int16_t)s;
  }
  if (rank == 0 && slice == 0 && tile % per_group == 0)
    for (int i = threadIdx.x; i <= count; i += kThreads) p.list[(long long)group * (1 + p.cap) + i] = i == 0 ? count : list[i];
  __syncthreads();

  const int first = slice * p.per_pass;  // of the list
  if (count <= first && warp == 0 && lane == 0)  // no adapter: the early copies must land before the CTA exits
    for (int i = 0; i < early; ++i) {
      mbar_arrive(&full_bar[i]);
      mbar_wait(&full_bar[i], 0, err, kKidLora, 50 + i, abort_flag);
    }

  int it = 0;  // stages used so far (all roles count alike)
  for (int j0 = first, pass = 0; j0 < count; j0 += p.slices * p.per_pass, ++pass) {
    const int nj = min(p.per_pass, count - j0), n = nj * p.rank;
    const int rows_per = (kBM + (int)ranks - 1) / (int)ranks, pitch = n + 4;
    if (warp == 0) {  // lane 0 copies x, each lane one adapter's rows (one thread alone takes 0.1 us a copy to issue them)
      bool ok = true;
      int i = it;
      for (int kb = kb0; kb < kb1; ++kb, ++i) {
        const int s = i % stages;
        uint8_t* sx = smem + s * stage_bytes;
        if (i >= early) ok = mbar_wait(&empty_bar[s], ((i / stages) & 1) ^ 1u, err, kKidLora, 20 + s, abort_flag);
        if (!__all_sync(0xffffffffu, ok)) break;
        if (lane == 0) {
          if (i >= early) {
            mbar_expect_tx(&full_bar[s], kXBytes);
            tma_load_2d(sx, &tx, &full_bar[s], kb * kBK, (int)row0);
          }
          mbar_arrive_expect_tx(&full_bar[s], n * kBK * 2);
        }
        __syncwarp();
        for (int j = lane; j < nj; j += 32)
          tma_load_2d(sx + kXBytes + j * p.rank * kBK * 2, &ta, &full_bar[s], kb * kBK, list[1 + j0 + j] * p.rank);
      }
      if (lane == 0 && i < it + kb1 - kb0)  // given up: our own copies must land before the CTA exits
        for (int k = max(0, i - stages); k < i; ++k)
          mbar_wait(&full_bar[k % stages], (k / stages) & 1, nullptr, 0, 0, nullptr, 200000000LL);
    } else if (warp == 1) {
      if (lane == 0) {
        const uint32_t idesc = make_idesc_bf16_f32(kBM, n);
        bool ok = true;
        int i = it;
        for (int kb = kb0; kb < kb1; ++kb, ++i) {
          const int s = i % stages;
          if (!mbar_wait(&full_bar[s], (i / stages) & 1, err, kKidLora, 30 + s, abort_flag)) { ok = false; break; }
          tc_fence_after();
          const uint32_t xa = smem_u32(smem + s * stage_bytes), aa = xa + kXBytes;
#pragma unroll
          for (int k = 0; k < kBK / 16; ++k)
            umma_f16_ss(tmem, make_sdesc_sw128(xa + k * 32, 16, 1024), make_sdesc_sw128(aa + k * 32, 16, 1024), idesc,
                        (kb > kb0 || k > 0) ? 1u : 0u);
          umma_commit(&empty_bar[s]);
        }
        if (ok) umma_commit(done_bar);
      }
    }
    // one row per thread of warps 2..5
    const int row = (warp & 3) * 32 + lane;
    const uint32_t t_row = tmem + ((uint32_t)((warp & 3) * 32) << 16);
    const long long trow0 = (long long)group * p.cap * p.tile_rows + (row0 - grow0);  // + j * tile_rows + row
    bool have = false;
    if (warp >= 2) {
      have = kb1 > kb0 && mbar_wait(done_bar, pass & 1, err, kKidLora, 40, abort_flag);
      tc_fence_after();
    }
    __syncwarp();
    if (ranks == 1) {
      if (warp >= 2) {
#pragma unroll 1
        for (int c = 0; c < n; c += 16) {
          const int j = j0 + c / p.rank;
          uint32_t v[16];
          tmem_ld_32x32b_x16(t_row + c, v);
          tmem_wait_ld();
          const float f = p.scale[list[1 + j]];
          const bool mine = have && slot[row] == j;
          uint32_t w[8];
#pragma unroll
          for (int e = 0; e < 8; ++e)
            w[e] = mine ? pack_bf16x2(f * __uint_as_float(v[2 * e]), f * __uint_as_float(v[2 * e + 1])) : 0u;
          uint4* dst = reinterpret_cast<uint4*>(p.t + (trow0 + (long long)j * p.tile_rows + row) * p.rank + c % p.rank);
          dst[0] = make_uint4(w[0], w[1], w[2], w[3]);
          dst[1] = make_uint4(w[4], w[5], w[6], w[7]);
        }
        tc_fence_before();
      }
    } else {
      __syncthreads();
      cluster_sync();  // every CTA is through with its stages: they take the partial sums
      if (warp >= 2) {
        // row -> the CTA that joins it: [source rank][row of the owner][column]
        const uint32_t owner = row / rows_per;
        float* dst = part + ((int)rank * rows_per + row % rows_per) * pitch;
#pragma unroll 1
        for (int c = 0; c < n; c += 16) {
          uint32_t v[16];
          tmem_ld_32x32b_x16(t_row + c, v);
          tmem_wait_ld();
#pragma unroll
          for (int e = 0; e < 16; ++e) v[e] = have ? v[e] : 0u;
#pragma unroll
          for (int q = 0; q < 4; ++q) st_cluster4(dst + c + 4 * q, owner, v + 4 * q);
        }
        tc_fence_before();
      }
      __syncwarp();
      cluster_sync();  // the partial sums of this CTA's rows have arrived
      const int r0 = (int)rank * rows_per, rows = min(rows_per, kBM - r0), half = n / 2;
      for (int e = threadIdx.x; e < rows * half; e += kThreads) {
        const int rl = e / half, c = 2 * (e % half), j = j0 + c / p.rank;
        float x = 0.f, y = 0.f;
#pragma unroll
        for (int k = 0; k < 8; ++k)
          if (k < (int)ranks) {  // in rank order
            const float2 f = *reinterpret_cast<const float2*>(part + (k * rows_per + rl) * pitch + c);
            x += f.x, y += f.y;
          }
        const bool mine = slot[r0 + rl] == j;
        const float f = p.scale[list[1 + j]];
        *reinterpret_cast<uint32_t*>(p.t + (trow0 + (long long)j * p.tile_rows + r0 + rl) * p.rank + c % p.rank) =
            mine ? pack_bf16x2(f * x, f * y) : 0u;
      }
    }
    it += kb1 - kb0;
    fence_proxy_async_shared();  // generic accesses to the stages before the next pass's copies
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
  }

  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == 1) tmem_dealloc(tmem, 128);
}

// ---------------------------------------------------------------------------
// Few rows (M <= 32): bound by reading W once (2 N K bytes).
//   lora_rows_t_kernel  T[m, r] = s_i x[m] . A_i[r] in f32, one warp per (m, r)
//   lora_rows_kernel    a CTA of 8 warps owns 16 output columns; its warps take 128-wide pieces of K in turn and
//                       multiply on the warp-level m16n8k16 instruction, W as the 16-row operand straight
//                       from global memory (both operands in the same permuted K order, so that a lane
//                       loads 16 contiguous bytes); partial sums are added in warp order, then T B^T and the epilogue,
//                       a thread per output (16 lanes to a product and a row at a time: 16 x 2048 x 2048 14.8 us, now 6.7).
// The second kernel is launched with programmatic serialisation: it streams W while T is computed and waits
// for T only before it is used.
// ---------------------------------------------------------------------------
constexpr int kRowsMax = 32;

struct RowsParams {
  const __nv_bfloat16* x; long long ldx;
  const __nv_bfloat16* w; long long ldw;
  const __nv_bfloat16* a;
  const __nv_bfloat16* b;
  const float* scale;
  const int* ids;
  int rows_per_id, n_adapters, rank;
  float* t;  // [M, rank]
  const __nv_bfloat16* bias;
  void* y; long long ldy;
  int out_f32, epi, act_lo, act_hi;
  const float* gate; long long gate_bs; int gate_rows;
  const __nv_bfloat16* resid; long long ldr;
  int M, N, K;
};

DFL_DEVICE int rows_id(const RowsParams& p, int m) {
  const int id = p.ids[p.rows_per_id > 0 ? m / p.rows_per_id : m];
  return id >= 0 && id < p.n_adapters ? id : -1;
}

DFL_DEVICE float dot8(const uint4& a, const uint4& b, float acc) {
  const uint32_t x[4] = {a.x, a.y, a.z, a.w}, y[4] = {b.x, b.y, b.z, b.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 u = unpack_bf16x2(x[i]), v = unpack_bf16x2(y[i]);
    acc = fmaf(u.x, v.x, acc);
    acc = fmaf(u.y, v.y, acc);
  }
  return acc;
}

__global__ void __launch_bounds__(256) lora_rows_t_kernel(RowsParams p, int* err) {
  griddep_wait();
  griddep_launch();
  const int m = blockIdx.x % p.M, r = blockIdx.x / p.M * 8 + threadIdx.x / 32, lane = threadIdx.x % 32;
  const int raw = p.ids[p.rows_per_id > 0 ? m / p.rows_per_id : m], id = rows_id(p, m);
  if (id < 0) {
    if (raw != -1 && r == 0 && lane == 0) record_error(err, kErrBounds, kKidLora, 11, m);
    return;  // (its T is not read)
  }
  if (r >= p.rank) return;
  const uint4* x = reinterpret_cast<const uint4*>(p.x + m * p.ldx);
  const uint4* a = reinterpret_cast<const uint4*>(p.a + ((long long)id * p.rank + r) * p.K);
  float acc[4] = {0.f, 0.f, 0.f, 0.f};
  const int nv = p.K / 8;
  int v = lane;
  for (; v + 96 < nv; v += 128) {
    uint4 xa[4], aa[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) xa[u] = __ldcg(x + v + 32 * u), aa[u] = __ldcg(a + v + 32 * u);
#pragma unroll
    for (int u = 0; u < 4; ++u) acc[u] = dot8(xa[u], aa[u], acc[u]);
  }
  for (; v < nv; v += 32) acc[0] = dot8(__ldcg(x + v), __ldcg(a + v), acc[0]);
  const float sum = warp_sum((acc[0] + acc[1]) + (acc[2] + acc[3]));
  if (lane == 0) p.t[m * p.rank + r] = sum * __ldcg(p.scale + id);
}

DFL_DEVICE void mma_bf16(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
DFL_DEVICE uint4 ld_stream16(const uint4* p) {  // read once: no L1 allocation
  uint4 r;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];"
               : "=r"(r.x), "=r"(r.y), "=r"(r.z), "=r"(r.w)
               : "l"(p));
  return r;
}

// NB: groups of 8 rows.
template <int NB>
__global__ void __launch_bounds__(256) lora_rows_kernel(RowsParams p) {
  __shared__ float red[8][16][8 * NB + 1];
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, quad = lane / 4, t = lane % 4;
  const int n0 = blockIdx.x * 16;
  const __nv_bfloat16* w0 = p.w + (long long)min(n0 + quad, p.N - 1) * p.ldw + 8 * t;
  const __nv_bfloat16* w1 = p.w + (long long)min(n0 + quad + 8, p.N - 1) * p.ldw + 8 * t;
  float c[NB][4];
#pragma unroll
  for (int g = 0; g < NB; ++g) c[g][0] = c[g][1] = c[g][2] = c[g][3] = 0.f;
  const uint4 zero = make_uint4(0u, 0u, 0u, 0u);
  int id = threadIdx.x / 16 < p.M ? rows_id(p, threadIdx.x / 16) : -1;  // of the row this thread stores
#pragma unroll 2
  for (int k0 = warp * 128; k0 < p.K; k0 += 8 * 128) {
    uint4 a[4][2], b[4][NB];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int k = k0 + 32 * u;
      const bool in = k + 8 * t < p.K;  // K is a multiple of 8: a lane's piece is inside or outside
      a[u][0] = in ? ld_stream16(reinterpret_cast<const uint4*>(w0 + k)) : zero;
      a[u][1] = in ? ld_stream16(reinterpret_cast<const uint4*>(w1 + k)) : zero;
#pragma unroll
      for (int g = 0; g < NB; ++g)
        b[u][g] = in && 8 * g + quad < p.M
                      ? __ldg(reinterpret_cast<const uint4*>(p.x + (8 * g + quad) * p.ldx + k + 8 * t)) : zero;
    }
#pragma unroll
    for (int u = 0; u < 4; ++u)
#pragma unroll
      for (int g = 0; g < NB; ++g) {
        mma_bf16(c[g], a[u][0].x, a[u][1].x, a[u][0].y, a[u][1].y, b[u][g].x, b[u][g].y);
        mma_bf16(c[g], a[u][0].z, a[u][1].z, a[u][0].w, a[u][1].w, b[u][g].z, b[u][g].w);
      }
  }
  // c[g][2 i + e]: column quad + 8 i, row 8 g + 2 t + e
#pragma unroll
  for (int g = 0; g < NB; ++g)
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int e = 0; e < 2; ++e) red[warp][quad + 8 * i][8 * g + 2 * t + e] = c[g][2 * i + e];
  // T B^T: a thread takes whole products, of one column and every 16th row
  const int n = threadIdx.x % 16, col = n0 + n;
  auto b_row = [&](int id) { return reinterpret_cast<const uint4*>(p.b + ((long long)id * p.N + col) * p.rank); };
  uint4 first[2];  // the adapter's first 16 values, on their way while the warps' sums are stored and T is waited for
  if (col >= p.N) id = -1;
  if (id >= 0) first[0] = __ldg(b_row(id)), first[1] = __ldg(b_row(id) + 1);
  griddep_wait();  // T is complete
  __syncthreads();
  if (col >= p.N) return;
  for (int m = threadIdx.x / 16; m < p.M; m += 16) {
    if (m >= 16) {
      id = rows_id(p, m);
      if (id >= 0) first[0] = __ldg(b_row(id)), first[1] = __ldg(b_row(id) + 1);
    }
    float v = 0.f;
#pragma unroll
    for (int k = 0; k < 8; ++k) v += red[k][n][m];
    if (id >= 0) {
      const uint4* bw = b_row(id);
      const float4* t4 = reinterpret_cast<const float4*>(p.t + m * p.rank);
      float acc[2] = {0.f, 0.f};
#pragma unroll 2
      for (int r = 0; r < p.rank / 8; r += 2)  // (a multiple of 16)
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          const uint4 w = r == 0 ? first[u] : __ldg(bw + r + u);
          const float4 t0 = __ldcg(t4 + 2 * (r + u)), t1 = __ldcg(t4 + 2 * (r + u) + 1);
          const float2 b0 = unpack_bf16x2(w.x), b1 = unpack_bf16x2(w.y), b2 = unpack_bf16x2(w.z), b3 = unpack_bf16x2(w.w);
          acc[u] += ((b0.x * t0.x + b0.y * t0.y) + (b1.x * t0.z + b1.y * t0.w)) +
                    ((b2.x * t1.x + b2.y * t1.y) + (b3.x * t1.z + b3.y * t1.w));
        }
      v += acc[0] + acc[1];
    }
    if (p.bias) v += __bfloat162float(p.bias[col]);
    if (col >= p.act_lo && col < p.act_hi) {
      if (p.epi == kEpiGelu) v = gelu_tanh(v);
      else if (p.epi == kEpiSilu) v = silu(v);
    }
    if (p.epi == kEpiGateResid)
      v = fmaf(p.gate[(long long)(m / p.gate_rows) * p.gate_bs + col], v, __bfloat162float(p.resid[m * p.ldr + col]));
    if (p.out_f32) reinterpret_cast<float*>(p.y)[m * p.ldy + col] = v;
    else reinterpret_cast<__nv_bfloat16*>(p.y)[m * p.ldy + col] = __float2bfloat16_rn(v);
  }
}

int lora_rows(const GemmArgs* a, cudaStream_t stream) {
  const LoraArgs* l = a->lora;
  if (a->gate_row_map || a->alpha != 1.f) return -27;
  if ((reinterpret_cast<uintptr_t>(a->B) & 15) || a->ldb % 8) return -4;
  RowsParams p{};
  p.x = reinterpret_cast<const __nv_bfloat16*>(a->A), p.ldx = a->lda;
  p.w = reinterpret_cast<const __nv_bfloat16*>(a->B), p.ldw = a->ldb;
  p.a = reinterpret_cast<const __nv_bfloat16*>(l->a);
  p.b = reinterpret_cast<const __nv_bfloat16*>(l->b);
  p.scale = l->scale;
  p.ids = l->ids;
  p.rows_per_id = l->rows_per_id, p.n_adapters = l->n_adapters, p.rank = l->rank;
  p.t = reinterpret_cast<float*>(l->t);
  p.bias = reinterpret_cast<const __nv_bfloat16*>(a->bias);
  p.y = a->D, p.ldy = a->ldd;
  p.out_f32 = a->out_f32, p.epi = a->epi, p.act_lo = a->act_lo, p.act_hi = a->act_hi;
  p.gate = a->gate, p.gate_bs = a->gate_bstride, p.gate_rows = a->rows_per_batch > 0 ? a->rows_per_batch : a->M;
  p.resid = reinterpret_cast<const __nv_bfloat16*>(a->resid), p.ldr = a->ldr;
  p.M = a->M, p.N = a->N, p.K = a->K;
  if (p.epi == kEpiGateResid && (!p.gate || !p.resid)) return -8;
  const cudaError_t e = dfl_host::launch_early(lora_rows_t_kernel, (unsigned)(p.M * ((p.rank + 7) / 8)), 256, 0, stream, p, a->err);
  if (e != cudaSuccess) return (int)e;
  const auto kern = p.M <= 8 ? lora_rows_kernel<1> : p.M <= 16 ? lora_rows_kernel<2> : lora_rows_kernel<4>;
  return (int)dfl_host::launch_early(kern, (unsigned)((p.N + 15) / 16), 256, 0, stream, p);
}

}  // namespace

extern "C" int dfl_lora_rows(int M) { return M <= kRowsMax; }

extern "C" int dfl_gemm_lora(const GemmArgs* a, cudaStream_t stream) {
  const LoraArgs* l = a->lora;
  if (!l || !l->a || !l->b || !l->scale || !l->ids || !l->t) return -20;
  if (l->n_adapters < 1 || l->n_adapters > kMaxAdapters) return -21;
  if (l->rank % 16 || l->rank < 16 || l->rank > 128 || (l->rank > 64 && l->rank != 128)) return -22;
  if (a->epi == kEpiSwiGLU || a->epi == kEpiQkv || a->out_world > 0) return -23;
  if (a->M > 0 && a->M <= kRowsMax) {
    if (a->K % 8 || (a->lda % 8) || ((reinterpret_cast<uintptr_t>(a->A) | reinterpret_cast<uintptr_t>(l->a) |
                                      reinterpret_cast<uintptr_t>(l->b) | reinterpret_cast<uintptr_t>(l->t)) & 15))
      return -25;
    return lora_rows(a, stream);
  }
  if (l->cap < 1 || l->cap > l->tile_rows || (l->tile_rows != 128 && l->tile_rows != 256)) return -24;
  if (!l->list || a->M <= 0 || a->K % 8 || (a->lda * 2) % 16 || (reinterpret_cast<uintptr_t>(a->A) & 15)) return -25;
  if ((reinterpret_cast<uintptr_t>(l->a) | reinterpret_cast<uintptr_t>(l->b) | reinterpret_cast<uintptr_t>(l->t)) & 15)
    return -26;
  int dev = 0;
  cudaGetDevice(&dev);
  // clusters of 1..8 CTAs, one CTA per SM, that are resident at once (a cluster stays inside one GPC)
  static int resident[16][9] = {{0}};
  int* fit = resident[dev & 15];
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.y = 1;
  at[0].val.clusterDim.z = 1;
  at[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.blockDim = dim3(kThreads, 1, 1);
  cfg.stream = stream;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  if (!fit[1]) {
    cudaError_t e = cudaFuncSetAttribute(lora_shrink_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kRegionOne + kTail);
    if (e != cudaSuccess) return (int)e;
    int found[9] = {0};
    for (int c = 2; c <= 8; ++c) {
      at[0].val.clusterDim.x = c;
      cfg.gridDim = dim3((unsigned)(c * 1024), 1, 1);
      cfg.dynamicSmemBytes = kRegionOne + kTail;
      e = cudaOccupancyMaxActiveClusters(&found[c], lora_shrink_kernel, &cfg);
      if (e != cudaSuccess) return (int)e;
    }
    for (int c = 2; c <= 8; ++c) fit[c] = found[c];
    fit[1] = dfl_host::num_sms(dev);
  }
  CUtensorMap tx, ta;
  int rc = dfl_host::make_tmap_2d_bf16(&tx, a->A, a->K, a->M, a->lda, kBK, kBM, true);
  if (rc) return 1000 + rc;
  rc = dfl_host::make_tmap_2d_bf16(&ta, l->a, a->K, (uint64_t)l->n_adapters * l->rank, a->K, kBK, l->rank, true);
  if (rc) return 2000 + rc;
  ShrinkParams p{};
  p.ids = l->ids;
  p.rows_per_id = l->rows_per_id;
  p.scale = l->scale;
  p.n_adapters = l->n_adapters;
  p.rank = l->rank;
  p.cap = l->cap;
  p.tile_rows = l->tile_rows;
  p.t = reinterpret_cast<__nv_bfloat16*>(l->t);
  p.list = l->list;
  p.sem = l->split_sem;
  p.sem_count = l->split_sem ? l->split_sem_count : 0;
  p.M = a->M;
  p.K = a->K;
  p.per_pass = std::max(1, std::min(l->cap, 128 / l->rank));
  // every 128-row tile of every M tile (the last M tile's second half may lie behind M: zeros)
  const long long tiles = ((long long)a->M + l->tile_rows - 1) / l->tile_rows * (l->tile_rows / kBM);
  // How many CTAs share a tile's K, and how many clusters its passes, all of them resident.  In 0.1 us: a K block takes 8
  // here and 3 in the GEMM, a join 30, launch and lists 60.  Where the GEMM's CTAs find SMs of their own beside, its loop
  // over x runs at the same time; else after.  12 tiles beside 96 CTAs, K 2048, 7 adapters: 8 CTAs a tile 32.7 us for both
  // kernels, 4 (beside) 25.9, 3 28.2, 2 32.5.  6 tiles of 12 passes, K 3648,
  // rank 128: one cluster of 8 a tile 147 us, six of 4 53 us.
  const int num_k = (a->K + kBK - 1) / kBK, passes = (l->cap + p.per_pass - 1) / p.per_pass;
  const long long room = fit[1] - dfl_gemm_ctas(a), gemm = 30 + 3ll * num_k;
  int ranks = 1;
  long long slices = 1, best = -1;
  for (int c = 1; c <= 8; ++c) {
    if (c > 1 && (tiles > fit[c] || num_k < 4 * c)) continue;
    auto consider = [&](long long sl, bool beside) {
      sl = std::max(1ll, std::min<long long>(passes, sl));
      const long long t = 60 + (passes + sl - 1) / sl * ((num_k + c - 1) / c * 8ll + (c > 1 ? 30 : 0));
      const long long cost = beside ? std::max(t, gemm) + t / 4 : t + gemm;
      if (best < 0 || cost < best) best = cost, ranks = c, slices = sl;
    };
    consider(fit[c] / tiles, false);
    if (tiles * c <= room) consider(std::min<long long>(room / (tiles * c), fit[c] / tiles), true);
  }
  p.tiles = (int)tiles;
  p.slices = (int)slices;
  const long long ctas = tiles * ranks * slices;
  p.region = ctas <= fit[1] ? kRegionOne : kRegionTwo;
  p.stages = std::min(kMaxStages, p.region / (kXBytes + p.per_pass * l->rank * kBK * 2));
  cfg.gridDim = dim3((unsigned)ctas, 1, 1);
  cfg.dynamicSmemBytes = p.region + kTail;
  at[0].val.clusterDim.x = ranks;
  cfg.numAttrs = 2;
  cudaError_t e = cudaLaunchKernelEx(&cfg, lora_shrink_kernel, tx, ta, p, a->err);
  if (e != cudaSuccess) return (int)e;
  return dfl_gemm_bf16(a, stream);
}
