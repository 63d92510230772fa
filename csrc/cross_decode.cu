// Attention of a few queries to many keys (single tokens, pooling queries): up to 16 query rows that share a key head
// to a CTA; more rows where the kernel of cross_attn.cuh would have too few tiles (dfl_cross_decode_takes).  sm_100a.
//
// Bound by reading K and V once: a 128-row tensor-memory tile would be nearly empty, so the keys are split over up
// to sixteen CTAs (one cluster per key head and batch row).  In each, one warp keeps a ring of 32-key stages full with
// tiled copies (64 KB in flight per CTA at dh 128, two CTAs per SM), and four warps walk 16-key blocks of them with
// a running maximum and sum on the warp-level m16n8k16 matrix instruction.  S = Q K^T takes Q and K with the head
// dimension in the same permuted order (lane t of a quad holds 8 contiguous values of every 32), 16 contiguous bytes
// a load.  O^T += V^T P^T: a lane's P, rounded to the inputs' type as the instruction asks, is its second operand as it
// stands, V is transposed on the way from shared memory, and eight query rows fill the instruction's narrow side.  The
// partial results are joined by log-sum-exp through distributed shared memory, in a fixed order.
//
// 8 x 8 key heads of 4096 keys x 128, four query heads each, nothing in L2: 23.8 us (134 MB, 5.6 TB/s; 20.8 us at the copy
// rate); 16384 keys 78 us (6.9 TB/s).  About 3.5 us are the launch, the first copies and the joins: 256 keys take 5 us.
// Measured and slower at 4096 keys: K and V loaded straight into registers with P V as f32 multiply-adds (40 us,
// bound by its instructions: 134 at 16384), the same arithmetic from the ring (41 us), eight such warps and a ring of
// 128 KB in one CTA per SM (25.5 us, and 11.4 instead of 10.0 at 1024), a ring of six stages (24.4 us; six warps
// on it 25.6 us), partial results read remotely instead of written (25.4 us; 17.5 instead of 6.3 for 16 rows of 64 keys).
#include <cuda_fp16.h>

#include <algorithm>

#include "common.cuh"
#include "found_once.h"
#include "kernels.h"

namespace {
using namespace dfl;

constexpr int kMaxSplits = 16, kMaxRows = 512;
constexpr int kKeys = 16;  // per warp and step
constexpr int kWarps = 4, kGroups = kWarps / 2;  // a pair of warps shares a stage, the pairs take the stages in turn
constexpr int kStageKeys = 2 * kKeys, kStages = 4;
static_assert(kStages % kGroups == 0, "a slot always serves the same warps, whose waits then follow every phase of it");
constexpr float kLog2e = 1.4426950408889634f;

DFL_DEVICE float exp2_sfu(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
DFL_DEVICE void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
DFL_DEVICE void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
// Stores to the same place in the shared memory of CTA `rank` of the cluster.
DFL_DEVICE uint32_t cluster_addr(const void* p, uint32_t rank) {
  uint32_t a;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem_u32(p)), "r"(rank));
  return a;
}
DFL_DEVICE void st_cluster(float2* p, uint32_t rank, float2 v) {
  asm volatile("st.shared::cluster.v2.f32 [%0], {%1, %2};" ::"r"(cluster_addr(p, rank)), "f"(v.x), "f"(v.y) : "memory");
}
DFL_DEVICE void st_cluster(float4* p, uint32_t rank, float4 v) {
  asm volatile("st.shared::cluster.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(cluster_addr(p, rank)), "f"(v.x), "f"(v.y), "f"(v.z),
               "f"(v.w)
               : "memory");
}

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

// Score of (row, key) after the mask: -inf when excluded.
DFL_DEVICE float masked_score(const DecodeArgs& a, float s, int b, int h, int q, int k) {
  const float z = s * a.scale;
  if (a.mask == nullptr) return z;
  const long long at = b * a.m_bs + h * a.m_hs + q * a.m_qs + k * a.m_ks;
  if (a.mask_dtype < 0) return reinterpret_cast<const uint8_t*>(a.mask)[at] ? z : -INFINITY;
  const float m = a.mask_dtype == kDtypeF32 ? reinterpret_cast<const float*>(a.mask)[at]
                  : a.mask_dtype == kDtypeBf16 ? __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(a.mask)[at])
                                               : __half2float(reinterpret_cast<const __half*>(a.mask)[at]);
  return fmaf(s, a.scale, m);
}

template <bool F16>
DFL_DEVICE uint32_t pack2(float lo, float hi) {
  if constexpr (F16) {
    __half2 v = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<uint32_t*>(&v);
  } else {
    return pack_bf16x2(lo, hi);
  }
}

// What a part of the keys with maximum m and sum l counts in a whole of maximum mu.
DFL_DEVICE float part_weight(float m, float l, float mu) { return m == -INFINITY && l == 0.f ? 0.f : exp2_sfu((m - mu) * kLog2e); }

// Joins the warps' results (maxima and sums s_ml, rows s_o) in this CTA, then the CTAs of the cluster, and stores the
// rows.  Every CTA writes its share of each quarter row into the CTA that stores it (c_o: R dh / splits values
// from each, c_ml: every CTA's maxima and sums), so one cluster barrier is waited for and nothing is read remotely.
template <int DH, bool F16, class SO>
DFL_DEVICE void decode_join(const DecodeArgs& a, int hk, int r0, int R, const float2 (&s_ml)[kWarps][16], SO s_o, float4* c_o,
                            float2 (&c_ml)[kMaxSplits][16]) {
  const int splits = gridDim.x, split = blockIdx.x, b = blockIdx.z, rep = a.H / a.Hk;
  const int n4 = R * (DH / 4), share = n4 / splits;  // splits divides dh / 4
  __syncthreads();
  if (splits > 1) cluster_wait();  // every CTA of the cluster has started
  for (int i = threadIdx.x; i < n4; i += blockDim.x) {
    const int r = i / (DH / 4), d = i % (DH / 4) * 4;
    float mx = s_ml[0][r].x;
#pragma unroll
    for (int w = 1; w < kWarps; ++w) mx = fmaxf(mx, s_ml[w][r].x);
    const float mu = mx == -INFINITY ? 0.f : mx;
    float4 ov = make_float4(0.f, 0.f, 0.f, 0.f);
    float lv = 0.f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const float f = part_weight(s_ml[w][r].x, s_ml[w][r].y, mu);
      const float4 x = *reinterpret_cast<const float4*>(&s_o[w][r][d]);
      ov.x += f * x.x, ov.y += f * x.y, ov.z += f * x.z, ov.w += f * x.w;
      lv += f * s_ml[w][r].y;
    }
    st_cluster(&c_o[split * share + i % share], i / share, ov);
    // a row's pieces tell one CTA each of its maximum and sum (there are as many pieces as that or more)
    if (d / 4 < splits) st_cluster(&c_ml[split][r], d / 4, make_float2(mx, lv));
  }
  if (splits > 1) {
    __syncwarp();
    cluster_arrive();
    cluster_wait();
  } else {
    __syncthreads();
  }
  for (int i = threadIdx.x; i < share; i += blockDim.x) {
    const int r = (split * share + i) / (DH / 4), d = (split * share + i) % (DH / 4) * 4;
    float mx = -INFINITY;
    for (int c = 0; c < splits; ++c) mx = fmaxf(mx, c_ml[c][r].x);
    const float mu = mx == -INFINITY ? 0.f : mx;
    float4 ov = make_float4(0.f, 0.f, 0.f, 0.f);
    float lv = 0.f;
#pragma unroll 4
    for (int c = 0; c < splits; ++c) {
      const float2 ml = c_ml[c][r];
      const float f = part_weight(ml.x, ml.y, mu);
      const float4 x = c_o[c * share + i];
      ov.x += f * x.x, ov.y += f * x.y, ov.z += f * x.z, ov.w += f * x.w;
      lv += f * ml.y;
    }
    const float inv = lv == 0.f ? 0.f : 1.f / lv;
    const int h = hk * rep + (r0 + r) / a.Sq, q = (r0 + r) % a.Sq;
    const uint2 y = make_uint2(pack2<F16>(ov.x * inv, ov.y * inv), pack2<F16>(ov.z * inv, ov.w * inv));
    *reinterpret_cast<uint2*>(reinterpret_cast<uint16_t*>(a.o) + b * a.o_bs + (long long)h * a.o_hs + (long long)q * a.o_ss + d) = y;
    if (a.lse && d == 0) a.lse[((long long)b * a.H + h) * a.Sq + q] = lv == 0.f ? -INFINITY : mx + logf(lv);
  }
}

DFL_DEVICE void tma_load_4d(uint8_t* dst, const CUtensorMap* map, uint64_t* bar, int c0, int c1, int c2, int c3) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%3, %4, %5, %6}], [%2];" ::"r"(smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(smem_u32(bar)), "r"(c0), "r"(c1), "r"(c2), "r"(c3)
      : "memory");
}
// Four 8 x 8 matrices of 16-bit values, transposed: lane l names row l % 8 of matrix l / 8.
DFL_DEVICE void ldmatrix_x4_trans(uint32_t (&r)[4], const uint8_t* p) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(smem_u32(p))
               : "memory");
}
// NB: blocks of eight query rows.  The last warp fills the ring.
template <int DH, bool F16, int NB>
__global__ void __launch_bounds__(32 * (kWarps + 1), 2)
    cross_decode_kernel(const __grid_constant__ CUtensorMap tk, const __grid_constant__ CUtensorMap tv, const DecodeArgs a) {
  constexpr int KC = DH / 32, DT = DH / 16;
  constexpr int kTile = kStageKeys * DH * 2, kChunk = kStageKeys * 128;
  static_assert(kWarps * 8 * NB * DH * 4 <= kStages * 2 * kTile, "the warps' results take the stages' place");
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  float(*s_o)[8 * NB][DH] = reinterpret_cast<float(*)[8 * NB][DH]>(smem);
  __shared__ float2 s_ml[kWarps][16], c_ml[kMaxSplits][16];
  __shared__ float4 c_o[2 * NB * DH];
  __shared__ uint64_t full[kStages], empty[kStages];
  __shared__ int aborted;
  volatile int* abort_flag = &aborted;

  if (gridDim.x > 1) cluster_arrive();  // waited for before the first remote write
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, quad = lane / 4, t = lane % 4;
  const int splits = gridDim.x, split = blockIdx.x, b = blockIdx.z;
  const int rep = a.H / a.Hk, groups = gridDim.y / a.Hk, hk = blockIdx.y / groups;
  const int r0 = blockIdx.y % groups * (8 * NB), R = min(8 * NB, rep * a.Sq - r0);  // this CTA's rows of the key head
  if (threadIdx.x == 0) {
    for (int i = 0; i < kStages; ++i) mbar_init(&full[i], 1), mbar_init(&empty[i], 2);
    aborted = 0;
    fence_barrier_init();
    fence_proxy_async_shared();
  }
  griddep_wait();  // (launched while the kernel before it ends)
  const int lo = a.kv_lo ? max(0, a.kv_lo[b]) : 0, hi = a.kv_hi ? min(a.Sk, a.kv_hi[b]) : a.Sk;
  const int nb = hi > lo ? (hi - lo + kStageKeys - 1) / kStageKeys : 0;
  __syncthreads();

  if (warp == kWarps) {
    if (lane == 0) {
      int i = 0;
      for (int blk = split; blk < nb; blk += splits, ++i) {
        const int slot = i % kStages, k0 = lo + blk * kStageKeys;
        if (!mbar_wait(&empty[slot], ((i / kStages) & 1) ^ 1u, a.err, kKidCross, 150 + slot, abort_flag)) break;
        uint8_t* st = smem + slot * 2 * kTile;
        mbar_arrive_expect_tx(&full[slot], 2 * kTile);
#pragma unroll
        for (int c = 0; c < DH / 64; ++c) tma_load_4d(st + c * kChunk, &tk, &full[slot], 64 * c, k0, hk, b);
#pragma unroll
        for (int c = 0; c < DH / 64; ++c) tma_load_4d(st + kTile + c * kChunk, &tv, &full[slot], 64 * c, k0, hk, b);
      }
      for (int k = max(0, i - kStages); k < i; ++k)  // every copy has landed before the stages are used otherwise
        mbar_wait(&full[k % kStages], (k / kStages) & 1, nullptr, 0, 0, nullptr, 200000000LL);
    }
    __syncwarp();
    __syncthreads();
  } else {
    uint4 qf[KC][NB];  // rows quad and quad + 8
    int hrow[NB], qrow[NB];
#pragma unroll
    for (int h = 0; h < NB; ++h) {
      const int r = quad + 8 * h;
      hrow[h] = hk * rep + (r0 + r) / a.Sq, qrow[h] = (r0 + r) % a.Sq;
      const uint16_t* qp = reinterpret_cast<const uint16_t*>(a.q) + b * a.q_bs + (long long)hrow[h] * a.q_hs +
                           (long long)qrow[h] * a.q_ss;
#pragma unroll
      for (int c = 0; c < KC; ++c)
        qf[c][h] = r < R ? *reinterpret_cast<const uint4*>(qp + 32 * c + 8 * t) : make_uint4(0u, 0u, 0u, 0u);
    }
    float m[NB], l[NB];
    float o[NB][DT][4];  // [2 j + e]: column 16 dt + quad + 8 j of row 8 h + 2 t + e
#pragma unroll
    for (int h = 0; h < NB; ++h) {
      m[h] = -INFINITY, l[h] = 0.f;
#pragma unroll
      for (int d = 0; d < DT; ++d) o[h][d][0] = o[h][d][1] = o[h][d][2] = o[h][d][3] = 0.f;
    }
    const bool by_bool = a.mask != nullptr && a.mask_dtype < 0;
    // row and 16-byte piece that this lane names to ldmatrix: columns + 0 | + 8 of keys 0-7, then of keys 8-15
    const int vrow = (lane / 16) * 8 + lane % 8, vcol = lane / 8 % 2;

    int i = 0;
    for (int blk = split; blk < nb; blk += splits, ++i) {
      if (i % kGroups != warp / 2) continue;
      const int slot = i % kStages, row0 = 16 * (warp % 2), k0 = lo + blk * kStageKeys + row0, left = hi - k0;
      if (!mbar_wait_warp(&full[slot], (i / kStages) & 1, a.err, kKidCross, 160 + slot, abort_flag)) break;
      if (left > 0) {
        // 128-byte rows in the copies' swizzle: 16-byte piece p of row r lies at p ^ (r % 8)
        uint8_t* st = smem + slot * 2 * kTile + row0 * 128;
        float s[2][4], s2[2][4];  // two chains of products each: the instruction's latency is what one alone would show
#pragma unroll
        for (int n = 0; n < 2; ++n) {
#pragma unroll
          for (int e = 0; e < 4; ++e) s[n][e] = s2[n][e] = 0.f;
#pragma unroll
          for (int c = 0; c < KC; ++c) {
            const uint4 k = *reinterpret_cast<const uint4*>(st + (c / 2) * kChunk + (8 * n + quad) * 128 + ((((c & 1) * 4 + t) ^ quad) * 16));
            const uint4 q0 = qf[c][0], q1 = NB == 2 ? qf[c][NB - 1] : make_uint4(0u, 0u, 0u, 0u);
            mma16816<F16>(s[n], q0.x, q1.x, q0.y, q1.y, k.x, k.y);
            mma16816<F16>(s2[n], q0.z, q1.z, q0.w, q1.w, k.z, k.w);
          }
#pragma unroll
          for (int e = 0; e < 2 * NB; ++e) s[n][e] += s2[n][e];
        }
        // s[n][2 h + e]: row quad + 8 h, key 8 n + 2 t + e
        const bool plain = a.mask == nullptr && left >= kKeys;  // (rows past R are not stored, whatever they hold)
        float f[NB];
        bool moved = false;
#pragma unroll
        for (int h = 0; h < NB; ++h) {
          float mx = -INFINITY;
#pragma unroll
          for (int n = 0; n < 2; ++n)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const int key = 8 * n + 2 * t + e;
              float& z = s[n][2 * h + e];
              if (plain) z *= a.scale;
              else z = quad + 8 * h < R && key < left ? masked_score(a, z, b, hrow[h], qrow[h], k0 + key) : -INFINITY;
              mx = fmaxf(mx, z);
            }
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
          mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
          // the old maximum serves until it is exceeded by 5 (P stays below 2^8, the sums are exact all the same)
          f[h] = 1.f;
          if (mx > m[h] + 5.f) {
            f[h] = m[h] == -INFINITY ? 0.f : exp2_sfu((m[h] - mx) * kLog2e);
            m[h] = mx;
            moved = true;
          }
        }
        uint32_t keep[2][2];
        if (by_bool) {
#pragma unroll
          for (int n = 0; n < 2; ++n)
#pragma unroll
            for (int e = 0; e < 2; ++e)
              keep[n][e] = __ballot_sync(0xffffffffu, s[n][e] != -INFINITY || (NB == 2 && s[n][2 + e] != -INFINITY));
        }
        uint32_t p[NB][2];
#pragma unroll
        for (int h = 0; h < NB; ++h) {
          const float mu = m[h] == -INFINITY ? 0.f : m[h];
          float sum = 0.f;
#pragma unroll
          for (int n = 0; n < 2; ++n) {
            const float p0 = exp2_sfu((s[n][2 * h] - mu) * kLog2e), p1 = exp2_sfu((s[n][2 * h + 1] - mu) * kLog2e);
            sum += p0 + p1;
            p[h][n] = pack2<F16>(p0, p1);
          }
          l[h] = l[h] * f[h] + sum;
        }
        if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
          for (int h = 0; h < NB; ++h) {
            const float f0 = __shfl_sync(0xffffffffu, f[h], 8 * t), f1 = __shfl_sync(0xffffffffu, f[h], 8 * t + 4);
#pragma unroll
            for (int d = 0; d < DT; ++d) o[h][d][0] *= f0, o[h][d][1] *= f1, o[h][d][2] *= f0, o[h][d][3] *= f1;
          }
        }
        uint8_t* sv = st + kTile;
        if (left < kKeys || by_bool) {
          // what V holds at keys that no row keeps is not used: those rows become 0 (a product with P = 0 would
          // pass a NaN on)
          bool drop = lane < 16 && lane >= left;
          if (by_bool && lane < 16) {
            const uint32_t any = lane < 8 ? (lane & 1 ? keep[0][1] : keep[0][0]) : (lane & 1 ? keep[1][1] : keep[1][0]);
            drop = drop || !(any & (0x11111111u << (lane % 8 / 2)));
          }
          if (drop)
#pragma unroll
            for (int c = 0; c < DH / 8; ++c)
              *reinterpret_cast<uint4*>(sv + (c / 8) * kChunk + lane * 128 + (c % 8) * 16) = make_uint4(0u, 0u, 0u, 0u);
          fence_proxy_async_shared();  // before the stage's next copy
          __syncwarp();
        }
        // O^T += V^T P^T: P is laid out as the instruction's second operand already, V is transposed on its way
#pragma unroll
        for (int d = 0; d < DT; ++d) {
          uint32_t v[4];
          const int piece = 2 * d + vcol;  // of 8 columns
          ldmatrix_x4_trans(v, sv + (piece / 8) * kChunk + vrow * 128 + (((piece % 8) ^ (vrow & 7)) * 16));
#pragma unroll
          for (int h = 0; h < NB; ++h) mma16816<F16>(o[h][d], v[0], v[1], v[2], v[3], p[h][0], p[h][1]);
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&empty[slot]);
    }
    __syncwarp();
    __syncthreads();  // every stage has been read: the results take their place
#pragma unroll
    for (int h = 0; h < NB; ++h) {
      l[h] += __shfl_xor_sync(0xffffffffu, l[h], 1);
      l[h] += __shfl_xor_sync(0xffffffffu, l[h], 2);
      if (t == 0) s_ml[warp][quad + 8 * h] = make_float2(m[h], l[h]);
#pragma unroll
      for (int d = 0; d < DT; ++d)
#pragma unroll
        for (int j = 0; j < 4; ++j) s_o[warp][8 * h + 2 * t + j % 2][16 * d + quad + 8 * (j / 2)] = o[h][d][j];
    }
  }
  decode_join<DH, F16>(a, hk, r0, R, s_ml, s_o, c_o, c_ml);
}

int decode_tmap(CUtensorMap* map, const void* base, const DecodeArgs* a, long long ss, long long hs, long long bs) {
  dfl_host::EncodeTiledFn fn = dfl_host::get_encode_tiled();
  if (!fn) return 999;
  cuuint64_t dims[4] = {(cuuint64_t)a->dh, (cuuint64_t)a->Sk, (cuuint64_t)a->Hk, (cuuint64_t)a->B};
  cuuint64_t strides[3] = {(cuuint64_t)ss * 2, (cuuint64_t)hs * 2, (cuuint64_t)bs * 2};
  cuuint32_t box[4] = {64, (cuuint32_t)kStageKeys, 1, 1};
  cuuint32_t estr[4] = {1, 1, 1, 1};
  return (int)fn(map, a->f16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, const_cast<void*>(base),
                 dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                 CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
}

// Clusters of 1, 2, 4, 8 or 16 CTAs that are resident together (0: this size cannot be launched), found once per device.
struct Resident {
  int clusters[5] = {0, 0, 0, 0, 0};
};

int rows_of(const DecodeArgs* a) { return a->H / a->Hk * a->Sq; }
int groups_of(const DecodeArgs* a) { return (rows_of(a) + 15) / 16; }
int smem_bytes(int dh) { return kStages * 2 * kStageKeys * dh * 2 + 1024; }

// How one call is laid out: CTAs per group of rows, and what that is expected to take, in 11 ns.
struct Plan {
  int splits;
  long long cost;
};

template <int DH, bool F16, int NB>
int plan_decode(const DecodeArgs* a, Plan* plan) {
  static dfl_host::FoundOnce<Resident> resident[16];
  int dev = 0;
  cudaGetDevice(&dev);
  Resident res;
  const int rc = resident[dev & 15].get(&res, [&](Resident* r) {
    auto kern = cross_decode_kernel<DH, F16, NB>;
    cudaLaunchConfig_t cfg = {};
    cfg.blockDim = dim3(32 * (kWarps + 1), 1, 1);
    cfg.dynamicSmemBytes = smem_bytes(DH);
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)cfg.dynamicSmemBytes);
    if (e == cudaSuccess) e = cudaFuncSetAttribute(kern, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    for (int i = 0; i < 5 && e == cudaSuccess; ++i) {
      at[0].val.clusterDim.x = 1 << i;
      cfg.gridDim = dim3((unsigned)(1 << i), 1024, 1);
      e = cudaOccupancyMaxActiveClusters(&r->clusters[i], kern, &cfg);
    }
    return (int)e;
  });
  if (rc) return rc;
  // CTAs per key head: each wave of clusters costs its keys per CTA and a launch, ramp and join worth about 300 keys of
  // 128 values; no CTA gets less than a turn of its warps.  64 heads of 4096 keys take 4 (1, 2, 4, 8, 16: 52, 30, 24, 28,
  // 42 us), 72 of 512 take 2 (9.0, 6.8, 9.6, 12.8, 25 us), 48 of 4096 x 64 take 8 (45, 25, 16, 12, 22 us), 480 of 1024
  // take 1 (43, 53, 60, 87, 172 us).
  const long long heads = (long long)a->B * a->Hk * groups_of(a);
  plan->cost = -1;
  for (int i = 0; i < 5; ++i) {
    const long long fit = res.clusters[i], keys = (a->Sk + (1 << i) - 1) >> i;
    if (fit <= 0 || (i > 0 && keys < kGroups * kStageKeys)) continue;
    const long long cost = (heads + fit - 1) / fit * (keys + 300 * 128 / DH);
    if (plan->cost < 0 || cost < plan->cost) plan->cost = cost, plan->splits = 1 << i;
  }
  return 0;
}

template <int DH, bool F16, int NB>
int launch_decode(const DecodeArgs* a, cudaStream_t stream) {
  Plan plan;
  int rc = plan_decode<DH, F16, NB>(a, &plan);
  if (rc) return rc;
  CUtensorMap tk, tv;
  rc = decode_tmap(&tk, a->k, a, a->k_ss, a->k_hs, a->k_bs);
  if (rc) return 1000 + rc;
  rc = decode_tmap(&tv, a->v, a, a->v_ss, a->v_hs, a->v_bs);
  if (rc) return 2000 + rc;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(plan.splits, a->Hk * groups_of(a), a->B);
  cfg.blockDim = dim3(32 * (kWarps + 1), 1, 1);
  cfg.dynamicSmemBytes = smem_bytes(DH);
  cfg.stream = stream;
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = plan.splits;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  at[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = 2;
  return (int)cudaLaunchKernelEx(&cfg, cross_decode_kernel<DH, F16, NB>, tk, tv, *a);
}

// Calls f<DH, F16, NB>(a, ...) for the call's head dim, type and rows.
#define DFL_DECODE(f, ...)                                                                              \
  (a->dh == 64 ? (a->f16 ? (rows_of(a) <= 8 ? f<64, true, 1>(a, __VA_ARGS__) : f<64, true, 2>(a, __VA_ARGS__))       \
                         : (rows_of(a) <= 8 ? f<64, false, 1>(a, __VA_ARGS__) : f<64, false, 2>(a, __VA_ARGS__)))    \
               : (a->f16 ? (rows_of(a) <= 8 ? f<128, true, 1>(a, __VA_ARGS__) : f<128, true, 2>(a, __VA_ARGS__))     \
                         : (rows_of(a) <= 8 ? f<128, false, 1>(a, __VA_ARGS__) : f<128, false, 2>(a, __VA_ARGS__))))

}  // namespace

extern "C" int dfl_cross_decode_takes(const DecodeArgs* a) {
  if ((a->dh != 64 && a->dh != 128) || a->B <= 0 || a->Hk <= 0 || a->Sq <= 0 || a->Sk <= 0 || a->H % a->Hk) return 0;
  const long long rows = (long long)a->H / a->Hk * a->Sq;
  if (rows > kMaxRows || a->B > 65535 || a->Hk * ((rows + 15) / 16) > 65535) return 0;
  if (rows <= 16) return 1;
  // More rows read the keys once per 16 of them, while the other kernel gives 128 rows of a head, or 256, to a CTA that walks
  // all the keys: that leaves SMs idle where there are few tiles.  In ns: a key takes 12.5 there (20% more with a mask, which
  // it lays out first) and 4300 go to the rest; here 17 or 11 by head dim (80% more with a mask, read value by value).
  //   16 heads x 78 x 2355 x 64: 32.2 us there, 13.5 here; 12 x 17 x 4096 x 128: 55.8, 13.6; 32 x 64 x 4096 x 128: 56.6, 38.7
  //   (additive mask 65.9, 76.0); 96 x 20 x 512 x 128: 11.0, 14.3; 128 x 17 x 2000 x 64: 29.0, 30.9
  if (rows > 128 && a->Sk < 1024) return 0;
  Plan plan;
  if (DFL_DECODE(plan_decode, &plan)) return 0;
  int dev = 0;
  cudaGetDevice(&dev);
  const long long tiles = (long long)a->B * a->H * (a->Sq > 128 ? (a->Sq + 255) / 256 : 1), sms = dfl_host::num_sms(dev);
  const double here = plan.cost * (a->dh == 64 ? 11. : 17.) * (a->mask ? 1.8 : 1.);
  const double there = (double)((tiles + sms - 1) / sms) * (4300. + 12.5 * a->Sk) * (a->mask ? 1.2 : 1.);
  return here < 0.95 * there;
}

extern "C" int dfl_cross_decode(const DecodeArgs* a, cudaStream_t stream) {
  if (a->dh != 64 && a->dh != 128) return -2;
  if (a->B <= 0 || a->H <= 0 || a->Hk <= 0 || a->Sq <= 0 || a->Sk <= 0 || a->H % a->Hk) return -3;
  if ((long long)a->H / a->Hk * a->Sq > kMaxRows || a->B > 65535 || (long long)a->Hk * groups_of(a) > 65535) return -8;
  auto al16 = [](const void* ptr) { return (reinterpret_cast<uintptr_t>(ptr) & 15) == 0; };
  if (!al16(a->q) || !al16(a->k) || !al16(a->v) || !al16(a->o)) return -4;
  if ((a->q_ss | a->q_hs | a->q_bs | a->k_ss | a->k_hs | a->k_bs | a->v_ss | a->v_hs | a->v_bs | a->o_ss | a->o_hs |
       a->o_bs) % 8)
    return -5;
  return DFL_DECODE(launch_decode, stream);
}
