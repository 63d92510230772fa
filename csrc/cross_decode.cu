// Attention of a few queries to many keys (single tokens, pooling queries): at most 16 query rows
// share a key head.  sm_100a.
//
// Bound by reading K and V once: a 128-row tensor-memory tile would be nearly empty, so the keys are
// split over up to eight CTAs (one cluster per key head and batch row) of four warps, and each warp walks
// its own 16-key blocks with a running maximum and sum.  Q K^T runs on the warp-level m16n8k16 matrix
// instruction straight from registers: both operands take the head dimension in the same permuted
// order (lane t of a quad holds 8 contiguous values of every 32), so every load is 16 contiguous bytes and nothing is
// staged.  P V is f32 multiply-adds, a lane holding dh / 32 columns of every row, with P unrounded.  The partial
// results are joined by log-sum-exp through distributed shared memory, in a fixed order.
//
// 8 x 8 key heads of up to 3276 keys x 128, four query heads each: 25 us (84 MB, 3.4 TB/s; 13 us at the copy rate).
// About 6 us of it are the launch and the joins; the rest runs at 4.4 TB/s, four CTAs of 128 registers per SM being
// what the loads in flight allow.  Measured and slower: 32-key blocks with fewer CTAs (31 us), the next block's
// loads issued into the registers as they come free (35 us).
#include <cuda_fp16.h>

#include "common.cuh"
#include "kernels.h"

namespace {
using namespace dfl;

constexpr int kWarps = 4, kMaxSplits = 8;
constexpr int kKeys = 16;  // per warp and step: its K and V (8 KB at dh 128) are in flight together
constexpr float kLog2e = 1.4426950408889634f;

DFL_DEVICE float exp2_sfu(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
DFL_DEVICE uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
DFL_DEVICE void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
DFL_DEVICE float ld_cluster(const float* p, uint32_t rank) {
  uint32_t a;
  float v;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"(smem_u32(p)), "r"(rank));
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(a));
  return v;
}

// Packed f32 pairs.
DFL_DEVICE uint64_t f2_pack(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
DFL_DEVICE uint64_t f2_fma(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
DFL_DEVICE uint64_t f2_mul(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
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

template <bool F16>
DFL_DEVICE float2 unpack2(uint32_t v) {
  if constexpr (F16) return __half22float2(*reinterpret_cast<__half2*>(&v));
  else return unpack_bf16x2(v);
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

// NR: rows held by the P V accumulators (4, 8 or 16).
template <int DH, bool F16, int NR>
__global__ void __launch_bounds__(32 * kWarps, NR == 4 ? 4 : NR == 8 ? 3 : 2) cross_decode_kernel(const DecodeArgs a) {
  constexpr int KC = DH / 32;  // 16-byte pieces of a key row per lane
  constexpr int DL = DH / 32;  // output columns per lane
  // P of the block a warp is at, every value twice (the packed multiply-add takes pairs); later this CTA's joined
  // rows, read by the cluster
  constexpr int kBuf = kWarps * NR * kKeys * 2 > NR * DH ? kWarps * NR * kKeys * 2 : NR * DH;
  __shared__ __align__(16) float s_buf[kBuf];
  float(*s_p)[NR][kKeys * 2] = reinterpret_cast<float(*)[NR][kKeys * 2]>(s_buf);
  float(*c_o)[DH] = reinterpret_cast<float(*)[DH]>(s_buf);
  __shared__ float s_f[kWarps][16];               // rescaling of the rows, then their maxima
  __shared__ float s_l[kWarps][16];
  __shared__ __align__(16) float s_o[kWarps][NR][DH];
  __shared__ float c_m[16], c_l[16];

  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32, quad = lane / 4, t = lane % 4;
  const int splits = gridDim.x, split = blockIdx.x, hk = blockIdx.y, b = blockIdx.z;
  const int rep = a.H / a.Hk, R = rep * a.Sq;
  const int lo = a.kv_lo ? max(0, a.kv_lo[b]) : 0, hi = a.kv_hi ? min(a.Sk, a.kv_hi[b]) : a.Sk;
  const uint16_t* kp = reinterpret_cast<const uint16_t*>(a.k) + b * a.k_bs + hk * a.k_hs;
  const uint16_t* vp = reinterpret_cast<const uint16_t*>(a.v) + b * a.v_bs + hk * a.v_hs;
  auto head_of = [&](int r) { return hk * rep + r / a.Sq; };
  auto query_of = [&](int r) { return r % a.Sq; };

  uint4 qf[KC][2];  // rows quad and quad + 8
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int r = quad + 8 * i;
    const uint16_t* qp = reinterpret_cast<const uint16_t*>(a.q) + b * a.q_bs + (long long)head_of(r) * a.q_hs +
                         (long long)query_of(r) * a.q_ss;
#pragma unroll
    for (int c = 0; c < KC; ++c)
      qf[c][i] = r < R ? *reinterpret_cast<const uint4*>(qp + 32 * c + 8 * t) : make_uint4(0u, 0u, 0u, 0u);
  }
  float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
  uint64_t o[NR][DL / 2];  // pairs of columns
#pragma unroll
  for (int r = 0; r < NR; ++r)
#pragma unroll
    for (int d = 0; d < DL / 2; ++d) o[r][d] = 0ull;

  // blocks of the window, dealt to the warps of all splits in turn
  const int nb = hi > lo ? (hi - lo + kKeys - 1) / kKeys : 0;
  for (int blk = split * kWarps + warp; blk < nb; blk += splits * kWarps) {
    const int k0 = lo + blk * kKeys, left = hi - k0;  // keys of this block (kKeys or more: all)
    uint4 kf[kKeys / 8][KC];
    const uint16_t* kb = kp + (long long)(k0 + quad) * a.k_ss + 8 * t;
#pragma unroll
    for (int n = 0; n < kKeys / 8; ++n)
#pragma unroll
      for (int c = 0; c < KC; ++c)
        kf[n][c] = 8 * n + quad < left ? __ldg(reinterpret_cast<const uint4*>(kb + 8 * n * a.k_ss + 32 * c)) : make_uint4(0u, 0u, 0u, 0u);
    uint32_t vf[kKeys][DL / 2];  // on its way during the scores
    const uint16_t* vb = vp + (long long)k0 * a.v_ss + lane * DL;
#pragma unroll
    for (int k = 0; k < kKeys; ++k) {
      if constexpr (DL == 4) {
        const uint2 x = k < left ? __ldg(reinterpret_cast<const uint2*>(vb + k * a.v_ss)) : make_uint2(0u, 0u);
        vf[k][0] = x.x, vf[k][1] = x.y;
      } else {
        vf[k][0] = k < left ? __ldg(reinterpret_cast<const uint32_t*>(vb + k * a.v_ss)) : 0u;
      }
    }
    float s[kKeys / 8][4];
#pragma unroll
    for (int n = 0; n < kKeys / 8; ++n) {
      s[n][0] = s[n][1] = s[n][2] = s[n][3] = 0.f;
#pragma unroll
      for (int c = 0; c < KC; ++c) {
        mma16816<F16>(s[n], qf[c][0].x, qf[c][1].x, qf[c][0].y, qf[c][1].y, kf[n][c].x, kf[n][c].y);
        mma16816<F16>(s[n], qf[c][0].z, qf[c][1].z, qf[c][0].w, qf[c][1].w, kf[n][c].z, kf[n][c].w);
      }
    }
    // s[n][2 i + e]: row quad + 8 i, key 8 n + 2 t + e
#pragma unroll
    for (int i = 0; i < (NR + 7) / 8; ++i) {
      const int r = quad + 8 * i;
      if (8 * i >= R) continue;  // (uniform: no row of this half exists)
      const int h = head_of(r), q = query_of(r);
      float mx = m[i];
#pragma unroll
      for (int n = 0; n < kKeys / 8; ++n)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int key = 8 * n + 2 * t + e;
          float& z = s[n][2 * i + e];
          z = r < R && key < left ? masked_score(a, z, b, h, q, k0 + key) : -INFINITY;
          mx = fmaxf(mx, z);
        }
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
      mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
      const float mu = mx == -INFINITY ? 0.f : mx;
      const float f = m[i] == -INFINITY ? 0.f : exp2_sfu((m[i] - mu) * kLog2e);
      m[i] = mx;
      l[i] *= f;
#pragma unroll
      for (int n = 0; n < kKeys / 8; ++n) {
        const float p0 = exp2_sfu((s[n][2 * i] - mu) * kLog2e), p1 = exp2_sfu((s[n][2 * i + 1] - mu) * kLog2e);
        l[i] += p0 + p1;
        if (r < NR) *reinterpret_cast<float4*>(&s_p[warp][r][2 * (8 * n + 2 * t)]) = make_float4(p0, p0, p1, p1);
      }
      if (t == 0) s_f[warp][r] = f;
    }
    __syncwarp();
    if (a.mask != nullptr && a.mask_dtype < 0) {
      // a key that no row keeps adds nothing, whatever V holds there
#pragma unroll
      for (int k = 0; k < kKeys; ++k) {
        float any = 0.f;
#pragma unroll
        for (int r = 0; r < NR; ++r)
          if (r < R) any += s_p[warp][r][2 * k];
#pragma unroll
        for (int d = 0; d < DL / 2; ++d) vf[k][d] = any == 0.f ? 0u : vf[k][d];
      }
    }
#pragma unroll
    for (int r = 0; r < NR; ++r) {
      if (r >= R) continue;
      const float f = s_f[warp][r];
#pragma unroll
      for (int d = 0; d < DL / 2; ++d) o[r][d] = f2_mul(o[r][d], f2_pack(f, f));
    }
#pragma unroll
    for (int k = 0; k < kKeys; k += 2) {
      uint64_t v0[DL / 2], v1[DL / 2];
#pragma unroll
      for (int d = 0; d < DL / 2; ++d) {
        const float2 x = unpack2<F16>(vf[k][d]), y = unpack2<F16>(vf[k + 1][d]);
        v0[d] = f2_pack(x.x, x.y), v1[d] = f2_pack(y.x, y.y);
      }
#pragma unroll
      for (int r = 0; r < NR; ++r) {
        if (r >= R) continue;
        const ulonglong2 p = *reinterpret_cast<const ulonglong2*>(&s_p[warp][r][2 * k]);
#pragma unroll
        for (int d = 0; d < DL / 2; ++d) o[r][d] = f2_fma(p.y, v1[d], f2_fma(p.x, v0[d], o[r][d]));
      }
    }
    __syncwarp();
  }

  // join the warps of this CTA, then the CTAs of the cluster
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    l[i] += __shfl_xor_sync(0xffffffffu, l[i], 1);
    l[i] += __shfl_xor_sync(0xffffffffu, l[i], 2);
    if (t == 0) s_f[warp][quad + 8 * i] = m[i], s_l[warp][quad + 8 * i] = l[i];
  }
#pragma unroll
  for (int r = 0; r < NR; ++r)
#pragma unroll
    for (int d = 0; d < DL / 2; ++d) *reinterpret_cast<uint64_t*>(&s_o[warp][r][lane * DL + 2 * d]) = o[r][d];
  __syncthreads();
  for (int i = threadIdx.x; i < R * DH; i += 32 * kWarps) {
    const int r = i / DH, d = i % DH;
    float mx = s_f[0][r];
#pragma unroll
    for (int w = 1; w < kWarps; ++w) mx = fmaxf(mx, s_f[w][r]);
    const float mu = mx == -INFINITY ? 0.f : mx;
    float ov = 0.f, lv = 0.f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      if (s_f[w][r] == -INFINITY && s_l[w][r] == 0.f) continue;
      const float f = exp2_sfu((s_f[w][r] - mu) * kLog2e);
      ov += f * s_o[w][r][d];
      lv += f * s_l[w][r];
    }
    c_o[r][d] = ov;
    if (d == 0) c_m[r] = mx, c_l[r] = lv;
  }
  __syncthreads();
  if (splits > 1) cluster_sync();
  for (int i = threadIdx.x + 32 * kWarps * split; i < R * DH; i += 32 * kWarps * splits) {
    const int r = i / DH, d = i % DH;
    // all remote reads first: they are independent, and each takes most of a microsecond
    float mc[kMaxSplits], lc[kMaxSplits], oc[kMaxSplits];
    float mx = -INFINITY;
#pragma unroll
    for (int c = 0; c < kMaxSplits; ++c) {
      const bool in = c < splits;
      mc[c] = in ? (splits > 1 ? ld_cluster(&c_m[r], c) : c_m[r]) : -INFINITY;
      lc[c] = in ? (splits > 1 ? ld_cluster(&c_l[r], c) : c_l[r]) : 0.f;
      oc[c] = in ? (splits > 1 ? ld_cluster(&c_o[r][d], c) : c_o[r][d]) : 0.f;
    }
#pragma unroll
    for (int c = 0; c < kMaxSplits; ++c) mx = fmaxf(mx, mc[c]);
    const float mu = mx == -INFINITY ? 0.f : mx;
    float ov = 0.f, lv = 0.f;
#pragma unroll
    for (int c = 0; c < kMaxSplits; ++c) {
      if (mc[c] == -INFINITY && lc[c] == 0.f) continue;
      const float f = exp2_sfu((mc[c] - mu) * kLog2e);
      ov += f * oc[c];
      lv += f * lc[c];
    }
    const float y = lv == 0.f ? 0.f : ov / lv;
    const long long at = b * a.o_bs + (long long)head_of(r) * a.o_hs + (long long)query_of(r) * a.o_ss + d;
    if constexpr (F16) reinterpret_cast<__half*>(a.o)[at] = __float2half_rn(y);
    else reinterpret_cast<__nv_bfloat16*>(a.o)[at] = __float2bfloat16_rn(y);
    if (a.lse && d == 0)
      a.lse[((long long)b * a.H + head_of(r)) * a.Sq + query_of(r)] = lv == 0.f ? -INFINITY : mx + logf(lv);
  }
  if (splits > 1) cluster_sync();  // no CTA leaves while its results may be read
}

template <int DH, bool F16, int NR>
int launch_decode(const DecodeArgs* a, int splits, cudaStream_t stream) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(splits, a->Hk, a->B);
  cfg.blockDim = dim3(32 * kWarps, 1, 1);
  cfg.stream = stream;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = splits;
  at[0].val.clusterDim.y = 1;
  at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  return (int)cudaLaunchKernelEx(&cfg, cross_decode_kernel<DH, F16, NR>, *a);
}

template <int DH, bool F16>
int decode_rows(const DecodeArgs* a, int splits, cudaStream_t stream) {
  const int R = a->H / a->Hk * a->Sq;
  if (R <= 4) return launch_decode<DH, F16, 4>(a, splits, stream);
  if (R <= 8) return launch_decode<DH, F16, 8>(a, splits, stream);
  return launch_decode<DH, F16, 16>(a, splits, stream);
}

}  // namespace

extern "C" int dfl_cross_decode(const DecodeArgs* a, cudaStream_t stream) {
  if (a->dh != 64 && a->dh != 128) return -2;
  if (a->B <= 0 || a->H <= 0 || a->Hk <= 0 || a->Sq <= 0 || a->Sk <= 0 || a->H % a->Hk || a->H / a->Hk * a->Sq > 16) return -3;
  if (a->B > 65535 || a->Hk > 65535) return -8;
  auto al16 = [](const void* ptr) { return (reinterpret_cast<uintptr_t>(ptr) & 15) == 0; };
  if (!al16(a->q) || !al16(a->k) || !al16(a->v)) return -4;
  if ((a->q_ss | a->q_hs | a->q_bs | a->k_ss | a->k_hs | a->k_bs | a->v_ss | a->v_hs | a->v_bs) % 8) return -5;
  int dev = 0;
  cudaGetDevice(&dev);
  // CTAs per key head: as many as fill the SMs a few times over, each warp keeping a block or more
  const long long heads = (long long)a->B * a->Hk, room = 4ll * dfl_host::num_sms(dev);
  int splits = 1;
  while (splits < kMaxSplits && heads * splits * 2 <= room && a->Sk >= splits * 2 * kWarps * kKeys) splits *= 2;
  if (a->dh == 64) return a->f16 ? decode_rows<64, true>(a, splits, stream) : decode_rows<64, false>(a, splits, stream);
  return a->f16 ? decode_rows<128, true>(a, splits, stream) : decode_rows<128, false>(a, splits, stream);
}
