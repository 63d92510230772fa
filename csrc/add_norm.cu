// Residual RMSNorm with an optional MXFP8 output, and the MX dequantiser (sm_100a).
//
//   s = x + resid                                   (f32; resid may be absent)
//   y = s / sqrt(mean(s^2) + eps) [* w] [* (1 + scale[b])] [+ shift[b]]
//
// s is stored in the tensors' type, y in the same type or as FP8 elements with one power-of-two
// scale per 32 columns.  One pass: a row is read once into registers (f32), its sum of
// squares is reduced over the threads that share it, and both outputs are stored from the
// registers.  The norm uses the unrounded sum, and y is rounded once: to the output type, or
// (MX) straight from f32 to FP8.
//
// Bound by HBM: 8 bytes per value in bf16 (x, resid, s, y), 7.03 with the FP8 output.  At 32760 x 5120 bf16 takes
// 200 us (6.7 TB/s; a plain copy reaches 6.5), with adaLN modulation into MXFP8 206 us (5.7 TB/s: two words of
// scales per 128 columns and 40 KB of modulation a row through L1).  Measured and slower: a register cap for six
// or more blocks per SM, no-allocate loads, a persistent form fed by bulk copies.
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include "common.cuh"
#include "kernels.h"

namespace {
using namespace dfl;

template <typename T>
struct Io;  // 16-byte vectors of T to and from f32

template <>
struct Io<float> {
  static constexpr int E = 4;
  static DFL_DEVICE float ld(float v) { return v; }
  static DFL_DEVICE float st(float v) { return v; }
  static DFL_DEVICE void unpack(const uint4& w, float (&f)[4]) {
    f[0] = __uint_as_float(w.x), f[1] = __uint_as_float(w.y), f[2] = __uint_as_float(w.z), f[3] = __uint_as_float(w.w);
  }
  static DFL_DEVICE uint4 pack(const float (&f)[4]) {
    return make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
  }
};

template <>
struct Io<__nv_bfloat16> {
  static constexpr int E = 8;
  static DFL_DEVICE float ld(__nv_bfloat16 v) { return __bfloat162float(v); }
  static DFL_DEVICE __nv_bfloat16 st(float v) { return __float2bfloat16_rn(v); }
  static DFL_DEVICE void unpack(const uint4& w, float (&f)[8]) {
    const uint32_t ws[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int h = 0; h < 4; ++h) {
      const float2 t = unpack_bf16x2(ws[h]);
      f[2 * h] = t.x, f[2 * h + 1] = t.y;
    }
  }
  static DFL_DEVICE uint4 pack(const float (&f)[8]) {
    return make_uint4(pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3]), pack_bf16x2(f[4], f[5]),
                      pack_bf16x2(f[6], f[7]));
  }
};

DFL_DEVICE uint32_t pack_f16x2(float lo, float hi) {
  __half2 v = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<uint32_t*>(&v);
}

template <>
struct Io<__half> {
  static constexpr int E = 8;
  static DFL_DEVICE float ld(__half v) { return __half2float(v); }
  static DFL_DEVICE __half st(float v) { return __float2half_rn(v); }
  static DFL_DEVICE void unpack(const uint4& w, float (&f)[8]) {
    uint32_t ws[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int h = 0; h < 4; ++h) {
      const float2 t = __half22float2(*reinterpret_cast<__half2*>(&ws[h]));
      f[2 * h] = t.x, f[2 * h + 1] = t.y;
    }
  }
  static DFL_DEVICE uint4 pack(const float (&f)[8]) {
    return make_uint4(pack_f16x2(f[0], f[1]), pack_f16x2(f[2], f[3]), pack_f16x2(f[4], f[5]), pack_f16x2(f[6], f[7]));
  }
};

DFL_DEVICE uint32_t fp8x4(const float* v, float inv, int e5m2) {
  const __nv_fp8_interpretation_t k = e5m2 ? __NV_E5M2 : __NV_E4M3;
  const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(v[0] * inv, v[1] * inv), __NV_SATFINITE, k);
  const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(v[2] * inv, v[3] * inv), __NV_SATFINITE, k);
  return lo | (hi << 16);
}

// NT threads share a row, every thread holding VPT groups of E values.  VEC: a group is 16
// contiguous bytes (D a multiple of E, 16-byte aligned rows); otherwise the group's values lie NT
// apart, which keeps single-value accesses coalesced for odd widths, strides and addresses.
template <typename T, int NT, int VPT, bool VEC>
__global__ void __launch_bounds__(NT < 128 ? 128 : NT) add_rms_norm_kernel(AddNormArgs a) {
  constexpr int E = Io<T>::E;
  constexpr int kRows = NT < 128 ? 128 / NT : 1;  // rows per block
  constexpr int kWarps = NT / 32;
  __shared__ float red[kWarps > 1 ? kWarps : 1];
  const int t = threadIdx.x % NT;
  const long long row = (long long)blockIdx.x * kRows + threadIdx.x / NT;
  griddep_wait();  // (launched while the kernel before it ends: 4 x 4096 bf16 in a row of calls 3.1 -> 2.9 us)
  if (row >= a.M) {
    // blocked scales cover whole 256-row groups: the rows behind the last one hold zeros
    if (a.quant && a.blocked && row < a.M_pad)
      for (int c = t; c < a.D / 128; c += NT) {
        const long long atom = (row / 128) * (a.D / 128) + c;
        *reinterpret_cast<uint32_t*>(a.sf + atom * 512 + (row % 32) * 16 + ((row % 128) / 32) * 4) = 0u;
      }
    return;  // uniform over the threads of a row, so no barrier below is left waiting
  }
  const T* x = reinterpret_cast<const T*>(a.x) + row * a.ldx;
  const T* rs = a.resid ? reinterpret_cast<const T*>(a.resid) + row * a.ldr : nullptr;
  auto col = [&](int i, int j) { return VEC ? (t + NT * i) * E + j : (i * E + j) * NT + t; };

  float v[VPT][E];
  if constexpr (VEC) {
    uint4 px[VPT], pr[VPT];
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const bool in = col(i, 0) < a.D;
      px[i] = in ? *reinterpret_cast<const uint4*>(x + col(i, 0)) : make_uint4(0u, 0u, 0u, 0u);
      pr[i] = in && rs ? *reinterpret_cast<const uint4*>(rs + col(i, 0)) : make_uint4(0u, 0u, 0u, 0u);
    }
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      float f[E];
      Io<T>::unpack(px[i], v[i]);
      Io<T>::unpack(pr[i], f);
#pragma unroll
      for (int j = 0; j < E; ++j) v[i][j] += f[j];
    }
  } else {
#pragma unroll
    for (int i = 0; i < VPT; ++i)
#pragma unroll
      for (int j = 0; j < E; ++j) {
        const int c = col(i, j);
        v[i][j] = c < a.D ? Io<T>::ld(x[c]) + (rs ? Io<T>::ld(rs[c]) : 0.f) : 0.f;
      }
  }
  float sq = 0.f;
#pragma unroll
  for (int i = 0; i < VPT; ++i)
#pragma unroll
    for (int j = 0; j < E; ++j) sq += v[i][j] * v[i][j];
  sq = warp_sum(sq);
  if constexpr (kWarps > 1) {
    if (t % 32 == 0) red[t / 32] = sq;
    __syncthreads();
    sq = 0.f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) sq += red[w];
  }
  const float rstd = __frsqrt_rn(sq / (float)a.D + a.eps);  // one rounding: it scales a whole row
  const float *sc = nullptr, *sh = nullptr;
  if (a.n_mod > 0) {
    const int b = a.row_map ? a.row_map[row] : (int)(row / a.rows_per_batch);
    if (b >= 0 && b < a.n_mod) {
      if (a.scale) sc = a.scale + (long long)b * a.scale_bs;
      if (a.shift) sh = a.shift + (long long)b * a.shift_bs;
    } else if (t == 0) {
      record_error(a.err, kErrBounds, kKidNorm, 90, (int)row);
    }
  }
  T* so = a.s_out ? reinterpret_cast<T*>(a.s_out) + row * a.lds : nullptr;

#pragma unroll
  for (int i = 0; i < VPT; ++i) {
    if constexpr (VEC) {
      const int c = col(i, 0);
      const bool in = c < a.D;
      if (!in && !a.quant) continue;  // (quant: every lane takes part in the block's shuffles)
      float y[E];
      if (in && so) *reinterpret_cast<uint4*>(so + c) = Io<T>::pack(v[i]);
#pragma unroll
      for (int j = 0; j < E; ++j) y[j] = v[i][j] * rstd;
      if (in && a.w) {
        if (a.w_f32) {
#pragma unroll
          for (int j = 0; j < E; ++j) y[j] *= reinterpret_cast<const float*>(a.w)[c + j];
        } else {
          float f[E];
          Io<T>::unpack(*reinterpret_cast<const uint4*>(reinterpret_cast<const T*>(a.w) + c), f);
#pragma unroll
          for (int j = 0; j < E; ++j) y[j] *= f[j];
        }
      }
      if (in && sc) {
#pragma unroll
        for (int j = 0; j < E; j += 4) {
          const float4 f = *reinterpret_cast<const float4*>(sc + c + j);
          y[j] *= 1.f + f.x, y[j + 1] *= 1.f + f.y, y[j + 2] *= 1.f + f.z, y[j + 3] *= 1.f + f.w;
        }
      }
      if (in && sh) {
#pragma unroll
        for (int j = 0; j < E; j += 4) {
          const float4 f = *reinterpret_cast<const float4*>(sh + c + j);
          y[j] += f.x, y[j + 1] += f.y, y[j + 2] += f.z, y[j + 3] += f.w;
        }
      }
      if (!a.quant) {
        *reinterpret_cast<uint4*>(reinterpret_cast<T*>(a.y) + row * a.ldy + c) = Io<T>::pack(y);
        continue;
      }
      // MX: 32 / E neighbouring lanes hold one block; its scale exponent is floor(log2(amax)) - emax
      float amax = 0.f;
#pragma unroll
      for (int j = 0; j < E; ++j) amax = fmaxf(amax, fabsf(y[j]));
      if (!in) amax = 0.f;
#pragma unroll
      for (int o = 1; o < 32 / E; o <<= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
      int e = (int)((__float_as_uint(amax) >> 23) & 0xFF) - 127 - (a.quant == 2 ? 15 : 8);
      e = amax > 0.f ? max(-127, e) : -127;
      const float inv = __uint_as_float((uint32_t)(127 - e) << 23);
      uint32_t byte = in ? (uint32_t)(e + 127) : 0u;
      if (a.blocked) {  // the four scales of 128 columns as one word
        constexpr int L = 32 / E;
        const uint32_t b1 = __shfl_down_sync(0xffffffffu, byte, L), b2 = __shfl_down_sync(0xffffffffu, byte, 2 * L),
                       b3 = __shfl_down_sync(0xffffffffu, byte, 3 * L);
        if (in && (c % 128) == 0) {
          const long long atom = (row / 128) * (a.D / 128) + c / 128;
          *reinterpret_cast<uint32_t*>(a.sf + atom * 512 + (row % 32) * 16 + ((row % 128) / 32) * 4) =
              byte | (b1 << 8) | (b2 << 16) | (b3 << 24);
        }
      } else if (in && (c % 32) == 0) {
        a.sf[row * (a.D / 32) + c / 32] = (uint8_t)byte;
      }
      if (in) {
        uint8_t* q = reinterpret_cast<uint8_t*>(a.y) + row * a.ldy + c;
        if constexpr (E == 8)
          *reinterpret_cast<uint2*>(q) = make_uint2(fp8x4(y, inv, a.quant == 2), fp8x4(y + 4, inv, a.quant == 2));
        else
          *reinterpret_cast<uint32_t*>(q) = fp8x4(y, inv, a.quant == 2);
      }
    } else {
#pragma unroll
      for (int j = 0; j < E; ++j) {
        const int c = col(i, j);
        if (c >= a.D) continue;
        if (so) so[c] = Io<T>::st(v[i][j]);
        float y = v[i][j] * rstd;
        if (a.w) y *= a.w_f32 ? reinterpret_cast<const float*>(a.w)[c] : Io<T>::ld(reinterpret_cast<const T*>(a.w)[c]);
        if (sc) y *= 1.f + sc[c];
        if (sh) y += sh[c];
        reinterpret_cast<T*>(a.y)[row * a.ldy + c] = Io<T>::st(y);
      }
    }
  }
}

template <typename T, int NT, int VPT>
int launch_norm(const AddNormArgs& a, bool vec, cudaStream_t stream) {
  constexpr int kRows = NT < 128 ? 128 / NT : 1;
  const long long rows = a.quant && a.blocked ? a.M_pad : a.M;
  const unsigned grid = (unsigned)((rows + kRows - 1) / kRows);
  return (int)dfl_host::launch_early(vec ? add_rms_norm_kernel<T, NT, VPT, true> : add_rms_norm_kernel<T, NT, VPT, false>, grid,
                                     NT < 128 ? 128 : NT, 0, stream, a);
}

template <typename T>
int dispatch_norm(const AddNormArgs& a, bool vec, cudaStream_t stream) {
  const int groups = (a.D + Io<T>::E - 1) / Io<T>::E;  // 16-byte groups per row
  if (groups <= 32) return launch_norm<T, 32, 1>(a, vec, stream);
  if (groups <= 64) return launch_norm<T, 32, 2>(a, vec, stream);
  if (groups <= 640) {
    switch ((groups + 127) / 128) {
      case 1: return launch_norm<T, 128, 1>(a, vec, stream);
      case 2: return launch_norm<T, 128, 2>(a, vec, stream);
      case 3: return launch_norm<T, 128, 3>(a, vec, stream);
      case 4: return launch_norm<T, 128, 4>(a, vec, stream);
      default: return launch_norm<T, 128, 5>(a, vec, stream);
    }
  }
  switch ((groups + 511) / 512) {
    case 1:
    case 2: return launch_norm<T, 512, 2>(a, vec, stream);
    case 3:
    case 4: return launch_norm<T, 512, 4>(a, vec, stream);
    default: return launch_norm<T, 512, 8>(a, vec, stream);
  }
}

// MX -> values, 8 elements per thread and step (lanes contiguous on both sides), four steps in flight.
template <typename T>
__global__ void __launch_bounds__(256) mx_dequant_kernel(const uint2* __restrict__ q, const uint8_t* __restrict__ sf,
                                                         T* __restrict__ out, long long n8, int e5m2) {
  constexpr int E = Io<T>::E, U = 4;
  const __nv_fp8_interpretation_t k = e5m2 ? __NV_E5M2 : __NV_E4M3;
  const long long i0 = (long long)blockIdx.x * (256 * U) + threadIdx.x;
  uint2 w[U];
  uint32_t s[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const long long i = i0 + 256 * u;
    w[u] = i < n8 ? __ldg(q + i) : make_uint2(0u, 0u);
    s[u] = i < n8 ? __ldg(sf + i / 4) : 0u;
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const long long i = i0 + 256 * u;
    if (i >= n8) break;
    // 2^(s - 127): the biased exponent is the f32 exponent field (s = 0: the subnormal 2^-127)
    const float f = s[u] ? __uint_as_float(s[u] << 23) : __uint_as_float(0x00400000u);
    const uint32_t ws[2] = {w[u].x, w[u].y};
    float v[8];
#pragma unroll
    for (int h = 0; h < 4; ++h) {
      const __half2_raw r = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(ws[h / 2] >> (16 * (h & 1))), k);
      const float2 p = __half22float2(*reinterpret_cast<const __half2*>(&r));
      v[2 * h] = p.x * f, v[2 * h + 1] = p.y * f;
    }
    uint4* o = reinterpret_cast<uint4*>(out + i * 8);
#pragma unroll
    for (int h = 0; h < 8 / E; ++h) o[h] = Io<T>::pack(*reinterpret_cast<float(*)[E]>(&v[h * E]));
  }
}

}  // namespace

extern "C" int dfl_add_rms_norm(const AddNormArgs* args, cudaStream_t stream) {
  AddNormArgs a = *args;
  if (a.M <= 0) return 0;
  if (a.D <= 0 || a.D > 16384) return -2;
  const int es = a.dtype == kDtypeF32 ? 4 : 2, E = 16 / es;
  a.M_pad = (a.M + 255) / 256 * 256;
  auto al = [](const void* p, int n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; };
  bool vec = a.D % E == 0 && al(a.x, 16) && al(a.resid, 16) && al(a.s_out, 16) && al(a.w, 16) && al(a.scale, 16) &&
             al(a.shift, 16) && a.ldx % E == 0 && (!a.resid || a.ldr % E == 0) && (!a.s_out || a.lds % E == 0) &&
             (!a.scale || a.scale_bs % 4 == 0) && (!a.shift || a.shift_bs % 4 == 0);
  vec = vec && al(a.y, a.quant ? 8 : 16) && a.ldy % E == 0;
  if (a.quant) {
    if (!vec || a.D % (a.blocked ? 128 : 32) || !al(a.sf, 4)) return -3;
  }
  switch (a.dtype) {
    case kDtypeF32: return dispatch_norm<float>(a, vec, stream);
    case kDtypeBf16: return dispatch_norm<__nv_bfloat16>(a, vec, stream);
    case kDtypeF16: return dispatch_norm<__half>(a, vec, stream);
    default: return -1;
  }
}

extern "C" int dfl_mx_dequantize(const void* q, const void* scales, void* out, long long n, int dtype, int e5m2,
                                 cudaStream_t stream) {
  if (n <= 0) return 0;
  if (n % 32 || ((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(out)) & 15)) return -2;
  const long long n8 = n / 8, blocks = (n8 + 1023) / 1024;
  if (blocks >= (1ll << 31)) return -3;
  const unsigned grid = (unsigned)blocks;
  const uint2* qp = reinterpret_cast<const uint2*>(q);
  const uint8_t* sp = reinterpret_cast<const uint8_t*>(scales);
  switch (dtype) {
    case kDtypeF32: mx_dequant_kernel<<<grid, 256, 0, stream>>>(qp, sp, reinterpret_cast<float*>(out), n8, e5m2); break;
    case kDtypeBf16:
      mx_dequant_kernel<<<grid, 256, 0, stream>>>(qp, sp, reinterpret_cast<__nv_bfloat16*>(out), n8, e5m2);
      break;
    case kDtypeF16: mx_dequant_kernel<<<grid, 256, 0, stream>>>(qp, sp, reinterpret_cast<__half*>(out), n8, e5m2); break;
    default: return -1;
  }
  return (int)cudaGetLastError();
}
