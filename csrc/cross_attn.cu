// Cross attention: bf16 variants, argument checks and the bit packing of boolean masks.
#include "cross_attn.cuh"

extern "C" int dfl_cross_attention_f16(const CrossArgs* a, cudaStream_t stream);

namespace {

// Bit rows of a boolean mask: one warp per (row, 32-key word), bits past the last key set (the key
// window excludes those keys).  Rows are [B, H, Q] of the mask's own (unbroadcast) extents.
__global__ void __launch_bounds__(256) cross_mask_bits_kernel(MaskBitsArgs a) {
  griddep_wait();
  griddep_launch();
  const long long n = (long long)a.B * a.H * a.Q * a.words;
  const int lane = threadIdx.x % 32;
  for (long long i = ((long long)blockIdx.x * blockDim.x + threadIdx.x) / 32; i < n;
       i += (long long)gridDim.x * blockDim.x / 32) {
    const int w = (int)(i % a.words);
    long long r = i / a.words;
    const int q = (int)(r % a.Q);
    r /= a.Q;
    const int h = (int)(r % a.H), b = (int)(r / a.H);
    const int k = w * 32 + lane;
    const bool keep = k >= a.Sk || a.mask[b * a.bs + h * a.hs + q * a.qs + k * a.ks] != 0;
    const uint32_t word = __ballot_sync(0xffffffffu, keep);
    if (lane == 0) a.bits[i] = word;
  }
}

// A key mask ([B, 1, 1, Sk]): one block per batch row writes its bit row and the key window [first kept
// key, last kept key + 1); a row that keeps nothing gets [0, 0).
__global__ void __launch_bounds__(256) cross_key_mask_kernel(MaskBitsArgs a) {
  griddep_wait();
  griddep_launch();  // the attention sets itself up meanwhile
  __shared__ int s_lo[8], s_hi[8];
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32, b = blockIdx.x;
  int lo = a.Sk, hi = 0;
  for (int w = warp; w < a.words; w += 8) {
    const int k = w * 32 + lane;
    const bool keep = k >= a.Sk || a.mask[b * a.bs + k * a.ks] != 0;
    uint32_t word = __ballot_sync(0xffffffffu, keep);
    if (lane == 0) a.bits[(long long)b * a.words + w] = word;
    const int left = a.Sk - w * 32;
    word = left <= 0 ? 0u : (left < 32 ? word & ((1u << left) - 1u) : word);
    if (word) {
      lo = min(lo, w * 32 + __ffs(word) - 1);
      hi = max(hi, w * 32 + 32 - __clz(word));
    }
  }
  if (lane == 0) s_lo[warp] = lo, s_hi[warp] = hi;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < 8; ++w) lo = min(lo, s_lo[w]), hi = max(hi, s_hi[w]);
    a.lo[b] = hi > 0 ? lo : 0;
    a.hi[b] = hi;
  }
}

DFL_DEVICE float mask_value(const void* p, int dtype, long long at) {
  if (dtype == kDtypeF32) return reinterpret_cast<const float*>(p)[at];
  if (dtype == kDtypeBf16) return __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(p)[at]);
  return __half2float(reinterpret_cast<const __half*>(p)[at]);
}

// One thread per 16-byte vector of a block: the main kernel then reads whole lines where the mask's own
// rows (any stride, any alignment) would cost a line per query and load.
template <bool F32>
__global__ void __launch_bounds__(256) cross_bias_tiles_kernel(BiasTileArgs a) {
  griddep_wait();
  griddep_launch();
  constexpr int E = F32 ? 4 : 8, V = 128 / E;
  const int rows = a.Q > 1 ? 32 : 1, nq = (a.Q + 31) / 32, nt = (a.Sk + 127) / 128;
  const long long n = (long long)a.B * a.H * nq * nt * V * rows;
  for (long long i = (long long)blockIdx.x * blockDim.x + threadIdx.x; i < n; i += (long long)gridDim.x * blockDim.x) {
    long long r = i;
    const int qi = (int)(r % rows);
    r /= rows;
    const int v = (int)(r % V);
    r /= V;
    const int t = (int)(r % nt);
    r /= nt;
    const int q = (int)(r % nq) * 32 + qi;
    r /= nq;
    const long long at = (r / a.H) * a.bs + (r % a.H) * a.hs + (long long)min(q, a.Q - 1) * a.qs;
    const int k0 = t * 128 + v * E;
    if constexpr (F32) {
      float f[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) f[e] = k0 + e < a.Sk ? mask_value(a.mask, a.dtype, at + (k0 + e) * a.ks) : 0.f;
      reinterpret_cast<float4*>(a.tiles)[i] = make_float4(f[0], f[1], f[2], f[3]);
    } else {
      const uint16_t* m = reinterpret_cast<const uint16_t*>(a.mask);
      uint32_t w[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const uint32_t x = k0 + 2 * e < a.Sk ? m[at + (k0 + 2 * e) * a.ks] : 0u;
        const uint32_t y = k0 + 2 * e + 1 < a.Sk ? m[at + (k0 + 2 * e + 1) * a.ks] : 0u;
        w[e] = x | (y << 16);
      }
      reinterpret_cast<uint4*>(a.tiles)[i] = make_uint4(w[0], w[1], w[2], w[3]);
    }
  }
}

}  // namespace

extern "C" int dfl_cross_bias_tiles(const BiasTileArgs* a, cudaStream_t stream) {
  if (a->B <= 0 || a->H <= 0 || a->Q <= 0 || a->Sk <= 0) return -2;
  const long long n = (long long)a->B * a->H * ((a->Q + 31) / 32) * ((a->Sk + 127) / 128) * (a->out_f32 ? 32 : 16) *
                      (a->Q > 1 ? 32 : 1);
  const long long blocks = (n + 255) / 256;
  const unsigned grid = (unsigned)(blocks < 148 * 32 ? blocks : 148 * 32);
  return (int)dfl_host::launch_early(a->out_f32 ? cross_bias_tiles_kernel<true> : cross_bias_tiles_kernel<false>, grid, 256, 0, stream, *a);
}

extern "C" int dfl_cross_mask_bits(const MaskBitsArgs* a, cudaStream_t stream) {
  if (a->B <= 0 || a->H <= 0 || a->Q <= 0 || a->Sk <= 0) return -2;
  if (a->words != (a->Sk + 127) / 128 * 4) return -3;
  if (a->lo) {
    if (a->H != 1 || a->Q != 1 || !a->hi) return -4;
    return (int)dfl_host::launch_early(cross_key_mask_kernel, (unsigned)a->B, 256, 0, stream, *a);
  }
  const long long warps = (long long)a->B * a->H * a->Q * a->words;
  const long long blocks = (warps + 7) / 8;
  return (int)dfl_host::launch_early(cross_mask_bits_kernel, (unsigned)(blocks < 148 * 32 ? blocks : 148 * 32), 256, 0, stream, *a);
}

// How a sliding window is laid out (q_tiles, splits): rounds of items, each of which costs its key tiles (a tile pair about 4300 cycles
// at head dim 128 and 3000 at 64, a lone tile 3600 and 2600) and about 4000 for its turn; parts cost their rows' way through L2
// and a launch.  The blocks are taken as equally long, as they are but for the first window.  1560 queries over 12 heads, 10920
// keys each: 144 us in 3 or 5 parts of pairs (1, 2, 4: 188, 206, 173; lone tiles 225 and more); 300 over 8 heads, 2004 keys
// each: 19 us in 8 parts of lone tiles (1, 2, 4: 38, 26, 20; pairs 46, 31, 23); 512 over 32 heads: 14 us lone and whole (16 in pairs).
extern "C" void dfl_cross_slide_plan(CrossArgs* a) {
  int dev = 0;
  cudaGetDevice(&dev);
  const long long sms = dfl_host::num_sms(dev), rows = (long long)a->B * a->H * a->Sq;
  double least = -1.;
  for (int qt = 1; qt <= 2; ++qt) {
    if (qt == 2 && a->Sq <= kBM) break;
    const long long items = ((long long)a->Sq + qt * kBM - 1) / (qt * kBM) * a->H * a->B;
    const long long span = std::min<long long>(a->Sk, (long long)a->slide + std::min(a->Sq, qt * kBM));
    const long long tiles = std::max<long long>(1, (span + kBN - 1) / kBN + (a->Sk > span ? (a->sinks + kBN - 1) / kBN : 0));
    const double step = qt == 2 ? (a->dh == 64 ? 3000. : 4300.) : (a->dh == 64 ? 2600. : 3600.);
    for (int s = 1; s <= kMaxParts && s <= tiles; ++s) {
      const double rounds = s == 1 && items > sms ? (double)items / sms : (double)((items * s + sms - 1) / sms);
      const double cost = rounds * ((tiles + s - 1) / s * step + 4000.) + (s > 1 ? 6000. + (double)s * rows * a->dh * 8 / 2600. : 0.);
      if (least < 0. || cost < least) least = cost, a->q_tiles = qt, a->splits = s;
    }
  }
}

extern "C" int dfl_cross_attention(const CrossArgs* a, cudaStream_t stream) {
  if (a->dh != 64 && a->dh != 128) return -2;
  if (a->B <= 0 || a->H <= 0 || a->Hk <= 0 || a->Sq <= 0 || a->Sk <= 0 || a->H % a->Hk) return -3;
  auto al16 = [](const void* ptr) { return (reinterpret_cast<uintptr_t>(ptr) & 15) == 0; };
  if (!al16(a->q) || !al16(a->k) || !al16(a->v) || !al16(a->o) || !al16(a->bits) || !al16(a->bias_tiles))
    return -4;
  if ((a->q_ss | a->q_hs | a->q_bs | a->k_ss | a->k_hs | a->k_bs | a->v_ss | a->v_hs | a->v_bs | a->o_ss | a->o_hs |
       a->o_bs) % 8)
    return -5;
  if (!(a->scale > 0.f)) return -6;
  if (a->bits && ((a->bits_bs | a->bits_hs | a->bits_qs) % 4 || a->bias_tiles)) return -7;
  if (a->p2 && (a->bits || a->bias_tiles)) return -8;
  if (a->slide && (a->slide < 0 || a->sinks < 0 || a->bits || a->bias_tiles || a->p2 || a->kv_lo)) return -9;
  if (a->slide && (a->splits < 1 || a->splits > kMaxParts || (a->splits > 1 && !a->parts) || !al16(a->parts) || (a->q_tiles != 1 && a->q_tiles != 2) || a->Sq >= (1 << 29) || a->Sk >= (1 << 29))) return -10;
  return a->f16 ? dfl_cross_attention_f16(a, stream) : cross_entry<false>(a, stream);
}
