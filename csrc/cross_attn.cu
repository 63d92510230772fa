// Cross attention: bf16 variants, argument checks and the bit packing of boolean masks.
#include "cross_attn.cuh"

extern "C" int dfl_cross_attention_f16(const CrossArgs* a, cudaStream_t stream);

namespace {

// Bit rows of a boolean mask: one warp per (row, 32-key word), bits past the last key set (the key
// window excludes those keys).  Rows are [B, H, Q] of the mask's own (unbroadcast) extents.
__global__ void __launch_bounds__(256) cross_mask_bits_kernel(MaskBitsArgs a) {
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

// Key window [first kept key, last kept key + 1) of every batch row of a key mask ([B, 1, 1, Sk]):
// one block per batch row.  A row that keeps nothing gets [0, 0).
__global__ void __launch_bounds__(256) cross_mask_window_kernel(MaskBitsArgs a) {
  __shared__ int s_lo, s_hi;
  if (threadIdx.x == 0) s_lo = a.Sk, s_hi = 0;
  __syncthreads();
  const uint32_t* row = a.bits + (long long)blockIdx.x * a.words;
  int lo = a.Sk, hi = 0;
  for (int w = threadIdx.x; w < a.words; w += blockDim.x) {
    uint32_t v = row[w];
    const int left = a.Sk - w * 32;
    if (left <= 0) continue;
    if (left < 32) v &= (1u << left) - 1u;
    if (v) {
      lo = min(lo, w * 32 + __ffs(v) - 1);
      hi = max(hi, w * 32 + 32 - __clz(v));
    }
  }
  atomicMin(&s_lo, lo);  // minima and maxima: the order of the updates does not matter
  atomicMax(&s_hi, hi);
  __syncthreads();
  if (threadIdx.x == 0) {
    a.lo[blockIdx.x] = s_hi > 0 ? s_lo : 0;
    a.hi[blockIdx.x] = s_hi;
  }
}

}  // namespace

extern "C" int dfl_cross_mask_bits(const MaskBitsArgs* a, cudaStream_t stream) {
  if (a->B <= 0 || a->H <= 0 || a->Q <= 0 || a->Sk <= 0) return -2;
  if (a->words != (a->Sk + 127) / 128 * 4) return -3;
  const long long warps = (long long)a->B * a->H * a->Q * a->words;
  const long long blocks = (warps + 7) / 8;
  cross_mask_bits_kernel<<<(unsigned)(blocks < 148 * 32 ? blocks : 148 * 32), 256, 0, stream>>>(*a);
  if (a->lo) cross_mask_window_kernel<<<(unsigned)a->B, 256, 0, stream>>>(*a);
  return (int)cudaGetLastError();
}

extern "C" int dfl_cross_attention(const CrossArgs* a, cudaStream_t stream) {
  if (a->dh != 64 && a->dh != 128) return -2;
  if (a->B <= 0 || a->H <= 0 || a->Hk <= 0 || a->Sq <= 0 || a->Sk <= 0 || a->H % a->Hk) return -3;
  auto al16 = [](const void* ptr) { return (reinterpret_cast<uintptr_t>(ptr) & 15) == 0; };
  if (!al16(a->q) || !al16(a->k) || !al16(a->v) || !al16(a->o) || !al16(a->bits)) return -4;
  if ((a->q_ss | a->q_hs | a->q_bs | a->k_ss | a->k_hs | a->k_bs | a->v_ss | a->v_hs | a->v_bs | a->o_ss | a->o_hs |
       a->o_bs) % 8)
    return -5;
  if (!(a->scale > 0.f)) return -6;
  if (a->bits && ((a->bits_bs | a->bits_hs | a->bits_qs) % 4 || a->bias)) return -7;
  return a->f16 ? dfl_cross_attention_f16(a, stream) : cross_entry<false>(a, stream);
}
