// Shared device helpers for the difflet_b200 sm_100a kernels.
//
// Everything here is written for Blackwell (sm_100a): mbarriers with bounded
// waits, TMA tile loads (plain per-CTA loads only), tcgen05
// tensor-memory allocation / MMA / loads, and the error-word protocol every
// kernel uses instead of __trap(): a wait that runs out of budget records a
// code in a device error word, the kernel unwinds, and the host raises.
#pragma once

#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#define DFL_DEVICE __device__ __forceinline__

namespace dfl {

// ---------------------------------------------------------------------------
// Error word.  Kernels receive `int* err` (a 4-int device buffer owned by the
// host runtime).  err[0] holds the first error code, err[1] the kernel id,
// err[2]/err[3] free-form detail (e.g. the stage or peer that timed out).
// ---------------------------------------------------------------------------
enum ErrCode : int {
  kErrNone = 0,
  kErrMbarTimeout = 1,     // an mbarrier wait exceeded its cycle budget
  kErrPeerTimeout = 2,     // a peer flag never arrived
  kErrBounds = 3,          // a bounds guard (debug builds) caught an index
  kErrBadArg = 4,          // device-side argument check
};

enum KernelId : int {
  kKidGemm = 1,
  kKidAttn = 2,
  kKidComm = 3,
  kKidNorm = 4,
  kKidMx = 5,
  kKidConv = 6,
  kKidCross = 7,
  kKidLora = 8,
};

DFL_DEVICE void record_error(int* err, int code, int kid, int d0, int d1) {
  if (err == nullptr) return;
  if (atomicCAS(err, 0, code) == 0) {
    err[1] = kid;
    err[2] = d0;
    err[3] = d1;
  }
}

// Default budget for waits inside one kernel (producer/consumer handshakes):
// ~4 s at 1.9 GHz.  A healthy wait is microseconds; running out means a bug.
constexpr long long kLocalWaitCycles = 8000000000LL;

// Debug builds (-DDFL_BOUNDS_CHECK, DIFFLET_BOUNDS_CHECK=1): index guards on values the host
// cannot check without a device read (per-row maps, peer owners).  A failed guard records
// kErrBounds with the kernel id and the offending index and the access is skipped; release
// builds compile the guard to `true`.
#ifdef DFL_BOUNDS_CHECK
#define DFL_GUARD(cond, err, kid, d0, d1) \
  ((cond) ? true : (::dfl::record_error((err), ::dfl::kErrBounds, (kid), (int)(d0), (int)(d1)), false))
#else
#define DFL_GUARD(cond, err, kid, d0, d1) true
#endif

// ---------------------------------------------------------------------------
// Shared-memory address helpers
// ---------------------------------------------------------------------------
DFL_DEVICE uint32_t smem_u32(const void* p) {
  return static_cast<uint32_t>(__cvta_generic_to_shared(p));
}

// ---------------------------------------------------------------------------
// mbarrier
// ---------------------------------------------------------------------------
DFL_DEVICE void mbar_init(uint64_t* bar, uint32_t count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(smem_u32(bar)), "r"(count));
}

DFL_DEVICE void fence_barrier_init() {
  asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
}

DFL_DEVICE void fence_proxy_async_shared() {
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
}

DFL_DEVICE void mbar_arrive_expect_tx(uint64_t* bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(smem_u32(bar)),
               "r"(bytes)
               : "memory");
}

DFL_DEVICE void mbar_arrive(uint64_t* bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
}

DFL_DEVICE bool mbar_try_wait(uint64_t* bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(smem_u32(bar)), "r"(parity)
      : "memory");
  return ok != 0;
}

// Bounded parity wait.  Returns false (and records an error) when the budget
// runs out, or immediately when `abort_flag` (shared) has been raised by a
// sibling role of the same CTA.
DFL_DEVICE bool mbar_wait(uint64_t* bar, uint32_t parity, int* err, int kid, int detail,
                          volatile int* abort_flag, long long budget = kLocalWaitCycles) {
  if (mbar_try_wait(bar, parity)) return true;
  long long t0 = clock64();
  for (uint32_t i = 1;; ++i) {
    if (mbar_try_wait(bar, parity)) return true;
    if ((i & 255u) == 0u) {
      if (abort_flag != nullptr && *abort_flag) return false;
      if (clock64() - t0 > budget) {
        record_error(err, kErrMbarTimeout, kid, detail, (int)parity);
        if (abort_flag != nullptr) *abort_flag = 1;
        return false;
      }
    }
  }
}

// The same by a whole warp, with one outcome for its lanes: a lane that gave up alone would be missing from the warp's next
// collective operation, which would then never end.
DFL_DEVICE bool mbar_wait_warp(uint64_t* bar, uint32_t parity, int* err, int kid, int detail, volatile int* abort_flag) {
  return __all_sync(0xffffffffu, mbar_wait(bar, parity, err, kid, detail, abort_flag));
}

// ---------------------------------------------------------------------------
// TMA (cp.async.bulk.tensor) -- plain loads only.  No cross-CTA broadcast form
// exists in this code base: a tile that several CTAs need is fetched by each.
// ---------------------------------------------------------------------------
DFL_DEVICE void tma_load_2d(void* smem_dst, const CUtensorMap* map, uint64_t* bar, int c0,
                            int c1) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%3, %4}], [%2];" ::"r"(smem_u32(smem_dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(smem_u32(bar)), "r"(c0), "r"(c1)
      : "memory");
}

DFL_DEVICE void tma_load_3d(void* smem_dst, const CUtensorMap* map, uint64_t* bar, int c0, int c1,
                            int c2) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(smem_u32(smem_dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(smem_u32(bar)), "r"(c0), "r"(c1), "r"(c2)
      : "memory");
}

DFL_DEVICE void prefetch_tmap(const CUtensorMap* map) {
  asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(map)) : "memory");
}

// ---------------------------------------------------------------------------
// tcgen05: tensor memory + 5th-generation MMA
// ---------------------------------------------------------------------------
DFL_DEVICE void tmem_alloc(uint32_t* smem_result, uint32_t ncols) {
  asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                   smem_u32(smem_result)),
               "r"(ncols)
               : "memory");
}

DFL_DEVICE void tmem_relinquish() {
  asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
}

DFL_DEVICE void tmem_dealloc(uint32_t taddr, uint32_t ncols) {
  asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(taddr), "r"(ncols)
               : "memory");
}

DFL_DEVICE void tc_fence_before() {
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
}
DFL_DEVICE void tc_fence_after() {
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
}

// Programmatic launch: let the next kernel of the stream start / wait until the previous one is complete (nothing
// to wait for in a launch without the attribute).
DFL_DEVICE void griddep_launch() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
DFL_DEVICE void griddep_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

// D[tmem] (+)= A[smem] * B[smem]^T, kind::f16 (bf16 or f16 inputs, same type for A and B).
DFL_DEVICE void umma_f16_ss(uint32_t tmem_d, uint64_t adesc, uint64_t bdesc, uint32_t idesc,
                            uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(tmem_d),
      "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate)
      : "memory");
}

// Arrive on an mbarrier once every previously issued tcgen05.mma of this thread completes.
DFL_DEVICE void umma_commit(uint64_t* bar) {
  asm volatile(
      "tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(
          smem_u32(bar))
      : "memory");
}

DFL_DEVICE void tmem_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
DFL_DEVICE void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// 32 lanes x 32 consecutive 32-bit columns: thread i of the warp receives row
// (lane_base + i), columns [col, col + 32).
DFL_DEVICE void tmem_ld_32x32b_x32(uint32_t taddr, uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
      "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
        "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]),
        "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]),
        "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]),
        "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr));
}

DFL_DEVICE void tmem_ld_32x32b_x16(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
        "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]),
        "=r"(r[14]), "=r"(r[15])
      : "r"(taddr));
}

DFL_DEVICE void tmem_st_32x32b_x16(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
      "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
      "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]),
      "r"(r[15])
      : "memory");
}

// ---------------------------------------------------------------------------
// UMMA descriptors
// ---------------------------------------------------------------------------
// Shared-memory matrix descriptor, 128-byte swizzle.
//   K-major: rows of 128 B (64 bf16 of K), 8-row atoms 1024 B apart (SBO);
//            LBO unused (1).
//   MN-major: 64 contiguous MN elements per 128-B row, rows step along K;
//            SBO = byte distance between 8-row K groups, LBO = byte distance
//            between 64-element MN chunks.
// Bits: start>>4 [0,14), LBO>>4 [16,30), SBO>>4 [32,46), version=1 [46,48),
// base offset 0 [49,52), layout type 2 = SWIZZLE_128B [61,64).
__host__ __device__ constexpr uint64_t make_sdesc_sw128(uint32_t smem_addr, uint32_t lbo_bytes, uint32_t sbo_bytes) {
  uint64_t d = 0;
  d |= (uint64_t)((smem_addr >> 4) & 0x3FFFu);
  d |= (uint64_t)((lbo_bytes >> 4) & 0x3FFFu) << 16;
  d |= (uint64_t)((sbo_bytes >> 4) & 0x3FFFu) << 32;
  d |= 1ull << 46;
  d |= 2ull << 61;
  return d;
}

// Instruction descriptor for kind::f16 with bf16 A/B and fp32 accumulation.
// a_mn_major / b_mn_major select MN-major operands (transposed smem tiles).
__host__ __device__ constexpr uint32_t make_idesc_bf16_f32(int M, int N, int a_mn_major = 0,
                                                          int b_mn_major = 0) {
  return (1u << 4)                      // D format: f32
         | (1u << 7)                    // A format: bf16
         | (1u << 10)                   // B format: bf16
         | ((uint32_t)a_mn_major << 15) // A major
         | ((uint32_t)b_mn_major << 16) // B major
         | ((uint32_t)(N >> 3) << 17)   // N / 8
         | ((uint32_t)(M >> 4) << 24);  // M / 16
}

// ---------------------------------------------------------------------------
// Small math helpers (all transcendental work goes through CUDA's own functions)
// ---------------------------------------------------------------------------
// tanh on the SFU (PTX tanh.approx.f32, max relative error ~2^-11): ample for
// activations that are rounded to bf16 (2^-8) right after.
DFL_DEVICE float tanh_sfu(float x) {
  float y;
  asm("tanh.approx.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

DFL_DEVICE float gelu_tanh(float x) {
  // GELU, tanh approximation: 0.5 x (1 + tanh(sqrt(2/pi) (x + 0.044715 x^3)))
  const float k0 = 0.7978845608028654f;  // sqrt(2/pi)
  const float k1 = 0.044715f;
  return 0.5f * x * (1.0f + tanh_sfu(k0 * (x + k1 * x * x * x)));
}

DFL_DEVICE float silu(float x) { return x / (1.0f + __expf(-x)); }

DFL_DEVICE uint32_t pack_bf16x2(float lo, float hi) {
  __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<uint32_t*>(&v);
}

DFL_DEVICE float2 unpack_bf16x2(uint32_t v) {
  __nv_bfloat162 b = *reinterpret_cast<__nv_bfloat162*>(&v);
  return __bfloat1622float2(b);
}

DFL_DEVICE float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

DFL_DEVICE float warp_max(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}

}  // namespace dfl

// ---------------------------------------------------------------------------
// Host side: driver entry point for tensor-map encoding (no -lcuda needed).
// ---------------------------------------------------------------------------
namespace dfl_host {
typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*,
                                  const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                                  const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                  CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
EncodeTiledFn get_encode_tiled();
// Returns 0 on success; non-zero CUresult otherwise.
int make_tmap_2d_bf16(CUtensorMap* map, const void* base, uint64_t inner, uint64_t outer,
                      uint64_t row_stride_elems, uint32_t box_inner, uint32_t box_outer,
                      bool swizzle128);
int make_tmap_3d_bf16(CUtensorMap* map, const void* base, uint64_t d0, uint64_t d1, uint64_t d2,
                      uint64_t stride1_elems, uint64_t stride2_elems, uint32_t b0, uint32_t b1,
                      uint32_t b2, bool swizzle128);
int num_sms(int device);
// A launch that may start while the kernel before it ends (the kernel waits for that itself: griddep_wait).
template <class... Params, class... Args>
cudaError_t launch_early(void (*kernel)(Params...), unsigned grid, int threads, size_t smem, cudaStream_t stream,
                         const Args&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid, 1, 1);
  cfg.blockDim = dim3((unsigned)threads, 1, 1);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, args...);
}
}  // namespace dfl_host
