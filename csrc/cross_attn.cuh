// Attention of queries to the states of an encoder (sm_100a, tcgen05): keys of another length
// than the queries, head dim 64 or 128, bf16 or fp16, heads that share keys, and masks.
//
//   z = scale q k^T [+ bias];  p = exp(z - max z) over the keys the mask leaves;  o = (p v) / sum p
//
// A row whose mask leaves no key is 0 (log-sum-exp -inf).  One pass over the keys with a running maximum
// and sum; statistics and accumulators are f32, P is rounded to the inputs' type for the P V
// product (the sum uses the unrounded values); callers that had f32 throughout before (LSE or a key window at
// head dim 64) take the variant that splits P into two such values.
//
// Persistent, one CTA per SM; a work item is a block of QT * 128 queries of one head:
//   TMA warp     Q tiles of the next item as soon as the last Q K^T of this one has read them;
//                K_j, V_j through a ring of shared-memory slots
//   MMA warp     steps s = (item, tile) as one sequence, PV0(s-1) QK0(s) PV1(s-1) QK1(s), so the scores of
//                the next item are computed while this item's rows are stored.  The fixed order also
//                keeps the two tiles out of step, one in its exponentials while the other multiplies (with a
//                warp per tile they fall into step and share the SFU: 402 us where this takes 349)
//   clean warp   zeroes the V rows of masked keys (what lies behind a sequence's length may be
//                anything; 0 * NaN would reach the sums), in the tiles that hold some
//   softmax      one warpgroup per Q tile, one query row per thread; P goes back to tensor memory
//                over S and is the A operand of P V; O is rescaled only when the maximum grew by
//                more than 2^8
// tcgen05 operations of an issuing thread complete in order: when S_g(s) is ready, P V_g(s-1) has
// finished, and P_g(first tile of an item) is signalled only after its warpgroup has read O_g of the
// item before, so neither P nor O needs a barrier of its own.
//
// 40 heads x 32760 queries x 512 keys x 128: 342 - 349 us in a loop over one state's tensors (1005 - 984 TFLOP/s), 413 (831) with
// three states' in turn (the products alone take 205 at the library's rate, the
// exponentials 180 at the SFU's).  What is left is the round trip of a Q tile (scores, exponentials, P, next
// scores: 3650 cycles for 2 x 1024 of products), which two tiles do not fill, and the turn of the items.  Measured
// and slower or equal: part of the exponentials on the FMA pipe (387 us), an MMA warp per Q tile (402), three K / V slots
// with a larger output buffer (388), the second half of a row kept in registers past the first P (348), the first
// quarter's exponentials under the old maximum while the new one is found (362), both P V before the new scores at
// the turn of an item (366).
//
// Masks: a key window [lo, hi) per batch row (tiles outside it are skipped), bits (kBits: packed
// by cross_mask_bits, per query or shared by all queries), an additive bias (kBias16 / kBias32), or a causal window that
// slides with the queries beside the first keys (kSlide: only the tiles that some query of the block sees are read).
#pragma once
#include <cuda_fp16.h>

#include <algorithm>
#include <cmath>

#include "common.cuh"
#include "kernels.h"

namespace {
using namespace dfl;

constexpr int kBM = 128;      // queries per Q tile
constexpr int kBN = 128;      // keys per tile
constexpr int kChunk = 16384;  // 128 rows x 64 values: one swizzle chunk
constexpr int kMaxParts = 8;   // of the keys of a block
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.69314718055994531f;

enum { kWindow = 0, kBits = 1, kBias16 = 2, kBias32 = 3, kSlide = 4 };  // kBias16: of the inputs' type, kBias32: f32
constexpr bool is_bias(int mask) { return mask == kBias16 || mask == kBias32; }

struct CrossParams {
  void* o;
  long long o_bs, o_hs, o_ss;
  float* lse;
  int B, H, Sq, Sk, rep;  // rep: query heads per key head
  int n_qb;               // query blocks per head
  float scale;
  const int* kv_lo;  // [B] or NULL
  const int* kv_hi;
  const uint32_t* bits;   // kBits: rows of `words` words, bit k of a row: key k is kept
  long long bits_bs, bits_hs, bits_qs;  // row strides (in words) by batch, head, query
  int key_bits;           // the bits do not vary over queries (V rows of masked keys are cleaned)
  // kBias16 / kBias32: blocks of 32 queries x 128 keys written by dfl_cross_bias_tiles (16-byte vectors,
  // [vector of keys][query], so a warp's loads are contiguous); strides in vectors (0: broadcast)
  const uint4* bias;
  long long bias_bs, bias_hs, bias_qs, bias_ts;  // batch, head, 32-query block, key tile
  int bias_rows;                                 // queries per block: 32, or 1 (one row for all)
  // kSlide: query i of batch row b stands at p = start[b] + i (start NULL: keys - Sq) and sees the keys up to p that are
  // among the last `slide` or the first `sinks`
  const int* start;
  int slide, sinks;
  // The key tiles of a block in `splits` parts, joined by cross_join_kernel: f32 rows and log-sum-exps (log2 units), [part][B, H, Sq]
  int splits;
  float* part_o;
  float* part_l;
};

template <int DH, int QT>
struct CrossCfg {
  static constexpr int kThreads = 128 * QT + 128;
  static constexpr int kProducerWarp = 4 * QT, kMmaWarp = 4 * QT + 1, kCleanWarp = 4 * QT + 2;
  static constexpr int kTile = 128 * DH * 2;
  static constexpr int kChunks = DH / 64;
  static constexpr int kRing = DH == 64 ? 8 : 4;  // (QT = 2, three slots: 360 -> 388 us at 512 keys)
  static constexpr int kQ = 0, kKV = QT * kTile;
  static constexpr int kOut = kKV + kRing * kTile;  // 4 KB per softmax warp: 32 rows x 64 columns on their way out
  static constexpr int kBar = kOut + 4 * QT * 4096;
  // q_full[2], q_empty[2], kv_full[R], kv_empty[R], s_full[2], p_full[2][2], o_full[2], v_clean[R]
  static constexpr int kNumBars = 4 + 3 * kRing + 2 + 4 + 2;
  static constexpr int kTotal = kBar + kNumBars * 8 + 16 + 1024;
  static constexpr uint32_t kTmemCols = QT == 2 ? 512 : 256;
  static constexpr uint32_t kOCol = 128 * QT;  // S_g at 128 g, O_g at kOCol + DH g
  static_assert(kTotal <= 232448, "shared memory budget");
  static_assert(kRing % 2 == 0, "a slot holds K or V for good: the cleaning warp then waits for every phase of a V slot");
  static_assert(kOCol + DH * QT <= kTmemCols, "tensor memory");
};

DFL_DEVICE float exp2_sfu(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
DFL_DEVICE uint64_t f2_pack(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
DFL_DEVICE void f2_unpack(uint64_t r, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(r)); }
DFL_DEVICE uint64_t f2_fma(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
DFL_DEVICE uint64_t f2_add(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
DFL_DEVICE float max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
DFL_DEVICE uint32_t first_bits(int n) {  // the n lowest bits set, n of any size and sign
  uint32_t r;
  asm("bmsk.clamp.b32 %0, 0, %1;" : "=r"(r) : "r"(max(n, 0)));
  return r;
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

// D[tmem] (+)= A[tmem] * B[smem]
DFL_DEVICE void umma_f16_ts(uint32_t tmem_d, uint32_t tmem_a, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(tmem_d),
      "r"(tmem_a), "l"(bdesc), "r"(idesc), "r"(accumulate)
      : "memory");
}

DFL_DEVICE void tma_load_4d(uint8_t* dst, const CUtensorMap* map, uint64_t* bar, int c0, int c1, int c2, int c3) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%3, %4, %5, %6}], [%2];" ::"r"(smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(smem_u32(bar)), "r"(c0), "r"(c1), "r"(c2), "r"(c3)
      : "memory");
}

DFL_DEVICE void tma_store_4d(const CUtensorMap* map, const uint8_t* src, int c0, int c1, int c2, int c3) {
  asm volatile("cp.async.bulk.tensor.4d.global.shared::cta.bulk_group [%0, {%2, %3, %4, %5}], [%1];" ::"l"(
                   reinterpret_cast<uint64_t>(map)),
               "r"(smem_u32(src)), "r"(c0), "r"(c1), "r"(c2), "r"(c3)
               : "memory");
}
DFL_DEVICE void bulk_commit() { asm volatile("cp.async.bulk.commit_group;" ::: "memory"); }
DFL_DEVICE void bulk_wait_read() { asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory"); }
DFL_DEVICE void bulk_wait_all() { asm volatile("cp.async.bulk.wait_group 0;" ::: "memory"); }

// The work items of one CTA: its query block, head, batch row, key window and key tiles, advanced by
// gridDim.x items without divisions (this stands on the issuing warps' critical path).
template <int QT>
struct CrossItems {
  int q0, h, b, lo, hi, t0, n;
  int qb, dq, dh, db;
  DFL_DEVICE explicit CrossItems(const CrossParams& p) {
    const int i = blockIdx.x, g = gridDim.x;
    qb = i % p.n_qb, h = (i / p.n_qb) % p.H, b = i / p.n_qb / p.H;
    dq = g % p.n_qb, dh = (g / p.n_qb) % p.H, db = g / p.n_qb / p.H;
    window(p);
  }
  DFL_DEVICE bool more(const CrossParams& p) const { return b < p.B; }
  DFL_DEVICE int tile(int j) const { return t0 + j; }
  DFL_DEVICE void next(const CrossParams& p) {
    const int was = b;
    qb += dq, h += dh, b += db;
    if (qb >= p.n_qb) qb -= p.n_qb, ++h;
    if (h >= p.H) h -= p.H, ++b;
    q0 = qb * (QT * kBM);
    if (b != was) window(p);
  }
  DFL_DEVICE void window(const CrossParams& p) {
    q0 = qb * (QT * kBM);
    if (b >= p.B) return;
    lo = p.kv_lo ? max(0, __ldcg(p.kv_lo + b)) : 0;
    hi = p.kv_hi ? min(p.Sk, __ldcg(p.kv_hi + b)) : p.Sk;
    t0 = lo / kBN;
    n = hi > lo ? (hi + kBN - 1) / kBN - t0 : 0;
  }
};

// The same where a window slides with the queries: the tiles of the first keys, then those of the window, or a part of them.
// Heads first, the last queries before the first ones: blocks with many keys lead, those with few fill the last round
// (12 heads x 32760 queries, window 9360: 2145 -> 1926 us).  Measured and slower: a window's tiles from its first key on,
// wherever that lies (24 heads x 8192, window 128: 95 -> 104 us), query tiles that pass over the tiles none of their rows sees (82 -> 87),
// a fifth slot in place of the buffers that rows leave through (32760 queries: 1646 -> 1713).
template <int QT>
struct SlideItems {
  int q0, h, b, n;
  int lo, hi, sinks;  // keys that a query of this block may see: [0, sinks) and [lo, hi)
  // Query i sees key j where j <= i + start and j > i - back (back = slide - start; both held to +- 2^29, beyond every length: the
  // launcher's limit, so 32 bits do)
  int start, back;
  int sp, qb, ds, dh, db, dq, len, n_sink, t_win, j0;
  DFL_DEVICE explicit SlideItems(const CrossParams& p) {
    const int i = blockIdx.x / p.splits, g = gridDim.x / p.splits;
    sp = blockIdx.x % p.splits, ds = gridDim.x % p.splits;
    h = i % p.H, b = i / p.H % p.B, qb = p.n_qb - 1 - i / p.H / p.B;
    dh = g % p.H, db = g / p.H % p.B, dq = g / p.H / p.B;
    row(p);
  }
  DFL_DEVICE bool more(const CrossParams& p) const { return qb >= 0; }
  DFL_DEVICE void next(const CrossParams& p) {
    const int was = b;
    sp += ds, h += dh, b += db, qb -= dq;
    if (sp >= p.splits) sp -= p.splits, ++h;
    if (h >= p.H) h -= p.H, ++b;
    if (b >= p.B) b -= p.B, --qb;
    if (b != was) row(p);
    else block(p);
  }
  DFL_DEVICE void row(const CrossParams& p) {
    if (qb < 0) return;
    len = p.kv_hi ? min(p.Sk, max(0, __ldcg(p.kv_hi + b))) : p.Sk;
    const long long first = p.start ? __ldcg(p.start + b) : len - p.Sq;
    start = (int)max(-(1ll << 29), min(1ll << 29, first));
    back = (int)max(-(1ll << 29), min(1ll << 29, p.slide - first));
    block(p);
  }
  DFL_DEVICE void block(const CrossParams& p) {
    q0 = qb * (QT * kBM);
    hi = max(0, min(len, start + min(q0 + QT * kBM, p.Sq)));
    lo = min(p.Sk, max(0, q0 - back + 1));
    sinks = min(p.sinks, hi);
    n_sink = (sinks + kBN - 1) / kBN;
    t_win = max(n_sink, lo / kBN);
    n = n_sink + (hi > lo ? max(0, (hi + kBN - 1) / kBN - t_win) : 0);
    j0 = 0;
    if (p.splits > 1) {
      const int per = (n + p.splits - 1) / p.splits;
      j0 = min(n, sp * per);
      n = min(per, n - j0);
    }
  }
  DFL_DEVICE int tile(int j) const { return j0 + j < n_sink ? j0 + j : t_win + j0 + j - n_sink; }
};
template <int MASK, int QT>
struct ItemsOf {
  using T = CrossItems<QT>;
};
template <int QT>
struct ItemsOf<kSlide, QT> {
  using T = SlideItems<QT>;
};

// The words of key tile k0 for one row of a bit mask (whole 128-key groups are stored).
template <class Item>
DFL_DEVICE uint4 cross_bits(const CrossParams& p, const Item& it, int q, int k0) {
  return __ldcg(reinterpret_cast<const uint4*>(p.bits + it.b * p.bits_bs + it.h * p.bits_hs + q * p.bits_qs + k0 / 32));
}

// Whether tile k0 holds V rows of keys that no query of this batch row may see.
template <int MASK, class Item>
DFL_DEVICE bool cross_dirty(const CrossParams& p, const Item& it, int k0) {
  if constexpr (MASK == kSlide) return it.hi < k0 + kBN || (it.lo > k0 && it.sinks < k0 + kBN);
  else if (it.lo > k0 || it.hi < min(k0 + kBN, p.Sk)) return true;
  if (MASK == kBits && p.key_bits) {
    const uint4 w = cross_bits(p, it, 0, k0);
    return (w.x & w.y & w.z & w.w) != 0xffffffffu;
  }
  return false;
}

// Packed pairs of two 16-bit values (bf16 or fp16) as f32.
template <bool F16>
DFL_DEVICE float2 unpack2(uint32_t v) {
  if constexpr (F16) return __half22float2(*reinterpret_cast<__half2*>(&v));
  else return unpack_bf16x2(v);
}
DFL_DEVICE uint64_t f2_mul(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}

// Register split for QT = 2: 128 threads with 64 and 256 with 216, or 88 and 208 where the items' state needs more
// (32760 queries: 1870 -> 1840 us).
template <int MASK>
DFL_DEVICE void fewer_registers() {
  if constexpr (MASK == kSlide) asm volatile("setmaxnreg.dec.sync.aligned.u32 88;");
  else asm volatile("setmaxnreg.dec.sync.aligned.u32 64;");
}
template <int MASK>
DFL_DEVICE void more_registers() {
  if constexpr (MASK == kSlide) asm volatile("setmaxnreg.inc.sync.aligned.u32 208;");
  else asm volatile("setmaxnreg.inc.sync.aligned.u32 216;");
}

// P2: P goes to the product as the sum of two values of the inputs' type (2^-16 of p in bf16 where one value keeps 2^-8).
template <int DH, bool F16, int QT, int MASK, bool P2>
__global__ void __launch_bounds__(CrossCfg<DH, QT>::kThreads, 1)
    cross_attn_kernel(const __grid_constant__ CUtensorMap tq, const __grid_constant__ CUtensorMap tk,
                      const __grid_constant__ CUtensorMap tv, const __grid_constant__ CUtensorMap to,
                      const CrossParams p, int* err) {
  using C = CrossCfg<DH, QT>;
  using Items = typename ItemsOf<MASK, QT>::T;
  constexpr int R = C::kRing;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + C::kBar);
  uint64_t* q_full = bars;
  uint64_t* q_empty = bars + 2;
  uint64_t* kv_full = bars + 4;
  uint64_t* kv_empty = kv_full + R;
  uint64_t* s_full = kv_empty + R;
  uint64_t* p_full = s_full + 2;  // p_full[2 g + h]: keys [64 h, 64 h + 64) of P_g stored
  uint64_t* o_full = p_full + 4;
  uint64_t* v_clean = o_full + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + C::kNumBars);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const bool cleaning = MASK != kSlide && (p.kv_lo || p.kv_hi || (MASK == kBits && p.key_bits));  // masked keys may hold anything
  uint64_t* v_raw = v_clean;  // kSlide: V tiles that the cleaning warp passes on (the others go straight to the products)

  if (threadIdx.x == 0) {
    for (int i = 0; i < C::kNumBars; ++i) {
      uint64_t* bar = &bars[i];
      mbar_init(bar, bar >= p_full && bar < p_full + 4 ? 128 : 1);
    }
    *abort_flag = 0;
    fence_barrier_init();
    fence_proxy_async_shared();
    prefetch_tmap(&tq);
    prefetch_tmap(&tk);
    prefetch_tmap(&tv);
  }
  if (warp == C::kMmaWarp) {
    tmem_alloc(tmem_slot, C::kTmemCols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  // (launched while the kernel before it, the mask's own among them, ends: what that writes is read past L1)
  griddep_wait();

  // Register split for QT = 2: 128 x 64 + 256 x 216 = 63488 (kSlide: 128 x 88 + 256 x 208 = 64512) <= 384 x 168 at launch
  // (checked by the launcher); every warp of a warpgroup executes its setmaxnreg.
  if (warp == C::kProducerWarp) {
    if constexpr (QT == 2) fewer_registers<MASK>();
    if (lane == 0) {
      // load L (K_s: 2 s, V_s: 2 s + 1 over all steps s) goes to slot L % R, use (L / R)
      bool issued[R], q_issued[2] = {false, false};
      uint32_t issued_par[R], raw = 0, raw_par = 0;  // raw: a bit per slot whose copy was counted on v_raw; raw_par: parity of its next phase
      for (int i = 0; i < R; ++i) issued[i] = false, issued_par[i] = 0;
      bool ok = true;
      int L = 0, used = 0;  // used: items with key tiles so far
      for (Items it(p); it.more(p) && ok; it.next(p)) {
        if (it.n == 0) continue;
        const int hk = it.h / p.rep;
        for (int j = 0; j < it.n && ok; ++j) {
          for (int which = 0; which < 2; ++which, ++L) {
            const int slot = L % R;
            const uint32_t par = (L / R) & 1;
            if (!mbar_wait(&kv_empty[slot], par ^ 1u, err, kKidCross, 100 + which, abort_flag)) { ok = false; break; }
            uint8_t* dst = smem + C::kKV + slot * C::kTile;
            uint64_t* full = &kv_full[slot];
            if constexpr (MASK == kSlide) {
              raw &= ~(1u << slot);
              if (which == 1 && cross_dirty<MASK>(p, it, it.tile(j) * kBN)) full = &v_raw[slot], raw |= 1u << slot, raw_par ^= 1u << slot;
            }
            mbar_arrive_expect_tx(full, C::kTile);
            for (int c = 0; c < C::kChunks; ++c)
              tma_load_4d(dst + c * kChunk, which == 0 ? &tk : &tv, full, c * 64, it.tile(j) * kBN, hk, it.b);
            issued[slot] = true;
            issued_par[slot] = par;
            if (j == 0 && which == 0) {  // the item's first keys are on their way: now its queries
              for (int g = 0; g < QT; ++g) {
                if (!mbar_wait(&q_empty[g], (used & 1) ^ 1u, err, kKidCross, 102 + g, abort_flag)) { ok = false; break; }
                mbar_arrive_expect_tx(&q_full[g], C::kTile);
                for (int c = 0; c < C::kChunks; ++c)
                  tma_load_4d(smem + C::kQ + g * C::kTile + c * kChunk, &tq, &q_full[g], c * 64, it.q0 + g * kBM, it.h, it.b);
                q_issued[g] = true;
              }
              if (!ok) { ++L; break; }
            }
          }
        }
        ++used;
      }
      if (!ok) {  // our own bulk copies must land before the CTA exits
        for (int g = 0; g < QT; ++g)
          if (q_issued[g]) mbar_wait(&q_full[g], 0, nullptr, 0, 0, nullptr, 200000000LL), mbar_wait(&q_full[g], 1, nullptr, 0, 0, nullptr, 200000000LL);
        for (int i = 0; i < R; ++i)
          if (issued[i]) {
            if constexpr (MASK == kSlide) {
              if ((raw >> i) & 1u) {
                mbar_wait(&v_raw[i], ((raw_par >> i) & 1u) ^ 1u, nullptr, 0, 0, nullptr, 200000000LL);
                continue;
              }
            }
            mbar_wait(&kv_full[i], issued_par[i], nullptr, 0, 0, nullptr, 200000000LL);
          }
      }
    }
  } else if (warp == C::kMmaWarp) {
    if constexpr (QT == 2) fewer_registers<MASK>();
    if (lane == 0) {
      constexpr uint32_t kF16Bits = F16 ? (1u << 7) | (1u << 10) : 0u;  // clears the two bf16 format bits
      constexpr uint32_t idesc_qk = make_idesc_bf16_f32(kBM, kBN, 0, 0) & ~kF16Bits;
      constexpr uint32_t idesc_pv = make_idesc_bf16_f32(kBM, DH, 0, 1) & ~kF16Bits;
      constexpr uint64_t kHiK = make_sdesc_sw128(0, 16, 1024);      // K-major Q / K tiles
      constexpr uint64_t kHiV = make_sdesc_sw128(0, kChunk, 1024);  // MN-major V tiles
      const uint32_t q_lo = smem_u32(smem + C::kQ) >> 4, kv_lo = smem_u32(smem + C::kKV) >> 4;
      auto slot_lo = [&](int L) { return kv_lo + (uint32_t)(L % R) * (C::kTile >> 4); };
      auto wait_load = [&](int L, int detail) {
        return mbar_wait(&kv_full[L % R], (L / R) & 1, err, kKidCross, detail, abort_flag);
      };
      auto issue_qk = [&](int g, int s) {
        const uint32_t qa = q_lo + (uint32_t)g * (C::kTile >> 4), ka = slot_lo(2 * s);
#pragma unroll
        for (int kk = 0; kk < DH / 16; ++kk) {
          const uint32_t o = (uint32_t)((((kk >> 2) * kChunk) + (kk & 3) * 32) >> 4);
          umma_f16_ss(tmem + 128u * g, kHiK | (qa + o), kHiK | (ka + o), idesc_qk, kk > 0 ? 1u : 0u);
        }
        umma_commit(&s_full[g]);
      };
      // P V of step s (first / last: of its item); P_g arrives in two halves of 64 keys
      auto issue_pv = [&](int g, int s, bool first, bool last) -> bool {
        const uint32_t va = slot_lo(2 * s + 1), o_t = tmem + C::kOCol + (uint32_t)(DH * g);
        for (int hf = 0; hf < 2; ++hf) {
          if (!mbar_wait(&p_full[2 * g + hf], s & 1, err, kKidCross, 130 + 2 * g + hf, abort_flag)) return false;
          tc_fence_after();
#pragma unroll
          for (int kq = 0; kq < kBN / 32; ++kq) {
            const int kk = hf * (kBN / 32) + kq;
            umma_f16_ts(o_t, tmem + 128u * g + kk * 8, kHiV | (va + (uint32_t)((kk * 2048) >> 4)), idesc_pv,
                        (!first || kk > 0) ? 1u : 0u);
          }
          if constexpr (P2) {  // the second terms lie behind the first, in the other half of S
#pragma unroll
            for (int kq = 0; kq < kBN / 32; ++kq) {
              const int kk = hf * (kBN / 32) + kq;
              umma_f16_ts(o_t, tmem + 128u * g + 64u + kk * 8, kHiV | (va + (uint32_t)((kk * 2048) >> 4)), idesc_pv, 1u);
            }
          }
        }
        if (last) umma_commit(&o_full[g]);
        return true;
      };
      bool ok = true, have = false, p_first = false, p_last = false;
      int s = 0, used = 0;
      uint32_t clean_par = 0;  // bit per slot: parity of its next v_clean phase
      // V_{s-1} must have landed, and (where keys may be masked) have passed the clean warp
      auto prev_ready = [&]() -> bool {
        const int slot = (2 * s - 1) % R;
        if (!wait_load(2 * s - 1, 114)) return false;
        if (!cleaning) return true;
        const uint32_t par = (clean_par >> slot) & 1u;
        clean_par ^= 1u << slot;
        return mbar_wait(&v_clean[slot], par, err, kKidCross, 116, abort_flag);
      };
      for (Items it(p); it.more(p) && ok; it.next(p)) {
        if (it.n == 0) continue;
        for (int j = 0; j < it.n && ok; ++j, ++s) {
          if (!wait_load(2 * s, 113)) { ok = false; break; }
          if (have && (!prev_ready() || !issue_pv(0, s - 1, p_first, p_last))) { ok = false; break; }
          if (j == 0 && !mbar_wait(&q_full[0], used & 1, err, kKidCross, 110, abort_flag)) { ok = false; break; }
          tc_fence_after();
          issue_qk(0, s);
          if (j == it.n - 1) umma_commit(&q_empty[0]);
          if (have) {
            if (QT == 2 && !issue_pv(1, s - 1, p_first, p_last)) { ok = false; break; }
            umma_commit(&kv_empty[(2 * s - 1) % R]);  // V_{s-1} consumed
          }
          if (QT == 2) {
            if (j == 0 && !mbar_wait(&q_full[1], used & 1, err, kKidCross, 111, abort_flag)) { ok = false; break; }
            tc_fence_after();
            issue_qk(1, s);
            if (j == it.n - 1) umma_commit(&q_empty[1]);
          }
          umma_commit(&kv_empty[(2 * s) % R]);  // K_s consumed
          have = true, p_first = j == 0, p_last = j == it.n - 1;
        }
        ++used;
      }
      if (ok && have) {
        if (prev_ready() && issue_pv(0, s - 1, p_first, p_last) && (QT == 1 || issue_pv(1, s - 1, p_first, p_last)))
          umma_commit(&kv_empty[(2 * s - 1) % R]);
      }
    }
  } else if (warp == C::kCleanWarp) {
    if constexpr (QT == 2) fewer_registers<MASK>();
    bool ok = true;
    int s = 0;
    if constexpr (MASK == kSlide) {
      // Only the tiles that hold keys which no query of the block sees pass here, a few at the window's ends: their copies are counted
      // on v_raw[slot], this warp's arrival completes kv_full[slot] in their place, and until it has the slot is not filled again, so
      // neither side can be a phase of it ahead.  (With every tile passing here, as below, 12 heads x 32760 queries took 1734 us instead of 1698.)
      uint32_t par = 0;  // a bit per slot: parity of its next phase
      for (Items it(p); it.more(p) && ok; it.next(p)) {
        for (int j = 0; j < it.n && ok; ++j, ++s) {
          const int k0 = it.tile(j) * kBN, slot = (2 * s + 1) % R;
          if (!cross_dirty<MASK>(p, it, k0)) continue;
          if (!mbar_wait_warp(&v_raw[slot], (par >> slot) & 1u, err, kKidCross, 141, abort_flag)) { ok = false; break; }
          par ^= 1u << slot;
          uint8_t* tile = smem + C::kKV + slot * C::kTile;
#pragma unroll
          for (int c = 0; c < 4; ++c) {  // as below
            const int r = 32 * c + lane, key = k0 + r;
            if (key >= it.hi || (key < it.lo && key >= it.sinks)) {
#pragma unroll
              for (int ch = 0; ch < C::kChunks; ++ch)
#pragma unroll
                for (int v = 0; v < 8; ++v)
                  *reinterpret_cast<uint4*>(tile + ch * kChunk + r * 128 + ((v + lane) & 7) * 16) = make_uint4(0u, 0u, 0u, 0u);
            }
          }
          fence_proxy_async_shared();
          __syncwarp();
          if (lane == 0) mbar_arrive(&kv_full[slot]);
        }
      }
    }
    // every V tile passes here in order (its phase of v_clean[slot] completes once), so neither this
    // warp nor the MMA warp can be a phase of a slot ahead of the other
    for (Items it(p); cleaning && it.more(p) && ok; it.next(p)) {
      for (int j = 0; j < it.n && ok; ++j, ++s) {
        const int k0 = it.tile(j) * kBN, L = 2 * s + 1;
        const bool dirty = cross_dirty<MASK>(p, it, k0);
        uint32_t w[4] = {~0u, ~0u, ~0u, ~0u};
        if (MASK == kBits && p.key_bits && dirty) {
          const uint4 b = cross_bits(p, it, 0, k0);
          w[0] = b.x, w[1] = b.y, w[2] = b.z, w[3] = b.w;
        }
        if (!mbar_wait_warp(&kv_full[L % R], (L / R) & 1, err, kKidCross, 140, abort_flag)) { ok = false; break; }
        uint8_t* tile = smem + C::kKV + (L % R) * C::kTile;
#pragma unroll
        for (int c = 0; c < 4 && dirty; ++c) {  // key row 32 c + lane: 128 bytes in every chunk (the swizzle stays inside)
          const int r = 32 * c + lane, key = k0 + r;
          if (key < it.lo || key >= it.hi || !((w[c] >> lane) & 1u)) {
#pragma unroll
            for (int ch = 0; ch < C::kChunks; ++ch)
#pragma unroll
              for (int v = 0; v < 8; ++v)
                *reinterpret_cast<uint4*>(tile + ch * kChunk + r * 128 + ((v + lane) & 7) * 16) = make_uint4(0u, 0u, 0u, 0u);
          }
        }
        fence_proxy_async_shared();
        __syncwarp();
        if (lane == 0) mbar_arrive(&v_clean[L % R]);
      }
    }
  } else if (warp >= C::kProducerWarp) {
    if constexpr (QT == 2) fewer_registers<MASK>();  // the idle warp
  } else {
    if constexpr (QT == 2) more_registers<MASK>();
    const int g = warp / 4;
    const int row = (warp & 3) * 32 + lane;  // row of the Q tile == tensor-memory lane
    const uint32_t lane_base = (uint32_t)((warp & 3) * 32) << 16;
    const uint32_t s_t = tmem + lane_base + 128u * g;
    const uint32_t o_t = tmem + lane_base + C::kOCol + (uint32_t)(DH * g);
    // window / bits: scores are scaled inside the exponent (scale > 0); bias: z is formed first
    const float sc = is_bias(MASK) ? kLog2e : p.scale * kLog2e;
    const float grow = is_bias(MASK) ? 8.f * kLn2 : 8.f;
    bool ok = true;
    int s = 0, used = 0;
    for (Items it(p); it.more(p) && ok; it.next(p)) {
      const int qrow = it.q0 + g * kBM + row;
      const bool live = qrow < p.Sq;
      float m = -INFINITY, l = 0.f;  // running maximum (log2 units; bias: natural units) and sum
      for (int j = 0; j < it.n; ++j, ++s) {
        const int k0 = it.tile(j) * kBN;
        uint4 keep = make_uint4(~0u, ~0u, ~0u, ~0u);
        if (MASK == kBits && live) keep = cross_bits(p, it, qrow, k0);
        // bias: 64 registers of it are on their way while the scores are awaited (16 bit: the whole
        // tile; f32: its first half, the second half follows as the first is used up)
        uint4 bv[is_bias(MASK) ? 16 : 1];
        const uint4* bp = nullptr;
        if constexpr (is_bias(MASK)) {
          const int qc = min(qrow, p.Sq - 1);  // (rows behind the last query read a valid one)
          bp = p.bias + it.b * p.bias_bs + it.h * p.bias_hs + (qc / 32) * p.bias_qs + it.tile(j) * p.bias_ts +
               (p.bias_rows > 1 ? qc % 32 : 0);
#pragma unroll
          for (int v = 0; v < 16; ++v) bv[v] = __ldcg(bp + v * p.bias_rows);
        }
        if (!mbar_wait_warp(&s_full[g], s & 1, err, kKidCross, 120 + g, abort_flag)) { ok = false; break; }
        tc_fence_after();
        float z[128];
        if constexpr (is_bias(MASK)) {
          const uint64_t scale2 = f2_pack(p.scale, p.scale);
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            tmem_ld_32x32b_x32(s_t + c * 32, *reinterpret_cast<uint32_t(*)[32]>(&z[c * 32]));
            tmem_wait_ld();
            float* zc = z + 32 * c;
            if constexpr (MASK == kBias16) {
#pragma unroll
              for (int v = 0; v < 4; ++v) {
                const uint32_t ws[4] = {bv[4 * c + v].x, bv[4 * c + v].y, bv[4 * c + v].z, bv[4 * c + v].w};
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                  const float2 f = unpack2<F16>(ws[e]);
                  float* zp = zc + 8 * v + 2 * e;
                  f2_unpack(f2_fma(f2_pack(zp[0], zp[1]), scale2, f2_pack(f.x, f.y)), zp[0], zp[1]);
                }
              }
            } else {
#pragma unroll
              for (int v = 0; v < 8; ++v) {
                uint4& b = bv[8 * (c & 1) + v];
                float* zp = zc + 4 * v;
                f2_unpack(f2_fma(f2_pack(zp[0], zp[1]), scale2, f2_pack(__uint_as_float(b.x), __uint_as_float(b.y))), zp[0], zp[1]);
                f2_unpack(f2_fma(f2_pack(zp[2], zp[3]), scale2, f2_pack(__uint_as_float(b.z), __uint_as_float(b.w))), zp[2], zp[3]);
                if (c < 2) b = __ldcg(bp + (16 + 8 * c + v) * p.bias_rows);
              }
            }
          }
        } else {
#pragma unroll
          for (int c = 0; c < 4; ++c) tmem_ld_32x32b_x32(s_t + c * 32, *reinterpret_cast<uint32_t(*)[32]>(&z[c * 32]));
          tmem_wait_ld();
        }
        if constexpr (MASK == kBits) {
          if ((keep.x & keep.y & keep.z & keep.w) != ~0u) {
            const uint32_t w[4] = {keep.x, keep.y, keep.z, keep.w};
#pragma unroll
            for (int c = 0; c < 128; ++c)
              if (!((w[c / 32] >> (c % 32)) & 1u)) z[c] = -INFINITY;
          }
        }
        if constexpr (MASK == kSlide) {
          // this row's keys, from k0 on: up to its own position, the last `slide` or the first `sinks` of them
          const int up = min(qrow + it.start + 1, it.hi) - k0, from = qrow - it.back + 1 - k0, sk = it.sinks - k0;
          if (up < kBN || (from > 0 && sk < kBN)) {
#pragma unroll
            for (int w = 0; w < 4; ++w) {  // (as bits: two instructions a score where the comparisons take five)
              const uint32_t keep = first_bits(up - 32 * w) & (~first_bits(from - 32 * w) | first_bits(sk - 32 * w));
#pragma unroll
              for (int c = 0; c < 32; ++c)
                if (!((keep >> c) & 1u)) z[32 * w + c] = -INFINITY;
            }
          }
        } else if (k0 < it.lo || k0 + kBN > it.hi) {
#pragma unroll
          for (int c = 0; c < 128; ++c)
            if (k0 + c < it.lo || k0 + c >= it.hi) z[c] = -INFINITY;
        }
        float mxa[8];
#pragma unroll
        for (int t = 0; t < 8; ++t) mxa[t] = fmaxf(z[t], z[8 + t]);
#pragma unroll
        for (int c = 16; c < 128; c += 16) {
#pragma unroll
          for (int t = 0; t < 8; ++t) mxa[t] = max3(mxa[t], z[c + t], z[c + 8 + t]);
        }
        const float mx = fmaxf(max3(mxa[0], mxa[1], mxa[2]), fmaxf(max3(mxa[3], mxa[4], mxa[5]), fmaxf(mxa[6], mxa[7])));
        const float m_new = fmaxf(m, is_bias(MASK) ? mx : mx * sc);
        // warp-uniform decision: tcgen05.ld / st are warp-collective
        const bool need = j > 0 && __any_sync(0xffffffffu, m_new > m + grow);
        const float m_old = m;
        if (j == 0 || need) m = m_new;
        const float m_use = m == -INFINITY ? 0.f : m;
        if (need) {  // O_g is stable: P V_g(s-1) completed before S_g(s)
          const float f = m_old == -INFINITY ? 0.f : exp2_sfu(is_bias(MASK) ? (m_old - m) * kLog2e : m_old - m);
#pragma unroll 1
          for (int c = 0; c < DH / 16; ++c) {
            uint32_t o_raw[16];
            tmem_ld_32x32b_x16(o_t + c * 16, o_raw);
            tmem_wait_ld();
#pragma unroll
            for (int e = 0; e < 16; ++e) o_raw[e] = __float_as_uint(__uint_as_float(o_raw[e]) * f);
            tmem_st_32x32b_x16(o_t + c * 16, o_raw);
          }
          l *= f;
        }
        uint64_t rs[2] = {f2_pack(0.f, 0.f), f2_pack(0.f, 0.f)};
        const uint64_t sc2 = f2_pack(sc, sc), nm2 = f2_pack(-m_use, -m_use);
#pragma unroll
        for (int qtr = 0; qtr < 4; ++qtr) {
          uint32_t pk[16], p2[P2 ? 16 : 1];
#pragma unroll
          for (int c = 0; c < 16; ++c) {
            const uint64_t zz = f2_pack(z[qtr * 32 + 2 * c], z[qtr * 32 + 2 * c + 1]);
            float x0, x1;
            if constexpr (is_bias(MASK)) {  // the difference first: a bias near the type's lowest value times log2(e) is -inf
              f2_unpack(f2_mul(f2_add(zz, nm2), sc2), x0, x1);
            } else {
              f2_unpack(f2_fma(zz, sc2, nm2), x0, x1);
            }
            const float e0 = exp2_sfu(x0), e1 = exp2_sfu(x1);
            rs[c & 1] = f2_add(rs[c & 1], f2_pack(e0, e1));
            pk[c] = pack2<F16>(e0, e1);
            if constexpr (P2) {
              const float2 first = unpack2<F16>(pk[c]);
              p2[c] = pack2<F16>(e0 - first.x, e1 - first.y);
            }
          }
          tmem_st_32x32b_x16(s_t + qtr * 16, pk);
          if constexpr (P2) tmem_st_32x32b_x16(s_t + 64 + qtr * 16, p2);
          if (qtr & 1) {
            tmem_wait_st();
            tc_fence_before();
            mbar_arrive(&p_full[2 * g + (qtr >> 1)]);
          }
        }
        float a0, a1, b0, b1;
        f2_unpack(rs[0], a0, a1);
        f2_unpack(rs[1], b0, b1);
        l += (a0 + a1) + (b0 + b1);
      }
      if (!ok) break;
      if constexpr (MASK == kSlide) {
        if (p.splits > 1) {  // a part: the row as it is weighted by its own maximum and sum, in f32; `to` addresses the parts
          if (it.n > 0) {
            if (!mbar_wait_warp(&o_full[g], used & 1, err, kKidCross, 122 + g, abort_flag)) { ok = false; break; }
            ++used;
            tc_fence_after();
            const float inv = l == 0.f ? 0.f : 1.f / l;
            uint8_t* stage = smem + C::kOut + warp * 4096;  // 32 rows x 32 values, swizzled as below
            const int r0 = it.q0 + g * kBM + (warp & 3) * 32;
#pragma unroll 1
            for (int c = 0; c < DH; c += 32) {
              if (lane == 0) bulk_wait_read();
              __syncwarp();
              uint32_t o_raw[32];
              tmem_ld_32x32b_x32(o_t + c, o_raw);
              tmem_wait_ld();
#pragma unroll
              for (int i = 0; i < 8; ++i)
                *reinterpret_cast<float4*>(stage + lane * 128 + ((i ^ (lane & 7)) * 16)) =
                    make_float4(__uint_as_float(o_raw[4 * i]) * inv, __uint_as_float(o_raw[4 * i + 1]) * inv,
                                __uint_as_float(o_raw[4 * i + 2]) * inv, __uint_as_float(o_raw[4 * i + 3]) * inv);
              fence_proxy_async_shared();
              __syncwarp();
              if (lane == 0 && r0 < p.Sq) {
                tma_store_4d(&to, stage, c, r0, it.h, it.sp * p.B + it.b);
                bulk_commit();
              }
            }
            tc_fence_before();  // O_g has been read before this thread's next P_g signal
          }
          if (live) p.part_l[(((long long)it.sp * p.B + it.b) * p.H + it.h) * p.Sq + qrow] = l == 0.f ? -INFINITY : m + log2f(l);
          continue;
        }
      }
      // this item's rows
      uint16_t* op = reinterpret_cast<uint16_t*>(p.o) + it.b * p.o_bs + it.h * p.o_hs + (long long)qrow * p.o_ss;
      if (it.n == 0) {
        if (live)
#pragma unroll 1
          for (int c = 0; c < DH / 8; ++c) reinterpret_cast<uint4*>(op)[c] = make_uint4(0u, 0u, 0u, 0u);
      } else {
        if (!mbar_wait_warp(&o_full[g], used & 1, err, kKidCross, 122 + g, abort_flag)) { ok = false; break; }
        ++used;
        tc_fence_after();
        const float inv = l == 0.f ? 0.f : 1.f / l;  // (a NaN sum stays NaN)
        const bool none = l == 0.f;
        // through shared memory (the store's swizzle: 16-byte piece i of row r at i ^ (r % 8)): a thread's own
        // row would cost a line per lane and store
        uint8_t* stage = smem + C::kOut + warp * 4096;
        const int r0 = it.q0 + g * kBM + (warp & 3) * 32;
#pragma unroll 1
        for (int ch = 0; ch < C::kChunks; ++ch) {
          if (lane == 0) bulk_wait_read();  // what left this buffer last has been read
          __syncwarp();
#pragma unroll
          for (int hf = 0; hf < 2; ++hf) {
            uint32_t o_raw[32];
            tmem_ld_32x32b_x32(o_t + ch * 64 + hf * 32, o_raw);
            tmem_wait_ld();
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              float o[8];
#pragma unroll
              for (int e = 0; e < 8; ++e) o[e] = none ? 0.f : __uint_as_float(o_raw[8 * i + e]) * inv;
              *reinterpret_cast<uint4*>(stage + lane * 128 + (((hf * 4 + i) ^ (lane & 7)) * 16)) =
                  make_uint4(pack2<F16>(o[0], o[1]), pack2<F16>(o[2], o[3]), pack2<F16>(o[4], o[5]), pack2<F16>(o[6], o[7]));
            }
          }
          fence_proxy_async_shared();
          __syncwarp();
          if (lane == 0 && r0 < p.Sq) {  // (rows past the last query are clipped)
            tma_store_4d(&to, stage, ch * 64, r0, it.h, it.b);
            bulk_commit();
          }
        }
        tc_fence_before();  // O_g has been read before this thread's next P_g signal
      }
      if (p.lse && live)
        p.lse[((long long)it.b * p.H + it.h) * p.Sq + qrow] =
            l == 0.f ? -INFINITY : (is_bias(MASK) ? m + logf(l) : (m + log2f(l)) * kLn2);
    }
    if (lane == 0) bulk_wait_all();  // this warp's stores have left shared memory
  }

  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == C::kMmaWarp) tmem_dealloc(tmem, C::kTmemCols);
}

// A block's rows from its parts, added in order; a thread takes 4 values of a row.
template <int DH, bool F16>
__global__ void __launch_bounds__(256) cross_join_kernel(const CrossParams p) {
  griddep_wait();
  constexpr int kRows = 256 / (DH / 4);
  const int d = threadIdx.x % (DH / 4) * 4;
  const long long rows = (long long)p.B * p.H * p.Sq;
  for (int bh = blockIdx.y; bh < p.B * p.H; bh += gridDim.y)
    for (int q = blockIdx.x * kRows + threadIdx.x / (DH / 4); q < p.Sq; q += gridDim.x * kRows) {
      const long long r = (long long)bh * p.Sq + q;
      float l[kMaxParts], top = -INFINITY;
#pragma unroll
      for (int s = 0; s < kMaxParts; ++s) {
        l[s] = s < p.splits ? __ldcg(p.part_l + s * rows + r) : -INFINITY;
        top = fmaxf(top, l[s]);
      }
      const float use = top == -INFINITY ? 0.f : top;
      float sum = 0.f;
      float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int s = 0; s < kMaxParts; ++s) {
        if (s >= p.splits || l[s] == -INFINITY) continue;  // (nothing was stored for it)
        const float f = exp2_sfu(l[s] - use);
        const float4 x = __ldcg(reinterpret_cast<const float4*>(p.part_o + (s * rows + r) * DH + d));
        o.x += f * x.x, o.y += f * x.y, o.z += f * x.z, o.w += f * x.w;
        sum += f;
      }
      const float inv = sum == 0.f ? 0.f : 1.f / sum;
      *reinterpret_cast<uint2*>(reinterpret_cast<uint16_t*>(p.o) + bh / p.H * p.o_bs + bh % p.H * p.o_hs + (long long)q * p.o_ss + d) =
          make_uint2(pack2<F16>(o.x * inv, o.y * inv), pack2<F16>(o.z * inv, o.w * inv));
      if (p.lse && d == 0) p.lse[r] = sum == 0.f ? -INFINITY : (use + log2f(sum)) * kLn2;
    }
}

inline int cross_tmap(CUtensorMap* map, const void* base, int D, long long S, int H, int B, long long ss, long long hs,
                      long long bs, bool f16, bool out = false, bool f32 = false) {
  dfl_host::EncodeTiledFn fn = dfl_host::get_encode_tiled();
  if (!fn) return 999;
  cuuint64_t dims[4] = {(cuuint64_t)D, (cuuint64_t)S, (cuuint64_t)H, (cuuint64_t)B};
  const cuuint64_t e = f32 ? 4 : 2;
  cuuint64_t strides[3] = {(cuuint64_t)ss * e, (cuuint64_t)hs * e, (cuuint64_t)bs * e};
  cuuint32_t box[4] = {f32 ? 32u : 64u, out ? 32u : 128u, 1, 1};
  cuuint32_t estr[4] = {1, 1, 1, 1};
  return (int)fn(map, f32 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : f16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4,
                 const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                 CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
}

template <int DH, bool F16, int QT, int MASK, bool P2>
int launch_cross(const CrossArgs* a, CrossParams p, cudaStream_t stream, int dev) {
  using C = CrossCfg<DH, QT>;
  auto kern = cross_attn_kernel<DH, F16, QT, MASK, P2>;
  static bool attr[16] = {false};
  if (!attr[dev & 15]) {
    cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kTotal);
    if (e != cudaSuccess) return (int)e;
    if (QT == 2) {
      cudaFuncAttributes fa;
      e = cudaFuncGetAttributes(&fa, kern);
      if (e != cudaSuccess) return (int)e;
      if (fa.numRegs * C::kThreads < (MASK == kSlide ? 128 * 88 + 256 * 208 : 128 * 64 + 256 * 216)) return -11;
    }
    attr[dev & 15] = true;
  }
  CUtensorMap tq, tk, tv, to;
  int rc = cross_tmap(&tq, a->q, DH, a->Sq, a->H, a->B, a->q_ss, a->q_hs, a->q_bs, F16);
  if (rc) return 1000 + rc;
  rc = cross_tmap(&tk, a->k, DH, a->Sk, a->Hk, a->B, a->k_ss, a->k_hs, a->k_bs, F16);
  if (rc) return 2000 + rc;
  rc = cross_tmap(&tv, a->v, DH, a->Sk, a->Hk, a->B, a->v_ss, a->v_hs, a->v_bs, F16);
  if (rc) return 3000 + rc;
  if (MASK == kSlide && p.splits > 1)
    rc = cross_tmap(&to, p.part_o, DH, a->Sq, a->H, a->B * p.splits, DH, (long long)a->Sq * DH, (long long)a->H * a->Sq * DH, F16, true, true);
  else
    rc = cross_tmap(&to, a->o, DH, a->Sq, a->H, a->B, a->o_ss, a->o_hs, a->o_bs, F16, true);
  if (rc) return 4000 + rc;
  p.n_qb = (a->Sq + QT * kBM - 1) / (QT * kBM);
  const long long items = (long long)p.n_qb * a->H * a->B * p.splits;
  const int sms = dfl_host::num_sms(dev);
  const cudaError_t e = dfl_host::launch_early(kern, (unsigned)(items < sms ? items : sms), C::kThreads, C::kTotal, stream, tq, tk, tv, to, p, a->err);
  if (MASK != kSlide || p.splits == 1 || e != cudaSuccess) return (int)e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)((a->Sq + 1024 / DH - 1) / (1024 / DH)), (unsigned)std::min<long long>((long long)a->B * a->H, 65535), 1);
  cfg.blockDim = dim3(256, 1, 1);
  cfg.stream = stream;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  return (int)cudaLaunchKernelEx(&cfg, cross_join_kernel<DH, F16>, p);
}

// Two ping-pong Q tiles per CTA unless one holds every query, or twice the items still fit the SMs.
template <int DH, bool F16, int MASK, bool P2 = false>
int launch_cross_qt(const CrossArgs* a, const CrossParams& p, cudaStream_t stream, int dev) {
  if constexpr (MASK == kSlide)
    return a->q_tiles == 1 ? launch_cross<DH, F16, 1, MASK, P2>(a, p, stream, dev) : launch_cross<DH, F16, 2, MASK, P2>(a, p, stream, dev);
  const long long items2 = (long long)((a->Sq + 2 * kBM - 1) / (2 * kBM)) * a->H * a->B;
  if (a->Sq <= kBM || items2 * 2 <= dfl_host::num_sms(dev)) return launch_cross<DH, F16, 1, MASK, P2>(a, p, stream, dev);
  return launch_cross<DH, F16, 2, MASK, P2>(a, p, stream, dev);
}

template <int DH, bool F16>
int launch_cross_mask(const CrossArgs* a, const CrossParams& p, cudaStream_t stream, int dev) {
  if (a->bias_tiles)
    return a->bias_f32 ? launch_cross_qt<DH, F16, kBias32>(a, p, stream, dev)
                       : launch_cross_qt<DH, F16, kBias16>(a, p, stream, dev);
  if (a->bits) return launch_cross_qt<DH, F16, kBits>(a, p, stream, dev);
  if (a->slide) return launch_cross_qt<DH, F16, kSlide>(a, p, stream, dev);
  if (a->p2) return launch_cross_qt<DH, F16, kWindow, true>(a, p, stream, dev);
  return launch_cross_qt<DH, F16, kWindow>(a, p, stream, dev);
}

template <bool F16>
int cross_entry(const CrossArgs* a, cudaStream_t stream) {
  CrossParams p{};
  p.o = a->o;
  p.o_bs = a->o_bs, p.o_hs = a->o_hs, p.o_ss = a->o_ss;
  p.lse = a->lse;
  p.B = a->B, p.H = a->H, p.Sq = a->Sq, p.Sk = a->Sk;
  p.rep = a->H / a->Hk;
  p.scale = a->scale;
  p.kv_lo = a->kv_lo, p.kv_hi = a->kv_hi;
  p.bits = a->bits;
  p.bits_bs = a->bits_bs, p.bits_hs = a->bits_hs, p.bits_qs = a->bits_qs;
  p.key_bits = a->key_bits;
  p.bias = reinterpret_cast<const uint4*>(a->bias_tiles);
  p.bias_bs = a->bias_bs, p.bias_hs = a->bias_hs, p.bias_qs = a->bias_qs, p.bias_ts = a->bias_ts;
  p.bias_rows = a->bias_rows;
  p.start = a->start;
  p.slide = a->slide, p.sinks = a->sinks;
  p.splits = a->slide ? a->splits : 1;
  p.part_o = a->parts;
  p.part_l = a->parts + (long long)p.splits * a->B * a->H * a->Sq * a->dh;
  int dev = 0;
  cudaGetDevice(&dev);
  return a->dh == 64 ? launch_cross_mask<64, F16>(a, p, stream, dev) : launch_cross_mask<128, F16>(a, p, stream, dev);
}

}  // namespace
