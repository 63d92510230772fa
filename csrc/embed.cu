// Embedding lookup y[i] = scale * W[ids[i]] and its gradient (sm_100a), f32, bf16 or fp16.
//
// Lookup: bound by its bytes; a thread moves 16-byte pieces (single values where a row is no multiple of them).  The product
// is formed in f32 and rounded once.
//
// Gradient: dW[v] = scale * sum of dy[i] over the tokens i with id v.  Every row of dW is written once, by the warp that sums it,
// zeros among them; f32 sums in ascending order of i, so the result does not depend on the order of atomics.
//   embed_sort_kernel  one cluster groups the tokens by id: count (a warp adds equal ids at once), give every id that occurs a
//                      range of the list, place.  Where the range lies and in which order tokens arrive there is left to chance;
//                      ids with more than 32 tokens are put in ascending order here, the rest by the warp that sums them.
//                      Their tokens are cut into items of 64.
//   embed_sum_kernel   warps take (item, 32 pieces of a row), then rows.  An item's sums are kept in f32 and the
//                      last warp of a row's piece adds them in order.
// A sort by value is not needed for that, and a scan over the vocabulary neither.
#include <algorithm>

#include <cuda_fp16.h>

#include "common.cuh"
#include "kernels.h"
#include "pair.cuh"

namespace {
using namespace dfl;

constexpr int kCluster = 8, kSortThreads = 1024, kFew = 32, kItem = 64, kByWarp = 256;
constexpr int kWindow = 1 << 18;  // tokens whose order a CTA finds by one bitmap in shared memory (32 KB)

struct Item {
  int row, begin, len, part;  // part: of the partial sums, -1 where the item is the whole row
  int first, items, ticket, pad;  // of the row: first part, items, index of its counters
};

struct EmbedWs {
  int* count;   // [V]
  int* start;   // [V]
  int* rank;    // [n]: of a token among its id's, in order of arrival
  int* list;    // [n]
  int* tmp;     // [n]
  int* many;    // [n / 32]: rows with more than kFew tokens
  Item* items;  // [n / 32]
  int* ticket;  // [n / 32][pieces]
  int* head;    // list length, rows in `many`, items, parts, tickets
  float* part;  // [n / 32][D]
};

__host__ __device__ inline long long up16(long long b) { return (b + 15) / 16 * 16; }
// (an item of at most 64 tokens belongs to a row of more than 32: there are at most n / 32 of them)
inline long long embed_layout(long long n, long long V, int D, char* base, EmbedWs* w) {
  long long at = 0;
  const long long m = n / kFew + 1, chunks = (D + 31) / 32;
  auto take = [&](long long bytes) {
    char* p = base + at;
    at += up16(bytes);
    return p;
  };
  EmbedWs r;
  r.count = reinterpret_cast<int*>(take(4 * V));
  r.start = reinterpret_cast<int*>(take(4 * V));
  r.rank = reinterpret_cast<int*>(take(4 * n));
  r.list = reinterpret_cast<int*>(take(4 * n));
  r.tmp = reinterpret_cast<int*>(take(4 * n));
  r.many = reinterpret_cast<int*>(take(4 * m));
  r.items = reinterpret_cast<Item*>(take((long long)sizeof(Item) * m));
  r.ticket = reinterpret_cast<int*>(take(4 * m * chunks));
  r.head = reinterpret_cast<int*>(take(64));
  r.part = reinterpret_cast<float*>(take(4 * m * D));
  if (w) *w = r;
  return at;
}

DFL_DEVICE long long id_at(const void* ids, int bytes, long long i) {
  return bytes == 8 ? __ldg(reinterpret_cast<const long long*>(ids) + i) : (long long)__ldg(reinterpret_cast<const int*>(ids) + i);
}

// Types: a piece is VEC values.
template <int DT>
struct Value;
template <>
struct Value<kDtypeF32> {
  using T = float;
  static constexpr int kWide = 4;
  static DFL_DEVICE float get(float v) { return v; }
  static DFL_DEVICE float put(float v) { return v; }
};
template <>
struct Value<kDtypeBf16> {
  using T = __nv_bfloat16;
  static constexpr int kWide = 8;
  static DFL_DEVICE float get(T v) { return __bfloat162float(v); }
  static DFL_DEVICE T put(float v) { return __float2bfloat16_rn(v); }
};
template <>
struct Value<kDtypeF16> {
  using T = __half;
  static constexpr int kWide = 8;
  static DFL_DEVICE float get(T v) { return __half2float(v); }
  static DFL_DEVICE T put(float v) { return __float2half_rn(v); }
};

template <class T, int VEC>
struct alignas(sizeof(T) * VEC) Piece {
  T v[VEC];
};

template <int DT, int VEC>
__global__ void __launch_bounds__(256) embed_kernel(EmbedArgs a, int lanes) {
  using V = Value<DT>;
  using P = Piece<typename V::T, VEC>;
  griddep_wait();
  const int pieces = a.D / VEC, sub = threadIdx.x / lanes, lane = threadIdx.x % lanes, rows = 256 / lanes;
  for (long long i = (long long)blockIdx.x * rows + sub; i < a.n; i += (long long)gridDim.x * rows) {
    const long long id = id_at(a.ids, a.id_bytes, i);
    const bool in = id >= 0 && id < a.V;
    if (!in && lane == 0) record_error(a.err, kErrBounds, kKidEmbed, 1, (int)i);
    const P* src = reinterpret_cast<const P*>(reinterpret_cast<const typename V::T*>(a.w) + (in ? id * a.ldw : 0));
    P* dst = reinterpret_cast<P*>(reinterpret_cast<typename V::T*>(a.y) + i * a.D);
#pragma unroll 4
    for (int c = lane; c < pieces; c += lanes) {
      P x;
      if (in) x = src[c];
#pragma unroll
      for (int e = 0; e < VEC; ++e) x.v[e] = in ? V::put(a.scale * V::get(x.v[e])) : V::put(0.f);
      dst[c] = x;
    }
  }
}

DFL_DEVICE int warp_add(int* p, int v) {  // exclusive sum over the lanes of what they add to *p
  int s = v;
  const int lane = threadIdx.x % 32;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int x = __shfl_up_sync(0xffffffffu, s, o);
    if (lane >= o) s += x;
  }
  int base = 0;
  if (lane == 31 && s) base = atomicAdd(p, s);
  return __shfl_sync(0xffffffffu, base, 31) + s - v;
}

__global__ void __cluster_dims__(kCluster, 1, 1) __launch_bounds__(kSortThreads, 1) embed_sort_kernel(EmbedGradArgs a, EmbedWs w) {
  __shared__ uint32_t bits[kWindow / 32];
  __shared__ int sums[kSortThreads / 32];
  griddep_wait();
  constexpr int kAll = kCluster * kSortThreads;
  const int me = blockIdx.x * kSortThreads + threadIdx.x, lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  auto sync = [] {
    __threadfence();
    cluster_sync();
  };
  for (long long v = me; v < a.V; v += kAll) w.count[v] = 0;
  if (me < 16) w.head[me] = 0;
  sync();
  // (whole warps walk the tokens, so that every lane takes part in the warp's operations)
  const long long rounds = (a.n + kAll - 1) / kAll;
  for (long long r = 0; r < rounds; ++r) {
    const long long i = r * kAll + me;
    int id = -1;
    if (i < a.n) {
      const long long raw = id_at(a.ids, a.id_bytes, i);
      id = raw >= 0 && raw < a.V && raw != a.pad ? (int)raw : -1;
    }
    const uint32_t same = __match_any_sync(0xffffffffu, id);
    const int before = __popc(same & ((1u << lane) - 1u)), leader = __ffs(same) - 1;
    int base = 0;
    if (lane == leader && id >= 0) base = atomicAdd(w.count + id, __popc(same));
    base = __shfl_sync(0xffffffffu, base, leader);
    if (i < a.n) w.rank[i] = id >= 0 ? base + before : -1;
  }
  sync();
  for (long long r = 0; r < rounds; ++r) {
    const long long i = r * kAll + me;
    const bool first = i < a.n && w.rank[i] == 0;
    const int id = first ? (int)id_at(a.ids, a.id_bytes, i) : 0;
    const int c = first ? __ldcg(w.count + id) : 0;
    const int at = warp_add(w.head, c);
    if (first) w.start[id] = at;
    const bool large = c > kFew;
    if (__any_sync(0xffffffffu, large)) {
      const int items = large ? (c + kItem - 1) / kItem : 0;
      const int slot = warp_add(w.head + 1, large), it = warp_add(w.head + 2, items), part = warp_add(w.head + 3, items > 1 ? items : 0);
      const int ticket = warp_add(w.head + 4, items > 1);
      if (large) {
        w.many[slot] = id;
        for (int k = 0; k < items; ++k)
          w.items[it + k] = Item{id, at + k * kItem, min(kItem, c - k * kItem), items > 1 ? part + k : -1, part, items, ticket, 0};
      }
    }
  }
  sync();
  for (long long i = me; i < a.n; i += kAll) {
    const int r = w.rank[i];
    if (r >= 0) w.list[__ldcg(w.start + id_at(a.ids, a.id_bytes, i)) + r] = (int)i;
  }
  const long long tickets = (long long)__ldcg(w.head + 4) * ((a.D + 31) / 32);
  for (long long i = me; i < tickets; i += kAll) w.ticket[i] = 0;
  sync();
  // rows with many tokens: a warp finds each token's place by counting, up to kByWarp of them; a CTA by a bitmap above
  const int rows = __ldcg(w.head + 1);
  for (int j = me / 32; j < rows; j += kAll / 32) {
    const int id = __ldcg(w.many + j), c = __ldcg(w.count + id), at = __ldcg(w.start + id);
    if (c > kByWarp) continue;
    for (int k = lane; k < c; k += 32) {
      const int mine = __ldcg(w.list + at + k);
      int place = 0;
      for (int o = 0; o < c; ++o) place += __ldcg(w.list + at + o) < mine;
      w.tmp[at + place] = mine;
    }
    __syncwarp();
    for (int k = lane; k < c; k += 32) w.list[at + k] = w.tmp[at + k];
  }
  for (int j = blockIdx.x; j < rows; j += kCluster) {
    const int id = __ldcg(w.many + j), c = __ldcg(w.count + id), at = __ldcg(w.start + id);
    if (c <= kByWarp) continue;
    int done = 0;
    for (long long w0 = 0; w0 < a.n; w0 += kWindow) {
      const int words = (int)((min((long long)kWindow, a.n - w0) + 31) / 32);
      for (int k = threadIdx.x; k < words; k += kSortThreads) bits[k] = 0u;
      __syncthreads();
      for (int k = threadIdx.x; k < c; k += kSortThreads) {
        const long long p = __ldcg(w.list + at + k) - w0;
        if (p >= 0 && p < kWindow) atomicOr(&bits[p / 32], 1u << (p % 32));
      }
      __syncthreads();
      // a thread takes consecutive words; how many tokens lie before them, by a sum over the threads
      const int per = (words + kSortThreads - 1) / kSortThreads, k0 = min(words, (int)threadIdx.x * per), k1 = min(words, k0 + per);
      int mine = 0;
      for (int k = k0; k < k1; ++k) mine += __popc(bits[k]);
      int s = mine;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int x = __shfl_up_sync(0xffffffffu, s, o);
        if (lane >= o) s += x;
      }
      if (lane == 31) sums[warp] = s;
      __syncthreads();
      int all = 0;
      for (int k = 0; k < kSortThreads / 32; ++k) {
        if (k == warp) s += all;
        all += sums[k];
      }
      int to = at + done + s - mine;
      for (int k = k0; k < k1; ++k)
        for (uint32_t b = bits[k]; b; b &= b - 1) w.tmp[to++] = (int)(w0 + k * 32 + __ffs(b) - 1);
      done += all;
      __syncthreads();
    }
    for (int k = threadIdx.x; k < c; k += kSortThreads) w.list[at + k] = w.tmp[at + k];
    __syncthreads();
  }
}

template <int DT, int VEC>
__global__ void __launch_bounds__(256) embed_sum_kernel(EmbedGradArgs a, EmbedWs w) {
  using V = Value<DT>;
  using P = Piece<typename V::T, VEC>;
  griddep_wait();
  const int lane = threadIdx.x % 32, pieces = a.D / VEC, chunks = (pieces + 31) / 32;
  const long long warps = (long long)gridDim.x * 8, me = (long long)blockIdx.x * 8 + threadIdx.x / 32;
  const typename V::T* dy = reinterpret_cast<const typename V::T*>(a.dy);
  typename V::T* dw = reinterpret_cast<typename V::T*>(a.dw);
  auto add = [&](float (&s)[VEC], const P& x) {
#pragma unroll
    for (int e = 0; e < VEC; ++e) s[e] += V::get(x.v[e]);
  };
  auto piece_of = [&](int token, int c) { return reinterpret_cast<const P*>(dy + (long long)token * a.D) + c; };
  auto put = [&](long long row, int c, const float (&s)[VEC]) {
    P x;
#pragma unroll
    for (int e = 0; e < VEC; ++e) x.v[e] = V::put(a.scale * s[e]);
    reinterpret_cast<P*>(dw + row * a.D)[c] = x;
  };

  const long long items = (long long)__ldcg(w.head + 2) * chunks;
  for (long long t = me; t < items; t += warps) {
    const Item it = w.items[t / chunks];
    const int chunk = (int)(t % chunks), c = chunk * 32 + lane;
    float s[VEC];
#pragma unroll
    for (int e = 0; e < VEC; ++e) s[e] = 0.f;
    const int t0 = lane < it.len ? __ldcg(w.list + it.begin + lane) : 0, t1 = lane + 32 < it.len ? __ldcg(w.list + it.begin + 32 + lane) : 0;
#pragma unroll 8
    for (int k = 0; k < it.len; ++k) {
      const int token = __shfl_sync(0xffffffffu, k < 32 ? t0 : t1, k % 32);
      if (c < pieces) add(s, *piece_of(token, c));
    }
    if (it.part < 0) {
      if (c < pieces) put(it.row, c, s);
      continue;
    }
    if (c < pieces)
#pragma unroll
      for (int e = 0; e < VEC; ++e) __stcg(w.part + (long long)it.part * a.D + c * VEC + e, s[e]);
    __threadfence();
    __syncwarp();
    int last = 0;
    if (lane == 0) last = atomicAdd(w.ticket + (long long)it.ticket * chunks + chunk, 1) == it.items - 1;
    if (!__shfl_sync(0xffffffffu, last, 0)) continue;
    __threadfence();
    if (c >= pieces) continue;
#pragma unroll
    for (int e = 0; e < VEC; ++e) s[e] = 0.f;
#pragma unroll 4
    for (int k = 0; k < it.items; ++k)
#pragma unroll
      for (int e = 0; e < VEC; ++e) s[e] += __ldcg(w.part + (long long)(it.first + k) * a.D + c * VEC + e);
    put(it.row, c, s);
  }

  for (long long v = me; v < a.V; v += warps) {
    const int n = __ldcg(w.count + v);
    if (n > kFew) continue;  // (an item's)
    int token = 0;
    if (n > 0) {  // this row's tokens in ascending order, one to a lane
      const int at = __ldcg(w.start + v);
      const int mine = lane < n ? __ldcg(w.list + at + lane) : 0x7fffffff;
      int place = 0;
      for (int k = 0; k < n; ++k) place += __shfl_sync(0xffffffffu, mine, k) < mine;
      for (int k = 0; k < n; ++k) {
        const int at_k = __shfl_sync(0xffffffffu, place, k), t = __shfl_sync(0xffffffffu, mine, k);
        if (at_k == lane) token = t;
      }
    }
#pragma unroll 2
    for (int c0 = 0; c0 < pieces; c0 += 32) {
      const int c = c0 + lane;
      float s[VEC];
#pragma unroll
      for (int e = 0; e < VEC; ++e) s[e] = 0.f;
#pragma unroll 4
      for (int k = 0; k < n; ++k) {
        const int t = __shfl_sync(0xffffffffu, token, k);
        if (c < pieces) add(s, *piece_of(t, c));
      }
      if (c < pieces) put(v, c, s);
    }
  }
}

bool al16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

template <int DT>
int launch_embed(const EmbedArgs* a, cudaStream_t stream) {
  constexpr int W = Value<DT>::kWide;
  const bool wide = a->D % W == 0 && a->ldw % W == 0 && al16(a->w) && al16(a->y);
  const int pieces = wide ? a->D / W : a->D;
  int lanes = 32;
  while (lanes < 256 && lanes < pieces) lanes *= 2;
  const long long rows = 256 / lanes, blocks = (a->n + rows - 1) / rows;
  const unsigned grid = (unsigned)std::min<long long>(blocks, 1 << 20);
  return (int)(wide ? dfl_host::launch_early(embed_kernel<DT, W>, grid, 256, 0, stream, *a, lanes)
                    : dfl_host::launch_early(embed_kernel<DT, 1>, grid, 256, 0, stream, *a, lanes));
}

template <int DT>
int launch_sum(const EmbedGradArgs* a, const EmbedWs& w, cudaStream_t stream) {
  constexpr int W = Value<DT>::kWide;
  const bool wide = a->D % W == 0 && al16(a->dy) && al16(a->dw);
  const long long work = a->V + a->n / kFew * ((a->D / (wide ? W : 1) + 31) / 32);
  const unsigned grid = (unsigned)std::min<long long>((work + 7) / 8, 148 * 8);
  return (int)(wide ? dfl_host::launch_early(embed_sum_kernel<DT, W>, grid, 256, 0, stream, *a, w)
                    : dfl_host::launch_early(embed_sum_kernel<DT, 1>, grid, 256, 0, stream, *a, w));
}

}  // namespace

extern "C" int dfl_embed(const EmbedArgs* a, cudaStream_t stream) {
  if (a->n <= 0 || a->D <= 0 || a->V < 0 || (a->id_bytes != 4 && a->id_bytes != 8)) return -2;
  switch (a->dtype) {
    case kDtypeF32: return launch_embed<kDtypeF32>(a, stream);
    case kDtypeBf16: return launch_embed<kDtypeBf16>(a, stream);
    case kDtypeF16: return launch_embed<kDtypeF16>(a, stream);
    default: return -1;
  }
}

extern "C" long long dfl_embed_grad_ws(long long n, long long V, int D) { return embed_layout(n, V, D, nullptr, nullptr); }

extern "C" int dfl_embed_grad(const EmbedGradArgs* a, cudaStream_t stream) {
  if (a->n <= 0 || a->D <= 0 || a->V <= 0 || a->n >= (1ll << 30) || a->V >= (1ll << 30) || (a->id_bytes != 4 && a->id_bytes != 8)) return -2;
  if (!al16(a->ws)) return -3;
  EmbedWs w;
  if (embed_layout(a->n, a->V, a->D, reinterpret_cast<char*>(a->ws), &w) > a->ws_bytes) return -4;
  const cudaError_t e = dfl_host::launch_early(embed_sort_kernel, kCluster, kSortThreads, 0, stream, *a, w);
  if (e != cudaSuccess) return (int)e;
  switch (a->dtype) {
    case kDtypeF32: return launch_sum<kDtypeF32>(a, w, stream);
    case kDtypeBf16: return launch_sum<kDtypeBf16>(a, w, stream);
    case kDtypeF16: return launch_sum<kDtypeF16>(a, w, stream);
    default: return -1;
  }
}
