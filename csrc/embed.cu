// Embedding lookup y[i] = scale * W[ids[i]] and its gradient (sm_100a), f32, bf16 or fp16.
//
// Lookup: bound by its bytes; a thread moves pieces of 16 bytes, or of 8, 4 or 2 where the rows' length or start asks for it.  The product
// is formed in f32 and rounded once.
//
// Gradient: dW[v] = scale * sum of dy[i] over the tokens i with id v: f32 sums in ascending order of i, so the result does not
// depend on the order of atomics, rounded once.  Bound by writing dW, nearly all of it zeros.
//   embed_sort_kernel  one cluster groups the tokens by id: count (a warp adds equal ids at once), give every id that occurs a
//                      range of the list, place.  Where the range lies and in which order tokens arrive there is left to chance;
//                      ids with more than 32 tokens are put in ascending order here, the rest by the warps that sum them.
//                      Meanwhile the other clusters fill dW with zeros.
//   embed_sum_kernel   a warp takes up to 1 KB of an item (an id's tokens, at most 64 of them).  The sums of an id's items are
//                      kept in f32 and added in order by the last warp of the piece.
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
  int row, begin, len, part;  // begin: in the list; part: of the partial sums, -1: none
  int first, items, ticket, order;  // of the row: first part, items, index of its counters
};

// An item's tokens: in any order, in ascending order, or the only one of its row, which `begin` is itself.
enum { kAnyOrder = 0, kInOrder = 1, kOnly = 2 };

struct EmbedWs {
  int* count;   // [V]
  int* start;   // [V]
  int* rank;    // [n]: of a token among its id's, in order of arrival
  int* list;    // [n]
  int* tmp;     // [n]
  int* many;    // [n / 32]: rows with more than kFew tokens
  Item* items;  // [n + n / 32]
  int* ticket;  // [n / 32][pieces]
  int* head;    // list length, rows in `many`, items, parts, tickets
  float* part;  // [n / 32][D]
};

__host__ __device__ inline long long up16(long long b) { return (b + 15) / 16 * 16; }
// (ids with more than 32 tokens have at most n / 32 items)
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
  r.items = reinterpret_cast<Item*>(take((long long)sizeof(Item) * (n + m)));
  r.ticket = reinterpret_cast<int*>(take(4 * m * chunks));
  r.head = reinterpret_cast<int*>(take(64));
  r.part = reinterpret_cast<float*>(take(4 * m * D));
  if (w) *w = r;
  return at;
}

DFL_DEVICE long long id_at(const void* ids, int bytes, long long i) {
  // (launched while the kernel before ends: what that writes is read past L1, here and below)
  return bytes == 8 ? __ldcg(reinterpret_cast<const long long*>(ids) + i) : (long long)__ldcg(reinterpret_cast<const int*>(ids) + i);
}

// A piece of a row: B = 16, 8, 4 or 2 bytes, the most that every row's start and length allow.
template <int B>
struct Bytes;
template <>
struct Bytes<16> {
  using R = uint4;
};
template <>
struct Bytes<8> {
  using R = uint2;
};
template <>
struct Bytes<4> {
  using R = uint32_t;
};
template <>
struct Bytes<2> {
  using R = uint16_t;
};

template <int DT, int B>
struct Piece {
  using R = typename Bytes<B>::R;
  static constexpr int kSize = DT == kDtypeF32 ? 4 : 2, N = B / kSize;  // values
  static_assert(B >= kSize, "a piece holds whole values");
  static DFL_DEVICE R load(const void* p) { return __ldcg(reinterpret_cast<const R*>(p)); }
  static DFL_DEVICE void values(R r, float (&v)[N]) {
    if constexpr (B == 2) {
      v[0] = DT == kDtypeBf16 ? __uint_as_float((uint32_t)r << 16) : __half2float(__ushort_as_half(r));
    } else {
      const uint32_t* w = reinterpret_cast<const uint32_t*>(&r);
#pragma unroll
      for (int i = 0; i < B / 4; ++i) {
        if constexpr (DT == kDtypeF32) {
          v[i] = __uint_as_float(w[i]);
        } else {
          const float2 f = DT == kDtypeBf16 ? unpack_bf16x2(w[i]) : __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
          v[2 * i] = f.x, v[2 * i + 1] = f.y;
        }
      }
    }
  }
  static DFL_DEVICE void store(void* p, const float (&v)[N], float scale) {  // scale * v, rounded once
    if constexpr (B == 2) {
      *reinterpret_cast<uint16_t*>(p) = DT == kDtypeBf16 ? __bfloat16_as_ushort(__float2bfloat16_rn(scale * v[0]))
                                                         : __half_as_ushort(__float2half_rn(scale * v[0]));
    } else {
      R r;
      uint32_t* w = reinterpret_cast<uint32_t*>(&r);
#pragma unroll
      for (int i = 0; i < B / 4; ++i) {
        if constexpr (DT == kDtypeF32) {
          w[i] = __float_as_uint(scale * v[i]);
        } else if constexpr (DT == kDtypeBf16) {
          w[i] = pack_bf16x2(scale * v[2 * i], scale * v[2 * i + 1]);
        } else {
          const __half2 h = __floats2half2_rn(scale * v[2 * i], scale * v[2 * i + 1]);
          w[i] = *reinterpret_cast<const uint32_t*>(&h);
        }
      }
      *reinterpret_cast<R*>(p) = r;
    }
  }
};

// Pieces that a thread has in flight: 64 bytes, or 16 loads.
template <int B>
constexpr int kFlight = B == 16 ? 4 : B == 8 ? 8 : 16;

// `lanes` threads to a row; the next row's id is on its way meanwhile.
template <int DT, int B>
__global__ void __launch_bounds__(256, 5) embed_kernel(EmbedArgs a, int lanes) {
  using P = Piece<DT, B>;
  constexpr int U = kFlight<B>;
  griddep_wait();
  const int pieces = a.D / P::N, lane = threadIdx.x % lanes, rows = 256 / lanes;
  const long long step = (long long)gridDim.x * rows;
  long long i = (long long)blockIdx.x * rows + threadIdx.x / lanes;
  if (i >= a.n) return;
  long long id = id_at(a.ids, a.id_bytes, i);
  for (; i < a.n; i += step) {
    const long long next = id_at(a.ids, a.id_bytes, min(i + step, a.n - 1));
    const bool in = id >= 0 && id < a.V;
    if (!in && lane == 0) record_error(a.err, kErrBounds, kKidEmbed, 1, (int)i);
    const uint8_t* src = reinterpret_cast<const uint8_t*>(a.w) + (in ? id * a.ldw * P::kSize : 0);
    uint8_t* dst = reinterpret_cast<uint8_t*>(a.y) + i * a.D * P::kSize;
    for (int c = lane; c < pieces; c += U * lanes) {
      typename P::R x[U];
#pragma unroll
      for (int u = 0; u < U; ++u) x[u] = in && c + u * lanes < pieces ? P::load(src + (long long)(c + u * lanes) * B) : typename P::R{};
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (c + u * lanes < pieces) {
          float v[P::N];
          P::values(x[u], v);
          P::store(dst + (long long)(c + u * lanes) * B, v, a.scale);
        }
    }
    id = next;
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
  if (blockIdx.x >= kCluster) {  // zeros
    const long long bytes = a.V * a.D * (a.dtype == kDtypeF32 ? 4 : 2), whole = bytes / 16, step = (long long)(gridDim.x - kCluster) * kSortThreads;
    const long long at = (long long)(blockIdx.x - kCluster) * kSortThreads + threadIdx.x;
    uint4* d = reinterpret_cast<uint4*>(a.dw);
    for (long long i = at; i < whole; i += step) d[i] = make_uint4(0u, 0u, 0u, 0u);
    if (at < bytes - whole * 16) reinterpret_cast<uint8_t*>(a.dw)[whole * 16 + at] = 0;
    return;
  }
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
    const int items = (c + kItem - 1) / kItem, it = warp_add(w.head + 2, items);
    int part = 0, ticket = 0;
    if (__any_sync(0xffffffffu, large)) {
      const int slot = warp_add(w.head + 1, large);
      part = warp_add(w.head + 3, items > 1 ? items : 0);
      ticket = warp_add(w.head + 4, items > 1);
      if (large) w.many[slot] = id;
    }
    for (int k = 0; k < items; ++k)
      w.items[it + k] = Item{id, c == 1 ? (int)i : at + k * kItem, min(kItem, c - k * kItem), items > 1 ? part + k : -1, part, items, ticket,
                           c == 1 ? kOnly : large ? kInOrder : kAnyOrder};
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
    int mine[kByWarp / 32], place[kByWarp / 32];
#pragma unroll
    for (int e = 0; e < kByWarp / 32; ++e) {
      mine[e] = e * 32 + lane < c ? __ldcg(w.list + at + e * 32 + lane) : 0x7fffffff;
      place[e] = 0;
    }
#pragma unroll
    for (int o = 0; o < kByWarp / 32; ++o) {
      if (o * 32 >= c) break;
      for (int s = 0; s < 32; ++s) {  // (what lies behind the last token is above all)
        const int x = __shfl_sync(0xffffffffu, mine[o], s);
#pragma unroll
        for (int e = 0; e < kByWarp / 32; ++e) place[e] += x < mine[e];
      }
    }
    __syncwarp();
#pragma unroll
    for (int e = 0; e < kByWarp / 32; ++e)
      if (e * 32 + lane < c) w.list[at + place[e]] = mine[e];
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

// A warp takes 32 U pieces of an item (lane l the pieces l, l + 32, ...), T tokens at a time; the next item is on its way meanwhile.  What counts is
// the loads in flight (most ids occur once): the whole gradient of 16384 tokens x 3584 over 152064 rows took 240 us with three CTAs an SM,
// U = 2 and four tokens in flight (two CTAs 247; U = 4 and two tokens 254, U = 1 and four 250, and eight 254), 32768 tokens
// x 4096 over 32000 rows 166 (181, 172, 186, 196); the pieces as whole words 221 and 164.
template <int B>
constexpr int kU = B == 16 ? 2 : B == 8 ? 4 : 8;
template <int B>
constexpr int kTokens = B >= 8 ? 4 : 2;

template <int DT, int B>
__global__ void __launch_bounds__(256, 3) embed_sum_kernel(EmbedGradArgs a, EmbedWs w) {
  using P = Piece<DT, B>;
  constexpr int VEC = P::N, U = kU<B>, T = kTokens<B>;
  griddep_wait();
  const int lane = threadIdx.x % 32, pieces = a.D / VEC, chunks = (pieces + 32 * U - 1) / (32 * U);
  const long long warps = (long long)gridDim.x * 8, me = (long long)blockIdx.x * 8 + threadIdx.x / 32;
  const uint8_t* dy = reinterpret_cast<const uint8_t*>(a.dy);
  uint8_t* dw = reinterpret_cast<uint8_t*>(a.dw);
  const long long row_bytes = (long long)a.D * P::kSize;

  // (item, chunk) by item * chunks + chunk, advanced without divisions
  const int items = __ldcg(w.head + 2), d_item = (int)(warps / chunks), d_chunk = (int)(warps % chunks);
  long long item = me / chunks;
  int chunk = (int)(me % chunks);
  Item it{};
  int t0 = 0, t1 = 0;
  auto tokens = [&] {  // the item's tokens, one or two to a lane
    t0 = it.order == kOnly ? it.begin : lane < it.len ? __ldcg(w.list + it.begin + lane) : 0x7fffffff;
    t1 = lane + 32 < it.len ? __ldcg(w.list + it.begin + 32 + lane) : 0;
  };
  if (item < items) {
    it = w.items[item];
    tokens();
  }
  while (item < items) {
    int to_chunk = chunk + d_chunk;
    item += d_item + (to_chunk >= chunks);
    to_chunk -= to_chunk >= chunks ? chunks : 0;
    const Item nx = w.items[min(item, items - 1ll)];
    const int c0 = chunk * 32 * U + lane;
    float s[U][VEC];
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int e = 0; e < VEC; ++e) s[u][e] = 0.f;
    if (it.order == kAnyOrder) {  // one token to a lane, in ascending order
      int place = 0;
      for (int k = 0; k < it.len; ++k) place += __shfl_sync(0xffffffffu, t0, k) < t0;
      const int mine = t0;
      for (int k = 0; k < it.len; ++k) {
        const int to = __shfl_sync(0xffffffffu, place, k), x = __shfl_sync(0xffffffffu, mine, k);
        if (to == lane) t0 = x;
      }
    }
    for (int k = 0; k < it.len; k += T) {
      typename P::R x[T][U];
#pragma unroll
      for (int j = 0; j < T; ++j) {
        if (k + j >= it.len) break;
        const uint8_t* src = dy + (long long)__shfl_sync(0xffffffffu, k < 32 ? t0 : t1, (k + j) % 32) * row_bytes;
#pragma unroll
        for (int u = 0; u < U; ++u) x[j][u] = P::load(src + (long long)min(c0 + 32 * u, pieces - 1) * B);  // (lanes past the row's end read it, and store nothing)
      }
#pragma unroll
      for (int j = 0; j < T; ++j) {
        if (k + j >= it.len) break;
#pragma unroll
        for (int u = 0; u < U; ++u) {
          float v[VEC];
          P::values(x[j][u], v);
#pragma unroll
          for (int e = 0; e < VEC; ++e) s[u][e] += v[e];
        }
      }
    }
    bool whole = true;
    if (it.part >= 0) {
      float* part = w.part + (long long)it.part * a.D;
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (c0 + 32 * u < pieces)
#pragma unroll
          for (int e = 0; e < VEC; ++e) __stcg(part + (long long)(c0 + 32 * u) * VEC + e, s[u][e]);
      __threadfence();
      __syncwarp();
      int last = 0;
      if (lane == 0) last = atomicAdd(w.ticket + (long long)it.ticket * chunks + chunk, 1) == it.items - 1;
      whole = __shfl_sync(0xffffffffu, last, 0);
      if (whole) __threadfence();
#pragma unroll
      for (int u = 0; u < U && whole; ++u) {
        const float* from = w.part + (long long)it.first * a.D + (long long)min(c0 + 32 * u, pieces - 1) * VEC;
#pragma unroll
        for (int e = 0; e < VEC; ++e) s[u][e] = 0.f;
#pragma unroll 4
        for (int k = 0; k < it.items; ++k)
#pragma unroll
          for (int e = 0; e < VEC; ++e) s[u][e] += __ldcg(from + (long long)k * a.D + e);
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (!whole || c0 + 32 * u >= pieces) break;
      P::store(dw + it.row * row_bytes + (long long)(c0 + 32 * u) * B, s[u], a.scale);
    }
    it = nx, chunk = to_chunk;
    tokens();
  }
}

bool al16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// Bytes of a piece: what divides the rows' length and pitch and both starts.
int piece_bytes(long long row, long long pitch, const void* a, const void* b) {
  const uintptr_t all = (uintptr_t)row | (uintptr_t)pitch | reinterpret_cast<uintptr_t>(a) | reinterpret_cast<uintptr_t>(b);
  return all % 16 == 0 ? 16 : all % 8 == 0 ? 8 : all % 4 == 0 ? 4 : 2;
}

template <int DT, int B>
int launch_embed(const EmbedArgs* a, cudaStream_t stream) {
  const int pieces = a->D / Piece<DT, B>::N;
  int lanes = 8;
  while (lanes < 256 && kFlight<B> * lanes < pieces) lanes *= 2;
  const long long rows = 256 / lanes, blocks = (a->n + rows - 1) / rows;
  return (int)dfl_host::launch_early(embed_kernel<DT, B>, (unsigned)std::min<long long>(blocks, 148 * 5), 256, 0, stream, *a, lanes);
}

template <int DT, int B>
int launch_sum(const EmbedGradArgs* a, const EmbedWs& w, cudaStream_t stream) {
  const int pieces = a->D / Piece<DT, B>::N;
  const long long work = (a->n + a->n / kFew) * ((pieces + 32 * kU<B> - 1) / (32 * kU<B>));  // (at most)
  return (int)dfl_host::launch_early(embed_sum_kernel<DT, B>, (unsigned)std::min<long long>((work + 7) / 8, 148 * 8), 256, 0, stream, *a, w);
}

// Calls f<type, bytes>(...).
#define DFL_EMBED(f, dtype, bytes, ...)                                                                           \
  ((dtype) == kDtypeF32                                                                                           \
       ? ((bytes) == 16 ? f<kDtypeF32, 16>(__VA_ARGS__) : (bytes) == 8 ? f<kDtypeF32, 8>(__VA_ARGS__) : f<kDtypeF32, 4>(__VA_ARGS__)) \
   : (dtype) == kDtypeBf16                                                                                        \
       ? ((bytes) == 16 ? f<kDtypeBf16, 16>(__VA_ARGS__) : (bytes) == 8 ? f<kDtypeBf16, 8>(__VA_ARGS__)           \
          : (bytes) == 4 ? f<kDtypeBf16, 4>(__VA_ARGS__) : f<kDtypeBf16, 2>(__VA_ARGS__))                         \
       : ((bytes) == 16 ? f<kDtypeF16, 16>(__VA_ARGS__) : (bytes) == 8 ? f<kDtypeF16, 8>(__VA_ARGS__)             \
          : (bytes) == 4 ? f<kDtypeF16, 4>(__VA_ARGS__) : f<kDtypeF16, 2>(__VA_ARGS__)))

}  // namespace

extern "C" int dfl_embed(const EmbedArgs* a, cudaStream_t stream) {
  if (a->n <= 0 || a->D <= 0 || a->V < 0 || (a->id_bytes != 4 && a->id_bytes != 8)) return -2;
  if (a->dtype != kDtypeF32 && a->dtype != kDtypeBf16 && a->dtype != kDtypeF16) return -1;
  const int size = a->dtype == kDtypeF32 ? 4 : 2, bytes = piece_bytes((long long)a->D * size, a->ldw * size, a->w, a->y);
  return DFL_EMBED(launch_embed, a->dtype, bytes, a, stream);
}

extern "C" long long dfl_embed_grad_ws(long long n, long long V, int D) { return embed_layout(n, V, D, nullptr, nullptr); }

extern "C" int dfl_embed_grad(const EmbedGradArgs* a, cudaStream_t stream) {
  if (a->n <= 0 || a->D <= 0 || a->V <= 0 || a->n >= (1ll << 30) || a->V >= (1ll << 30) || (a->id_bytes != 4 && a->id_bytes != 8)) return -2;
  if (a->dtype != kDtypeF32 && a->dtype != kDtypeBf16 && a->dtype != kDtypeF16) return -1;
  if (!al16(a->ws) || !al16(a->dw)) return -3;
  EmbedWs w;
  if (embed_layout(a->n, a->V, a->D, reinterpret_cast<char*>(a->ws), &w) > a->ws_bytes) return -4;
  const int size = a->dtype == kDtypeF32 ? 4 : 2, bytes = piece_bytes((long long)a->D * size, 0, a->dy, a->dw);
  // (14 clusters for the zeros; fewer where dW is small)
  const long long fill = (a->V * a->D * size + 16 * kCluster * kSortThreads - 1) / (16 * kCluster * kSortThreads);
  const unsigned clusters = 1 + (unsigned)std::min<long long>(fill, 14);
  const cudaError_t e = dfl_host::launch_early(embed_sort_kernel, clusters * kCluster, kSortThreads, 0, stream, *a, w);
  return e != cudaSuccess ? (int)e : DFL_EMBED(launch_sum, a->dtype, bytes, a, w, stream);
}
