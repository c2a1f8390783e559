// Eviction: of each sequence and head the heaviest tokens are kept, and their rows move together.
//
// Chosen exactly, by three passes over the weights' bits (11, 11, 10): each counts the numbers that share the digits found so far by their next digit, until the weight of the last kept
// token and how many of that weight are kept is known; a last pass numbers the kept ones in order.  A cluster of up to eight CTAs takes a sequence's head, and adds its counts up
// through distributed shared memory; the weights are read from L2 after the first pass.
//
// Moved by another kernel, bound by the bytes of the kept rows, read and written once.  In place: a kept token's new place is never behind its old one, so rows that are taken in order
// and written when all rows up to them have been read overwrite nothing that is still to be read.  One block, or a cluster whose blocks keep step, takes a piece of up to 64 bytes of all rows of one part of a head (the
// parts, heads and pieces of rows are independent), with the next tile's rows on their way while one is written.
// Measured: 8 x 16 heads of 64, float16 codes, from 8191 tokens to 4096 118 us (chosen 13, moved 105: 5.0 TB/s); 16 heads of 128 from 65001 to 16384 132 us (23, 108);
// with L2 flushed before the call 121 and 135, and in place 127 and 154 (clusters' barriers);
// 4 x 8 heads of 64, e4m3, from 700 to 512 15 us.  Moved in pieces of 32 bytes without clusters the second took 220 us, by clusters whose barrier waited for the next tile's loads 128; pieces of 128 bytes take 2 % less, eight loads a thread in
// place of four 18 % more (registers); chosen by weights read again
// for each pass by clusters of eight 49.
#include "tritt_weigh.cuh"

#include <cooperative_groups.h>

namespace tritt {
namespace {
namespace cg = cooperative_groups;

constexpr int kSms = 148;
constexpr int kSelectThreads = 1024, kBins = 2048, kMostCluster = 8;

struct Params {
  CacheArgs cache;
  tritt_weights_t w;
  const int* table_out;   // null: in place
  long long table_out_stride;
  int table_out_pages;
  int keep, first, recent;
  int* context_out;
  int* kept;
  int ranks;              // CTAs of a cluster that moves rows
};

// Tokens of a sequence, negative: it is not used.  (Those that have no weights are reported and left out.)
__device__ __forceinline__ int tokens_of(const Params& p, int b) {
  const int given = __ldg(p.cache.c.context + b);
  if (given < 0) return given;
  const int ctx = context_of(p.cache, b);
  if (ctx > p.w.before_length && p.cache.status) atomicOr(p.cache.status, kStatusPlace);
  return ctx < p.w.before_length ? ctx : p.w.before_length;
}

// A weight's bits in the order of the weights: a NaN as the largest, zeros of either sign alike.  (Bits from the load on: as a number the smallest would be taken for a zero, whose comparisons with
// fast arithmetic they are.)
__device__ __forceinline__ uint32_t order_of(uint32_t u) {
  const uint32_t size = u & 0x7fffffffu;
  if (size > 0x7f800000u) return 0xffffffffu;
  if (size == 0u) return 0x80000000u;
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// Inclusive sum over the block's threads (1024), and the sum of all.
__device__ __forceinline__ uint32_t scan1024(uint32_t v, uint32_t* tmp, uint32_t& total) {
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint32_t u = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += u;
  }
  __syncthreads();
  if (lane == 31) tmp[warp] = v;
  __syncthreads();
  uint32_t t = tmp[lane];
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint32_t u = __shfl_up_sync(0xffffffffu, t, o);
    if (lane >= o) t += u;
  }
  total = __shfl_sync(0xffffffffu, t, 31);
  const uint32_t before = __shfl_sync(0xffffffffu, t, warp ? warp - 1 : 0);
  return v + (warp ? before : 0u);
}

// HELD: a thread's weights, kHeld neighbours of them, stay in its registers (a CTA has at most kHeld * 1024); else they are read again for each pass.
constexpr int kHeld = 16;
template <bool HELD> __global__ void __launch_bounds__(kSelectThreads) evict_select_kernel(const __grid_constant__ Params p) {
  __shared__ __align__(8) uint32_t hist[3][kBins], tmp[32], found[2], counts[2];
  let_next_start();
  const CacheArgs& a = p.cache;
  const cg::cluster_group cluster = cg::this_cluster();
  const int rank = blockIdx.x, ranks = gridDim.x, tid = threadIdx.x;
  const int bh = blockIdx.y, b = bh / a.c.N, head = bh - b * a.c.N;
  const int ctx = tokens_of(p, b);
  if (rank == 0 && head == 0 && tid == 0) p.context_out[b] = ctx < p.keep ? ctx : p.keep;
  int* const kept = p.kept + (size_t)bh * p.keep;
  if (ctx <= p.keep) {   // (all of a cluster's CTAs)
    for (int r = rank * kSelectThreads + tid; r < p.keep; r += ranks * kSelectThreads) kept[r] = r < ctx ? r : -1;
    return;
  }
  const uint32_t* const w = reinterpret_cast<const uint32_t*>(p.w.before) + b * p.w.before_stride_b + head * p.w.before_stride_n;
  auto key = [&](int x) { return order_of(__ldg(w + x)); };
  const int lo = p.first, hi = ctx - p.recent, need = p.keep - p.first - p.recent;
  const int each = (hi - lo + ranks - 1) / ranks, x0 = lo + rank * each, x1 = x0 + each < hi ? x0 + each : hi;   // this CTA's tokens
  const int own = (each + kSelectThreads - 1) / kSelectThreads, own0 = x0 + tid * own;                           // HELD: this thread's, from own0 on
  uint32_t held[HELD ? kHeld : 1];
  if constexpr (HELD) {
#pragma unroll
    for (int i = 0; i < kHeld; ++i)
      if (i < own && own0 + i < x1) held[i] = key(own0 + i);
  }
  auto each_key = [&](auto&& f) {
    if constexpr (HELD) {
#pragma unroll
      for (int i = 0; i < kHeld; ++i)
        if (i < own && own0 + i < x1) f(held[i]);
    } else {
      for (int x = x0 + tid; x < x1; x += kSelectThreads) f(key(x));
    }
  };
  for (int r = rank * kSelectThreads + tid; r < p.first; r += ranks * kSelectThreads) kept[r] = r;
  for (int r = rank * kSelectThreads + tid; r < p.recent; r += ranks * kSelectThreads) kept[p.keep - p.recent + r] = ctx - p.recent + r;
  if (need == 0) return;

  const bool few = HELD && ranks == 1 && own == 1;
  if (!few)
    for (int i = tid; i < 3 * kBins; i += kSelectThreads) (&hist[0][0])[i] = 0;
  if (tid < 2) counts[tid] = 0;
  __syncthreads();
  uint32_t prefix = 0, mask = 0, left = (uint32_t)need;   // digits found so far; tokens still to be found among those that have them
  if (few) {   // a weight a thread: bit by bit, the block counted by its barrier
    const bool mine = own0 < x1;
    for (int bit = 31; bit >= 0; --bit) {
      const uint32_t next = prefix | 1u << bit;
      if (__syncthreads_count(mine && held[0] >= next) >= need) prefix = next;
    }
    left = (uint32_t)(need - __syncthreads_count(mine && held[0] > prefix));
  }
#pragma unroll 1
  for (int pass = few ? 3 : 0; pass < 3; ++pass) {
    const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0, bins = pass == 2 ? 1024 : 2048;
    uint32_t* const h = hist[pass];
    each_key([&](uint32_t k) {
      if ((k & mask) == prefix) atomicAdd(&h[k >> shift & (bins - 1)], 1u);
    });
    if (ranks > 1)
      cluster.sync();
    else
      __syncthreads();
    // the counts of all CTAs, from the largest digit down: two digits a thread
    const int d = bins - 1 - 2 * tid;
    uint32_t n0 = 0, n1 = 0;
    if (d > 0)
#pragma unroll 8
      for (int i = 0; i < ranks; ++i) {
        const uint2 other = *reinterpret_cast<const uint2*>(cluster.map_shared_rank(h, i) + (d - 1));
        n0 += other.y;
        n1 += other.x;
      }
    uint32_t total;
    const uint32_t behind = scan1024(n0 + n1, tmp, total), before = behind - n0 - n1;
    if (before < left && left <= behind) {
      const bool upper = left <= before + n0;
      found[0] = upper ? d : d - 1;
      found[1] = left - (upper ? before : before + n0);
    }
    __syncthreads();
    prefix |= found[0] << shift;
    mask |= (uint32_t)(bins - 1) << shift;
    left = found[1];
  }
  // kept: weights above `prefix`, and the first `left` tokens of that weight.  Those of the CTAs before this one:
  uint32_t more = 0, same = 0;
  each_key([&](uint32_t k) {
    more += k > prefix;
    same += k == prefix;
  });
  const uint32_t own_more = more, own_same = same;
  if (ranks > 1) {
    more = __reduce_add_sync(0xffffffffu, more);
    same = __reduce_add_sync(0xffffffffu, same);
    if (tid % 32 == 0) {
      atomicAdd(&counts[0], more);   // (whole numbers: in any order)
      atomicAdd(&counts[1], same);
    }
    cluster.sync();
    more = same = 0;
#pragma unroll 8
    for (int i = 0; i < rank; ++i) {
      const uint2 other = *reinterpret_cast<const uint2*>(cluster.map_shared_rank(&counts[0], i));
      more += other.x;
      same += other.y;
    }
  } else {
    more = same = 0;
  }
  uint32_t total;
  if constexpr (HELD) {
    const uint32_t scan = scan1024(own_more | own_same << 16, tmp, total);   // (kHeld * 1024 of either at most)
    more += (scan & 0xffffu) - own_more;
    same += (scan >> 16) - own_same;
#pragma unroll
    for (int i = 0; i < kHeld; ++i)
      if (i < own && own0 + i < x1) {
        const bool is_more = held[i] > prefix, is_same = held[i] == prefix;
        if (is_more || (is_same && same < left)) kept[p.first + more + (same < left ? same : left)] = own0 + i;
        more += is_more;
        same += is_same;
      }
  } else {
    for (int x = x0; x < x1; x += kSelectThreads) {
      const uint32_t k = x + tid < x1 ? key(x + tid) : 0u;
      const bool is_more = x + tid < x1 && k > prefix, is_same = x + tid < x1 && k == prefix;
      const uint32_t scan = scan1024((uint32_t)is_more | (uint32_t)is_same << 16, tmp, total);   // (1024 of either at most)
      const uint32_t m = more + (scan & 0xffffu) - is_more, s = same + (scan >> 16) - is_same;   // before this token
      if (is_more || (is_same && s < left)) kept[p.first + m + (s < left ? s : left)] = x + tid;
      more += total & 0xffffu;
      same += total >> 16;
    }
  }
  if (ranks > 1) cluster.sync();   // (the others read this CTA's counts)
}

// ---------------------------------------------------------------- moving
constexpr int kMoveThreads = 256, kRing = 4, kMoveCtas = 4 * kSms;

template <int W> struct Move {   // pieces of W bytes of a row
  static constexpr int kLanes = W / 16, kAtOnce = kMoveThreads / kLanes;
  static constexpr int kLoads = kAtOnce * 4 <= 512 ? 4 : 512 / kAtOnce, kRows = kAtOnce * kLoads;   // rows of a tile
  static constexpr int kOwn = (kRows + kMoveThreads - 1) / kMoveThreads;                            // of which a thread finds the places
};
__device__ __forceinline__ Place place_in(const int* table, int pages, const CacheArgs& a, int token) {
  const int i = token >> a.page_log2;
  Place at{-1, token & (a.c.page_size - 1)};
  if (i < pages) {
    const int page = __ldg(table + i);
    if (page >= 0 && page < a.c.pages) at.page = page;
  }
  return at;
}

// Number of a row's log-sum-exp by the row's number in part 0.
__device__ __forceinline__ size_t lse_row(const CacheArgs& a, long long row, int head) {
  const long long page = (row >> a.page_log2) / (4LL * a.c.N);
  return (((size_t)page * a.c.N + head) << a.page_log2) + (row & (a.c.page_size - 1));
}

template <int W> __global__ void __launch_bounds__(kMoveThreads) evict_move_kernel(const __grid_constant__ Params p) {
  using M = Move<W>;
  __shared__ long long from[kRing][M::kRows], to[kRing][M::kRows];   // numbers of a tile's rows, -1: none
  wait_for_previous();
  const CacheArgs& a = p.cache;
  const cg::cluster_group cluster = cg::this_cluster();
  const int ranks = p.ranks, rank = blockIdx.x % ranks;
  const int tid = threadIdx.x, piece = blockIdx.x / ranks, part = blockIdx.y, bh = blockIdx.z, b = bh / a.c.N, head = bh - b * a.c.N;
  const int ctx = tokens_of(p, b), count = ctx < p.keep ? ctx : p.keep;
  if (ctx < 0) return;
  const bool in_place = p.table_out == nullptr;
  const float* const before = p.w.before + b * p.w.before_stride_b + head * p.w.before_stride_n;
  float* const after = p.w.after + b * p.w.after_stride_b + head * p.w.after_stride_n;
  if (in_place && ctx <= p.keep && before == after) return;
  const int* const kept = p.kept + (size_t)bh * p.keep;
  const int* const table = a.c.table + b * a.c.table_stride;
  const int* const table_out = in_place ? table : p.table_out + b * p.table_out_stride;
  const int pages_out = in_place ? a.c.table_pages : p.table_out_pages;
  const size_t row_bytes = (size_t)a.c.D * (a.c.code == TRITT_CODE_F16 ? 2 : 1);
  uint8_t* const codes = (uint8_t*)a.c.codes + piece * W + tid % M::kLanes * 16;
  const int mine = tid / M::kLanes;
  // what rows have besides: with the first piece of each part its exponent, of part 0 the log-sum-exp too, of part 1 the weight
  const bool exponents = piece == 0, lse = piece == 0 && part == 0 && a.c.lse != nullptr, weights = piece == 0 && part == 1;

  uint4 v[2][M::kLoads];
  uint8_t e[2][M::kOwn];
  float l[2][M::kOwn], wt[2][M::kOwn];
  auto find = [&](int tile) {   // places of a tile's rows
#pragma unroll
    for (int k = 0; k < M::kOwn; ++k) {
      const int at = tid + k * kMoveThreads, r = (tile * ranks + rank) * M::kRows + at;
      if (at >= M::kRows) break;
      long long f = -1, t = -1;
      if (r < count) {
        const int x = __ldcg(kept + r);   // (written by the kernel before)
        const Place src = place_in(table, a.c.table_pages, a, x), dst = place_in(table_out, pages_out, a, r);
        if (src.page >= 0 && dst.page >= 0) {
          f = (long long)row_of(a, src, part, head);
          t = (long long)row_of(a, dst, part, head);
          if (f == t) f = t = -1;
        } else if (a.status) {
          atomicOr(a.status, kStatusPlace);
        }
      }
      from[tile % kRing][at] = f;
      to[tile % kRing][at] = t;
    }
  };
  // (loads that may not be moved behind the stores of other threads: not through the read-only path)
  auto load = [&](int tile, uint4 (&u)[M::kLoads], uint8_t (&ex)[M::kOwn], float (&lx)[M::kOwn], float (&wx)[M::kOwn]) {
    const long long* at = from[tile % kRing];
#pragma unroll
    for (int k = 0; k < M::kLoads; ++k) {
      const long long f = at[mine + k * M::kAtOnce];
      if (f >= 0) u[k] = __ldcg(reinterpret_cast<const uint4*>(codes + f * row_bytes));
    }
#pragma unroll
    for (int k = 0; k < M::kOwn; ++k) {
      const int i = tid + k * kMoveThreads, r = (tile * ranks + rank) * M::kRows + i;
      if (i >= M::kRows) break;
      const long long f = at[i];
      if (f >= 0 && exponents) ex[k] = __ldcg(a.c.exponents + f);
      if (f >= 0 && lse) lx[k] = __ldcg(a.c.lse + lse_row(a, f, head));
      if (weights && r < count) {
        wx[k] = __ldcg(before + __ldcg(kept + r));
      }
    }
  };
  auto store = [&](int tile, const uint4 (&u)[M::kLoads], const uint8_t (&ex)[M::kOwn], const float (&lx)[M::kOwn], const float (&wx)[M::kOwn]) {
    const long long* at = to[tile % kRing];
#pragma unroll
    for (int k = 0; k < M::kLoads; ++k) {
      const long long t = at[mine + k * M::kAtOnce];
      if (t >= 0) *reinterpret_cast<uint4*>(codes + t * row_bytes) = u[k];
    }
#pragma unroll
    for (int k = 0; k < M::kOwn; ++k) {
      const int i = tid + k * kMoveThreads, r = (tile * ranks + rank) * M::kRows + i;
      if (i >= M::kRows) break;
      const long long t = at[i];
      if (t >= 0 && exponents) a.c.exponents[t] = ex[k];
      if (t >= 0 && lse) a.c.lse[lse_row(a, t, head)] = lx[k];
      if (weights && r < count) after[r] = wx[k];
    }
  };
  const int tiles = (count + M::kRows * ranks - 1) / (M::kRows * ranks);
  if (tiles == 0) return;
  // Before a tile is written its rows, and those of all tiles before it, have been read by all threads of the block, or in place of the cluster (the barrier behind their loads); the next tile's, on their way
  // then, lie behind what is written.  The ring's place that `find` fills was last read by the stores of two tiles ago, before the last barrier.
  // A cluster's barrier waits for the thread's loads, so the next tile's are sent behind it; a block's does not, and they are sent ahead of it.
  // (Weights in place are such a case too where the rows go to other pages.)
  const bool clustered = ranks > 1 && (in_place || (weights && before == after));
  find(0);
  __syncthreads();
  load(0, v[0], e[0], l[0], wt[0]);
  if (tiles > 1) find(1);
  __syncthreads();
  for (int i = 0; i < tiles; i += 2) {
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      if (i + k >= tiles) break;
      const bool more = i + k + 1 < tiles;
      if (more && !clustered) load(i + k + 1, v[1 - k], e[1 - k], l[1 - k], wt[1 - k]);
      if (i + k + 2 < tiles) find(i + k + 2);
      if (clustered)
        cluster.sync();
      else
        __syncthreads();
      if (more && clustered) load(i + k + 1, v[1 - k], e[1 - k], l[1 - k], wt[1 - k]);
      store(i + k, v[k], e[k], l[k], wt[k]);
    }
  }
}

template <int W> int launch_move(Params p, int row_bytes, cudaStream_t stream) {
  const int pieces = row_bytes / W;
  // as many CTAs as keep all SMs' loads in flight, while each has two tiles
  const long long streams = 4LL * p.cache.c.B * p.cache.c.N * pieces;
  while (p.ranks < kMostCluster && streams * p.ranks < kMoveCtas && p.keep > 2 * Move<W>::kRows * p.ranks) p.ranks *= 2;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(pieces * p.ranks, 4, p.cache.c.B * p.cache.c.N);
  cfg.blockDim = dim3(kMoveThreads);
  cfg.stream = stream;
  cudaLaunchAttribute attr[2]{};
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = p.ranks;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  TRITT_CUDA_OK(cudaLaunchKernelEx(&cfg, evict_move_kernel<W>, p));
  count_launch();
  return 0;
}

int check(const tritt_cache_t* c, const tritt_weights_t* w, const Params& p) {
  if (p.keep < 1 || p.first < 0 || p.recent < 0 || p.first > p.keep - p.recent) {
    set_error("keep must be at least 1 and first + recent, each at least 0, at most keep: got %d, %d and %d", p.keep, p.first, p.recent);
    return -10;
  }
  if (w->after_length < p.keep) {
    set_error("weights of %d tokens to keep, room for %d", p.keep, w->after_length);
    return -1;
  }
  if (!p.context_out || !p.kept) {
    set_error("null tensor pointer");
    return -4;
  }
  if (((uintptr_t)p.context_out | (uintptr_t)p.kept | (uintptr_t)p.table_out) & 3) {
    set_error("a pointer to contexts, kept tokens or a table is not aligned");
    return -5;
  }
  if ((const int*)p.context_out == c->context) {
    set_error("context_out must be another array than context");
    return -4;
  }
  if (p.table_out && (p.table_out_pages < 1 || (long long)p.table_out_pages * c->page_size > (1LL << 28) || (long long)p.table_out_pages * c->page_size < p.keep)) {
    set_error("a table of %d pages for %d tokens to keep", p.table_out_pages, p.keep);
    return -12;
  }
  if ((long long)c->B * c->N * p.keep > (1LL << 40)) {
    set_error("too many tokens for one call; split the batch");
    return -11;
  }
  return 0;
}

}  // namespace
}  // namespace tritt

using namespace tritt;

extern "C" int tritt_cache_evict(const tritt_cache_t* c, const tritt_weights_t* w, const int* table_out, long long table_out_stride, int table_out_pages, int keep,
                                 int first, int recent, int* context_out, int* kept, int* status_word, tritt_stream_t stream) {
  if (int rc = check_cache(c)) return rc;
  if (int rc = check_weights(c, w)) return rc;
  Params p{cache_args(*c, status_word), *w, table_out, table_out_stride, table_out_pages, keep, first, recent, context_out, kept, 1};
  if (int rc = check(c, w, p)) return rc;
  if (table_out && table_out == c->table && (c->B == 1 || table_out_stride == c->table_stride)) p.table_out = nullptr;   // (in place, after all)
  p.cache.c.n = 1;   // (places are reported of every sequence in use)
  p.cache.c.counts = nullptr;
  // A cluster for a head as far as the weights do not fit in one CTA's registers (fewer and larger clusters: eight CTAs a head of 65001 weights took 39 us, some of them behind others), and not more CTAs
  // than the chip holds at once.
  long long tokens = (long long)c->table_pages * c->page_size;
  if (w->before_length < tokens) tokens = w->before_length;
  int ranks = 1;
  while (ranks < kMostCluster && tokens > (long long)kHeld * kSelectThreads * ranks && 2LL * ranks * c->B * c->N <= kSms) ranks *= 2;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(ranks, c->B * c->N);
  cfg.blockDim = dim3(kSelectThreads);
  cfg.stream = (cudaStream_t)stream;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = ranks;
  attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  if (tokens <= (long long)kHeld * kSelectThreads * ranks)
    TRITT_CUDA_OK(cudaLaunchKernelEx(&cfg, evict_select_kernel<true>, p));
  else
    TRITT_CUDA_OK(cudaLaunchKernelEx(&cfg, evict_select_kernel<false>, p));
  count_launch();
  const int row_bytes = c->D * code_bytes(c->code);
  switch (row_bytes < 64 ? row_bytes : 64) {
    case 16: return launch_move<16>(p, row_bytes, (cudaStream_t)stream);
    case 32: return launch_move<32>(p, row_bytes, (cudaStream_t)stream);
    default: return launch_move<64>(p, row_bytes, (cudaStream_t)stream);
  }
}
