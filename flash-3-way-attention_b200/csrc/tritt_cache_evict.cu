// Eviction: of each sequence and head the heaviest tokens are kept, and their rows move together.
//
// Chosen exactly, by three passes over the weights' bits (11, 11, 10): each counts the numbers that share the digits found so far by their next digit, until the weight of the last kept
// token and how many of that weight are kept is known; a last pass numbers the kept ones in order.  A cluster of up to eight CTAs takes a sequence's head, and adds its counts up
// through distributed shared memory; the weights are read from L2 after the first pass.
//
// Moved by another kernel, bound by the bytes of the kept rows, read and written once.  In place: a kept token's new place is never behind its old one, so rows that are taken in order
// and written when all rows up to them have been read overwrite nothing that is still to be read.  One block takes a piece of 32 to 128 bytes of all rows of one part of a head (the
// parts, heads and pieces of rows are independent), with the next tile's rows on their way while one is written.
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
};

// A weight's bits in the order of the weights: a NaN as the largest, zeros of either sign alike.
__device__ __forceinline__ uint32_t order_of(float v) {
  const uint32_t u = __float_as_uint(v);   // (comparisons of numbers would take the smallest for zeros)
  if ((u & 0x7fffffffu) > 0x7f800000u) return 0xffffffffu;
  if (u << 1 == 0u) return 0x80000000u;
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

__global__ void __launch_bounds__(kSelectThreads) evict_select_kernel(const __grid_constant__ Params p) {
  __shared__ uint32_t hist[3][kBins], tmp[32], found[2], counts[2];
  let_next_start();
  const CacheArgs& a = p.cache;
  const cg::cluster_group cluster = cg::this_cluster();
  const int rank = blockIdx.x, ranks = gridDim.x, tid = threadIdx.x;
  const int bh = blockIdx.y, b = bh / a.c.N, head = bh - b * a.c.N;
  const int given = __ldg(a.c.context + b), ctx = given < 0 ? given : context_of(a, b);
  if (rank == 0 && head == 0 && tid == 0) p.context_out[b] = ctx < p.keep ? ctx : p.keep;
  int* const kept = p.kept + (size_t)bh * p.keep;
  if (ctx <= p.keep) {   // (all of a cluster's CTAs)
    for (int r = rank * kSelectThreads + tid; r < p.keep; r += ranks * kSelectThreads) kept[r] = r < ctx ? r : -1;
    return;
  }
  if (ctx > p.w.before_length && a.status) atomicOr(a.status, kStatusPlace);
  const float* const w = p.w.before + b * p.w.before_stride_b + head * p.w.before_stride_n;
  auto key = [&](int x) { return order_of(x < p.w.before_length ? __ldg(w + x) : 0.f); };
  const int lo = p.first, hi = ctx - p.recent, need = p.keep - p.first - p.recent;
  const int each = (hi - lo + ranks - 1) / ranks, x0 = lo + rank * each, x1 = x0 + each < hi ? x0 + each : hi;   // this CTA's tokens
  for (int r = rank * kSelectThreads + tid; r < p.first; r += ranks * kSelectThreads) kept[r] = r;
  for (int r = rank * kSelectThreads + tid; r < p.recent; r += ranks * kSelectThreads) kept[p.keep - p.recent + r] = ctx - p.recent + r;
  if (need == 0) return;

  for (int i = tid; i < 3 * kBins; i += kSelectThreads) (&hist[0][0])[i] = 0;
  __syncthreads();
  uint32_t prefix = 0, mask = 0, left = (uint32_t)need;   // digits found so far; tokens still to be found among those that have them
  for (int pass = 0; pass < 3; ++pass) {
    const int shift = pass == 0 ? 21 : pass == 1 ? 10 : 0, bins = pass == 2 ? 1024 : 2048;
    for (int x = x0 + tid; x < x1; x += kSelectThreads) {
      const uint32_t k = key(x);
      if ((k & mask) == prefix) atomicAdd(&hist[pass][k >> shift & (bins - 1)], 1u);
    }
    cluster.sync();
    // the counts of all CTAs, from the largest digit down: two digits a thread
    const int d = bins - 1 - 2 * tid;
    uint32_t n0 = 0, n1 = 0;
    if (d > 0)
      for (int i = 0; i < ranks; ++i) {
        const uint32_t* other = cluster.map_shared_rank(&hist[pass][0], i);
        n0 += other[d];
        n1 += other[d - 1];
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
  if (tid < 2) counts[tid] = 0;
  __syncthreads();
  uint32_t more = 0, same = 0;
  for (int x = x0 + tid; x < x1; x += kSelectThreads) {
    const uint32_t k = key(x);
    more += k > prefix;
    same += k == prefix;
  }
  more = __reduce_add_sync(0xffffffffu, more);
  same = __reduce_add_sync(0xffffffffu, same);
  if (tid % 32 == 0) {
    atomicAdd(&counts[0], more);   // (whole numbers: in any order)
    atomicAdd(&counts[1], same);
  }
  cluster.sync();
  more = same = 0;
  for (int i = 0; i < rank; ++i) {
    const uint32_t* other = cluster.map_shared_rank(&counts[0], i);
    more += other[0];
    same += other[1];
  }
  for (int x = x0; x < x1; x += kSelectThreads) {
    const uint32_t k = x + tid < x1 ? key(x + tid) : 0u;
    const bool is_more = x + tid < x1 && k > prefix, is_same = x + tid < x1 && k == prefix;
    uint32_t total;
    const uint32_t scan = scan1024((uint32_t)is_more | (uint32_t)is_same << 16, tmp, total);   // (1024 of either at most)
    const uint32_t m = more + (scan & 0xffffu) - is_more, s = same + (scan >> 16) - is_same;   // before this token
    if (is_more || (is_same && s < left)) kept[p.first + m + (s < left ? s : left)] = x + tid;
    more += total & 0xffffu;
    same += total >> 16;
  }
  cluster.sync();   // (the others read this CTA's counts)
}

// ---------------------------------------------------------------- moving
constexpr int kMoveThreads = 256, kRing = 4;

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
  const int tid = threadIdx.x, piece = blockIdx.x, part = blockIdx.y, bh = blockIdx.z, b = bh / a.c.N, head = bh - b * a.c.N;
  if (__ldg(a.c.context + b) < 0) return;
  const int ctx = context_of(a, b), count = ctx < p.keep ? ctx : p.keep;
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
      const int at = tid + k * kMoveThreads, r = tile * M::kRows + at;
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
      const int i = tid + k * kMoveThreads, r = tile * M::kRows + i;
      if (i >= M::kRows) break;
      const long long f = at[i];
      if (f >= 0 && exponents) ex[k] = __ldcg(a.c.exponents + f);
      if (f >= 0 && lse) lx[k] = __ldcg(a.c.lse + lse_row(a, f, head));
      if (weights && r < count) {
        const int x = __ldcg(kept + r);
        wx[k] = x < p.w.before_length ? __ldcg(before + x) : 0.f;
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
      const int i = tid + k * kMoveThreads, r = tile * M::kRows + i;
      if (i >= M::kRows) break;
      const long long t = at[i];
      if (t >= 0 && exponents) a.c.exponents[t] = ex[k];
      if (t >= 0 && lse) a.c.lse[lse_row(a, t, head)] = lx[k];
      if (weights && r < count) after[r] = wx[k];
    }
  };
  const int tiles = (count + M::kRows - 1) / M::kRows;
  if (tiles == 0) return;
  // Before a tile is written its rows, and those of all tiles before it, have been read by all threads (the barrier behind their loads); the next tile's, on their way then, lie behind what is written.
  // The ring's place that `find` fills was last read by the stores of two tiles ago, before the last barrier.
  find(0);
  __syncthreads();
  load(0, v[0], e[0], l[0], wt[0]);
  if (tiles > 1) find(1);
  __syncthreads();
  for (int i = 0; i < tiles; i += 2) {
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      if (i + k >= tiles) break;
      if (i + k + 1 < tiles) load(i + k + 1, v[1 - k], e[1 - k], l[1 - k], wt[1 - k]);
      if (i + k + 2 < tiles) find(i + k + 2);
      __syncthreads();
      store(i + k, v[k], e[k], l[k], wt[k]);
    }
  }
}

template <int W> int launch_move(const Params& p, int row_bytes, cudaStream_t stream) {
  return launch_kernel_after(evict_move_kernel<W>, dim3(row_bytes / W, 4, p.cache.c.B * p.cache.c.N), kMoveThreads, 0, stream, true, p);
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
  Params p{cache_args(*c, status_word), *w, table_out, table_out_stride, table_out_pages, keep, first, recent, context_out, kept};
  if (int rc = check(c, w, p)) return rc;
  p.cache.c.n = 1;   // (places are reported of every sequence in use)
  p.cache.c.counts = nullptr;
  // A cluster for a head: a CTA takes a few thousand weights, and there are no more of them than the chip holds at once.
  long long tokens = (long long)c->table_pages * c->page_size;
  if (w->before_length < tokens) tokens = w->before_length;
  int ranks = 1;
  while (ranks < kMostCluster && tokens > 4096LL * ranks && 2LL * ranks * c->B * c->N <= 2 * kSms) ranks *= 2;
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
  TRITT_CUDA_OK(cudaLaunchKernelEx(&cfg, evict_select_kernel, p));
  count_launch();
  // Pieces of rows: the widest with which there are blocks enough to keep all SMs' loads in flight (each block takes all of a head's kept tokens, one tile after the other).
  const int row_bytes = c->D * code_bytes(c->code);
  const long long parts = 4LL * c->B * c->N;
  int piece = row_bytes < 128 ? row_bytes : 128;
  while (piece > 32 && parts * (row_bytes / piece) < 4 * kSms) piece /= 2;
  switch (piece) {
    case 16: return launch_move<16>(p, row_bytes, (cudaStream_t)stream);
    case 32: return launch_move<32>(p, row_bytes, (cudaStream_t)stream);
    case 64: return launch_move<64>(p, row_bytes, (cudaStream_t)stream);
    default: return launch_move<128>(p, row_bytes, (cudaStream_t)stream);
  }
}
