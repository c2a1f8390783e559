// The attention weight of cached tokens in the triple dot product where the rows that new tokens attend to fit in shared memory: narrow windows, or short tables.
//
// (What is computed: tritt_tdp_weigh.cu.)  A cluster of blocks takes a sequence's head with all its new tokens; each block stages a part of the tokens k, as fp16 codes of K2, and the tokens j that a band leaves
// those, of K1.  A warp takes 16 tokens k, some columns j and some new tokens at a time: the operand q * K2 is formed in registers, as two fp16 numbers (22 bits), K1's codes are the other operand, and
// the exponentials add up along both sides in registers over the new tokens.  Only the 32-column blocks that a window and a band reach are looked at.  The units' sums stand in shared memory,
// added up in order there and over the cluster, each token's by one thread, with the weights of before: one launch, no scratch.
//
// What bounds it: the way from a unit's operand to its sums with 14 warps an SM (38 % of the issue slots, the tensor pipe 23 %), and units that do not come out even over warps and blocks (a fifth of the time).
// 16 tokens of 8 x 16 heads of 64, windows 128/128/32/32, int8: 50 us, where tiles of 128 x 128 take 110 and whole columns of 128 a unit 53; 55 by eight tokens a unit.  Forming the operand in fp16 where the query is exact as
// that (5 to 11 % of few tokens' time; 2 instructions a pair of elements instead of 10) leaves the same 22 bits.
#include "tritt_weigh.cuh"

#include <cooperative_groups.h>

#include <type_traits>

namespace tritt {
namespace {
namespace cg = cooperative_groups;

constexpr int kWarps = 8, kThreads = kWarps * 32, kMostCluster = 8;
constexpr int kMostSmem = 200 * 1024;
constexpr int kWide = 64;                     // columns of a unit
template <int CODE> constexpr int kDown = CODE == TRITT_CODE_F16 ? 2 : 0;   // (q is below 4, codes below 2^15, 448, 127)

struct WindowParams {
  TdpWeighArgs a;
  int rows, cols;    // places of a block for tokens k and j: multiples of 16 and of kWide
  int group;         // new tokens of a unit
};

// Byte offset of a 16-byte chunk of a staged row: two rows' four chunks lie in different banks.
template <int D> __device__ __forceinline__ int staged(int row, int chunk) { return row * (2 * D) + ((chunk ^ ((row & 1) << 2 | (row >> 1 & 3))) << 4); }
__device__ __forceinline__ float2 pair_of(uint32_t w) { return __half22float2(*reinterpret_cast<const __half2*>(&w)); }

struct Layout {   // of a block's shared memory
  int k1, k2, e1, e2, q, q16, scale, lse, there, rows_part, cols_part, rows_sum, cols_sum, counter, size;
};
template <int D> __host__ __device__ inline Layout layout_of(int rows, int cols, int n, int group) {
  const int groups = (n + group - 1) / group;
  Layout l;
  int at = 0;
  auto take = [&](int bytes) {
    const int was = at;
    at += (bytes + 15) / 16 * 16;
    return was;
  };
  l.k1 = take(cols * 2 * D);
  l.k2 = take(rows * 2 * D);
  l.e1 = take(cols * 4);
  l.e2 = take(rows);
  l.q = take(n * D * 4);
  l.q16 = take(n * D * 2);
  l.scale = take(n * 4);
  l.lse = take(n * 4);
  l.there = take(cols / 8);
  l.rows_part = take(cols / kWide * groups * rows * 4);
  l.cols_part = take(rows / 16 * groups * cols * 4);
  l.rows_sum = take(rows * 4);
  l.cols_sum = take(cols * 4);
  l.counter = take(16);
  l.size = at;
  return l;
}
// The tokens k (from a multiple of 16 on) and j (of 32) that a block of the cluster has.
struct Part {
  int k0, k1, j0, j1;   // the first and one behind the last
};
struct Head {
  int ctx, cnt, last, lo_j, lo_k;
};
__device__ __forceinline__ Part part_of(const TdpWeighArgs& a, const Head& h, int rank, int ranks) {
  const int first = h.lo_k / 16, tiles = h.cnt && h.last >= h.lo_k ? h.last / 16 - first + 1 : 0;
  const int t0 = tiles * rank / ranks, t1 = tiles * (rank + 1) / ranks;
  Part p{(first + t0) * 16, (first + t1) * 16, 0, 0};
  if (t0 == t1) return p;
  const int least = p.k0 - a.kkl, most = a.kkr < h.last ? p.k1 - 1 + a.kkr : h.last;
  p.j0 = (least > h.lo_j ? least : h.lo_j) / 32 * 32;
  p.j1 = (most < h.last ? most : h.last) + 1;
  if (p.j1 < p.j0) p.j1 = p.j0;
  return p;
}

template <typename T, int D, int CODE> __global__ void __launch_bounds__(kThreads, D == 64 ? 2 : 1) tdp_weigh_window_kernel(const __grid_constant__ WindowParams p) {
  constexpr int W = kWide, kBlocks = W / 32;
  constexpr size_t kRow = D * (CODE == TRITT_CODE_F16 ? 2 : 1);
  extern __shared__ __align__(128) uint8_t smem[];
  const TdpWeighArgs& a = p.a;
  const CacheArgs& ca = a.cache;
  const cg::cluster_group cluster = cg::this_cluster();
  const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32, g = lane / 4, t = lane % 4;
  const int rank = blockIdx.x, ranks = gridDim.x, bh = blockIdx.y, b = bh / ca.c.N, head = bh - b * ca.c.N;
  if (__ldg(ca.c.context + b) < 0) return;   // (all of the cluster)
  Head hd;
  hd.ctx = context_of(ca, b), hd.cnt = new_tokens(ca, b);
  const int places = ca.c.table_pages << ca.page_log2;
  hd.last = (hd.cnt < places - hd.ctx ? hd.ctx + hd.cnt : places) - 1;
  hd.lo_j = hd.ctx - (a.k1w < hd.ctx ? a.k1w : hd.ctx), hd.lo_k = hd.ctx - (a.k2w < hd.ctx ? a.k2w : hd.ctx);
  if (rank == 0 && tid == 0 && hd.cnt > places - hd.ctx && ca.status) atomicOr(ca.status, kStatusPlace);
  const Part own = part_of(a, hd, rank, ranks);
  const int nk = own.k1 - own.k0, nj = own.j1 - own.j0;   // at most p.rows, p.cols
  const Layout l = layout_of<D>(p.rows, p.cols, ca.c.n, p.group);
  uint8_t *const sK1 = smem + l.k1, *const sK2 = smem + l.k2, *const sE2 = smem + l.e2;
  float *const sScale1 = (float*)(smem + l.e1), *const sQ = (float*)(smem + l.q), *const sScale = (float*)(smem + l.scale), *const sLse = (float*)(smem + l.lse);
  __half* const sQ16 = (__half*)(smem + l.q16);
  uint32_t* const sThere = (uint32_t*)(smem + l.there);
  float *const rows_part = (float*)(smem + l.rows_part), *const cols_part = (float*)(smem + l.cols_part);
  float *const rows_sum = (float*)(smem + l.rows_sum), *const cols_sum = (float*)(smem + l.cols_sum);
  int *const counter = (int*)(smem + l.counter), *const largest = counter + 1;
  if (tid < 2) counter[tid] = 0;
  __syncthreads();

  // --- rows as fp16 codes, zeros where there are none; K1's exponent bytes stand in the place of their scales at first (-1: not there), and in that of the sums of K2's rows whether they are there
  constexpr int L = D / 8, kStep = kThreads / L, kBatch = 4;
  auto stage = [&](int part, int lo, int n, int padded, uint8_t* to, auto&& exponent) {
    const uint8_t* const codes = (const uint8_t*)ca.c.codes;
    const int ch = tid % L;
    for (int r0 = tid / L; r0 < padded; r0 += kStep * kBatch) {
      int page[kBatch], e[kBatch];
      Codes8<CODE> c[kBatch];
#pragma unroll
      for (int k = 0; k < kBatch; ++k) {
        const int r = r0 + k * kStep;
        page[k] = r < n ? place_of(ca, b, lo + r).page : -1;
      }
#pragma unroll
      for (int k = 0; k < kBatch; ++k) {
        const size_t at = row_of(ca, Place{page[k] < 0 ? 0 : page[k], (lo + r0 + k * kStep) & (ca.c.page_size - 1)}, part, head);
        c[k].load(codes + at * kRow, ch * 8);
        e[k] = ch == 0 ? __ldg(ca.c.exponents + at) : 0;
      }
#pragma unroll
      for (int k = 0; k < kBatch; ++k) {
        const int r = r0 + k * kStep;
        if (r >= padded) break;
        uint32_t w[4];
        c[k].halves(w);
        const uint32_t on = page[k] >= 0 ? 0xffffffffu : 0u;
        *reinterpret_cast<uint4*>(to + staged<D>(r, ch)) = make_uint4(w[0] & on, w[1] & on, w[2] & on, w[3] & on);
        if (ch == 0) exponent(r, page[k] >= 0 ? e[k] : -1);
      }
    }
  };
  const int padded_j = (nj + W - 1) / W * W;
  stage(kPartK1, own.j0, own.j1 <= hd.last ? nj : hd.last + 1 - own.j0, padded_j, sK1, [&](int r, int e) {
    reinterpret_cast<int*>(sScale1)[r] = e;
    if (e >= 0 && e != 255) atomicMax(largest, e);
  });
    stage(kPartK2, own.k0, hd.last + 1 - own.k0 < nk ? hd.last + 1 - own.k0 : nk, nk, sK2, [&](int r, int e) {
    sE2[r] = (uint8_t)(e < 0 ? 0 : e);
    rows_sum[r] = e < 0 ? 0.f : 1.f;   // (its sums come later)
  });
  for (int i = warp; i < hd.cnt; i += kWarps) {   // q, its largest element brought to [2, 4)
    const T* row = (const T*)a.q.p + rows_at(a.q, b, head, i);
    float4 f = lane < D / 4 ? load4(row + lane * 4) : make_float4(0.f, 0.f, 0.f, 0.f);
    const int field = (int)(largest_of_row<32>(largest4(f)) >> 23);
    const float up = to_operand(field) * (1.f / (1 << kDown<CODE>));
    f = field == 255 ? make_float4(0.f, 0.f, 0.f, 0.f) : make_float4(f.x * up, f.y * up, f.z * up, f.w * up);
    const uint2 h = make_uint2(pack_halves(f.x, f.y), pack_halves(f.z, f.w));
    if (lane < D / 4) {
      *reinterpret_cast<float4*>(sQ + i * D + lane * 4) = f;
      *reinterpret_cast<uint2*>(sQ16 + i * D + lane * 4) = h;
    }
    const float2 a0 = pair_of(h.x), a1 = pair_of(h.y);
    const bool exact = __all_sync(0xffffffffu, a0.x == f.x && a0.y == f.y && a1.x == f.z && a1.y == f.w);
    if (lane == 0) {
      sScale[i] = __int_as_float(field | (exact ? 256 : 0));
      sLse[i] = __ldg(a.lse + (size_t)bh * ca.c.n + i);
    }
  }
  __syncthreads();
  const int middle = middle_byte<CODE>(*largest);
  for (int x = warp; x < padded_j / 32; x += kWarps) {   // scales of K1's rows, and words of those that are there
    const int e = reinterpret_cast<const int*>(sScale1)[x * 32 + lane];
    const uint32_t there = __ballot_sync(0xffffffffu, e >= 0);
    sScale1[x * 32 + lane] = e < 0 ? 0.f : e == 255 ? __uint_as_float(0x7fffffffu) : relative_power(e - middle);
    if (lane == 0) sThere[x] = there;
  }
  __syncthreads();

  // --- units: 16 tokens k, W columns j, a group of new tokens
  const int tiles = nk / 16, wides = padded_j / W, groups = (hd.cnt + p.group - 1) / p.group;
  // the wide columns that a tile of k reaches
  auto reach = [&](int tile, int& c0, int& c1) {
    const int k0 = own.k0 + tile * 16, most = a.kkr < hd.last ? k0 + 15 + a.kkr : hd.last;
    const int lo = k0 - a.kkl > own.j0 ? k0 - a.kkl : own.j0, hi = most < own.j1 - 1 ? most : own.j1 - 1;
    c0 = (lo - own.j0) / W;
    c1 = hi < lo ? c0 : (hi - own.j0) / W + 1;
  };
  const int units = tiles * wides * groups;
  for (;;) {
    int u = 0;
    if (lane == 0) u = atomicAdd(counter, 1);   // (whichever warp takes a unit, its sums are the same)
    u = __shfl_sync(0xffffffffu, u, 0);
    if (u >= units) break;
    const int tile = u / (wides * groups), wide = u / groups % wides, group = u % groups;
    int w0, w1;
    reach(tile, w0, w1);
    if (wide < w0 || wide >= w1) continue;
    const int kt = own.k0 + tile * 16, jt = own.j0 + wide * W;
    // this thread's rows g and g + 8
    int k_at[2], e2[2];
    bool there2[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int r = tile * 16 + g + 8 * h;
      k_at[h] = own.k0 + r;
      e2[h] = sE2[r];
      there2[h] = rows_sum[r] != 0.f;
    }
    float row_sum[2] = {0.f, 0.f}, column[W / 8][2];
#pragma unroll
    for (int n = 0; n < W / 8; ++n) column[n][0] = column[n][1] = 0.f;
    const int i1 = (group + 1) * p.group < hd.cnt ? (group + 1) * p.group : hd.cnt;
    for (int i = group * p.group; i < i1; ++i) {
      const int pos = hd.ctx + i, k_lo = pos - (a.k2w < pos ? a.k2w : pos), j_lo = pos - (a.k1w < pos ? a.k1w : pos);
      const float lse = sLse[i];
      if (lse == -INFINITY || kt > pos || kt + 15 < k_lo) continue;
      // what the rows attend to, and of the columns those that any of the 16 does
      int from[2], to[2];
      float scale[2];
      const int field = __float_as_int(sScale[i]) & 255;
      const bool exact = __float_as_int(sScale[i]) >> 8;   // (as fp16)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const bool seen = k_at[h] >= k_lo && k_at[h] <= pos, on = seen && there2[h];
        if (seen && !on && t == 0 && ca.status) atomicOr(ca.status, kStatusPlace);
        from[h] = on ? (k_at[h] - a.kkl > j_lo ? k_at[h] - a.kkl : j_lo) : 1 << 30;
        to[h] = !on ? -1 : a.kkr < pos - k_at[h] ? k_at[h] + a.kkr : pos;
        // 2^e of the row, that of the columns' in the middle, q and the operand
        int power = e2[h] + middle - 254 + field - 128 + kDown<CODE>;
        power = power < -126 ? -126 : power > 127 ? 127 : power;
        scale[h] = e2[h] == 255 || field == 255 ? __uint_as_float(0x7fffffffu) : field == 0 ? 0.f : a.scale2 * power_of_two(power);
      }
      const int any_from = (kt - a.kkl > j_lo ? kt - a.kkl : j_lo) - jt, any_to = (a.kkr < pos - kt - 15 ? kt + 15 + a.kkr : pos) - jt;
      if (any_to < 0 || any_from >= W || any_to < any_from) continue;
      // q * K2: elements 32 j + 8 t + 4 s + {0, 1 | 2, 3} of rows g, g + 8 in steps 2 j + s
      uint32_t hi[D / 16][4], rest[D / 16][4];
#pragma unroll
      for (int j = 0; j < D / 32; ++j) {
        uint32_t w[2][4];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const uint4 v = *reinterpret_cast<const uint4*>(sK2 + staged<D>(tile * 16 + g + 8 * h, j * 4 + t));
          w[h][0] = v.x, w[h][1] = v.y, w[h][2] = v.z, w[h][3] = v.w;
        }
        if (exact) {   // the rounded product, and what it leaves, from one multiplication and addition
          const uint4 q = *reinterpret_cast<const uint4*>(sQ16 + i * D + j * 32 + t * 8);
          const uint32_t qw[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
          for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const __half2 c = *reinterpret_cast<const __half2*>(&w[h][e]), qq = *reinterpret_cast<const __half2*>(&qw[e]);
              const __half2 product = __hmul2(c, qq), left = __hfma2(c, qq, __hneg2(product));
              hi[2 * j + e / 2][2 * (e % 2) + h] = *reinterpret_cast<const uint32_t*>(&product);
              rest[2 * j + e / 2][2 * (e % 2) + h] = *reinterpret_cast<const uint32_t*>(&left);
            }
        } else {
          const float4 qa = *reinterpret_cast<const float4*>(sQ + i * D + j * 32 + t * 8), qb = *reinterpret_cast<const float4*>(sQ + i * D + j * 32 + t * 8 + 4);
          const float q[8] = {qa.x, qa.y, qa.z, qa.w, qb.x, qb.y, qb.z, qb.w};
#pragma unroll
          for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const float2 c = pair_of(w[h][e]);
              const float x = q[2 * e] * c.x, y = q[2 * e + 1] * c.y;
              const uint32_t top16 = pack_halves(x, y);
              hi[2 * j + e / 2][2 * (e % 2) + h] = top16;
              rest[2 * j + e / 2][2 * (e % 2) + h] = pack_rests(x, y, top16);
            }
        }
      }
      const float lse2 = lse * kLog2e;
#pragma unroll
      for (int blk = 0; blk < kBlocks; ++blk) {
        if (any_to < blk * 32 || any_from >= blk * 32 + 32) continue;
        const int c0 = wide * W + blk * 32, j0 = jt + blk * 32;
        uint32_t mask[2];
        const uint32_t there = sThere[c0 / 32];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int lo = from[h] - j0 > 0 ? from[h] - j0 : 0, hi_c = to[h] - j0 < 31 ? to[h] - j0 : 31;
          const uint32_t w = lo > 31 || hi_c < lo ? 0u : (0xffffffffu << lo) & (0xffffffffu >> (31 - hi_c));
          if ((w & ~there) && t == 0 && ca.status) atomicOr(ca.status, kStatusPlace);
          mask[h] = w & there;
        }
        if (!__any_sync(0xffffffffu, mask[0] | mask[1])) continue;
        const bool all = !__any_sync(0xffffffffu, (mask[0] & mask[1]) != 0xffffffffu);
#pragma unroll
        for (int n = 0; n < 4; ++n) {
          float s[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int j = 0; j < D / 32; ++j) {
            const uint4 k = *reinterpret_cast<const uint4*>(sK1 + staged<D>(c0 + n * 8 + g, j * 4 + t));
            mma_16816(s, hi[2 * j], make_uint2(k.x, k.y));
            mma_16816(s, hi[2 * j + 1], make_uint2(k.z, k.w));
            mma_16816(s, rest[2 * j], make_uint2(k.x, k.y));
            mma_16816(s, rest[2 * j + 1], make_uint2(k.z, k.w));
          }
          const float2 by = *reinterpret_cast<const float2*>(sScale1 + c0 + n * 8 + 2 * t);
          float x[4];
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            x[2 * h] = scaled_score(s[2 * h], by.x, scale[h], lse2);
            x[2 * h + 1] = scaled_score(s[2 * h + 1], by.y, scale[h], lse2);
            if (!all) {
              x[2 * h] = mask[h] >> (n * 8 + 2 * t) & 1 ? x[2 * h] : -INFINITY;
              x[2 * h + 1] = mask[h] >> (n * 8 + 2 * t + 1) & 1 ? x[2 * h + 1] : -INFINITY;
            }
            x[2 * h] = exp2f(x[2 * h]), x[2 * h + 1] = exp2f(x[2 * h + 1]);
            row_sum[h] += x[2 * h] + x[2 * h + 1];
          }
          column[blk * 4 + n][0] += x[0] + x[2];
          column[blk * 4 + n][1] += x[1] + x[3];
        }
      }
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      row_sum[h] += __shfl_xor_sync(0xffffffffu, row_sum[h], 1);
      row_sum[h] += __shfl_xor_sync(0xffffffffu, row_sum[h], 2);
    }
    if (t < 2) rows_part[(wide * groups + group) * p.rows + tile * 16 + g + 8 * t] = t ? row_sum[1] : row_sum[0];
    float* const to = cols_part + (size_t)(tile * groups + group) * p.cols + wide * W;
#pragma unroll
    for (int n = 0; n < W / 8; ++n)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float v = column[n][e];
        v += __shfl_xor_sync(0xffffffffu, v, 4);
        v += __shfl_xor_sync(0xffffffffu, v, 8);
        v += __shfl_xor_sync(0xffffffffu, v, 16);
        if (g == 0) to[n * 8 + 2 * t + e] = v;
      }
  }
  __syncthreads();

  // --- the block's sums, of its units in order
  for (int r = tid; r < nk; r += kThreads) {
    int w0, w1;
    reach(r / 16, w0, w1);
    float v = 0.f;
    for (int w = w0; w < w1; ++w)
      for (int i = 0; i < groups; ++i) v += rows_part[(w * groups + i) * p.rows + r];
    rows_sum[r] = v;
  }
  for (int x = tid; x < padded_j; x += kThreads) {
    float v = 0.f;
    for (int tile = 0; tile < tiles; ++tile) {
      int w0, w1;
      reach(tile, w0, w1);
      if (x / W < w0 || x / W >= w1) continue;
      for (int i = 0; i < groups; ++i) v += cols_part[(size_t)(tile * groups + i) * p.cols + x];
    }
    cols_sum[x] = v;
  }
  cluster.sync();
  // --- a token's, of the cluster's blocks in order, and the weight of before
  const int end = weighed_tokens(ca, a.w, hd.ctx + hd.cnt);
  for (int x = rank * kThreads + tid; x < end; x += ranks * kThreads) {
    float v = x < hd.ctx ? faded(a.w, b, head, x) : 0.f, sum = 0.f;
    if (x <= hd.last && (x >= hd.lo_j || x >= hd.lo_k)) {
      for (int r = 0; r < ranks; ++r) {
        const Part part = part_of(a, hd, r, ranks);
        if (x >= part.k0 && x < part.k1) sum += cluster.map_shared_rank(rows_sum, r)[x - part.k0];
        if (x >= part.j0 && x < part.j1) sum += cluster.map_shared_rank(cols_sum, r)[x - part.j0];
      }
    }
    *weight_of(a.w, b, head, x) = v + sum;
  }
  cluster.sync();   // (the others read this block's sums)
}

// Of the two kernels this one is the faster where the cells (tokens k by the columns that a band leaves 16 of them) times 2.2, or 2.8 at head dimension 128, are fewer than those of the tiles of 128 x 128 that the other
// goes through; few cells more, half a million in all, are made up for by the launch that it saves.  With one block an SM (head dimension 128, or more than half the shared memory), its heads have to fit on the SMs at once.
// us, the other / this; bfloat16 queries, int8 codes at 64 and float16 at 128; windows (band to either side) of
//                      one token, 4 x 8   one token, 32 x 16   4 tokens, 2 x 16   16 tokens, 8 x 16
//   64   64 (64)       14 / 10            52 / 29              20 / 13            114 / 37
//        128 (32)      15 / 11            52 / 37              20 / 16            115 / 51
//        128           14 / 13            52 / 46              20 / 19            114 / 81
//        256 (32)      17 / 12            72 / 63              24 / 17            186 / 89
//        256           16 / 19            77 / 103             26 / 32            203 / 218
//        512 (32)      19 / 14            108 / -              32 / 23            315 / 220
//   128  64 (64)       15 / 11            53 / 55              22 / 15            119 / 49
//        128 (32)      15 / 12            55 / 70              23 / 17            127 / 74
//        128           15 / 14            54 / 85              23 / 20            128 / 118
//        256 (32)      18 / 14            84 / 131             28 / 22            194 / -
bool faster(const tritt_cache_t& c, long long places, long long reach_k, long long reach_j, long long band) {
  auto least = [](long long x, long long y) { return x < y ? x : y; };
  auto tiled = [&](long long tokens) { return tokens < places ? tokens + 127 : (tokens + 127) / 128 * 128; };   // (a window begins anywhere in a tile)
  const long long others = tiled(reach_k) * least(tiled(reach_j), 128 + band + 127);
  const long long cells = (reach_k + 15) / 16 * 16 * ((least(reach_j, 16 + band) + 31) / 32 * 32) * (c.D == 64 ? 22 : 28) / 10;
  return cells <= others || (cells - others) * c.B * c.N * c.n <= 500000;
}
// Blocks of a cluster, and the places that each needs: false, it is not a call for this kernel.
bool plan(const TdpWeighArgs& a, WindowParams& p, int& ranks) {
  const tritt_cache_t& c = a.cache.c;
  if (c.D != 64 && c.D != 128) return false;
  const long long places = (long long)c.page_size * c.table_pages;
  auto reach = [&](int w) { return (long long)w + c.n < places ? (long long)w + c.n : places; };
  const long long tiles = (reach(a.k2w) + 30) / 16, seen = reach(a.k1w);
  if (tiles > 256 || seen > 4096 || !faster(c, places, reach(a.k2w), seen, (long long)a.kkl + a.kkr)) return false;
  p.a = a;
  for (int per_sm = c.D == 64 ? 2 : 1; per_sm > 0; --per_sm) {   // blocks of an SM
    ranks = 1;
    while (ranks < kMostCluster && 2LL * ranks * c.B * c.N <= per_sm * kWeighCtas && 2 * ranks <= tiles) ranks *= 2;
    const long long rows = (tiles + ranks - 1) / ranks * 16, band = rows + a.kkl + a.kkr;
    p.rows = (int)rows;
    p.cols = (int)(((band < seen ? band : seen) + 31 + kWide - 1) / kWide * kWide);
    // small units share out better (128, band 32 above: 51 us by four tokens, 55 by eight), as far as their sums leave room for as many blocks (256, band 32: 116 by four, one block an SM, 89 by eight)
    for (p.group = 4; p.group <= 8; p.group *= 2) {
      const long long groups = (c.n + p.group - 1) / p.group;
      if (groups * p.rows / 16 * p.cols > 1 << 18 || (long long)c.n * c.D > 1 << 15) continue;   // (no overflow below)
      const int bytes = (c.D == 64 ? layout_of<64>(p.rows, p.cols, c.n, p.group) : layout_of<128>(p.rows, p.cols, c.n, p.group)).size;
      if (bytes <= kMostSmem / per_sm && (per_sm == 2 || (long long)c.B * c.N <= kWeighCtas)) return true;
    }
  }
  return false;
}

template <typename T, int D, int CODE> int launch(const WindowParams& p, int ranks, cudaStream_t stream) {
  const tritt_cache_t& c = p.a.cache.c;
  const int bytes = layout_of<D>(p.rows, p.cols, c.n, p.group).size;
  TRITT_CUDA_OK(cudaFuncSetAttribute(tdp_weigh_window_kernel<T, D, CODE>, cudaFuncAttributeMaxDynamicSharedMemorySize, kMostSmem));
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(ranks, c.B * c.N);
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = bytes;
  cfg.stream = stream;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = ranks;
  attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  TRITT_CUDA_OK(cudaLaunchKernelEx(&cfg, tdp_weigh_window_kernel<T, D, CODE>, p));
  count_launch();
  return 0;
}
template <typename T, int CODE> int by_size(const WindowParams& p, int ranks, cudaStream_t stream) {
  return p.a.cache.c.D == 64 ? launch<T, 64, CODE>(p, ranks, stream) : launch<T, 128, CODE>(p, ranks, stream);
}
template <typename T> int by_code(const WindowParams& p, int ranks, cudaStream_t stream) {
  switch (p.a.cache.c.code) {
    case TRITT_CODE_F16: return by_size<T, TRITT_CODE_F16>(p, ranks, stream);
    case TRITT_CODE_E4M3: return by_size<T, TRITT_CODE_E4M3>(p, ranks, stream);
    default: return by_size<T, TRITT_CODE_INT8>(p, ranks, stream);
  }
}

}  // namespace

bool window_tdp_weigh_applies(const TdpWeighArgs& a) {
  WindowParams p{};
  int ranks;
  return plan(a, p, ranks);
}

int window_tdp_weigh(const TdpWeighArgs& a, cudaStream_t stream) {
  WindowParams p{};
  int ranks;
  plan(a, p, ranks);
  if (a.dtype == TRITT_F32) return by_code<float>(p, ranks, stream);
  return a.dtype == TRITT_F16 ? by_code<__half>(p, ranks, stream) : by_code<__nv_bfloat16>(p, ranks, stream);
}

}  // namespace tritt
