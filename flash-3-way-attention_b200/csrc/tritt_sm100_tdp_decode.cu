// Triple-dot-product attention of new tokens over the quantised cache on Blackwell tensor cores (tcgen05 + TMEM).
//
// For a new token q and one k the scores are those of an ordinary attention with the query A[k] = alpha q*K2[k]:
//   S[k, j] = A[k].K1[j],   acc[k] = sum_j P[k, j] SiLU(V1)[j],   o = sum_k 2^(m[k] - m) acc[k]*V2[k]
// so one token is flash attention with as many query rows as it attends to tokens k.  Rows are taken in groups of 32 of one new
// token (a warp, so that the last sum crosses no warps), four groups a tile of 128 rows, two tiles at a time, which share every slab
// of 128 columns j.  Bound by the products (4 D flops a pair) and the exponentials (one a pair).
//
// The line of all (sequence, head, pair of tiles, slab) steps is cut in equal parts, one for each CTA: contexts may differ in length, one
// short sequence still uses all SMs, and nothing of it is known to the host.  A part that begins or ends inside a pair of tiles leaves its
// groups' maxima, sums and results all the same; a second kernel joins all groups and pieces of a row in a fixed order.
//
// Codes become fp16 operands: a slab's rows, whose exponents differ, are brought to the largest one's by exact multiplications by powers of
// two, whatever lies 2^-38 below is lost.  K1's exponent joins the scale of the scores, for each 32 columns; V1's runs along with the
// accumulator, which is multiplied where it grows.  A is rounded once to 11 bits, P (times 2^7, fp16's lower range) once.
//
//   warp 0        issues tcgen05.mma: S_x = A_x K1^T, acc_x += P_x V1 for the tiles x = a, b in turn, P_x read from TMEM over S_x
//   warps 4-7     producers: a warp loads 32 rows of a slab (pages, exponents, codes), converts and stores them with the 128-byte
//                 swizzle; the loads of a tile are in flight before its stage is free
//   warps 8-15    one row a thread: form A, then maximum, exponentials, P; at the end of a piece the group's sum
#include "tritt_cache.cuh"
#include "tritt_sm100.cuh"
#include "tritt_sm100_tdp.cuh"

namespace tritt {
namespace {
using namespace sm100;

constexpr int kThreads = 512;
constexpr float kGap = 8.f;      // the accumulator is rescaled when a row's maximum grew by more than 2^8
constexpr float kLift = 7.f;     // P is formed times 2^7: at most 2^15, normal down to 2^-21 of the reference
constexpr int kMetas = 6;        // slabs whose descriptions are kept: two more than the ring's depth (one is overwritten when S of the slab
                                 // kMetas back is done, and the rows have then read that of the slab before it)
constexpr int kUnlimited = 1 << 30;

template <int D> struct Cfg {
  static constexpr int kTile = 128 * D * 2;
  static constexpr int kStages = D == 128 ? 2 : 4;                 // of keys, and as many of values
  static constexpr int kOffA = 0;                                  // two tiles
  static constexpr int kOffK = 2 * kTile;
  static constexpr int kOffV = kOffK + kStages * kTile;
  static constexpr int kOffQ = kOffV + kStages * kTile;            // [8 warps][D] fp32
  static constexpr int kOffMisc = kOffQ + 8 * D * 4;
  static constexpr int kSmem = kOffMisc + 1024;
  static constexpr int kTmemO = 256;                               // S_a | S_b | acc_a | acc_b
};

struct Meta {             // of one slab, by the warp that loaded 32 of its rows
  uint32_t there[4];      // rows that have a place
  uint32_t nan[4];        // rows that read as NaN (K1 or V1)
  float scale[4];         // of the 32 columns' scores
  int v_exp[4];           // largest exponent byte of V1's rows
};

struct Misc {
  uint64_t k_full[4], k_empty[4], v_full[4], v_empty[4];
  uint64_t meta_full[kMetas], a_ready[2], s_ready[2], p_ready[2], o_done[2];
  Meta meta[kMetas];
  uint32_t tmem_base;
  int abort_flag;
  int first_b;
  long long first_base, total;
};
static_assert(sizeof(Misc) <= 1024, "shared memory of the barriers");

// What the line of steps has of one sequence.
struct Line {
  int ctx, cnt;          // tokens before the new ones, new ones
  int groups;            // of 32 rows, of each new token
  int pairs, slabs;      // pairs of tiles of a head; slabs of a pair (the most of any)
};
struct LineEntry {       // in the workspace, for the kernel that joins
  long long base, pair_base;
  Line line;
  int pad;
};

struct Params {
  TdpDecodeArgs a;
  LineEntry* table;      // [B]
  float* part;           // [pieces][8][D + 2]
  int ctas;
};

// Columns that a pair's groups may attend to, by their numbers in the sequence (whatever the tree: its tokens are told apart by masks).
struct Columns {
  int lo, hi;
};

__host__ __device__ inline int least(int x, int y) { return x < y ? x : y; }
__host__ __device__ inline int most(int x, int y) { return x > y ? x : y; }

__device__ __forceinline__ Line line_of(const TdpDecodeArgs& a, int b) {
  Line l;
  l.ctx = context_of(a.cache, b);
  l.cnt = new_tokens(a.cache, b);
  if (l.cnt == 0) {
    l.groups = l.pairs = l.slabs = 0;
    return l;
  }
  l.groups = (least(l.ctx + l.cnt - 1, a.k2w) + 32) / 32;   // (rows: the window and the token itself)
  l.pairs = (l.cnt * l.groups + 7) / 8;
  l.slabs = (least(l.ctx, a.k1w) + l.cnt + 127) / 128;
  return l;
}
__device__ __forceinline__ Columns columns_of(const TdpDecodeArgs& a, const Line& l, int pair) {
  Columns c{kUnlimited, -1};
  const int g1 = least(pair * 8 + 8, l.cnt * l.groups);
  for (int g = pair * 8; g < g1; ++g) {
    // positions of the group's rows, whatever the token's depth in a tree (0 to i)
    const int i = g / l.groups, r = (g - i * l.groups) * 32;
    const int ka = most(0, l.ctx - a.k2w) + r, kb = most(0, l.ctx + i - a.k2w) + r + 31;
    c.lo = least(c.lo, most(most(0, l.ctx - a.k1w), ka - least(ka, a.kkl)));
    c.hi = most(c.hi, kb + least(a.kkr, kUnlimited - 1) < l.ctx ? kb + a.kkr : l.ctx + i);
  }
  c.lo = least(c.lo, l.ctx);
  return c;
}

// Steps of a CTA: walks the line from the CTA's first step to its last.
struct Walk {
  long long x, end, base;   // present step, behind the last, first step of sequence b
  long long pair_base;      // pairs before sequence b's
  int b;
  Line l;
};
struct Piece {
  int b, head, pair, s0, s1;
  long long id;             // pieces are numbered by pair + CTA: each new pair and each cut makes one
};
__device__ __forceinline__ bool next_piece(const Params& p, Walk& w, Piece& s) {
  if (w.x >= w.end) return false;
  while (true) {
    const long long here = (long long)w.l.pairs * w.l.slabs * p.a.cache.c.N;
    if (w.x < w.base + here) break;
    if (w.b + 1 >= p.a.cache.c.B) return false;   // (contexts that changed under the kernel)
    w.base += here;
    w.pair_base += (long long)w.l.pairs * p.a.cache.c.N;
    w.l = line_of(p.a, ++w.b);
  }
  const long long rel = w.x - w.base, pair = rel / w.l.slabs;
  s.b = w.b;
  s.head = (int)(pair / w.l.pairs);
  s.pair = (int)(pair % w.l.pairs);
  s.s0 = (int)(rel % w.l.slabs);
  s.s1 = (int)least((int)(w.l.slabs - s.s0 < w.end - w.x ? w.l.slabs - s.s0 : w.end - w.x), w.l.slabs) + s.s0;
  s.id = w.pair_base + pair + blockIdx.x;
  w.x += s.s1 - s.s0;
  return true;
}

// Four fp16 pairs times a power of two (exact above 2^-24).
__device__ __forceinline__ uint4 times(uint4 v, uint32_t f) {
  const __half2 h = *reinterpret_cast<const __half2*>(&f);
  uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const __half2 r = __hmul2(*reinterpret_cast<__half2*>(&w[i]), h);
    w[i] = *reinterpret_cast<const uint32_t*>(&r);
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}
// 2^e as a pair of fp16 (0 below its range; e <= 15)
__device__ __forceinline__ uint32_t half_power(int e) {
  const uint32_t h = e >= -14 ? (uint32_t)(e + 15) << 10 : e >= -24 ? 1u << (e + 24) : 0u;
  return h | h << 16;
}
// codes times 2^kUp use fp16's range: 2^15 is the largest
template <int CODE> constexpr int kUp = CODE == TRITT_CODE_F16 ? 0 : CODE == TRITT_CODE_E4M3 ? 5 : 7;
// q (largest element in [1, 2)) times a code times 2^-kDown is at most 2^9
template <int CODE> constexpr int kDown = CODE == TRITT_CODE_F16 ? 7 : 0;

template <int D, int CODE> struct TileLoader {   // a warp's 32 rows of one part of a slab
  static constexpr int kChunks = CODE == TRITT_CODE_F16 ? D / 8 : D / 16;   // of 16 bytes of codes, a row
  uint4 v[kChunks];
  // page: of the lane's own row, -1: none (zeros)
  __device__ __forceinline__ void load(const CacheArgs& a, int part, int head, int token0, int page, int lane) {
#pragma unroll
    for (int it = 0; it < kChunks; ++it) {
      const int idx = it * 32 + lane, row = idx / kChunks, ch = idx % kChunks;
      const int pg = __shfl_sync(0xffffffffu, page, row);
      v[it] = make_uint4(0u, 0u, 0u, 0u);
      if (pg >= 0) {
        const size_t at = row_of(a, Place{pg, (token0 + row) & (a.c.page_size - 1)}, part, head);
        v[it] = __ldg(reinterpret_cast<const uint4*>((const uint8_t*)a.c.codes + at * (size_t)(kChunks * 16)) + ch);
      }
    }
  }
  // to rows row0 .. row0 + 31 of a tile, each times the power of two of its lane
  __device__ __forceinline__ void store(uint8_t* tile, int row0, uint32_t factor, int lane) {
#pragma unroll
    for (int it = 0; it < kChunks; ++it) {
      const int idx = it * 32 + lane, row = idx / kChunks, ch = idx % kChunks;
      const uint32_t f = __shfl_sync(0xffffffffu, factor, row);
      if constexpr (CODE == TRITT_CODE_F16) {
        *reinterpret_cast<uint4*>(tile + (ch >> 3) * 16384 + swz128(row0 + row, ch & 7)) = times(v[it], f);
      } else {
        uint4 lo, hi;
        bytes_to_halves<CODE>(v[it].x, lo.x, lo.y);
        bytes_to_halves<CODE>(v[it].y, lo.z, lo.w);
        bytes_to_halves<CODE>(v[it].z, hi.x, hi.y);
        bytes_to_halves<CODE>(v[it].w, hi.z, hi.w);
        lo = times(lo, f);
        hi = times(hi, f);
        // (lanes whose chunks lie in the second 64 columns store in the other order, off the first ones' banks)
        const int swap = D == 128 ? ch >> 2 & 1 : 0, c0 = 2 * ch + swap, c1 = 2 * ch + 1 - swap;
        *reinterpret_cast<uint4*>(tile + (c0 >> 3) * 16384 + swz128(row0 + row, c0 & 7)) = swap ? hi : lo;
        *reinterpret_cast<uint4*>(tile + (c1 >> 3) * 16384 + swz128(row0 + row, c1 & 7)) = swap ? lo : hi;
      }
    }
  }
};

template <typename T16, int D, int CODE>
__global__ void __launch_bounds__(kThreads, 1) tdp_decode_kernel(const __grid_constant__ Params p) {
  using C = Cfg<D>;
  constexpr int NS = C::kStages;
  extern __shared__ __align__(1024) uint8_t smem[];
  Misc& ms = *reinterpret_cast<Misc*>(smem + C::kOffMisc);
  const TdpDecodeArgs& a = p.a;
  const CacheArgs& ca = a.cache;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (smem_u32(smem) & 1023u) {
    if (tid == 0 && ca.status) atomicOr(ca.status, 8);
    return;
  }
  if (tid == 32) {
    ms.abort_flag = 0;
    for (int i = 0; i < NS; ++i) {
      mbar_init(&ms.k_full[i], 128);
      mbar_init(&ms.k_empty[i], 1);
      mbar_init(&ms.v_full[i], 128);
      mbar_init(&ms.v_empty[i], 1);
    }
    for (int i = 0; i < kMetas; ++i) mbar_init(&ms.meta_full[i], 4);
    for (int x = 0; x < 2; ++x) {
      mbar_init(&ms.a_ready[x], 128);
      mbar_init(&ms.s_ready[x], 1);
      mbar_init(&ms.p_ready[x], 128);
      mbar_init(&ms.o_done[x], 1);
    }
    fence_barrier_init();
  }
  if (warp == 0) {
    tmem_alloc(&ms.tmem_base, 512);
    tmem_relinquish();
  }
  if (warp == 2) {
    // the whole line's length, and the sequence of this CTA's first step: 32 sequences at a time
    long long total = 0, pairs = 0;
    for (int b0 = 0; b0 < ca.c.B; b0 += 32) {
      const int b = b0 + lane;
      Line l{};
      if (b < ca.c.B) l = line_of(a, b);
      const long long np = (long long)l.pairs * ca.c.N, steps = np * l.slabs;
      long long s = steps, q = np;   // sums up to this lane
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const long long s2 = __shfl_up_sync(0xffffffffu, s, o), q2 = __shfl_up_sync(0xffffffffu, q, o);
        if (lane >= o) s += s2, q += q2;
      }
      if (blockIdx.x == 0 && b < ca.c.B) p.table[b] = LineEntry{total + s - steps, pairs + q - np, l, 0};
      total += __shfl_sync(0xffffffffu, s, 31);
      pairs += __shfl_sync(0xffffffffu, q, 31);
    }
    if (lane == 0) ms.total = total;
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = ms.tmem_base;
  volatile int* abort_flag = &ms.abort_flag;
  const long long total = ms.total;
  Walk walk;
  walk.x = (long long)blockIdx.x * total / p.ctas;
  walk.end = ((long long)blockIdx.x + 1) * total / p.ctas;
  walk.base = walk.pair_base = 0;
  walk.b = 0;
  Piece s;
  if (walk.x < walk.end) walk.l = line_of(a, 0);

  if (warp == 0) {
    // ------------------------------------------------------------------ products
    const bool leader = elect_one();
    auto wait_all = [&](uint64_t* bar, uint32_t parity) { return __all_sync(0xffffffffu, mbar_wait(bar, parity, abort_flag)); };
    auto commit = [&](uint64_t* bar) {
      if (leader) mma_commit(bar);
    };
    constexpr uint32_t idesc_pv = make_idesc_f16(128, D, 0, false, true);
    constexpr uint32_t kHi = desc_hi(1024);
    const uint32_t aLo = desc_lo(smem_u32(smem + C::kOffA), 16);
    int slab = 0, pieces[2] = {0, 0}, pcount[2] = {0, 0};   // slabs so far, each tile's pieces and P's
    bool alive = true;
    while (alive && next_piece(p, walk, s)) {
      const Columns col = columns_of(a, walk.l, s.pair);
      const int n = least(s.s1, (col.hi - col.lo + 128) / 128) - s.s0;
      if (n <= 0) continue;
      const int tiles = least(8, walk.l.cnt * walk.l.groups - s.pair * 8) > 4 ? 2 : 1;
      auto width = [&](int i) { return least(128, col.hi + 1 - (col.lo + (s.s0 + i) * 128)); };
      // S_x of slab i
      auto issue_s = [&](int x, int i) {
        const int pos = slab + i, st = pos % NS;
        if (x == 0 && !wait_all(&ms.k_full[st], (pos / NS) & 1)) return false;
        tc_fence_after();
        const uint32_t bLo = desc_lo(smem_u32(smem + C::kOffK + st * C::kTile), 16);
        const uint32_t idesc = make_idesc_f16(128, (width(i) + 31) / 32 * 32, 0, false, false);
#pragma unroll
        for (int k = 0; k < D / 16; ++k) {
          const uint32_t kk = (k >> 2) * (16384 >> 4) + (k & 3) * 2;
          if (leader) mma_ss_lo(tmem + x * 128, aLo + x * (C::kTile >> 4) + kk, bLo + kk, kHi, idesc, k > 0);
        }
        commit(&ms.s_ready[x]);
        if (x == tiles - 1) commit(&ms.k_empty[st]);
        return true;
      };
      auto issue_pv = [&](int x, int i) {
        const int pos = slab + i, st = pos % NS;
        if (x == 0 && !wait_all(&ms.v_full[st], (pos / NS) & 1)) return false;
        tc_fence_after();
        const uint32_t bLo = desc_lo(smem_u32(smem + C::kOffV + st * C::kTile), 16384);
        const int steps = (width(i) + 15) / 16;
#pragma unroll
        for (int k = 0; k < 8; ++k)
          if (leader && k < steps)
            mma_ts_lo(tmem + C::kTmemO + x * D, tmem + x * 128 + k * 8, bLo + k * (2048 >> 4), kHi, idesc_pv, k > 0 || i > 0);
        if (x == tiles - 1) commit(&ms.v_empty[st]);
        if (i == n - 1) commit(&ms.o_done[x]);
        return true;
      };
      for (int x = 0; x < tiles && alive; ++x) alive = wait_all(&ms.a_ready[x], pieces[x] & 1) && issue_s(x, 0);
      for (int i = 0; i < n && alive; ++i)
        for (int x = 0; x < tiles && alive; ++x) {
          alive = wait_all(&ms.p_ready[x], pcount[x] & 1);
          if (!alive) break;
          pcount[x] += 1;
          tc_fence_after();
          // (S_x of the next slab overwrites P_x: the pipe runs it behind P_x V)
          alive = issue_pv(x, i) && (i + 1 >= n || issue_s(x, i + 1));
        }
      slab += n;
      ++pieces[0];
      pieces[1] += tiles - 1;
    }
  } else if (warp >= 4 && warp < 8) {
    // ------------------------------------------------------------------ producers
    const int w = warp - 4;
    int slab = 0;
    bool alive = true;
    while (alive && next_piece(p, walk, s)) {
      const Columns col = columns_of(a, walk.l, s.pair);
      const int n = least(s.s1, (col.hi - col.lo + 128) / 128) - s.s0;
      int v_exp = 0;   // the largest exponent byte of V1's rows in this piece so far
      int token = col.lo + s.s0 * 128 + w * 32 + lane;
      auto page_of = [&](int t) { return t <= col.hi ? place_of(ca, s.b, t).page : -1; };
      int page = n > 0 ? page_of(token) : -1;
      for (int i = 0; i < n && alive; ++i, token += 128) {
        const int pos = slab + i, st = pos % NS, mt = pos % kMetas;
        const int token0 = token - lane;
        const bool any = token0 <= col.hi;   // (32 columns that no row looks at are not loaded)
        TileLoader<D, CODE> tile;
        int ek = 0, ev = 0;
        if (page >= 0) {
          const Place at{page, token & (ca.c.page_size - 1)};
          ek = __ldg(ca.c.exponents + row_of(ca, at, kPartK1, s.head));
          ev = __ldg(ca.c.exponents + row_of(ca, at, kPartV1, s.head));
        }
        if (any) tile.load(ca, kPartK1, s.head, token0, page, lane);
        const int next = i + 1 < n ? page_of(token + 128) : -1;
        const uint32_t there = __ballot_sync(0xffffffffu, page >= 0), nan = __ballot_sync(0xffffffffu, page >= 0 && (ek == 255 || ev == 255));
        if (ek == 255) ek = 0;   // (its codes are zeros)
        if (ev == 255) ev = 0;
        const int ek_most = __reduce_max_sync(0xffffffffu, ek), ev_most = __reduce_max_sync(0xffffffffu, ev);
        if (!__all_sync(0xffffffffu, mbar_wait(&ms.k_empty[st], ((pos / NS) & 1) ^ 1, abort_flag))) {
          alive = false;
          break;
        }
        if (lane == 0) {
          Meta& m = ms.meta[mt];
          m.there[w] = there;
          m.nan[w] = nan;
          m.scale[w] = ek_most > kUp<CODE> ? __uint_as_float((uint32_t)(ek_most - kUp<CODE>) << 23) : 0.f;
          m.v_exp[w] = ev_most;
          mbar_arrive(&ms.meta_full[mt]);
        }
        if (any) tile.store(smem + C::kOffK + st * C::kTile, w * 32, half_power(kUp<CODE> + ek - ek_most), lane);
        fence_async_smem();
        mbar_arrive(&ms.k_full[st]);
        if (any) tile.load(ca, kPartV1, s.head, token0, page, lane);
        if (!__all_sync(0xffffffffu, mbar_wait(&ms.meta_full[mt], (pos / kMetas) & 1, abort_flag)) ||
            !__all_sync(0xffffffffu, mbar_wait(&ms.v_empty[st], ((pos / NS) & 1) ^ 1, abort_flag))) {
          alive = false;
          break;
        }
        const volatile Meta& m = ms.meta[mt];
        v_exp = max(max(max(v_exp, m.v_exp[0]), m.v_exp[1]), max(m.v_exp[2], m.v_exp[3]));
        if (any) tile.store(smem + C::kOffV + st * C::kTile, w * 32, half_power(kUp<CODE> + ev - v_exp), lane);
        fence_async_smem();
        mbar_arrive(&ms.v_full[st]);
        page = next;
      }
      if (n > 0) slab += n;
    }
  } else if (warp >= 8) {
    // ------------------------------------------------------------------ soft-max, one row a thread
    const int x = (warp - 8) >> 2, wq = warp & 3;
    const uint32_t lane_base = (uint32_t)(wq * 32) << 16;
    const uint32_t tS = tmem + lane_base + x * 128, tO = tmem + lane_base + C::kTmemO + x * D;
    float* sq = reinterpret_cast<float*>(smem + C::kOffQ) + (warp - 8) * D;
    int slab = 0, scount = 0, piece = 0;   // slabs so far, this tile's, its pieces
    bool alive = true;
    while (alive && next_piece(p, walk, s)) {
      const Line l = walk.l;
      const Columns col = columns_of(a, l, s.pair);
      const int n = least(s.s1, (col.hi - col.lo + 128) / 128) - s.s0;
      const int groups = l.cnt * l.groups, g = s.pair * 8 + x * 4 + wq;
      float* out = p.part + (size_t)(s.id * 8 + x * 4 + wq) * (D + 2);
      if (n <= 0) {
        if (lane == 0 && g < groups) out[0] = -INFINITY, out[1] = 0.f;
        continue;
      }
      if (s.pair * 8 + x * 4 >= groups) {   // (no second tile)
        slab += n;
        continue;
      }
      // --- this thread's row: token k of new token i
      const int i = g < groups ? g / l.groups : 0;
      const unsigned long long word = ca.c.ancestors ? seen_word(ca, s.b, i) : 0;
      const int pos_q = l.ctx + (ca.c.ancestors ? __popcll(word) - 1 : i);
      const int pk = most(0, pos_q - a.k2w) + (g % l.groups) * 32 + lane;
      bool on = g < groups && pk <= pos_q;
      int token = pk;
      if (ca.c.ancestors && pk >= l.ctx) {
        unsigned long long left = word;
        for (int c = l.ctx; c < pk && left; ++c) left &= left - 1;
        token = l.ctx + (left ? __ffsll(left) - 1 : 0);
      }
      int byte = 0, byte2 = 0;
      Place at{-1, 0};
      if (on) {
        at = place_of(ca, s.b, token);
        if (at.page < 0) {
          on = false;
          if (ca.status) atomicOr(ca.status, kStatusPlace);
        }
      }
      if (on) {
        byte = __ldg(ca.c.exponents + row_of(ca, at, kPartK2, s.head));
        byte2 = __ldg(ca.c.exponents + row_of(ca, at, kPartV2, s.head));
      }
      // columns that the row attends to: numbers c_lo .. c_hi, and of a tree's tokens a word
      const int c_lo = on ? most(most(0, pos_q - a.k1w), pk - least(pk, a.kkl)) : kUnlimited;
      const int last = pk < kUnlimited - a.kkr ? least(pos_q, pk + a.kkr) : pos_q;
      const int c_hi = !on ? -1 : ca.c.ancestors ? least(l.ctx - 1, last) : last;
      unsigned long long tree = 0;
      if (on && ca.c.ancestors) {
        unsigned long long left = word;
        for (int c = l.ctx; left; ++c, left &= left - 1)
          if (c >= c_lo && c <= last) tree |= left & (~left + 1);
      }
      // --- A = 2^-kDown q * code, q brought to [1, 2); the powers of two and alpha go to the scores' scale
      float row_scale;
      {
        const T16* q = (const T16*)a.q.p + rows_at(a.q, s.b, s.head, i);
        constexpr int E = D / 32;
        float f[E];
        uint32_t big = 0;
#pragma unroll
        for (int e = 0; e < E; ++e) {
          f[e] = to_f(q[lane * E + e]);
          big = max(big, __float_as_uint(f[e]) & 0x7fffffffu);
        }
        big = __reduce_max_sync(0xffffffffu, big);
        const int power = max(min(254 - (int)(big >> 23), 253), 1);   // (the largest numbers are brought to [2, 4))
        const float up = __uint_as_float((uint32_t)power << 23);
        const float sign = a.scale2 < 0.f ? -1.f : 1.f;
        __syncwarp();
#pragma unroll
        for (int e = 0; e < E; ++e) sq[lane * E + e] = f[e] * up * sign;
        __syncwarp();
        row_scale = fabsf(a.scale2) * (on && byte != 255 ? __uint_as_float((uint32_t)byte << 23) : 0.f) * (float)(1 << kDown<CODE>);
        row_scale *= __uint_as_float((uint32_t)(254 - power) << 23);
      }
      {
        uint8_t* tile = smem + C::kOffA + x * C::kTile;
        const uint8_t* codes = (const uint8_t*)ca.c.codes + (on ? row_of(ca, at, kPartK2, s.head) : 0) * (size_t)(D * (CODE == TRITT_CODE_F16 ? 2 : 1));
#pragma unroll 4
        for (int ch = 0; ch < D / 8; ++ch) {
          uint32_t h[4] = {0u, 0u, 0u, 0u};
          if (on) {
            Codes8<CODE> c8;
            c8.load(codes, ch * 8);
            c8.halves(h);
          }
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float2 c = __half22float2(*reinterpret_cast<const __half2*>(&h[e]));
            const float2 q = *reinterpret_cast<const float2*>(sq + ch * 8 + 2 * e);
            constexpr float down = 1.f / (1 << kDown<CODE>);
            h[e] = pack2<__half>(q.x * (c.x * down), q.y * (c.y * down));
          }
          *reinterpret_cast<uint4*>(tile + (ch >> 3) * 16384 + swz128(wq * 32 + lane, ch & 7)) = make_uint4(h[0], h[1], h[2], h[3]);
        }
      }
      fence_async_smem();
      mbar_arrive(&ms.a_ready[x]);
      // --- slabs
      float m_used = -INFINITY, l_sum = 0.f;
      int v_exp = 0;
      for (int t = 0; t < n; ++t, ++scount) {
        const int pos = slab + t, c0 = col.lo + (s.s0 + t) * 128, wid = least(128, col.hi + 1 - c0);
        const volatile Meta& m = ms.meta[pos % kMetas];
        if (!__all_sync(0xffffffffu, mbar_wait(&ms.meta_full[pos % kMetas], (pos / kMetas) & 1, abort_flag)) ||
            !__all_sync(0xffffffffu, mbar_wait(&ms.s_ready[x], scount & 1, abort_flag))) {
          alive = false;
          break;
        }
        tc_fence_after();
        float f[4];
        bool clean = wid == 128;
        int v_now = v_exp;
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          f[c] = row_scale * m.scale[c];
          clean = clean && m.there[c] == 0xffffffffu && m.nan[c] == 0u;
          v_now = max(v_now, m.v_exp[c]);
        }
        const bool full = __all_sync(0xffffffffu, clean && c_lo <= c0 && c_hi >= c0 + 127);
        // columns that count, and those of them that read as NaN
        uint32_t mask[4], bad[4];
        float mx = -INFINITY;
        if (full) {
#pragma unroll
          for (int hf = 0; hf < 2; ++hf) {
            uint32_t sr[64];
            tmem_ld64(tS + hf * 64, sr);
            tmem_wait_ld();
#pragma unroll
            for (int q = 0; q < 2; ++q) {
              float m0 = -INFINITY, m1 = -INFINITY;
#pragma unroll
              for (int c = 0; c < 32; c += 2) {
                m0 = fmaxf(m0, __uint_as_float(sr[q * 32 + c]));
                m1 = fmaxf(m1, __uint_as_float(sr[q * 32 + c + 1]));
              }
              mx = fmaxf(mx, fmaxf(m0, m1) * f[hf * 2 + q]);
            }
          }
        } else {
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            const int c1 = c0 + c * 32;
            const int lo = most(c_lo - c1, 0), hi = least(c_hi - c1, 31);
            uint32_t b = lo > 31 || hi < lo ? 0u : (0xffffffffu << lo) & (0xffffffffu >> (31 - hi));
            const int off = l.ctx - c1;   // of the first new token
            if (tree && off < 32 && off > -64) b |= (uint32_t)(off >= 0 ? tree << off : tree >> -off);
            mask[c] = b & m.there[c];
            if (mask[c] != b && ca.status) atomicOr(ca.status, kStatusPlace);
            bad[c] = mask[c] & m.nan[c];
            if (c * 32 < wid) {
              uint32_t sr[32];
              tmem_ld32(tS + c * 32, sr);
              tmem_wait_ld();
              float m0 = -INFINITY;
#pragma unroll
              for (int e = 0; e < 32; ++e)
                if (mask[c] >> e & 1) m0 = fmaxf(m0, __uint_as_float(sr[e]));
              if (m0 != -INFINITY) mx = fmaxf(mx, m0 * f[c]);
            }
          }
        }
        if (t == 0) {
          m_used = mx;
        } else {
          const bool grow = mx > m_used + kGap;
          if (__any_sync(0xffffffffu, grow) || v_now != v_exp) {
            // (s_ready of this slab was committed behind the previous slab's P V)
            float corr = grow ? exp2f(m_used - mx) : 1.f;
            if (grow) {
              m_used = mx;
              l_sum *= corr;
            }
            corr *= v_now - v_exp < 126 ? __uint_as_float((uint32_t)(127 - (v_now - v_exp)) << 23) : 0.f;
#pragma unroll
            for (int ch = 0; ch < D / 32; ++ch) {
              uint32_t o[32];
              tmem_ld32(tO + ch * 32, o);
              tmem_wait_ld();
#pragma unroll
              for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * corr);
              tmem_st32(tO + ch * 32, o);
            }
          }
        }
        v_exp = v_now;
        const float shift = kLift - m_used;
        float psum = 0.f;
        if (full) {
#pragma unroll
          for (int hf = 0; hf < 2; ++hf) {
            uint32_t sr[64], pk2[32];
            tmem_ld64(tS + hf * 64, sr);
            tmem_wait_ld();
            float p0 = 0.f, p1 = 0.f;
#pragma unroll
            for (int c = 0; c < 64; c += 2) {
              const float e0 = exp2f(fmaf(__uint_as_float(sr[c]), f[hf * 2 + c / 32], shift));
              const float e1 = exp2f(fmaf(__uint_as_float(sr[c + 1]), f[hf * 2 + c / 32], shift));
              p0 += e0;
              p1 += e1;
              pk2[c >> 1] = pack2<__half>(e0, e1);
            }
            psum += p0 + p1;
            tmem_st32(tS + hf * 32, pk2);
          }
        } else {
#pragma unroll
          for (int c = 0; c < 4; ++c)
            if (c * 32 < wid) {
              uint32_t sr[32], pk2[16];
              tmem_ld32(tS + c * 32, sr);
              tmem_wait_ld();
#pragma unroll
              for (int e = 0; e < 32; e += 2) {
                const float e0 = mask[c] >> e & 1 ? exp2f(fmaf(__uint_as_float(sr[e]), f[c], shift)) : 0.f;
                const float e1 = mask[c] >> (e + 1) & 1 ? exp2f(fmaf(__uint_as_float(sr[e + 1]), f[c], shift)) : 0.f;
                psum += e0 + e1;
                pk2[e >> 1] = pack2<__half>(e0, e1);
              }
              if (bad[c]) psum = __uint_as_float(0x7fffffffu);
              tmem_st16(tS + c * 16, pk2);
            }
        }
        l_sum += psum;
        tmem_wait_st();
        tc_fence_before();
        mbar_arrive(&ms.p_ready[x]);
      }
      if (!alive) break;
      slab += n;
      // --- the group's sum: sum over its rows of 2^(m_row - m) acc V2, and of the sums
      if (on && (byte == 255 || byte2 == 255) && l_sum > 0.f) l_sum = __uint_as_float(0x7fffffffu);
      float m_all = m_used;
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) m_all = fmaxf(m_all, __shfl_xor_sync(0xffffffffu, m_all, o));
      const float weight = m_used == -INFINITY ? 0.f : exp2f(m_used - m_all - kLift);
      float l_all = m_used == -INFINITY ? (l_sum != l_sum ? l_sum : 0.f) : l_sum * weight;
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) l_all += __shfl_xor_sync(0xffffffffu, l_all, o);
      // V1's and V2's powers of two (fp32's range is that of the result's own type and more)
      const float vscale = weight == 0.f || byte2 == 255 ? 0.f : weight * exp2f((float)(v_exp - 127 - kUp<CODE>)) * exp2f((float)(byte2 - 127));
      if (!__all_sync(0xffffffffu, mbar_wait(&ms.o_done[x], piece & 1, abort_flag))) {
        alive = false;
        break;
      }
      ++piece;
      tc_fence_after();
      const uint8_t* codes = (const uint8_t*)ca.c.codes + (on ? row_of(ca, at, kPartV2, s.head) : 0) * (size_t)(D * (CODE == TRITT_CODE_F16 ? 2 : 1));
#pragma unroll 1
      for (int ch = 0; ch < D / 32; ++ch) {
        uint32_t o[32];
        float v[32];
        tmem_ld32(tO + ch * 32, o);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          float c[8];
#pragma unroll
          for (int k = 0; k < 8; ++k) c[k] = 0.f;
          if (on) {
            Codes8<CODE> c8;
            c8.load(codes, ch * 32 + e * 8);
            code_values<CODE>(c8, vscale, c);
          }
#pragma unroll
          for (int k = 0; k < 8; ++k) v[e * 8 + k] = c[k];
        }
        tmem_wait_ld(o);
#pragma unroll
        for (int e = 0; e < 32; ++e) v[e] = weight == 0.f ? 0.f : v[e] * __uint_as_float(o[e]);
        // column sums over the warp: halves change hands until each lane has one column
#pragma unroll
        for (int h = 16; h > 0; h >>= 1) {
          const bool upper = lane & h;
#pragma unroll
          for (int e = 0; e < h; ++e) {
            const float give = upper ? v[e] : v[e + h], keep = upper ? v[e + h] : v[e];
            v[e] = keep + __shfl_xor_sync(0xffffffffu, give, h);
          }
        }
        if (g < groups) out[2 + ch * 32 + lane] = v[0];
      }
      if (g < groups && lane == 0) out[0] = m_all, out[1] = l_all;
      tc_fence_before();
    }
  }

  // ------------------------------------------------------------------ teardown
  tc_fence_before();
  __syncthreads();
  if (warp == 0) tmem_dealloc(tmem, 512);
  if (tid == 0 && ms.abort_flag && ca.status) atomicOr(ca.status, kStatusTdpDecode);
}

struct TdpJoinParams {
  TdpDecodeArgs a;
  const LineEntry* table;
  const float* part;
  void* o;
  float* lse;
  int ctas;
};

// One block a row: its eight warps take the row's groups in turn, each all pieces of its group; then the warps' results are added up in order.
template <typename T, int D>
__global__ void __launch_bounds__(256) tdp_join_kernel(const __grid_constant__ TdpJoinParams j) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  __shared__ float sm[8], sl[8], so[8][D];
  const CacheArgs& ca = j.a.cache;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const long long row = blockIdx.x;
  const int i = (int)(row % ca.c.n), head = (int)(row / ca.c.n % ca.c.N), b = (int)(row / ca.c.n / ca.c.N);
  const LineEntry e = j.table[b];
  const LineEntry end = j.table[ca.c.B - 1];
  const long long total = end.base + (long long)end.line.pairs * end.line.slabs * ca.c.N;
  constexpr int E = D / 32;
  float m = -INFINITY, l = 0.f, acc[E];
#pragma unroll
  for (int k = 0; k < E; ++k) acc[k] = 0.f;
  if (i < e.line.cnt)
    for (int g = i * e.line.groups + warp; g < (i + 1) * e.line.groups; g += 8) {
      const long long pair = (long long)head * e.line.pairs + g / 8, first = e.base + pair * e.line.slabs;
      // CTA c has the steps from c total / ctas to the next one's
      for (long long x = first; x < first + e.line.slabs;) {
        const long long c = ((x + 1) * j.ctas - 1) / total;
        x = (c + 1) * total / j.ctas;
        const float* p = j.part + (size_t)((e.pair_base + pair + c) * 8 + g % 8) * (D + 2);
        const float mp = p[0], lp = p[1];
        if (mp == -INFINITY && lp == 0.f) continue;
        const float mn = fmaxf(m, mp), w0 = m == -INFINITY ? 0.f : exp2f(m - mn), w1 = mp == -INFINITY ? 1.f : exp2f(mp - mn);
        l = l * w0 + lp * w1;
#pragma unroll
        for (int k = 0; k < E; ++k) acc[k] = acc[k] * w0 + p[2 + k * 32 + lane] * w1;
        m = mn;
      }
    }
  if (lane == 0) sm[warp] = m, sl[warp] = l;
#pragma unroll
  for (int k = 0; k < E; ++k) so[warp][k * 32 + lane] = acc[k];
  __syncthreads();
  float top = -INFINITY, sum = 0.f;
#pragma unroll
  for (int w = 0; w < 8; ++w) top = fmaxf(top, sm[w]);
#pragma unroll
  for (int w = 0; w < 8; ++w) sum += sm[w] == -INFINITY ? (sl[w] != sl[w] ? sl[w] : 0.f) : sl[w] * exp2f(sm[w] - top);
  const bool none = top == -INFINITY && sum == 0.f;
  for (int c = threadIdx.x; c < D; c += 256) {
    float v = 0.f;
#pragma unroll
    for (int w = 0; w < 8; ++w) v += sm[w] == -INFINITY ? 0.f : so[w][c] * exp2f(sm[w] - top);
    ((T*)j.o)[(size_t)row * D + c] = from_f<T>(none ? 0.f : sum != sum ? sum : v * (1.f / sum));
  }
  if (j.lse && threadIdx.x == 0) j.lse[row] = none ? -INFINITY : sum != sum ? sum : (top + log2f(sum)) * kLn2;
}

template <typename T16, int D, int CODE>
int launch(const Params& p, const TdpJoinParams& j, cudaStream_t stream) {
  auto kern = tdp_decode_kernel<T16, D, CODE>;
  TRITT_CUDA_OK(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg<D>::kSmem));
  kern<<<p.ctas, kThreads, Cfg<D>::kSmem, stream>>>(p);
  count_launch();
  TRITT_CUDA_OK(cudaGetLastError());
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)((long long)p.a.cache.c.B * p.a.cache.c.N * p.a.cache.c.n));
  cfg.blockDim = dim3(256);
  cfg.stream = stream;
  TRITT_CUDA_OK(cudaLaunchKernelEx(&cfg, tdp_join_kernel<T16, D>, j));
  count_launch();
  return 0;
}

template <typename T16> int by_size(const Params& p, const TdpJoinParams& j, cudaStream_t s) {
  const int code = p.a.cache.c.code;
  if (p.a.cache.c.D == 64) {
    if (code == TRITT_CODE_F16) return launch<T16, 64, TRITT_CODE_F16>(p, j, s);
    return code == TRITT_CODE_E4M3 ? launch<T16, 64, TRITT_CODE_E4M3>(p, j, s) : launch<T16, 64, TRITT_CODE_INT8>(p, j, s);
  }
  if (code == TRITT_CODE_F16) return launch<T16, 128, TRITT_CODE_F16>(p, j, s);
  return code == TRITT_CODE_E4M3 ? launch<T16, 128, TRITT_CODE_E4M3>(p, j, s) : launch<T16, 128, TRITT_CODE_INT8>(p, j, s);
}

}  // namespace

bool sm100_tdp_decode_supported(int D, int dtype) { return (D == 64 || D == 128) && (dtype == TRITT_F16 || dtype == TRITT_BF16); }

size_t sm100_tdp_decode_workspace(const tritt_cache_t& c, int k2_window) {
  const long long rows = (long long)c.page_size * c.table_pages + c.n, window = (long long)k2_window + 1;
  const long long groups = ((rows < window ? rows : window) + 31) / 32, pairs = (c.n * groups + 7) / 8;
  return align_up((size_t)c.B * sizeof(LineEntry), 256) + align_up((size_t)((long long)c.B * c.N * pairs + num_sms()) * 8 * (c.D + 2) * 4, 256);
}

int sm100_tdp_decode(const TdpDecodeArgs& a, void* workspace, void* o, float* lse, cudaStream_t stream) {
  Params p{a, (LineEntry*)workspace, (float*)((char*)workspace + align_up((size_t)a.cache.c.B * sizeof(LineEntry), 256)), num_sms()};
  const TdpJoinParams j{a, p.table, p.part, o, lse, p.ctas};
  return a.dtype == TRITT_F16 ? by_size<__half>(p, j, stream) : by_size<__nv_bfloat16>(p, j, stream);
}

}  // namespace tritt
