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
// Codes become fp16 operands: a slab's rows, whose exponents differ, are brought to the largest one's by multiplications by powers of
// two.  K1's exponent joins the scale of the scores, for each 32 columns; V1's runs along with the
// accumulator, which is multiplied where it grows.  A is rounded once to 11 bits, P (times 2^7, fp16's lower range) once.
// Where exponents lie further apart than 2^14 to 2^24, by the codes (of 32 rows of K1, or of a piece's rows of V1), whoever attends to them, V1's rows keep their own from there to
// the piece's end, and K1's those of the 32: the soft-max warps multiply scores by K1's before they use them, and P by V1's, relative to the largest one that the row
// attends to.  (Below, the 8 tokens over 2040 with one row 2^40 larger, 20 tokens before the end: 870 us instead of 356.)
//
//   warp 1        walks the line and tells the others each piece (a pair of tiles, a range of slabs) by a ring in shared memory: what each
//                 role kept of the walk before cost it registers that it had not, and spills go to L2 beside 213 KB of shared memory
//   warp 0        issues tcgen05.mma: S_x = A_x K1^T, acc_x += P_x V1 for the tiles x = a, b in turn, P_x read from TMEM over S_x
//   warps 4-7     keys: a warp loads 32 rows of a slab (pages, exponents, codes), converts and stores them with the 128-byte swizzle;
//                 the loads of a tile are in flight before its stage is free.  They form tile b's A, and tell its rows' masks and scales
//   warps 8-11    values in the same way, and tile a's A
//   warps 12-19   one row a thread: maximum, exponentials, P; at the end of a piece the group's sum
// Measured: 8 tokens over 2040, 16 heads of 128, float16 codes 356 us (products alone would take 166, exponentials 122; 346 before it looked at how far
// exponents lie apart); one token over up to 700, 4 sequences of 8 heads of 64, e4m3 31 us.
// Stamps of an earlier form, which took 374 us for the first: a pair of tiles' slab 5.1 thousand cycles, of them 3.2 in a tile's soft-max (a
// warp a scheduler works alone for most of it) and 1.9 from its P to the next scores; the change of pieces 17 thousand a piece, the
// group's sums 8 and the rows' A 13 of them, side by side.  Of the second 10 of the first 19 thousand cycles are the way to the first A.
// Tried on forms of 344 to 374 us.  Registers: with 32 rows of 256 bytes at a time the loading warps need more than 112 (104: 407 us, 112: 374, and the soft-max
// warps at 104: 421); with 16 rows 96 do, and the soft-max warps take 120 (344 us; 88 / 136: 397).
// Keys and values from the same warps: 1.3 us a slab that nothing hid (690 us then).  A formed by the soft-max warps: 15 us a piece.  P in quarters
// with the next quarter's scores on their way: 388 us instead of 345 (more votes).  A's codes on their way before the tile is free: 387 to 400, its
// rows loaded side by side: 500 (registers of the warps that form it).  What follows a slab whose exponents lie apart inside the common code: 366.
#include "tritt_cache.cuh"
#include "tritt_sm100.cuh"
#include "tritt_sm100_tdp.cuh"

#include <atomic>

namespace tritt {
namespace {
using namespace sm100;

constexpr int kThreads = 640;
constexpr int kRegsLaunch = 96;   // a thread; the soft-max warps take what the others give up
constexpr int kRegsIssue = 32, kRegsLoad = 96, kRegsSoftmax = 120;
static_assert(kRegsIssue + 2 * kRegsLoad + 2 * kRegsSoftmax <= 5 * kRegsLaunch, "more registers than the launch has");
constexpr float kGap = 8.f;      // the accumulator is rescaled when a row's maximum grew by more than 2^8
constexpr float kLift = 7.f;     // P is formed times 2^7: at most 2^15, normal down to 2^-21 of the reference
constexpr int kMetas = 6;        // slabs whose descriptions are kept: two more than the ring's depth (one is overwritten when S of the slab
                                 // kMetas back is done, and the rows have then read that of the slab before it)
constexpr int kUnlimited = 1 << 30;
// The most of one sequence's head: groups of rows, whose numbers are 32-bit (65536 new tokens behind a million come to 2^31), and steps of the line, so that
// those of all 65535 heads times the CTAs stay below 2^63 (2^39 steps of 2 us take two hours on all SMs).
constexpr long long kMostGroups = 1ll << 30, kMostSteps = 1ll << 39;

template <int D> struct Cfg {
  static constexpr int kTile = 128 * D * 2;
  static constexpr int kStages = D == 128 ? 2 : 4;                 // of keys, and as many of values
  static constexpr int kOffA = 0;                                  // two tiles
  static constexpr int kOffK = 2 * kTile;
  static constexpr int kOffV = kOffK + kStages * kTile;
  static constexpr int kOffQ = kOffV + kStages * kTile;            // [8 warps][D] fp16
  static constexpr int kOffRows = kOffQ + 8 * D * 2;               // [256] RowInfo
  static constexpr int kOffRun = kOffRows + 256 * 32;          // [8 warps][D] fp32
  static constexpr int kOffOwn = kOffRun + 8 * D * 4;              // [256] rows' own exponents of V1
  static constexpr int kOffMisc = kOffOwn + 1024;
  static constexpr int kSmem = kOffMisc + 2816;
  static constexpr int kTmemO = 256;                               // S_a | S_b | acc_a | acc_b
};

struct __align__(16) Meta {   // of one slab, by the warp that loaded 32 of its rows
  uint32_t there[4];      // rows that have a place
  uint32_t nan[4];        // rows that read as NaN (K1 or V1)
  float scale[4];         // of the 32 columns' scores
  uint32_t span[4];       // exponent bytes of V1's rows
  uint8_t ek[128], ev[128];
};
// The largest and the least of some exponent bytes in one word, of which the larger halves of two are those of both: the largest in the upper half, 255
// less the least one (of rows of zeros: none) in the lower.  kApart: K1's rows have kept their own, which counts like V1's being too far apart.
constexpr uint32_t kApart = 4096;
__device__ __forceinline__ uint32_t span_of(int largest, int least) { return (uint32_t)largest << 16 | (uint32_t)(255 - least); }
__device__ __forceinline__ uint32_t span_with(uint32_t a, uint4 b) { return __vmaxu2(__vmaxu2(__vmaxu2(a, b.x), b.y), __vmaxu2(b.z, b.w)); }
__device__ __forceinline__ bool too_wide(uint32_t span, int spread) { return (span >> 16) + (span & 0xffffu) > 255u + spread; }

// A row of a tile, by the thread that formed its A for the one that works on its scores.
struct __align__(16) RowInfo {
  unsigned long long tree;   // of a tree's tokens, those that it attends to
  size_t v2_row;             // its V2's number in the cache
  float scale;               // of its scores
  int c_lo, c_hi;            // columns that it attends to, by their numbers
  int flags;                 // V2's exponent byte; kRowNan: it reads as NaN
};
static_assert(sizeof(RowInfo) == 32, "two 16-byte accesses");
constexpr int kRowNan = 256;

// A piece, as the roles see it.  n = 0: there is no more.
struct __align__(16) Item {
  int n, tiles, first, behind;       // slabs, tiles; columns first .. behind - 1, 128 a slab
  int b, head, g0, groups;           // groups g0 .. of the sequence's line; groups of a new token
  int all_groups, ctx;               // groups of all its new tokens
  int token[8];                      // of the soft-max warps' groups
};
constexpr int kItems = 4;
constexpr int kConsumers = 17;       // warps that read them

struct Misc {
  uint64_t k_full[4], k_empty[4], v_full[4], v_empty[4];
  uint64_t meta_full[kMetas], a_ready[2], a_free[2], s_ready[2], p_ready[2], o_done[2], item_full[kItems], item_free[kItems];
  Meta meta[kMetas];
  Item items[kItems];
  uint32_t tmem_base;
  int abort_flag;
};
static_assert(sizeof(Misc) <= 2816, "shared memory of the barriers");

// What the line of steps has of one sequence.
struct Line {
  int ctx, cnt;          // tokens before the new ones, new ones
  int groups;            // of 32 rows, of each new token
  int pairs, slabs;      // pairs of tiles of a head; slabs of a pair (the most of any)
};
struct LineEntry {       // in the workspace, for the kernel that joins
  long long base;
  Line line;
};

struct Params {
  TdpDecodeArgs a;
  LineEntry* table;      // [B]
  float* part;           // [new tokens of all heads + CTAs][8][D + 2]: each of a CTA's soft-max warps' maximum, sum and result of one new
                         // token; the CTAs that share a token, and the tokens that share a CTA, follow one another, so their sum numbers them
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
  l.slabs = (least(l.ctx, a.k1w) + l.cnt + 127) / 128;
  const long long all = (long long)l.cnt * l.groups, pairs = (all + 7) / 8;
  if (all > kMostGroups || pairs * l.slabs > kMostSteps) {   // too much: reported, and left out like a sequence without new tokens
    if (a.cache.status) atomicOr(a.cache.status, kStatusTdpDecode);
    l.cnt = l.groups = l.pairs = l.slabs = 0;
    return l;
  }
  l.pairs = (int)pairs;
  return l;
}
__device__ __forceinline__ Columns columns_of(const TdpDecodeArgs& a, const Line& l, int pair) {
  const int g0 = pair * 8, g1 = least(g0 + 8, l.cnt * l.groups);
  int i = g0 / l.groups, r = (g0 - i * l.groups) * 32;
  const int lo = most(0, l.ctx - a.k1w);
  if (a.kkl >= l.ctx + l.cnt && a.kkr >= l.ctx + l.cnt) return Columns{lo, l.ctx + (g1 - 1) / l.groups};   // (no band)
  Columns c{l.ctx, -1};
  for (int g = g0; g < g1; ++g, r += 32) {
    if (r == l.groups * 32) r = 0, ++i;
    // positions of the group's rows, whatever the token's depth in a tree (0 to i)
    const int ka = most(0, l.ctx - a.k2w) + r, kb = most(0, l.ctx + i - a.k2w) + r + 31;
    c.lo = least(c.lo, most(lo, ka - least(ka, a.kkl)));
    c.hi = most(c.hi, kb + least(a.kkr, kUnlimited - 1) < l.ctx ? kb + a.kkr : l.ctx + i);
  }
  return c;
}

// Steps of a CTA: walks the line from the CTA's first step to its last.  (Where it stands is found by division once, then by counting.)
struct Walk {
  long long left;           // steps
  int b, head, pair, slab;
  Line l;
};
struct Piece {
  int b, head, pair, s0, s1;
};
__device__ __forceinline__ Walk start_walk(const Params& p, long long total, int b, long long base) {
  long long x = (long long)blockIdx.x * total / p.ctas;
  Walk w{((long long)blockIdx.x + 1) * total / p.ctas - x, b, 0, 0, 0, {}};
  if (w.left == 0) return w;
  w.l = line_of(p.a, b);
  x -= base;
  if (x >= (long long)w.l.pairs * p.a.cache.c.N * w.l.slabs) {   // (contexts that changed under the kernel)
    w.left = 0;
    return w;
  }
  const long long pair = x / w.l.slabs;
  w.slab = (int)(x - pair * w.l.slabs);
  w.head = (int)(pair / w.l.pairs);
  w.pair = (int)(pair - (long long)w.head * w.l.pairs);
  return w;
}
__device__ __forceinline__ bool next_piece(const Params& p, Walk& w, Piece& s) {
  if (w.left <= 0) return false;
  while (w.slab == w.l.slabs) {   // the next pair, head, sequence (that has any)
    if (w.l.slabs) ++w.pair;
    w.slab = 0;
    if (w.pair < w.l.pairs) break;
    w.pair = 0;
    if (w.l.slabs && ++w.head < p.a.cache.c.N) break;
    w.head = 0;
    if (w.b + 1 >= p.a.cache.c.B) return false;
    w.l = line_of(p.a, ++w.b);
    if (w.l.slabs) break;
  }
  s.b = w.b;
  s.head = w.head;
  s.pair = w.pair;
  s.s0 = w.slab;
  s.s1 = w.l.slabs - w.slab < w.left ? w.l.slabs : w.slab + (int)w.left;
  w.left -= s.s1 - s.s0;
  w.slab = s.s1;
  return true;
}

// Two fp32 numbers an instruction.
__device__ __forceinline__ float2 fma_pair(float2 a, float b, float c) {
  float2 r;
  asm("{\n\t.reg .b64 x, y, z;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %4};\n\tmov.b64 z, {%5, %5};\n\t"
      "fma.rn.ftz.f32x2 x, x, y, z;\n\tmov.b64 {%0, %1}, x;\n\t}"
      : "=f"(r.x), "=f"(r.y)
      : "f"(a.x), "f"(a.y), "f"(b), "f"(c));
  return r;
}
__device__ __forceinline__ float2 add_pair(float2 a, float2 b) {
  float2 r;
  asm("{\n\t.reg .b64 x, y;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tadd.rn.ftz.f32x2 x, x, y;\n\tmov.b64 {%0, %1}, x;\n\t}"
      : "=f"(r.x), "=f"(r.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return r;
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

__device__ __forceinline__ uint4 load16_if(const void* p, bool on) {   // zeros where not (a predicate: a branch would keep loads from overlapping)
  uint4 v;
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %5, 0;\n\tmov.b32 %0, 0;\n\tmov.b32 %1, 0;\n\tmov.b32 %2, 0;\n\tmov.b32 %3, 0;\n\t"
      "@p ld.global.nc.v4.b32 {%0, %1, %2, %3}, [%4];\n\t}"
      : "=&r"(v.x), "=&r"(v.y), "=&r"(v.z), "=&r"(v.w)
      : "l"(p), "r"((int)on));
  return v;
}

template <int D, int CODE> struct TileLoader {   // a warp's 32 rows of one part of a slab
  static constexpr int kChunks = CODE == TRITT_CODE_F16 ? D / 8 : D / 16;   // of 16 bytes of codes, a row
  static constexpr int kRows = kChunks > 8 ? 16 : 32;                       // at a time: 32 registers
  static constexpr int kLoads = kChunks * kRows / 32;
  uint4 v[kLoads];
  // mine: the lane's own row, null: none (zeros)
  __device__ __forceinline__ void load(const uint8_t* mine, int lane, int from) {
    const uint32_t lo = (uint32_t)(size_t)mine, hi = (uint32_t)((size_t)mine >> 32);
    // rows that follow one another in a page (all 32, where a tile does not start or end in the middle of one)
    const size_t first = (size_t)__shfl_sync(0xffffffffu, hi, 0) << 32 | __shfl_sync(0xffffffffu, lo, 0);
    if (__all_sync(0xffffffffu, mine != nullptr && (size_t)mine == first + lane * (kChunks * 16))) {
#pragma unroll
      for (int it = 0; it < kLoads; ++it) v[it] = __ldg(reinterpret_cast<const uint4*>(first) + from * kChunks + it * 32 + lane);
      return;
    }
#pragma unroll
    for (int it = 0; it < kLoads; ++it) {
      const int idx = it * 32 + lane, row = from + idx / kChunks, ch = idx % kChunks;
      const uint32_t l = __shfl_sync(0xffffffffu, lo, row), h = __shfl_sync(0xffffffffu, hi, row);
      const size_t at = (size_t)h << 32 | l;
      v[it] = load16_if((const uint8_t*)at + ch * 16, at != 0);
    }
  }
  // to rows row0 .. row0 + 31 of a tile, each times the power of two of its lane
  __device__ __forceinline__ void store(uint8_t* tile, int row0, uint32_t factor, int lane, int from) {
#pragma unroll
    for (int it = 0; it < kLoads; ++it) {
      const int idx = it * 32 + lane, row = from + idx / kChunks, ch = idx % kChunks;
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

// A row's slab where rows of K1 or V1 keep their exponents, and of large scores: what the soft-max warps do otherwise, column by column in two passes.
// (Not inlined: rare, and registers are few.)  -> the row's reference, what its sum is multiplied by, what is added to it
struct SlabApart {
  uint32_t tS, tO;
  int chunks, wid, up, spread;   // of 16 columns of the accumulator; columns; kUp, kSpread
  uint32_t before, span;     // V1's exponents up to the slab before, and to this one
  bool later;                // (the accumulator holds something)
};
__device__ __noinline__ float4 slab_apart(const Meta& m, SlabApart a, uint4 mask, float scale, float m_used, int* own) {
  auto attended = [&](int c) { return (c < 64 ? c < 32 ? mask.x : mask.y : c < 96 ? mask.z : mask.w) >> (c & 31) & 1; };
  auto score = [&](uint32_t s, int c) {   // in log2 units
    const float block = m.scale[c >> 5];
    // (rounded, as the maximum was: not taken into the subtraction)
    return __fmul_rn(__uint_as_float(s), scale * (block < 0.f ? power_of_two(m.ek[c] - 127 - a.up) : block));
  };
  const bool wide = too_wide(a.span, a.spread);
  const int common = (int)(a.before >> 16);   // V1's exponent so far
  // (0: nothing attended so far.  A common exponent may be of rows that this one does not attend to: then the least that all of them have)
  const int old = !wide ? common : m_used == -INFINITY ? 0 : *own;
  int now = !wide ? (int)(a.span >> 16) : m_used == -INFINITY ? 0 : too_wide(a.before, a.spread) ? *own : most(common - a.spread, 1);
  float mx = -INFINITY;
#pragma unroll 1
  for (int c0 = 0; c0 < 128 && c0 < a.wid; c0 += 16) {
    uint32_t s[16];
    __syncwarp();
    tmem_ld16(a.tS + c0, s);
    tmem_wait_ld(s);
#pragma unroll
    for (int e = 0; e < 16; ++e)
      if (attended(c0 + e)) {
        mx = fmaxf(mx, score(s[e], c0 + e));
        if (wide && m.ev[c0 + e] != 255) now = most(now, m.ev[c0 + e]);
      }
  }
  const bool grow = mx > m_used + kGap;
  const float corr = grow ? exp2f(m_used - mx) : 1.f;
  if (grow) m_used = mx;
  *own = now;
  __syncwarp();
  if (a.later) {
    const float f = corr * power_of_two(old - now);
#pragma unroll 1
    for (int ch = 0; ch < a.chunks; ++ch) {
      uint32_t o[16];
      tmem_ld16(a.tO + ch * 16, o);
      tmem_wait_ld(o);
#pragma unroll
      for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
      tmem_st16(a.tO + ch * 16, o);
    }
  }
  const float base = m_used == -INFINITY ? 0.f : m_used;
  float sum = 0.f;
#pragma unroll 1
  for (int c0 = 0; c0 < 128 && c0 < a.wid; c0 += 32) {   // (P of 32 columns over the first half of theirs and before)
    uint32_t pk[16];
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      uint32_t s[16];
      __syncwarp();
      tmem_ld16(a.tS + c0 + half * 16, s);
      tmem_wait_ld(s);
#pragma unroll
      for (int e = 0; e < 16; e += 2) {
        float v[2];
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const int c = c0 + half * 16 + e + k;
          v[k] = attended(c) ? exp2f(score(s[e + k], c) - base + kLift) : 0.f;
          sum += v[k];
          if (wide) v[k] *= power_of_two(least(0, m.ev[c] - now));
        }
        pk[half * 8 + e / 2] = pack2<__half>(v[0], v[1]);
      }
    }
    __syncwarp();
    tmem_st16(a.tS + c0 / 2, pk);
  }
  return make_float4(m_used, corr, sum, 0.f);
}

// A warp's 32 rows of a tile: token k of new token i each.  A = 2^-kDown q * code, q brought to [1, 2); the powers of two and alpha go to
// the scores' scale.
template <typename T16, int D, int CODE>
__device__ __noinline__ void form_rows(const TdpDecodeArgs& a, const Item& s, int x, int wq, int lane, uint8_t* tile, __half* sq, RowInfo* info) {
  const CacheArgs& ca = a.cache;
  const int g = s.g0 + x * 4 + wq, ctx = s.ctx;
  const bool any = g < s.all_groups;
  const int i = any ? g / s.groups : 0;
  const T16* qp = (const T16*)a.q.p + rows_at(a.q, s.b, s.head, i);
  constexpr int E = D / 32;
  float f[E];
#pragma unroll
  for (int e = 0; e < E; ++e) f[e] = to_f(qp[lane * E + e]);
  const unsigned long long word = ca.c.ancestors ? seen_word(ca, s.b, i) : 0;
  const int pos_q = ctx + (ca.c.ancestors ? __popcll(word) - 1 : i);
  const int pk = most(0, pos_q - a.k2w) + (g - i * s.groups) * 32 + lane;
  bool on = any && pk <= pos_q;
  int token = pk;
  if (ca.c.ancestors && pk >= ctx) {
    unsigned long long left = word;
    for (int c = ctx; c < pk && left; ++c) left &= left - 1;
    token = ctx + (left ? __ffsll(left) - 1 : 0);
  }
  RowInfo r{0, 0, 0.f, kUnlimited, -1, 0};
  const uint8_t* codes = (const uint8_t*)ca.c.codes;
  int byte = 0;
  if (on) {
    const Place at = place_of(ca, s.b, token);
    if (at.page < 0) {
      on = false;
      if (ca.status) atomicOr(ca.status, kStatusPlace);
    } else {
      const size_t row = row_of(ca, at, kPartK2, s.head);
      r.v2_row = row_of(ca, at, kPartV2, s.head);
      codes += row * (size_t)(D * (CODE == TRITT_CODE_F16 ? 2 : 1));
      byte = __ldg(ca.c.exponents + row);
      const int byte2 = __ldg(ca.c.exponents + r.v2_row);
      r.flags = byte2 | (byte == 255 || byte2 == 255 ? kRowNan : 0);
      // columns that the row attends to: numbers c_lo .. c_hi, and of a tree's tokens a word
      const int last = pk < kUnlimited - a.kkr ? least(pos_q, pk + a.kkr) : pos_q;
      r.c_lo = most(most(0, pos_q - a.k1w), pk - least(pk, a.kkl));
      r.c_hi = ca.c.ancestors ? least(ctx - 1, last) : last;
      if (ca.c.ancestors) {
        unsigned long long left = word;
        for (int c = ctx; left; ++c, left &= left - 1)
          if (c >= r.c_lo && c <= last) r.tree |= left & (~left + 1);
      }
    }
  }
  uint32_t big = 0;
#pragma unroll
  for (int e = 0; e < E; ++e) big = max(big, __float_as_uint(f[e]) & 0x7fffffffu);
  big = __reduce_max_sync(0xffffffffu, big);
  const int power = max(min(254 - (int)(big >> 23), 253), 1);   // (the largest numbers are brought to [2, 4))
  const float up = __uint_as_float((uint32_t)power << 23) * (a.scale2 < 0.f ? -1.f : 1.f);
  __syncwarp();
#pragma unroll
  for (int e = 0; e < E; e += 2) *reinterpret_cast<uint32_t*>(sq + lane * E + e) = pack2<__half>(f[e] * up, f[e + 1] * up);
  __syncwarp();
  r.scale = fabsf(a.scale2) * (on && byte != 255 ? __uint_as_float((uint32_t)byte << 23) : 0.f) * (float)(1 << kDown<CODE>) *
            __uint_as_float((uint32_t)(254 - power) << 23);
  const int row = wq * 32 + lane;
  // (q as fp16 is exact, and so is a code times 2^-kDown; their product is rounded once)
  constexpr int kBytes = CODE == TRITT_CODE_F16 ? 16 : 8, kBatch = CODE == TRITT_CODE_F16 ? 4 : 8;   // of eight codes; chunks whose loads overlap
  auto form_chunk = [&](int ch, uint32_t (&h)[4]) {
    uint4 q = *reinterpret_cast<const uint4*>(sq + ch * 8);
    const uint32_t qw[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      __half2 c = *reinterpret_cast<const __half2*>(&h[e]);
      if (kDown<CODE> > 0) c = __hmul2(c, __float2half2_rn(1.f / (1 << kDown<CODE>)));
      c = __hmul2(c, *reinterpret_cast<const __half2*>(&qw[e]));
      h[e] = *reinterpret_cast<const uint32_t*>(&c);
    }
    *reinterpret_cast<uint4*>(tile + (ch >> 3) * 16384 + swz128(row, ch & 7)) = make_uint4(h[0], h[1], h[2], h[3]);
  };
#pragma unroll 1
  for (int c0 = 0; c0 < D / 8; c0 += kBatch) {
    uint4 v[kBatch * kBytes / 16];
#pragma unroll
    for (int k = 0; k < kBatch * kBytes / 16; ++k) v[k] = load16_if(codes + c0 * kBytes + k * 16, on);
#pragma unroll
    for (int k = 0; k < kBatch * kBytes / 16; ++k) {
      if constexpr (CODE == TRITT_CODE_F16) {
        uint32_t h[4] = {v[k].x, v[k].y, v[k].z, v[k].w};
        form_chunk(c0 + k, h);
      } else {
        uint32_t h[4];
        bytes_to_halves<CODE>(v[k].x, h[0], h[1]);
        bytes_to_halves<CODE>(v[k].y, h[2], h[3]);
        form_chunk(c0 + 2 * k, h);
        bytes_to_halves<CODE>(v[k].z, h[0], h[1]);
        bytes_to_halves<CODE>(v[k].w, h[2], h[3]);
        form_chunk(c0 + 2 * k + 1, h);
      }
    }
  }
  info[row] = r;
}

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
    for (int i = 0; i < kItems; ++i) {
      mbar_init(&ms.item_full[i], 1);
      mbar_init(&ms.item_free[i], kConsumers);
    }
    for (int x = 0; x < 2; ++x) {
      mbar_init(&ms.a_ready[x], 128);
      mbar_init(&ms.a_free[x], 5);   // its last products, and four warps that have read what its rows are
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
  Walk walk{};
  if (warp == 1) {
    // the whole line's length, 32 sequences at a time, and the sequence of this CTA's first step (a walk from sequence to sequence took 200
    // cycles each)
    long long total = 0, behind = 0, here = 0;   // steps; of the lane's sequence: those up to its end, its own
    auto sums = [&](int b0, bool write) {
      const int b = b0 + lane;
      Line l{};
      if (b < ca.c.B) l = line_of(a, b);
      here = (long long)l.pairs * ca.c.N * l.slabs;
      long long s = here;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const long long s2 = __shfl_up_sync(0xffffffffu, s, o);
        if (lane >= o) s += s2;
      }
      behind = total + s;
      if (write && blockIdx.x == 0 && b < ca.c.B) p.table[b] = LineEntry{behind - here, l};
      total = __shfl_sync(0xffffffffu, behind, 31);
    };
    for (int b0 = 0; b0 < ca.c.B; b0 += 32) sums(b0, true);
    const long long steps = total, x = (long long)blockIdx.x * steps / p.ctas;
    int b0 = 0;
    if (ca.c.B > 32) {
      total = 0;
      for (; b0 < ca.c.B; b0 += 32) {
        sums(b0, false);
        if (x < total) break;
      }
    }
    const uint32_t found = __ballot_sync(0xffffffffu, x < behind);
    const int at = found ? __ffs(found) - 1 : 0;
    walk = start_walk(p, found ? steps : 0, b0 + at, __shfl_sync(0xffffffffu, behind - here, at));
  }
  let_next_start();
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = ms.tmem_base;
  volatile int* abort_flag = &ms.abort_flag;
  uint8_t* const sA = smem + C::kOffA;
  RowInfo* const sRows = reinterpret_cast<RowInfo*>(smem + C::kOffRows);
  __half* const sQ = reinterpret_cast<__half*>(smem + C::kOffQ);
  // (every lane has the same; the reduction tells the compiler so, which keeps what follows from it on the uniform datapath)
  auto uniform = [](int v) -> int { return __reduce_max_sync(0xffffffffu, v); };
  // the next piece; 0: there is none, or a wait ran out.  The warp gives its place in the ring back when it has read what it needs.
  auto next_item = [&](int count) -> int {
    if (!__all_sync(0xffffffffu, mbar_wait(&ms.item_full[count % kItems], (count / kItems) & 1, abort_flag))) return 0;
    return uniform(ms.items[count % kItems].n);
  };
  auto free_item = [&](int count) {
    __syncwarp();
    if (lane == 0) mbar_arrive(&ms.item_free[count % kItems]);
  };

  if (warp < 4) {
    set_regs<kRegsLaunch, kRegsIssue>();
    if (warp == 1) {
      // ------------------------------------------------------------------ pieces
      Piece s;
      int count = 0;
      bool more = true;
      long long last = -1;   // (lanes 0 to 7: of the soft-max warp with that number) where its previous group's results are
      while (more) {
        more = next_piece(p, walk, s);
        Item it{};
        if (more) {
          const Columns col = columns_of(a, walk.l, s.pair);
          it.n = least(s.s1, (col.hi - col.lo + 128) / 128) - s.s0;
          it.g0 = s.pair * 8;
          it.groups = walk.l.groups;
          it.all_groups = walk.l.cnt * walk.l.groups;
          it.tiles = it.all_groups - it.g0 > 4 ? 2 : 1;
          it.first = col.lo + s.s0 * 128;
          it.behind = col.hi + 1;
          it.b = s.b;
          it.head = s.head;
          it.ctx = walk.l.ctx;
          const int group = it.g0 + (lane & 7), token = least(group, it.all_groups - 1) / it.groups;
#pragma unroll
          for (int k = 0; k < 8; ++k) it.token[k] = __shfl_sync(0xffffffffu, token, k);
          const long long at = ((long long)s.b * ca.c.N + s.head) * ca.c.n + token + blockIdx.x;
          if (lane < 8 && group < it.all_groups && at != last) {   // nothing seen so far
            float* out = p.part + (size_t)(at * 8 + lane) * (D + 2);
            out[0] = -INFINITY;
            out[1] = 0.f;
            last = at;
          }
          __syncwarp();
          if (it.n <= 0) continue;   // (its slabs lie behind all columns)
        }
        if (!__all_sync(0xffffffffu, mbar_wait(&ms.item_free[count % kItems], ((count / kItems) & 1) ^ 1, abort_flag))) break;
        if (lane == 0) {
          ms.items[count % kItems] = it;
          mbar_arrive(&ms.item_full[count % kItems]);
        }
        ++count;
      }
    } else if (warp == 0) {
      // ------------------------------------------------------------------ products
      // (the whole warp walks the schedule converged and one elected lane issues)
      const bool leader = elect_one();
      auto wait_all = [&](uint64_t* bar, uint32_t parity) { return __all_sync(0xffffffffu, mbar_wait(bar, parity, abort_flag)); };
      auto commit = [&](uint64_t* bar) {
        if (leader) mma_commit(bar);
      };
      constexpr uint32_t idesc_s = make_idesc_f16(128, 128, 0, false, false), idesc_pv = make_idesc_f16(128, D, 0, false, true);
      constexpr uint32_t kHi = desc_hi(1024);
      const uint32_t aLo = desc_lo(smem_u32(sA), 16), kLo = desc_lo(smem_u32(smem + C::kOffK), 16), vLo = desc_lo(smem_u32(smem + C::kOffV), 16384);
      int kst = 0, kph = 0, vst = 0, vph = 0;   // the rings' next stages
      int pieces[2] = {0, 0}, pcount[2] = {0, 0};
      bool alive = true;
      for (int count = 0; alive; ++count) {
        const int n = next_item(count);
        if (n == 0) break;
        const Item& it = ms.items[count % kItems];
        const int tiles = uniform(it.tiles), wide = uniform(it.behind - it.first);   // columns from the first slab on
        free_item(count);
        // step i: P_x V of slab i (all of its columns, or as many blocks of 16 as there are), S_x of slab i + 1 (as many of 32), for the
        // tiles in turn.  (S_x overwrites P_x: the pipe runs it behind P_x V.  One copy of the code: the instruction caches are small)
        for (int i = -1; i < n && alive; ++i)
#pragma unroll 1
          for (int x = 0; x < tiles && alive; ++x) {
            if (i < 0) {
              alive = wait_all(&ms.a_ready[x], pieces[x] & 1);
              if (!alive) break;
            } else {
              alive = wait_all(&ms.p_ready[x], pcount[x] & 1) && (x > 0 || wait_all(&ms.v_full[vst], vph));
              if (!alive) break;
              ++pcount[x];
              tc_fence_after();
              const uint32_t bLo = vLo + vst * (C::kTile >> 4), acc = tmem + C::kTmemO + x * D, pT = tmem + x * 128;
              const int w = wide - i * 128;
              if (w > 112) {
                if (leader) {
#pragma unroll
                  for (int k = 0; k < 8; ++k) mma_ts_lo(acc, pT + k * 8, bLo + k * (2048 >> 4), kHi, idesc_pv, k > 0 || i > 0);
                }
              } else {
#pragma unroll 1
                for (int k = 0; k * 16 < w; ++k)
                  if (leader) mma_ts_lo(acc, pT + k * 8, bLo + k * (2048 >> 4), kHi, idesc_pv, k > 0 || i > 0);
              }
              if (i == n - 1) commit(&ms.o_done[x]);
              if (x == tiles - 1) {
                commit(&ms.v_empty[vst]);
                if (++vst == NS) vst = 0, vph ^= 1;
              }
            }
            if (i + 1 < n) {
              if (x == 0) {
                alive = wait_all(&ms.k_full[kst], kph);
                if (!alive) break;
              }
              tc_fence_after();
              const uint32_t bLo = kLo + kst * (C::kTile >> 4), aL = aLo + x * (C::kTile >> 4), sT = tmem + x * 128;
              const int w = wide - (i + 1) * 128;
              const uint32_t idesc = w > 96 ? idesc_s : make_idesc_f16(128, (w + 31) / 32 * 32, 0, false, false);
              if (leader) {
#pragma unroll
                for (int k = 0; k < D / 16; ++k) {
                  const uint32_t kk = (k >> 2) * (16384 >> 4) + (k & 3) * 2;
                  mma_ss_lo(sT, aL + kk, bLo + kk, kHi, idesc, k > 0);
                }
              }
              commit(&ms.s_ready[x]);
              if (i + 2 >= n) commit(&ms.a_free[x]);
              if (x == tiles - 1) {
                commit(&ms.k_empty[kst]);
                if (++kst == NS) kst = 0, kph ^= 1;
              }
            }
          }
        ++pieces[0];
        pieces[1] += tiles - 1;
      }
    }
  } else if (warp < 12) {
    set_regs<kRegsLaunch, kRegsLoad>();
    // ------------------------------------------------------------------ keys and tile b's A (warps 4-7), values and tile a's A
    const bool keys = warp < 8;
    const int w = warp & 3, mine = keys ? 1 : 0;   // this warpgroup's tile
    uint64_t* const full = keys ? ms.k_full : ms.v_full;
    uint64_t* const empty = keys ? ms.k_empty : ms.v_empty;
    uint8_t* const ring = smem + (keys ? C::kOffK : C::kOffV);
    int slab = 0, st = 0, ph = 0, formed = 0;   // slabs so far, the ring's next stage, A's formed
    bool alive = true;
    for (int count = 0; alive; ++count) {
      const int n = next_item(count);
      if (n == 0) break;
      const Item& it = ms.items[count % kItems];
      const int b = uniform(it.b), head = uniform(it.head), first = uniform(it.first), behind = uniform(it.behind);
      const bool forms = mine < uniform(it.tiles);
      const size_t part_rows = (size_t)ca.c.N << ca.page_log2, head_rows = (size_t)head << ca.page_log2;
      constexpr int kRowBytes = TileLoader<D, CODE>::kChunks * 16;
      const size_t load_rows = (keys ? kPartK1 : kPartV1) * part_rows + head_rows, v_rows = kPartV1 * part_rows + head_rows;
      auto form = [&]() {
        if (!__all_sync(0xffffffffu, mbar_wait(&ms.a_free[mine], (formed & 1) ^ 1, abort_flag))) return false;
        form_rows<T16, D, CODE>(a, it, mine, w, lane, sA + mine * C::kTile, sQ + (mine * 4 + w) * D, sRows + mine * 128);
        fence_async_smem();
        mbar_arrive(&ms.a_ready[mine]);
        ++formed;
        return true;
      };
      if (!keys && forms) alive = form();
      uint32_t span = 0;   // of V1's rows in this piece so far
      int token = first + w * 32 + lane;
      auto page_of = [&](int t) { return t < behind ? place_of(ca, b, t).page : -1; };
      int page = page_of(token);
      for (int i = 0; i < n && alive; ++i, token += 128) {
        const int pos = slab + i, mt = pos % kMetas, token0 = token - lane;
        const bool any = token0 < behind;   // (32 columns that no row looks at are not loaded)
        TileLoader<D, CODE> tile;
        int ek = 0, ev = 0;
        const size_t row = (size_t)page * (4 * part_rows) + (token & (ca.c.page_size - 1));   // (but for the part and head)
        if (page >= 0) {
          if (keys) ek = __ldg(ca.c.exponents + row + load_rows);
          ev = __ldg(ca.c.exponents + row + v_rows);
        }
        const uint8_t* const codes = page >= 0 ? (const uint8_t*)ca.c.codes + (row + load_rows) * kRowBytes : nullptr;
        if (any) tile.load(codes, lane, 0);
        const int next = i + 1 < n ? page_of(token + 128) : -1;
        int up;   // the row's power of two
        if (keys) {
          const uint32_t there = __ballot_sync(0xffffffffu, page >= 0), nan = __ballot_sync(0xffffffffu, page >= 0 && (ek == 255 || ev == 255));
          if (ek == 255) ek = 0;   // (its codes are zeros)
          if (ev == 255) ev = 0;
          const int ek_most = __reduce_max_sync(0xffffffffu, ek), ev_most = __reduce_max_sync(0xffffffffu, ev);
          const int ev_least = __reduce_min_sync(0xffffffffu, least_byte(ev));
          const bool apart = __any_sync(0xffffffffu, least_byte(ek) < ek_most - kSpread<CODE>);
          alive = __all_sync(0xffffffffu, mbar_wait(&empty[st], ph ^ 1, abort_flag));
          if (!alive) break;
          Meta& m = ms.meta[mt];
          m.ek[w * 32 + lane] = (uint8_t)ek;
          m.ev[w * 32 + lane] = (uint8_t)ev;
          __syncwarp();
          if (lane == 0) {
            m.there[w] = there;
            m.nan[w] = nan;
            m.scale[w] = apart ? -1.f : ek_most > kUp<CODE> ? __uint_as_float((uint32_t)(ek_most - kUp<CODE>) << 23) : 0.f;
            m.span[w] = span_of(ev_most, ev_least) | (apart ? kApart : 0u);
            mbar_arrive(&ms.meta_full[mt]);
          }
          up = apart ? kUp<CODE> : kUp<CODE> + ek - ek_most;
        } else {
          if (ev == 255) ev = 0;
          alive = __all_sync(0xffffffffu, mbar_wait(&ms.meta_full[mt], (pos / kMetas) & 1, abort_flag)) &&
                  __all_sync(0xffffffffu, mbar_wait(&empty[st], ph ^ 1, abort_flag));
          if (!alive) break;
          const volatile Meta& m = ms.meta[mt];
          span = span_with(span, make_uint4(m.span[0], m.span[1], m.span[2], m.span[3]));
          up = too_wide(span, kSpread<CODE>) ? kUp<CODE> : kUp<CODE> + ev - (int)(span >> 16);
        }
        if (any) {
          tile.store(ring + st * C::kTile, w * 32, half_power(up), lane, 0);
          if constexpr (TileLoader<D, CODE>::kRows == 16) {
            tile.load(codes, lane, 16);
            tile.store(ring + st * C::kTile, w * 32, half_power(up), lane, 16);
          }
        }
        fence_async_smem();
        mbar_arrive(&full[st]);
        if (++st == NS) st = 0, ph ^= 1;
        page = next;
        if (keys && i == 0 && forms) alive = form();   // (the first keys are on their way before)
      }
      slab += n;
      free_item(count);
    }
  } else {
    set_regs<kRegsLaunch, kRegsSoftmax>();
    // ------------------------------------------------------------------ soft-max, one row a thread
    const int x = (warp - 12) >> 2, wq = warp & 3;
    const uint32_t lane_base = (uint32_t)(wq * 32) << 16;
    const uint32_t tS = tmem + lane_base + x * 128, tO = tmem + lane_base + C::kTmemO + x * D;
    int slab = 0, scount = 0, mine = 0;   // slabs so far; this tile's, and its pieces
    // what the warp has of a new token runs along its pieces: maximum and sum here, the result in shared memory, a column a lane
    float* const run = reinterpret_cast<float*>(smem + C::kOffRun) + (x * 4 + wq) * D + lane;
    int* const own = reinterpret_cast<int*>(smem + C::kOffOwn) + x * 128 + wq * 32 + lane;   // the exponent that this row's results count in
    long long last = -1;
    float m_run = -INFINITY, l_run = 0.f;
    bool alive = true;
    for (int count = 0; alive; ++count) {
      const int n = next_item(count);
      if (n == 0) break;
      const Item& it = ms.items[count % kItems];
      const int first = uniform(it.first), behind = uniform(it.behind), ctx = uniform(it.ctx);
      const bool used = it.g0 + x * 4 + wq < it.all_groups;   // (the warp's rows are of a new token)
      const long long at = ((long long)it.b * ca.c.N + it.head) * ca.c.n + it.token[x * 4 + wq] + blockIdx.x;
      const bool second = uniform(it.tiles) == 2;
      free_item(count);
      if (x == 1 && !second) {
        slab += n;
        continue;
      }
      alive = __all_sync(0xffffffffu, mbar_wait(&ms.a_ready[x], mine & 1, abort_flag));
      if (!alive) break;
      const RowInfo r = sRows[x * 128 + wq * 32 + lane];
      __syncwarp();
      // (without this the A of the next piece, and of the one behind it, might come while this warp is at the previous piece's sums: it would
      // find the barrier two phases on, and other rows)
      if (lane == 0) mbar_arrive(&ms.a_free[x]);
      // --- slabs: a half of 64 columns at a time is read once, its maximum taken, and the row's reference raised where that is 2^8 above it
      float m_used = -INFINITY, l_sum = 0.f;
      uint32_t span = 0;   // as the loading warps have it
      *own = 0;
      for (int t = 0; t < n; ++t, ++scount) {
        const int pos = slab + t, c0 = first + t * 128, wid = behind - c0;
        const Meta& m = ms.meta[pos % kMetas];
        if (!__all_sync(0xffffffffu, mbar_wait(&ms.meta_full[pos % kMetas], (pos / kMetas) & 1, abort_flag))) {
          alive = false;
          break;
        }
        const uint4 there = *reinterpret_cast<const uint4*>(m.there), nan = *reinterpret_cast<const uint4*>(m.nan);
        const float4 ks = *reinterpret_cast<const float4*>(m.scale);
        const uint4 spans = *reinterpret_cast<const uint4*>(m.span);
        const bool clean = wid >= 128 && (there.x & there.y & there.z & there.w) == 0xffffffffu && (nan.x | nan.y | nan.z | nan.w) == 0u;
        const bool full = __all_sync(0xffffffffu, clean && r.c_lo <= c0 && r.c_hi >= c0 + 127);
        uint32_t mask[4] = {0u, 0u, 0u, 0u};   // columns that count
        bool bad = false;                      // one of them reads as NaN
        int some = 3;                          // halves with one, of any row of the warp
        if (!full) {
          const uint32_t th[4] = {there.x, there.y, there.z, there.w}, na[4] = {nan.x, nan.y, nan.z, nan.w};
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            const int c1 = c0 + c * 32;
            const int lo = most(r.c_lo - c1, 0), hi = least(r.c_hi - c1, 31);
            uint32_t b = lo > 31 || hi < lo ? 0u : (0xffffffffu << lo) & (0xffffffffu >> (31 - hi));
            const int off = ctx - c1;   // of the first new token
            if (r.tree && off < 32 && off > -64) b |= (uint32_t)(off >= 0 ? r.tree << off : r.tree >> -off);
            mask[c] = b & th[c];
            if (mask[c] != b && ca.status) atomicOr(ca.status, kStatusPlace);
            bad = bad || (mask[c] & na[c]);
          }
          some = (__any_sync(0xffffffffu, mask[0] | mask[1]) ? 1 : 0) | (__any_sync(0xffffffffu, mask[2] | mask[3]) ? 2 : 0);
        }
        // (a scale of 0, of rows of zeros: any small one, so that masked columns' -infinity stays one)
        const float f[4] = {fmaxf(r.scale * ks.x, 1e-37f), fmaxf(r.scale * ks.y, 1e-37f), fmaxf(r.scale * ks.z, 1e-37f), fmaxf(r.scale * ks.w, 1e-37f)};
        const uint32_t before = span;
        span = span_with(span, spans);
        const bool wide = too_wide(span, kSpread<CODE>);   // rows keep their exponents, in this slab and those behind it
        const bool odd = __any_sync(0xffffffffu, wide || fmaxf(fmaxf(f[0], f[1]), fmaxf(f[2], f[3])) > kLargeFactor);
        alive = __all_sync(0xffffffffu, mbar_wait(&ms.s_ready[x], scount & 1, abort_flag));
        if (!alive) break;
        tc_fence_after();
        // the accumulator times `corr` (s_ready of this slab was committed behind the previous slab's P V)
        auto correct = [&](float corr) {
          tmem_wait_st();   // (it may be for the second or third time in this slab: what the last one wrote is read)
#pragma unroll 1
          for (int ch = 0; ch < D / 16; ++ch) {
            uint32_t o[16];
            tmem_ld16(tO + ch * 16, o);
            tmem_wait_ld();
#pragma unroll
            for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * corr);
            tmem_st16(tO + ch * 16, o);
          }
        };
        float psum = 0.f;
        if (odd) {
          const uint4 attended = full ? make_uint4(~0u, ~0u, ~0u, ~0u) : make_uint4(mask[0], mask[1], mask[2], mask[3]);
          const float4 v = slab_apart(m, SlabApart{tS, tO, D / 16, wid, kUp<CODE>, kSpread<CODE>, before, span, t > 0}, attended, r.scale, m_used, own);
          m_used = v.x;
          l_sum *= v.y;
          psum = v.z;
        } else {
          if (span >> 16 != before >> 16) {
            const int by = (int)(span >> 16) - (int)(before >> 16);
            *own = (int)(span >> 16);
            if (t > 0) correct(by < 126 ? __uint_as_float((uint32_t)(127 - by) << 23) : 0.f);
          }
#pragma unroll 1
          for (int hf = 0; hf < 2; ++hf) {   // (one copy of the code)
            const float f0 = hf ? f[2] : f[0], f1 = hf ? f[3] : f[1];
            if (some >> hf & 1) {
              uint32_t sr[64];
              tmem_ld64(tS + hf * 64, sr);
              tmem_wait_ld();
              if (!full) {
                const uint32_t m0 = hf ? mask[2] : mask[0], m1 = hf ? mask[3] : mask[1];
#pragma unroll
                for (int e = 0; e < 64; ++e) sr[e] = (e < 32 ? m0 : m1) >> (e % 32) & 1 ? sr[e] : 0xff800000u;
              }
              float mx;
              {
                float q[4];
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                  q[k] = fmaxf(__uint_as_float(sr[k * 16]), __uint_as_float(sr[k * 16 + 1]));
#pragma unroll
                  for (int e = 2; e < 16; e += 2) q[k] = fmaxf(q[k], fmaxf(__uint_as_float(sr[k * 16 + e]), __uint_as_float(sr[k * 16 + e + 1])));
                }
                mx = fmaxf(fmaxf(q[0], q[1]) * f0, fmaxf(q[2], q[3]) * f1);
              }
              const bool grow = mx > m_used + kGap;
              if (__any_sync(0xffffffffu, grow)) {
                const float corr = grow ? exp2f(m_used - mx) : 1.f;
                if (grow) {
                  m_used = mx;
                  l_sum *= corr;
                  psum *= corr;
                }
                if (t > 0) correct(corr);
                if (hf == 1) {   // (this slab's first half, formed already)
#pragma unroll 1
                  for (int q = 0; q < 2; ++q) {
                    uint32_t o[16];
                    tmem_wait_st();
                    tmem_ld16(tS + q * 16, o);
                    tmem_wait_ld();
#pragma unroll
                    for (int e = 0; e < 16; ++e) {
                      const float2 v = unpack2<__half>(o[e]);
                      o[e] = pack2<__half>(v.x * corr, v.y * corr);
                    }
                    tmem_st16(tS + q * 16, o);
                  }
                }
              }
              const float shift = kLift - (m_used == -INFINITY ? 0.f : m_used);
              float2 sum[2] = {{0.f, 0.f}, {0.f, 0.f}};
#pragma unroll
              for (int q = 0; q < 2; ++q) {
                uint32_t pk[16];
#pragma unroll
                for (int c = 0; c < 32; c += 2) {
                  const float2 z = fma_pair(make_float2(__uint_as_float(sr[q * 32 + c]), __uint_as_float(sr[q * 32 + c + 1])), q ? f1 : f0, shift);
                  const float2 e = make_float2(exp2f(z.x), exp2f(z.y));
                  sum[c >> 1 & 1] = add_pair(sum[c >> 1 & 1], e);
                  pk[c >> 1] = pack2<__half>(e.x, e.y);
                }
                tmem_st16(tS + hf * 32 + q * 16, pk);
              }
              psum += (sum[0].x + sum[0].y) + (sum[1].x + sum[1].y);
            } else if (hf * 64 < wid) {
              uint32_t pk[16];
#pragma unroll
              for (int e = 0; e < 16; ++e) pk[e] = 0u;
              tmem_st16(tS + hf * 32, pk);
              tmem_st16(tS + hf * 32 + 16, pk);
            }
          }
        }
        l_sum += bad ? __uint_as_float(0x7fffffffu) : psum;
        tmem_wait_st();
        tc_fence_before();
        mbar_arrive(&ms.p_ready[x]);
      }
      if (!alive) break;
      slab += n;
      // --- the group's sum: sum over its rows of 2^(m_row - m) acc V2, and of the sums.  V2's codes come while the last products run
      const uint8_t* codes = (const uint8_t*)ca.c.codes + r.v2_row * (size_t)(D * (CODE == TRITT_CODE_F16 ? 2 : 1));
      // (a row that is not there has number 0 and weight 0)
      constexpr int kWords = CODE == TRITT_CODE_F16 ? 4 : 2;   // 16-byte words of 32 columns' codes
      uint4 even[kWords], odd[kWords];   // two blocks ahead: a row's codes lie apart from its neighbours', and come from L2
      auto load_codes = [&](uint4 (&v)[kWords], int ch) {
#pragma unroll
        for (int k = 0; k < kWords; ++k) v[k] = __ldg(reinterpret_cast<const uint4*>(codes) + ch * kWords + k);
      };
      load_codes(even, 0);
      load_codes(odd, 1);
      if ((r.flags & kRowNan) && l_sum > 0.f) l_sum = __uint_as_float(0x7fffffffu);
      const bool more = at == last;   // (of the token that the previous piece was of)
      last = at;
      float m_all = more ? fmaxf(m_used, m_run) : m_used;
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) m_all = fmaxf(m_all, __shfl_xor_sync(0xffffffffu, m_all, o));
      const float weight = m_used == -INFINITY ? 0.f : exp2f(m_used - m_all - kLift);
      float l_all = m_used == -INFINITY ? (l_sum != l_sum ? l_sum : 0.f) : l_sum * weight;
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) l_all += __shfl_xor_sync(0xffffffffu, l_all, o);
      const float keep_run = !more || m_run == -INFINITY ? 0.f : exp2f(m_run - m_all);
      if (more) l_all += m_run == -INFINITY ? l_run : l_run * keep_run;
      m_run = m_all;
      l_run = l_all;
      float* const out = p.part + (size_t)(at * 8 + x * 4 + wq) * (D + 2);
      // V1's and V2's powers of two (fp32's range is that of the result's own type and more)
      const int byte2 = r.flags & 255;
      const float vscale =
          weight == 0.f || byte2 == 255 ? 0.f : weight * exp2f((float)(*own - 127 - kUp<CODE>)) * exp2f((float)(byte2 - 127));
      if (!__all_sync(0xffffffffu, mbar_wait(&ms.o_done[x], mine & 1, abort_flag))) {
        alive = false;
        break;
      }
      ++mine;
      tc_fence_after();
      auto fold = [&](uint4 (&c)[kWords], int ch) {
        uint32_t o[32];
        tmem_ld32(tO + ch * 32, o);
        tmem_wait_ld(o);
        float v[32];
        auto times_codes = [&](uint32_t h, int at) {
          const float2 f = unpack2<__half>(h);
          v[at] = weight == 0.f ? 0.f : f.x * vscale * __uint_as_float(o[at]);
          v[at + 1] = weight == 0.f ? 0.f : f.y * vscale * __uint_as_float(o[at + 1]);
        };
#pragma unroll
        for (int k = 0; k < kWords; ++k) {
          const uint32_t w[4] = {c[k].x, c[k].y, c[k].z, c[k].w};
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            if constexpr (CODE == TRITT_CODE_F16) {
              times_codes(w[e], k * 8 + e * 2);
            } else {
              uint32_t h0, h1;
              bytes_to_halves<CODE>(w[e], h0, h1);
              times_codes(h0, k * 16 + e * 4);
              times_codes(h1, k * 16 + e * 4 + 2);
            }
          }
        }
        if (ch + 2 < D / 32) load_codes(c, ch + 2);
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
        if (keep_run != 0.f) v[0] = fmaf(run[ch * 32], keep_run, v[0]);
        run[ch * 32] = v[0];
        if (used) out[2 + ch * 32 + lane] = v[0];
      };
#pragma unroll 1
      for (int ch = 0; ch < D / 32; ch += 2) {
        fold(even, ch);
        fold(odd, ch + 1);
      }
      if (used && lane == 0) out[0] = m_all, out[1] = l_all;
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

// CTA c has the steps from c total / ctas to the next one's.  The first step behind CTA c's, and the CTA of a step.  (Not inlined: a
// division of 64 bits is long.)
__device__ __noinline__ long long behind_cta(long long c, long long total, int ctas) {
  if (total < 1 << 20) return (uint32_t)(c + 1) * (uint32_t)total / (uint32_t)ctas;
  return (c + 1) * total / ctas;
}
__device__ __noinline__ long long cta_of(long long x, long long total, int ctas) {
  if (total < 1 << 20) return ((uint32_t)(x + 1) * (uint32_t)ctas - 1) / (uint32_t)total;
  return ((x + 1) * ctas - 1) / total;
}

// One block a row.  The results of a row are those of the warps of the CTAs that have steps of it: a thread looks at one's maximum, then the warps
// add them up in order, four loads in flight, and their sums are added in order.
template <typename T, int D>
__global__ void __launch_bounds__(256) tdp_join_kernel(const __grid_constant__ TdpJoinParams j) {
  wait_for_previous();
  constexpr int E = D / 32;
  __shared__ float s_top[8], s_sum[8], so[8][D];
  __shared__ float s_max[256];   // -infinity: none
  const CacheArgs& ca = j.a.cache;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const long long row = blockIdx.x;
  const int i = (int)(row % ca.c.n), head = (int)(row / ca.c.n % ca.c.N), b = (int)(row / ca.c.n / ca.c.N);
  const LineEntry e = j.table[b], end = j.table[ca.c.B - 1];
  const long long total = end.base + (long long)end.line.pairs * end.line.slabs * ca.c.N;
  float top = -INFINITY, sum = 0.f, acc[E];   // of this warp's results
#pragma unroll
  for (int k = 0; k < E; ++k) acc[k] = 0.f;
  if (i < e.line.cnt) {
    // the row's groups, its pairs' steps, and the CTAs of those
    const int ga = i * e.line.groups, gb = ga + e.line.groups, slabs = e.line.slabs;
    const long long base = e.base + (long long)head * e.line.pairs * slabs;   // of the head
    const long long xa = base + (long long)(ga / 8) * slabs, xb = base + (long long)((gb + 7) / 8) * slabs;
    auto pair_of = [&](long long x) {   // (a division of 64 bits is long)
      return (int)(xb - base < 1ll << 32 ? (uint32_t)(x - base) / (uint32_t)slabs : (x - base) / slabs);
    };
    const long long ca0 = cta_of(xa, total, j.ctas);
    const int count = (int)(cta_of(xb - 1, total, j.ctas) - ca0 + 1) * 8;
    const float* part = j.part + (size_t)(row + ca0) * 8 * (D + 2);
    for (int k0 = 0; k0 < count; k0 += 256) {
      const int k = k0 + tid;
      float m = -INFINITY;
      if (k < count) {
        const long long c = ca0 + k / 8, x0 = behind_cta(c - 1, total, j.ctas), x1 = behind_cta(c, total, j.ctas);
        const long long lo = x0 > xa ? x0 : xa, hi = x1 < xb ? x1 : xb;   // its steps of the row's pairs
        if (lo < hi) {
          // its groups of the row; the warp has one of them if there are eight, or a group of its number among fewer
          const int g0 = most(ga, pair_of(lo) * 8), g1 = least(gb, pair_of(hi - 1) * 8 + 8);
          if (((k - g0) & 7) < g1 - g0) m = part[(size_t)k * (D + 2)];
          // (a maximum of -infinity with a sum of NaN is of a row that reads as NaN)
          if (((k - g0) & 7) < g1 - g0 && m == -INFINITY) {
            const float l = part[(size_t)k * (D + 2) + 1];
            if (l != l) sum = l;
          }
        }
      }
      __syncthreads();
      s_max[tid] = m;
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
      if (lane == 0) s_top[warp] = m;
      __syncthreads();
      float now = top;
#pragma unroll
      for (int w = 0; w < 8; ++w) now = fmaxf(now, s_top[w]);
      const float w0 = top == -INFINITY ? 0.f : exp2f(top - now);
      if (top != -INFINITY) sum *= w0;
#pragma unroll
      for (int q = 0; q < E; ++q) acc[q] *= w0;
      top = now;
      const int here = least(count - k0, 256);
#pragma unroll 1
      for (int q0 = warp; q0 < here; q0 += 32) {
        float w[4], l[4], v[4][E];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          const int q = q0 + u * 8;
          const float mq = q < here ? s_max[q] : -INFINITY;
          w[u] = mq == -INFINITY ? 0.f : exp2f(mq - top);
          const float* p = part + (size_t)(k0 + q) * (D + 2);
          l[u] = mq == -INFINITY ? 0.f : p[1];
#pragma unroll
          for (int c = 0; c < E; ++c) v[u][c] = mq == -INFINITY ? 0.f : p[2 + c * 32 + lane];
        }
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          if (lane == 0) sum += l[u] * w[u];   // (a thread's own NaN stays in its sum)
#pragma unroll
          for (int c = 0; c < E; ++c) acc[c] += w[u] == 0.f ? 0.f : v[u][c] * w[u];
        }
      }
    }
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  if (lane == 0) s_sum[warp] = sum;
#pragma unroll
  for (int k = 0; k < E; ++k) so[warp][k * 32 + lane] = acc[k];
  __syncthreads();
  float all = 0.f;
#pragma unroll
  for (int w = 0; w < 8; ++w) all += s_sum[w];
  const bool none = top == -INFINITY && all == 0.f;
  for (int c = tid; c < D; c += 256) {
    float v = 0.f;
#pragma unroll
    for (int w = 0; w < 8; ++w) v += so[w][c];
    ((T*)j.o)[(size_t)row * D + c] = from_f<T>(none ? 0.f : all != all ? all : v * (1.f / all));
  }
  if (j.lse && tid == 0) j.lse[row] = none ? -INFINITY : all != all ? all : (top + log2f(all)) * kLn2;
}

template <typename T16, int D, int CODE>
int launch(const Params& p, const TdpJoinParams& j, cudaStream_t stream) {
  auto kern = tdp_decode_kernel<T16, D, CODE>;
  // (the registers' split is of what the kernel is launched with: setmaxnreg.inc waits without a limit for more)
  static std::atomic<int> regs{0};
  if (regs.load(std::memory_order_relaxed) == 0) {
    cudaFuncAttributes attr;
    TRITT_CUDA_OK(cudaFuncGetAttributes(&attr, kern));
    regs.store(attr.numRegs, std::memory_order_relaxed);
  }
  if (regs.load(std::memory_order_relaxed) != kRegsLaunch) {
    set_error("the kernel over the cache was built with %d registers per thread, its split needs %d", regs.load(), kRegsLaunch);
    return -30;
  }
  TRITT_CUDA_OK(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg<D>::kSmem));
  if (int rc = launch_kernel_after(kern, dim3(p.ctas), kThreads, Cfg<D>::kSmem, stream, false, p)) return rc;
  return launch_kernel_after(tdp_join_kernel<T16, D>, dim3((unsigned)((long long)p.a.cache.c.B * p.a.cache.c.N * p.a.cache.c.n)), 256, 0, stream, true, j);
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

size_t sm100_tdp_decode_workspace(const tritt_cache_t& c) {
  return align_up((size_t)c.B * sizeof(LineEntry), 256) + align_up((size_t)((long long)c.B * c.N * c.n + num_sms()) * 8 * (c.D + 2) * 4, 256);
}

int sm100_tdp_decode(const TdpDecodeArgs& a, void* workspace, void* o, float* lse, cudaStream_t stream) {
  Params p{a, (LineEntry*)workspace, (float*)((char*)workspace + align_up((size_t)a.cache.c.B * sizeof(LineEntry), 256)), num_sms()};
  const TdpJoinParams j{a, p.table, p.part, o, lse, p.ctas};
  return a.dtype == TRITT_F16 ? by_size<__half>(p, j, stream) : by_size<__nv_bfloat16>(p, j, stream);
}

}  // namespace tritt
