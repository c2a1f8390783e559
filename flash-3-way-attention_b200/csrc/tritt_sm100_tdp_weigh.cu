// The attention weight of cached tokens in the triple dot product on Blackwell tensor cores (tcgen05 + TMEM), head dimensions 64 and 128.
//
//   P[j, k] = exp(alpha sum_h q[h] K1[j, h] K2[k, h] - lse);   of each new token its row sums go to the tokens j, its column sums to the tokens k
// For one new token and a tile of 128 tokens k the operand Q[k] = q * K2[k] is formed once; tiles of 128 tokens j then stream by as S = K1 Q^T.  K1's codes are exact as fp16 numbers, Q is held in two (22 bits: of
// 16-bit queries and any codes exact), which doubles the products and costs nothing at head dimension 64, where the exponentials take twice as long as they do.  The rows' powers of two stay out of the operands: a
// score is multiplied by its column's, relative to the largest of 32 (or, where those are far apart, to one in the middle), and by its row's.  A row's sum is one thread's, over its 32 columns, and leaves after each tile; a column's is kept in registers by 128 threads, a number each, until the tokens j have all
// been, and then added up over them.  No row needs another's maximum: lse is known.
// What bounds it: exponentials, one a pair (16 a clock and SM), take 1024 clocks a tile of 128 x 128, the products 512 at D = 64 and 1024 at D = 128; a tile takes 1500 and 1700.  930 instructions a scheduler and tile
// fill 57 % of the issue slots, the rest is the way of each warp from one tile's scores to the next.  At D = 128 with fp16 codes the tiles of K1, 32 KB each, come from L2 at 4.9 TB/s.
// Measured: one token of 2 x 16 heads of 64 over 4095 and 3098 tokens, int8 codes 172 us (exponentials alone 94, products 33, both numbers of Q 65); 8 tokens over 2040, 16 heads of 128, float16 codes 224 to
// 230 us (119, 84, 165) at 1965 MHz, and 260 in a run of more than a third of a second, when the power limit (990 W) has taken the clock to 1570 MHz; one token of 4 x 8 heads over up to 700 24 us, of which the way to the first
// scores takes 7.
//
// The line of steps (tritt_weigh.cuh) is cut in equal parts, one for each CTA.
//   warp 1        walks the line and tells the others each piece (a new token, a tile of k, a range of tiles of j) by a ring in shared memory
//   warp 0        issues tcgen05.mma: eight or sixteen for a tile, K1 from tensor memory, into three buffers of scores in turn
//   warps 2, 3    fetch tiles of K1 in turn, several ahead: pages, exponents, and the codes of what lies in one page by a TMA copy
//   warps 4-7     turn a row a thread into fp16 and store it in tensor memory (with both operands in shared memory its bandwidth would be all that the products leave nothing of)
//   warps 8-11    Q for the piece after the present one, and its columns' powers of two
//   warps 12-27   four warpgroups, 32 columns each: exponentials and sums.  Four warps a scheduler: with two, of 64 columns each, registers and the way from a tile's scores to the
//                 next one's left half of the exponentials' time unused
// Before (us, the first two of these cases, ten calls each, before the power limit counts): warp-level products, all in a block of eight warps 631 / 1149; two warpgroups that sum 64 columns, K1 through registers or by copies into shared memory 220 / 298; K1
// through tensor memory by four warps that also fetched it 250 / 367; four warpgroups of 32 columns 193 / 264; fetched by two warps in turn, fewer instructions in the sums 188 / 238; one barrier for a tile's scores
// and its rows' exponents 177 / 227.  Tried: halves of 16 columns with the next half on its way 193 / 263 (registers); a polynomial on the multiply-add units for 2, 4, 8 of 16 pairs - / 236, 196 / 261, 237 / 307
// (instructions); no exponentials at all, wrong, for the time: 135 / 213.
#include "tritt_sm100.cuh"
#include "tritt_weigh.cuh"

namespace tritt {
namespace {
using namespace sm100;

constexpr int kThreads = 896;
constexpr int kRegsLaunch = 72;   // a thread; the warps that sum take what the others give up
constexpr int kRegsIssue = 40, kRegsConvert = 56, kRegsForm = 56, kRegsSum = 88;
static_assert(kRegsIssue + kRegsConvert + kRegsForm + 4 * kRegsSum <= 7 * kRegsLaunch, "more registers than the launch has");
constexpr int kMetas = 16;        // tiles whose rows are described
constexpr int kItems = 4;
constexpr int kScores = 3;        // buffers of scores

// Columns' powers of two join Q as long as the exponents of a warpgroup's 32 lie no further apart than this: Q then has its 22 bits, counted from the largest product of a row, down to fp16's smallest numbers.  Beyond,
// and where a row is not finite, scores are multiplied column by column.
template <int CODE> constexpr int kSpread = CODE == TRITT_CODE_F16 ? 13 : CODE == TRITT_CODE_E4M3 ? 9 : 8;
// q (below 4) times a code times 2^-kDown fits fp16
template <int CODE> constexpr int kDown = CODE == TRITT_CODE_F16 ? 2 : 0;

struct __align__(16) Item {       // a piece; n < 0: there is no more
  int n, s0, kg, fresh;           // tiles of j, the first; tile of k; whether the slot is to be cleared
  int b, head, i, pos;            // the new token
  int k_lo, j_lo, base, last;
  float minus;                    // lse in log2 units
  int pad[3];
};
struct __align__(16) Meta {       // of a tile of K1
  uint16_t row[128];              // exponent byte; kOff: the new token does not attend to it; kPlain: it attends to all of the tile's, and they are finite
};
constexpr int kOff = 256, kPlain = 512;
struct __align__(16) Columns {    // of a tile of Q
  float scale[128];               // (apart) of scores
  uint32_t there[4];              // of 32 columns: those that have a place and are attended to
  int middle[4];                  // the exponent byte that their powers of two are relative to
  int apart[4];                   // whether each has its own power of two
  int field;                      // q's exponent
  int pad[3];
};
template <int D, int CODE> struct Cfg {
  static constexpr int kTile = 128 * D * 2;
  static constexpr int kRow = D * (CODE == TRITT_CODE_F16 ? 2 : 1);                      // bytes of a row of codes
  static constexpr int kPitch = kRow < 128 ? kRow : 128, kBoxes = kRow / kPitch;         // as TMA leaves it: boxes of 64 or 128 bytes
  static constexpr int kRaw = 128 * kRow;                                                // a tile of codes
  static constexpr int kDepth = CODE == TRITT_CODE_F16 ? (D == 128 ? 2 : 6) : (D == 128 ? 5 : 8);   // tiles of codes on their way
  static constexpr int kOperands = 2, kOperandCols = D / 2;                                // tiles of K1 in tensor memory, behind the scores
  static constexpr int kTmemA = kScores * 128;
  static_assert(kTmemA + kOperands * kOperandCols <= 512, "tensor memory");
  // (the warps that convert say with the barrier of a tile's scores that it is described: they get there when the products of kOperands tiles back are done, and so the barrier's phase before)
  static_assert(kOperands < kScores, "arrivals in the phase of another tile");
  // Tile t is described when its codes may be fetched: those of kDepth tiles back have been converted then, so the products of kOperands further back are done, which had waited for the scores of kScores further
  // back to be read.
  static_assert(kDepth + kOperands + kScores <= kMetas, "descriptions of tiles in use");
  static constexpr int kOffQ = 0;                      // [2][hi, lo]
  static constexpr int kOffRaw = 4 * kTile;            // [kDepth]
  static constexpr int kOffMisc = kOffRaw + kDepth * kRaw;
};
struct Misc {
  uint64_t raw_full[8], raw_free[8], a_full[4], a_free[4], q_full[2], q_free[2], s_full[kScores], s_free[kScores], item_full[kItems],
      item_free[kItems];
  Item items[kItems];
  Meta meta[kMetas];
  Columns columns[2];
  float sums[4][2][4][32];        // [warpgroup][parity of the piece][warp][column]
  uint32_t tmem_base;
  int abort_flag;
};
template <int D, int CODE> constexpr int kSmem = Cfg<D, CODE>::kOffMisc + (int)sizeof(Misc);
constexpr int kConsumers = 1 + 2 + 4 + 4 + 16;   // warps that read an item

__device__ __forceinline__ int most(int x, int y) { return x > y ? x : y; }
__device__ __forceinline__ int least_of(int x, int y) { return x < y ? x : y; }

// (with numbers below fp32's normal ones: see scaled_score)
__device__ __forceinline__ float2 mul_pair(float2 a, float2 b) {
  float2 r;
  asm("{\n\t.reg .b64 x, y;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tmul.rn.f32x2 x, x, y;\n\tmov.b64 {%0, %1}, x;\n\t}"
      : "=f"(r.x), "=f"(r.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return r;
}
__device__ __forceinline__ float2 fma_pair(float2 a, float b, float c) {
  float2 r;
  asm("{\n\t.reg .b64 x, y, z;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %4};\n\tmov.b64 z, {%5, %5};\n\t"
      "fma.rn.f32x2 x, x, y, z;\n\tmov.b64 {%0, %1}, x;\n\t}"
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

// 32 rows of codes that a warp loads together: lane's chunk (16 bytes) of rows lane / kChunks, + 32 / kChunks, ...
template <int D, int CODE> struct RowChunks {
  static constexpr int kBytes = D * (CODE == TRITT_CODE_F16 ? 2 : 1), kChunks = kBytes / 16, kStep = 32 / kChunks;
  // the address of row `row`, which lane `row` has as `mine` (null: the row is not there)
  static __device__ __forceinline__ const uint8_t* row(const uint8_t* mine, int row) {
    const uint32_t lo = __shfl_sync(0xffffffffu, (uint32_t)(size_t)mine, row), hi = __shfl_sync(0xffffffffu, (uint32_t)((size_t)mine >> 32), row);
    return (const uint8_t*)((size_t)hi << 32 | lo);
  }
};
__device__ __forceinline__ uint4 load16_if(const void* p, bool on) {   // zeros where not (a predicate: a branch would keep loads from overlapping)
  uint4 v;
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %5, 0;\n\tmov.b32 %0, 0;\n\tmov.b32 %1, 0;\n\tmov.b32 %2, 0;\n\tmov.b32 %3, 0;\n\t"
      "@p ld.global.nc.v4.b32 {%0, %1, %2, %3}, [%4];\n\t}"
      : "=&r"(v.x), "=&r"(v.y), "=&r"(v.z), "=&r"(v.w)
      : "l"(p), "r"((int)on));
  return v;
}
template <typename T, int D, int CODE>
__global__ void __launch_bounds__(kThreads, 1) tdp_weigh_sm100_kernel(const __grid_constant__ TdpWeighArgs p, const __grid_constant__ CUtensorMap map) {
  using C = Cfg<D, CODE>;
  using R = RowChunks<D, CODE>;
  extern __shared__ __align__(1024) uint8_t smem[];
  Misc& ms = *reinterpret_cast<Misc*>(smem + C::kOffMisc);
  const CacheArgs& a = p.cache;
  const uint8_t* const codes = (const uint8_t*)a.c.codes;
  const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32;
  if (tid == 32) {
    ms.abort_flag = (smem_u32(smem) & 1023u) != 0;
    for (int i = 0; i < C::kDepth; ++i) {
      mbar_init(&ms.raw_full[i], 1);
      mbar_init(&ms.raw_free[i], 4);
    }
    for (int i = 0; i < C::kOperands; ++i) {
      mbar_init(&ms.a_full[i], 128);
      mbar_init(&ms.a_free[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&ms.q_full[i], 128);
      mbar_init(&ms.q_free[i], 17);   // its last products, and sixteen warps that have read its columns
    }
    for (int i = 0; i < kScores; ++i) {
      mbar_init(&ms.s_full[i], 5);   // the products, and four warps that have seen the tile's description
      mbar_init(&ms.s_free[i], 16);
    }
    for (int i = 0; i < kItems; ++i) {
      mbar_init(&ms.item_full[i], 1);
      mbar_init(&ms.item_free[i], kConsumers);
    }
    fence_barrier_init();
  }
  if (warp == 0) {
    tmem_alloc(&ms.tmem_base, 512);
    tmem_relinquish();
  }
  WeighWalk walk{};
  if (warp == 1) walk = weigh_start(p, weigh_part(p));   // (beside the others' preparations; a CTA without a part has no pieces)
  let_next_start();
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  auto uniform = [](int v) -> int { return __reduce_max_sync(0xffffffffu, v); };
  const uint32_t tmem = (uint32_t)uniform((int)ms.tmem_base);   // (every lane has the same: told so, the compiler keeps the products' addresses on the uniform datapath)
  volatile int* const abort_flag = &ms.abort_flag;
  auto wait_all = [&](uint64_t* bar, uint32_t parity) { return __all_sync(0xffffffffu, mbar_wait(bar, parity, abort_flag)); };
  // the next piece's tiles; negative: there is none, or a wait ran out.  The warp gives its place in the ring back when it has read what it needs.
  auto next_item = [&](int count) -> int {
    if (!wait_all(&ms.item_full[count % kItems], (count / kItems) & 1)) return -1;
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
      WeighPiece s;
      bool more = !*abort_flag;
      for (int count = 0; more; ++count) {
        more = weigh_next(p, walk, s);
        Item it{};
        it.n = -1;
        if (more) {
          const float lse = __ldg(p.lse + ((size_t)s.b * a.c.N + s.head) * a.c.n + s.i);
          it.n = lse == -INFINITY ? 0 : s.s1 - s.s0;
          it.s0 = s.s0;
          it.kg = s.kg;
          it.fresh = s.fresh;
          it.b = s.b;
          it.head = s.head;
          it.i = s.i;
          it.pos = s.l.ctx + s.i;
          it.k_lo = it.pos - (p.k2w < it.pos ? p.k2w : it.pos);
          it.j_lo = it.pos - (p.k1w < it.pos ? p.k1w : it.pos);
          it.base = s.l.base;
          it.last = s.l.last;
          it.minus = lse * kLog2e;
        }
        if (!wait_all(&ms.item_free[count % kItems], ((count / kItems) & 1) ^ 1)) break;
        if (lane == 0) {
          ms.items[count % kItems] = it;
          mbar_arrive(&ms.item_full[count % kItems]);
        }
      }
    } else if (warp == 0) {
      // ------------------------------------------------------------------ products
      // (the whole warp walks the schedule converged and one elected lane issues)
      const bool leader = elect_one();
      auto commit = [&](uint64_t* bar) {
        if (leader) mma_commit(bar);
      };
      constexpr uint32_t idesc = make_idesc_f16(128, 128, 0, false, false);
      constexpr uint32_t kHi = desc_hi(1024);
      const uint32_t qLo = desc_lo(smem_u32(smem + C::kOffQ), 16);
      int pieces = 0;
      uint32_t tiles = 0;
      bool alive = true;
      for (int count = 0; alive; ++count) {
        const int n = next_item(count);
        if (n < 0) break;
        free_item(count);
        if (n == 0) continue;
        const int buf = pieces & 1;
        alive = wait_all(&ms.q_full[buf], (pieces >> 1) & 1);
        for (int i = 0; i < n && alive; ++i, ++tiles) {
          const uint32_t sb = tiles % kScores, ab = tiles % C::kOperands;
          alive = wait_all(&ms.a_full[ab], (tiles / C::kOperands) & 1) && wait_all(&ms.s_free[sb], ((tiles / kScores) & 1) ^ 1);
          if (!alive) break;
          tc_fence_after();
          const uint32_t a_at = tmem + C::kTmemA + ab * C::kOperandCols, bLo = qLo + buf * (2 * C::kTile >> 4), to = tmem + sb * 128;
          if (leader) {
#pragma unroll
            for (int k = 0; k < D / 8; ++k) {
              const uint32_t s = k % (D / 16);
              mma_ts_lo(to, a_at + s * 8, bLo + (k / (D / 16)) * (C::kTile >> 4) + (s >> 2) * (16384 >> 4) + (s & 3) * 2, kHi, idesc, k > 0);
            }
          }
          commit(&ms.a_free[ab]);
          commit(&ms.s_full[sb]);
          if (i == n - 1) commit(&ms.q_free[buf]);
        }
        ++pieces;
      }
    } else {
      // ------------------------------------------------------------------ K1 on its way
      // A lane has four rows.  Of the warp's tiles pages are looked up three ahead of the copies, exponents read one ahead.
      const int r0 = lane * 4, mine = warp - 2;
      const int seg_log2 = a.page_log2 < 7 ? a.page_log2 : 7, seg = 1 << seg_log2;   // rows that lie in one page, ...
      const int lanes = seg / 4, lane0 = lane & ~(lanes - 1);                        // ... which neighbouring lanes have
      const uint32_t mask = lanes == 32 ? 0xffffffffu : (1u << lanes) - 1;
      uint32_t before = 0;   // tiles of the pieces so far
      bool alive = true;
      if (lane == 0) tma_prefetch_desc(&map);
      for (int count = 0; alive; ++count) {
        const int n = next_item(count);
        if (n < 0) break;
        const Item it = ms.items[count % kItems];
        free_item(count);
        const int f = (int)((before ^ mine) & 1), own = (n - f + 1) / 2;   // the warp's first tile of the piece, and how many it has
        const int x0 = (it.s0 + f) * 128 + r0, row_in_page = (kPartK1 * a.c.N + it.head) << a.page_log2;
        // the page of the lane's rows of the warp's i-th tile, as the table has it (not looked at here, so that nothing waits for it); -1: nobody looks at them, or the table has none
        auto attended = [&](int i) { return i < own && x0 + i * 256 + 3 >= it.j_lo && x0 + i * 256 <= it.pos; };
        auto page_of = [&](int i) {
          const int at = (x0 + i * 256) >> a.page_log2;
          int page = -1;
          if (attended(i) && at < a.c.table_pages) page = __ldg(a.c.table + it.b * a.c.table_stride + at);
          return page;
        };
        struct Four {
          int page;
          uint32_t exponents;
          bool there;
        };
        auto read = [&](int i, int page) {
          Four t{page, 0, page >= 0 && page < a.c.pages};
          if (t.there) {
            t.exponents = __ldg(reinterpret_cast<const uint32_t*>(a.c.exponents + row_of(a, Place{page, (x0 + i * 256) & (a.c.page_size - 1)}, kPartK1, it.head)));
          } else if (attended(i) && a.status) {
            atomicOr(a.status, kStatusPlace);
          }
          return t;
        };
        // (four steps a round, so that what is on its way stays in the registers that it comes to: a move would wait for it)
        int page[4] = {page_of(0), page_of(1), page_of(2), -1};
        Four four[2];
        four[0] = read(0, page[0]);
        for (int i0 = 0; i0 < own && alive; i0 += 4) {
#pragma unroll
          for (int u = 0; u < 4; ++u) {
            const int i = i0 + u;
            if (i >= own || !alive) break;
            page[(u + 3) % 4] = page_of(i + 3);
            four[(u + 1) % 2] = read(i + 1, page[(u + 1) % 4]);
            const Four& now = four[u % 2];
            const uint32_t tile = before + f + 2 * i, slot = tile % C::kDepth;
            alive = wait_all(&ms.raw_free[slot], ((tile / C::kDepth) & 1) ^ 1);
            if (!alive) break;
            const uint32_t found = __ballot_sync(0xffffffffu, now.there);
            uint32_t bytes = 128 * C::kRow;
            if (found != 0xffffffffu) {
              bytes = 0;
              for (int l = 0; l < 32; l += lanes)
                if (found >> l & mask) bytes += seg * C::kRow;
            }
            // the tile's description; who has seen the codes come has seen it
            const int x = x0 + i * 256;
            uint32_t e[4];
            bool plain = now.there && x >= it.j_lo && x + 3 <= it.pos;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              e[k] = now.exponents >> 8 * k & 255;
              plain = plain && e[k] != 255;
              if (!now.there || x + k < it.j_lo || x + k > it.pos) e[k] = kOff;
            }
            const uint32_t flag = __all_sync(0xffffffffu, plain) ? kPlain | kPlain << 16 : 0u;
            *reinterpret_cast<uint2*>(&ms.meta[tile % kMetas].row[r0]) = make_uint2(e[0] | e[1] << 16 | flag, e[2] | e[3] << 16 | flag);
            __syncwarp();
            if (lane == 0) mbar_arrive_expect_tx(&ms.raw_full[slot], bytes);
            const uint32_t of = found >> lane0 & mask;
            if (of && lane == lane0 + __ffs(of) - 1) {   // (all of the page's rows that the tile has may be read, whether somebody looks at them or not)
              const int at = r0 & ~(seg - 1);
              uint8_t* const to = smem + C::kOffRaw + slot * C::kRaw + at * C::kPitch;
#pragma unroll
              for (int c = 0; c < C::kBoxes; ++c)   // (rows are numbered within their page: the cache may have more than an int)
                tma_load_3d(to + c * 128 * C::kPitch, &map, &ms.raw_full[slot], c * 64, row_in_page + (x & (a.c.page_size - 1)) - (r0 - at), now.page);
            }
          }
        }
        before += n;
      }
      if (*abort_flag) {   // give copies still in flight a bounded chance to land before the CTA retires
        const long long t0 = clock64();
        while (clock64() - t0 < 2000000) {
        }
      }
    }
  } else if (warp < 8) {
    set_regs<kRegsLaunch, kRegsConvert>();
    // ------------------------------------------------------------------ codes to fp16 in tensor memory: a row a thread
    const int row = tid - 128;
    const uint32_t t_lane = (uint32_t)(warp & 3) << 21;
    uint32_t tiles = 0;
    bool alive = true;
    for (int count = 0; alive; ++count) {
      const int n = next_item(count);
      if (n < 0) break;
      free_item(count);
      for (int i = 0; i < n && alive; ++i, ++tiles) {
        const uint32_t ab = tiles % C::kOperands, slot = tiles % C::kDepth, sb = tiles % kScores;
        alive = wait_all(&ms.raw_full[slot], (tiles / C::kDepth) & 1) && wait_all(&ms.a_free[ab], ((tiles / C::kOperands) & 1) ^ 1);
        if (!alive) break;
        tc_fence_after();
        const uint8_t* const from = smem + C::kOffRaw + slot * C::kRaw;
        const uint32_t to = tmem + C::kTmemA + ab * C::kOperandCols + t_lane;
        auto chunk = [&](int c) {   // 16 bytes of the thread's row
          const uint32_t off = (c * 16 / C::kPitch) * (128 * C::kPitch) + row * C::kPitch + c * 16 % C::kPitch;
          return *reinterpret_cast<const uint4*>(from + (off ^ (off >> 7 & (C::kPitch / 16 - 1)) << 4));   // (swizzled)
        };
        constexpr int kParts = D / 32;   // of 32 elements, 16 columns of tensor memory
#pragma unroll
        for (int h = 0; h < kParts; ++h) {
          uint32_t v[16];
          constexpr int kEach = C::kRow / kParts / 16;
#pragma unroll
          for (int c = 0; c < kEach; ++c) {
            const uint4 x = chunk(h * kEach + c);
            if constexpr (CODE == TRITT_CODE_F16) {
              v[4 * c] = x.x, v[4 * c + 1] = x.y, v[4 * c + 2] = x.z, v[4 * c + 3] = x.w;
            } else {
              bytes_to_halves<CODE>(x.x, v[8 * c], v[8 * c + 1]);
              bytes_to_halves<CODE>(x.y, v[8 * c + 2], v[8 * c + 3]);
              bytes_to_halves<CODE>(x.z, v[8 * c + 4], v[8 * c + 5]);
              bytes_to_halves<CODE>(x.w, v[8 * c + 6], v[8 * c + 7]);
            }
          }
          tmem_st16(to + h * 16, v);
        }
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(&ms.raw_free[slot]);
          mbar_arrive(&ms.s_full[sb]);
        }
        tmem_wait_st();
        tc_fence_before();
        mbar_arrive(&ms.a_full[ab]);
      }
    }
  } else if (warp < 12) {
    set_regs<kRegsLaunch, kRegsForm>();
    // ------------------------------------------------------------------ Q
    const int w = warp & 3, chunk = lane % R::kChunks, row0 = lane / R::kChunks;
    constexpr int kEach = CODE == TRITT_CODE_F16 ? 8 : 16, kAtOnce = 4;   // elements of a chunk; chunks on their way together
    int pieces = 0;
    bool alive = true;
    for (int count = 0; alive; ++count) {
      const int n = next_item(count);
      if (n < 0) break;
      const Item it = ms.items[count % kItems];
      free_item(count);
      if (n == 0) continue;
      const int buf = pieces & 1, k = it.kg * 128 + w * 32 + lane;
      // q: its largest element's exponent, and the elements of the lane's chunk
      const T* const q_row = (const T*)p.q.p + rows_at(p.q, it.b, it.head, it.i);
      float q[kEach];
#pragma unroll
      for (int e = 0; e < kEach; e += 4) {
        const float4 f = load4(q_row + chunk * kEach + e);
        q[e] = f.x, q[e + 1] = f.y, q[e + 2] = f.z, q[e + 3] = f.w;
      }
      Place at{-1, 0};
      if (k >= it.k_lo && k <= it.pos) {
        at = place_of(a, it.b, k);
        if (at.page < 0 && a.status) atomicOr(a.status, kStatusPlace);
      }
      const uint8_t* mine = nullptr;
      int byte = 0;
      if (at.page >= 0) {
        const size_t r = row_of(a, at, kPartK2, it.head);
        mine = codes + r * R::kBytes;
        byte = __ldg(a.c.exponents + r);
      }
      uint32_t top = 0;
#pragma unroll
      for (int e = 0; e < kEach; ++e) top = max(top, __float_as_uint(q[e]) & 0x7fffffffu);
      const int field = (int)(__reduce_max_sync(0xffffffffu, top) >> 23);
      const float up = to_operand(field) * (1.f / (1 << kDown<CODE>));
#pragma unroll
      for (int e = 0; e < kEach; ++e) q[e] = field == 255 ? 0.f : q[e] * up;
      const uint32_t there = __ballot_sync(0xffffffffu, mine != nullptr);
      alive = wait_all(&ms.q_free[buf], ((pieces >> 1) & 1) ^ 1);
      if (!alive) break;
      // byte 1 is that of rows of zeros, which do not count, and of all that are too small for a lower one: their codes may be as large as any
      if (__any_sync(0xffffffffu, byte == 1)) {
        uint32_t bits = byte == 1 ? 0u : 1u;
        if (byte == 1)
#pragma unroll 1
          for (int c = 0; c < R::kChunks; ++c) {
            const uint4 x = __ldg(reinterpret_cast<const uint4*>(mine) + c);
            bits |= x.x | x.y | x.z | x.w;
          }
        if (bits == 0) byte = 0;
      }
      const int largest = uniform(byte == 255 ? 0 : byte), least = -uniform(byte == 0 ? -255 : -byte);   // (of rows that are finite; least: 255 if all are zeros)
      const bool apart = __any_sync(0xffffffffu, byte == 255) || (least < 255 && largest - least > kSpread<CODE>);
      const int middle = apart ? middle_byte<CODE>(largest) : largest;
      const float own_scale = byte == 0 ? 0.f : byte == 255 ? __uint_as_float(0x7fffffffu) : relative_power(byte - middle);
      Columns& col = ms.columns[buf];
      col.scale[w * 32 + lane] = own_scale;
      if (lane == 0) {
        col.there[w] = there;
        col.middle[w] = middle;
        col.apart[w] = apart;
        col.field = field;   // (all four warps the same)
      }
      uint8_t* const hi_tile = smem + C::kOffQ + buf * 2 * C::kTile;
      uint8_t* const lo_tile = hi_tile + C::kTile;
      auto put = [&](int row, int at16, const uint32_t (&h)[4], int e0, float by) {   // eight elements, 16 bytes of either number
        uint32_t hi[4], lo[4];
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h[x]));
          const float va = q[e0 + 2 * x] * f.x * by, vb = q[e0 + 2 * x + 1] * f.y * by;
          hi[x] = pack_halves(va, vb);
          lo[x] = pack_rests(va, vb, hi[x]);
        }
        const uint32_t off = (at16 >> 3) * 16384 + swz128(row, at16 & 7);
        *reinterpret_cast<uint4*>(hi_tile + off) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
        *reinterpret_cast<uint4*>(lo_tile + off) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
      };
#pragma unroll 1
      for (int k0 = 0; k0 < R::kChunks; k0 += kAtOnce) {
        uint4 v[kAtOnce];
#pragma unroll
        for (int x = 0; x < kAtOnce; ++x) {
          const uint8_t* from = R::row(mine, row0 + (k0 + x) * R::kStep);
          v[x] = load16_if(from + chunk * 16, from != nullptr);
        }
#pragma unroll
        for (int x = 0; x < kAtOnce; ++x) {
          const int row = w * 32 + row0 + (k0 + x) * R::kStep;
          const float by = __shfl_sync(0xffffffffu, apart ? 1.f : own_scale, row0 + (k0 + x) * R::kStep);
          if constexpr (CODE == TRITT_CODE_F16) {
            const uint32_t h[4] = {v[x].x, v[x].y, v[x].z, v[x].w};
            put(row, chunk, h, 0, by);
          } else {
            uint32_t h[4];
            bytes_to_halves<CODE>(v[x].x, h[0], h[1]);
            bytes_to_halves<CODE>(v[x].y, h[2], h[3]);
            put(row, 2 * chunk, h, 0, by);
            bytes_to_halves<CODE>(v[x].z, h[0], h[1]);
            bytes_to_halves<CODE>(v[x].w, h[2], h[3]);
            put(row, 2 * chunk + 1, h, kEach / 2, by);
          }
        }
      }
      fence_async_smem();
      mbar_arrive(&ms.q_full[buf]);
      ++pieces;
    }
  } else {
    set_regs<kRegsLaunch, kRegsSum>();
    // ------------------------------------------------------------------ sums: a row a thread, 32 columns
    const int wg = (warp - 12) / 4, wq = warp & 3, row = wq * 32 + lane;
    const uint32_t t_col = tmem + wg * 32 + ((uint32_t)(wq * 32) << 16);
    int pieces = 0, sb = 0, sph = 0, mt = 0;   // the next buffer of scores, the next description
    bool alive = true;
    for (int count = 0; alive; ++count) {
      const int n = next_item(count);
      if (n < 0) break;
      const Item& it = ms.items[count % kItems];
      const int pos = it.pos, base = it.base, last = it.last, s0 = it.s0, k0 = it.kg * 128 + wg * 32, k_lo = it.k_lo;
      const float minus = -it.minus;
      float* const slot = weigh_slot(p, it.b, it.head);
      float* const row_sums = slot + (size_t)wg * p.span;   // (each thread's own rows, here and where they are cleared)
      float* const col_sums = slot + (size_t)4 * p.span;
      if (it.fresh) {
        for (int x = row; x <= last - base; x += 128) row_sums[x] = 0.f;
        if (row < 32)
          for (int x = wg * 32 + row; x <= last - base; x += 128) col_sums[x] = 0.f;
      }
      free_item(count);
      if (n == 0) continue;
      const int buf = pieces & 1;
      alive = wait_all(&ms.q_full[buf], (pieces >> 1) & 1);
      if (!alive) break;
      const Columns& col = ms.columns[buf];
      const uint32_t there = col.there[wg];
      const int field = col.field;
      const bool apart = col.apart[wg];
      // what a row's scores are multiplied by: its power of two with that of the columns, q and Q (beyond fp32's range scores have no use for), and the scale
      const int power = col.middle[wg] + field - 382 + 127 + kDown<CODE>;
      const float scale = field == 255 ? __uint_as_float(0x7fffffffu) : field == 0 ? 0.f : p.scale2;
      // whether the rows of a plain tile have pairs with all of the 32 columns
      const bool plain = there == 0xffffffffu && !apart && field != 255 && k0 >= k_lo && k0 + 31 <= pos && p.kkl >= pos && p.kkr >= pos;
      float2 column[16];
#pragma unroll
      for (int c = 0; c < 16; ++c) column[c] = make_float2(0.f, 0.f);
      float* to = row_sums + (s0 * 128 + row - base);   // (a slot has room for all of a tile's rows)
      for (int i = 0; i < n; ++i, to += 128) {
        alive = wait_all(&ms.s_full[sb], sph);
        if (!alive) break;
        tc_fence_after();
        uint32_t s[32];
        tmem_ld32(t_col + sb * 128, s);
        const int e = ms.meta[mt].row[row];   // (the thread's row, beside the load)
        float factor = scale * __uint_as_float((uint32_t)least_of(most((e & 255) + power, 1), 254) << 23);
        tmem_wait_ld(s);
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&ms.s_free[sb]);
        float2 x[16];
#pragma unroll
        for (int c = 0; c < 16; ++c) x[c] = make_float2(__uint_as_float(s[2 * c]), __uint_as_float(s[2 * c + 1]));
        if (plain && (e & kPlain)) {   // (all of the warp's rows alike)
#pragma unroll
          for (int c = 0; c < 16; ++c) x[c] = fma_pair(x[c], factor, minus);
        } else {   // scores of pairs that there are not become minus infinity; where columns' exponents are apart, each has its own factor
          const int j = (s0 + i) * 128 + row;
          const int c_lo = most(k_lo, j - p.kkr) - k0, c_hi = !(e & kOff) ? (p.kkl < pos - j ? j + p.kkl : pos) - k0 : -1;   // columns that the row has pairs with
          uint32_t seen = there;
          if (c_lo > 0) seen &= c_lo > 31 ? 0u : 0xffffffffu << c_lo;
          if (c_hi < 31) seen &= c_hi < 0 ? 0u : 0xffffffffu >> (31 - c_hi);
          if ((e & 255) == 255) factor = __uint_as_float(0x7fffffffu);
          if (apart) {
            const float2* by = reinterpret_cast<const float2*>(col.scale + wg * 32);
#pragma unroll
            for (int c = 0; c < 16; ++c) x[c] = mul_pair(x[c], by[c]);
          }
#pragma unroll
          for (int c = 0; c < 16; ++c) {
            x[c] = fma_pair(x[c], factor, minus);
            x[c].x = seen >> (2 * c) & 1 ? x[c].x : -INFINITY;
            x[c].y = seen >> (2 * c + 1) & 1 ? x[c].y : -INFINITY;
          }
        }
        float2 sum[2];
#pragma unroll
        for (int c = 0; c < 16; ++c) {
          x[c].x = exp2f(x[c].x), x[c].y = exp2f(x[c].y);
          sum[c % 2] = c < 2 ? x[c] : add_pair(sum[c % 2], x[c]);
          column[c] = add_pair(column[c], x[c]);
        }
        const float2 both = add_pair(sum[0], sum[1]);
        // (no thread but this one adds to the place, in order)
        asm volatile("red.relaxed.gpu.global.add.f32 [%0], %1;" ::"l"(to), "f"(both.x + both.y) : "memory");
        if (++sb == kScores) sb = 0, sph ^= 1;
        mt = (mt + 1) % kMetas;
      }
      if (!alive) break;
      __syncwarp();
      if (lane == 0) mbar_arrive(&ms.q_free[buf]);
      // the columns' sums over the rows: halves change hands within the warp until a lane has one column; then over the four warps
      float* v = reinterpret_cast<float*>(column);
#pragma unroll
      for (int h = 16; h > 0; h >>= 1) {
        const bool upper = lane & h;
#pragma unroll
        for (int x = 0; x < h; ++x) {
          const float give = upper ? v[x] : v[x + h], keep = upper ? v[x + h] : v[x];
          v[x] = keep + __shfl_xor_sync(0xffffffffu, give, h);
        }
      }
      float(&sums)[4][32] = ms.sums[wg][buf];
      sums[wq][lane] = v[0];
      named_bar_sync(1 + wg, 128);   // (the other parity's numbers have been read by then)
      if (__any_sync(0xffffffffu, *abort_flag)) break;
      if (row < 32 && k0 + row <= last) col_sums[k0 + row - base] += (sums[0][row] + sums[1][row]) + (sums[2][row] + sums[3][row]);
      ++pieces;
    }
    // The warpgroup's barrier has no limit of its own.  A warp whose wait ran out arrives, once, at the one that it leaves out, after the flag is set; the others see the flag behind that barrier, leave, and arrive at the next in
    // the same way, which nobody waits at without having seen it.
    if (__any_sync(0xffffffffu, *abort_flag)) named_bar_arrive(1 + wg, 128);
  }

  // ------------------------------------------------------------------ teardown
  tc_fence_before();
  __syncthreads();
  if (warp == 0) tmem_dealloc(tmem, 512);
  if (tid == 0 && ms.abort_flag && a.status) atomicOr(a.status, kStatusTdpDecode);
}

template <typename T, int D, int CODE> int launch(const TdpWeighArgs& p, cudaStream_t stream) {
  using C = Cfg<D, CODE>;
  const tritt_cache_t& c = p.cache.c;
  // all pages of the cache, boxes of what one has of 128 rows
  if (4LL * c.N * c.page_size >= 1LL << 31) {
    set_error("pages of %d heads and %d tokens have too many rows for one call", c.N, c.page_size);
    return -11;
  }
  CUtensorMap map{};
  if (int rc = make_tmap_codes(&map, c.codes, C::kRow, (uint64_t)4 * c.N * c.page_size, c.pages, C::kPitch, c.page_size < 128 ? c.page_size : 128)) return rc;
  // (warpgroups share out the registers that the kernel is launched with: with fewer those that raise their count would wait for good)
  cudaFuncAttributes attr;
  TRITT_CUDA_OK(cudaFuncGetAttributes(&attr, tdp_weigh_sm100_kernel<T, D, CODE>));
  if (attr.numRegs != kRegsLaunch) {
    set_error("the weights' kernel was built for %d registers a thread instead of %d", attr.numRegs, kRegsLaunch);
    return -30;
  }
  TRITT_CUDA_OK(cudaFuncSetAttribute(tdp_weigh_sm100_kernel<T, D, CODE>, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem<D, CODE>));
  tdp_weigh_sm100_kernel<T, D, CODE><<<p.ctas, kThreads, kSmem<D, CODE>, stream>>>(p, map);
  count_launch();
  TRITT_CUDA_OK(cudaGetLastError());
  return 0;
}
template <typename T, int CODE> int by_size(const TdpWeighArgs& p, cudaStream_t stream) {
  return p.cache.c.D == 64 ? launch<T, 64, CODE>(p, stream) : launch<T, 128, CODE>(p, stream);
}
template <typename T> int by_code(const TdpWeighArgs& p, cudaStream_t stream) {
  switch (p.cache.c.code) {
    case TRITT_CODE_F16: return by_size<T, TRITT_CODE_F16>(p, stream);
    case TRITT_CODE_E4M3: return by_size<T, TRITT_CODE_E4M3>(p, stream);
    default: return by_size<T, TRITT_CODE_INT8>(p, stream);
  }
}

}  // namespace

bool sm100_tdp_weigh_supported(int D) { return D == 64 || D == 128; }

int sm100_tdp_weigh(const TdpWeighArgs& p, cudaStream_t stream) {
  if (p.dtype == TRITT_F32) return by_code<float>(p, stream);
  return p.dtype == TRITT_F16 ? by_code<__half>(p, stream) : by_code<__nv_bfloat16>(p, stream);
}

}  // namespace tritt
