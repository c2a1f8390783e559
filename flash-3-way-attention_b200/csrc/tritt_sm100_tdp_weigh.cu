// The attention weight of cached tokens in the triple dot product on Blackwell tensor cores (tcgen05 + TMEM), head dimensions 64 and 128.
//
//   P[j, k] = exp(alpha sum_h q[h] K1[j, h] K2[k, h] - lse);   of each new token its row sums go to the tokens j, its column sums to the tokens k
// For one new token and a tile of 128 tokens k the operand Q[k] = q * K2[k] is formed once; tiles of 128 tokens j then stream by as S = K1 Q^T.  K1's codes are exact as fp16 numbers, Q is held in two (22 bits: of
// 16-bit queries and any codes exact), which doubles the products and costs nothing at head dimension 64, where the exponentials take twice as long as they do.  The rows' powers of two stay out of the operands: a
// score is multiplied by its column's, relative to the largest of 32, and by its row's.  A row's sum is one thread's, over its 64 columns, and leaves after each tile; a column's is kept in registers by 128 threads, a number each, until the tokens j have all
// been, and then added up over them.  No row needs another's maximum: lse is known.
// Bound by the exponentials, one a pair (16 a clock and SM), at D = 128 by the products as well (128 x 128 x 16 takes 64 clocks).
//
// The line of steps (tritt_weigh.cuh) is cut in equal parts, one for each CTA.
//   warp 1        walks the line and tells the others each piece (a new token, a tile of k, a range of tiles of j) by a ring in shared memory
//   warp 0        issues tcgen05.mma: eight or sixteen for a tile, into four buffers of scores in tensor memory in turn
//   warps 4-7     tiles of K1: 8-bit codes through registers, the next tile's on their way while one is converted; fp16 codes by asynchronous copies
//   warps 8-11    Q for the piece after the present one, and its columns' powers of two
//   warps 12-19   two warpgroups, 64 columns each: exponentials and sums
#include "tritt_sm100.cuh"
#include "tritt_weigh.cuh"

namespace tritt {
namespace {
using namespace sm100;

constexpr int kThreads = 640;
constexpr int kRegsLaunch = 96;   // a thread; the warps that sum take what the others give up
constexpr int kRegsIssue = 40, kRegsLoad = 80, kRegsForm = 88, kRegsSum = 136;
static_assert(kRegsIssue + kRegsLoad + kRegsForm + 2 * kRegsSum <= 5 * kRegsLaunch, "more registers than the launch has");
constexpr int kMetas = 8;         // tiles whose rows are described: a stage is written when the products of the tile `stages` back are done, which had waited for the sums of the one four further back
constexpr int kItems = 4, kConsumers = 17;
constexpr int kScores = 4;        // buffers of scores

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
  uint8_t exponent[128];
  uint32_t there[4];
};
struct __align__(16) Columns {    // of a tile of Q
  float scale[128];
  uint32_t there[4];
  int largest[4], field, pad[3];  // exponent bytes that 32 columns' are relative to; q's
};
struct Misc {
  uint64_t k_full[4], k_empty[4], meta_full[kMetas], q_full[2], q_free[2], s_full[kScores], s_free[kScores], item_full[kItems], item_free[kItems];
  Item items[kItems];
  Meta meta[kMetas];
  Columns columns[2];
  float sums[2][2][4][64];        // [warpgroup][parity of the piece][warp][column]
  long long scan[33], at[2];
  uint32_t tmem_base;
  int abort_flag;
};
template <int D> struct Cfg {
  static constexpr int kTile = 128 * D * 2;
  static constexpr int kStages = D == 128 ? 2 : 4;
  static_assert(kStages + kScores <= kMetas, "descriptions of tiles in use");
  static constexpr int kOffQ = 0;                      // [2][hi, lo]
  static constexpr int kOffK = 4 * kTile;
  static constexpr int kOffMisc = kOffK + kStages * kTile;
  static constexpr int kSmem = kOffMisc + (int)sizeof(Misc);
  static_assert(kSmem <= 227 * 1024, "shared memory");
};

__device__ __forceinline__ float2 mul_pair(float2 a, float2 b) {
  float2 r;
  asm("{\n\t.reg .b64 x, y;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tmul.rn.ftz.f32x2 x, x, y;\n\tmov.b64 {%0, %1}, x;\n\t}"
      : "=f"(r.x), "=f"(r.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return r;
}
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
// 16 bytes to shared memory, zeros where not (src is then any address that can be read)
__device__ __forceinline__ void copy16_if(void* dst, const void* src, bool on) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(dst)), "l"(src), "r"(on ? 16 : 0) : "memory");
}

template <typename T, int D, int CODE>
__global__ void __launch_bounds__(kThreads, 1) tdp_weigh_sm100_kernel(const __grid_constant__ TdpWeighArgs p) {
  using C = Cfg<D>;
  using R = RowChunks<D, CODE>;
  constexpr int NS = C::kStages;
  extern __shared__ __align__(1024) uint8_t smem[];
  Misc& ms = *reinterpret_cast<Misc*>(smem + C::kOffMisc);
  const CacheArgs& a = p.cache;
  const uint8_t* const codes = (const uint8_t*)a.c.codes;
  const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32;
  const long long total = all_steps(p, ms.scan);
  if ((int)blockIdx.x >= weigh_parts(p, total)) return;
  find_sequence(p, (long long)blockIdx.x * total / weigh_parts(p, total), ms.scan, ms.at);
  if (tid == 32) {
    ms.abort_flag = (smem_u32(smem) & 1023u) != 0;
    for (int i = 0; i < NS; ++i) {
      mbar_init(&ms.k_full[i], 128);
      mbar_init(&ms.k_empty[i], 1);
    }
    for (int i = 0; i < kMetas; ++i) mbar_init(&ms.meta_full[i], 4);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&ms.q_full[i], 128);
      mbar_init(&ms.q_free[i], 9);   // its last products, and eight warps that have read its columns
    }
    for (int i = 0; i < kScores; ++i) {
      mbar_init(&ms.s_full[i], 1);
      mbar_init(&ms.s_free[i], 8);
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
  let_next_start();
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = ms.tmem_base;
  volatile int* const abort_flag = &ms.abort_flag;
  auto wait_all = [&](uint64_t* bar, uint32_t parity) { return __all_sync(0xffffffffu, mbar_wait(bar, parity, abort_flag)); };
  auto uniform = [](int v) -> int { return __reduce_max_sync(0xffffffffu, v); };
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
      WeighWalk walk = weigh_start(p, total, (int)ms.at[0], ms.at[1]);
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
      const uint32_t qLo = desc_lo(smem_u32(smem + C::kOffQ), 16), kLo = desc_lo(smem_u32(smem + C::kOffK), 16);
      int kst = 0, kph = 0, pieces = 0;
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
          const uint32_t sb = tiles % kScores;
          alive = wait_all(&ms.k_full[kst], kph) && wait_all(&ms.s_free[sb], ((tiles / kScores) & 1) ^ 1);
          if (!alive) break;
          tc_fence_after();
          const uint32_t aLo = kLo + kst * (C::kTile >> 4), bLo = qLo + buf * (2 * C::kTile >> 4), to = tmem + sb * 128;
          if (leader) {
#pragma unroll
            for (int k = 0; k < D / 8; ++k) {
              const uint32_t s = k % (D / 16), kk = (s >> 2) * (16384 >> 4) + (s & 3) * 2;
              mma_ss_lo(to, aLo + kk, bLo + (k / (D / 16)) * (C::kTile >> 4) + kk, kHi, idesc, k > 0);
            }
          }
          commit(&ms.k_empty[kst]);
          commit(&ms.s_full[sb]);
          if (i == n - 1) commit(&ms.q_free[buf]);
          if (++kst == NS) kst = 0, kph ^= 1;
        }
        ++pieces;
      }
    }
  } else if (warp < 8) {
    set_regs<kRegsLaunch, kRegsLoad>();
    // ------------------------------------------------------------------ tiles of K1
    const int w = warp & 3;
    uint8_t* const ring = smem + C::kOffK;
    const int chunk = lane % R::kChunks, row0 = lane / R::kChunks;
    int st = 0, ph = 0;
    uint32_t tiles = 0;
    bool alive = true;
    // a lane's own row of a tile: its address (null: not there, or nobody looks at it), its exponent, and where it is described
    const uint8_t* mine = nullptr;
    int exponent = 0;
    auto find = [&](const Item& it, int x) {
      Place at{-1, 0};
      if (x >= it.j_lo && x <= it.pos) {
        at = place_of(a, it.b, x);
        if (at.page < 0 && a.status) atomicOr(a.status, kStatusPlace);
      }
      mine = nullptr;
      exponent = 0;
      if (at.page >= 0) {
        const size_t r = row_of(a, at, kPartK1, it.head);
        mine = codes + r * R::kBytes;
        exponent = __ldg(a.c.exponents + r);
      }
    };
    auto describe = [&](bool there, int e) {
      Meta& m = ms.meta[tiles % kMetas];
      m.exponent[w * 32 + lane] = (uint8_t)e;
      const uint32_t word = __ballot_sync(0xffffffffu, there);
      if (lane == 0) m.there[w] = word;
      __syncwarp();
      if (lane == 0) mbar_arrive(&ms.meta_full[tiles % kMetas]);
    };
    if constexpr (CODE == TRITT_CODE_F16) {
      // the codes are the operand: copied as they are, a tile behind the one that is waited for
      bool waiting = false;
      auto finish = [&](int stage, bool last) {   // the tile of that stage has come
        if (last)
          asm volatile("cp.async.wait_group 0;" ::: "memory");
        else
          asm volatile("cp.async.wait_group 1;" ::: "memory");
        fence_async_smem();
        mbar_arrive(&ms.k_full[stage]);
      };
      for (int count = 0; alive; ++count) {
        const int n = next_item(count);
        if (n < 0) break;
        const Item it = ms.items[count % kItems];
        free_item(count);
        for (int i = 0; i < n && alive; ++i, ++tiles) {
          find(it, (it.s0 + i) * 128 + w * 32 + lane);
          if (waiting && NS == 2 && !__all_sync(0xffffffffu, mbar_test(&ms.k_empty[st], ph ^ 1))) {   // (with two stages the one to be filled may wait for the one on its way)
            finish(st ? st - 1 : NS - 1, true);
            waiting = false;
          }
          alive = wait_all(&ms.k_empty[st], ph ^ 1);
          if (!alive) break;
          uint8_t* const tile = ring + st * C::kTile;
#pragma unroll
          for (int k = 0; k < R::kChunks; ++k) {
            const int row = row0 + k * R::kStep;
            const uint8_t* from = R::row(mine, row);
            copy16_if(tile + (chunk >> 3) * 16384 + swz128(w * 32 + row, chunk & 7), from ? from + chunk * 16 : codes, from != nullptr);
          }
          asm volatile("cp.async.commit_group;" ::: "memory");
          describe(mine != nullptr, exponent);
          if (waiting) finish(st ? st - 1 : NS - 1, false);
          waiting = true;
          if (++st == NS) st = 0, ph ^= 1;
        }
        // (a piece's last tile is not left waiting for the next piece)
        if (waiting && alive) finish(st ? st - 1 : NS - 1, true);
        waiting = false;
      }
      asm volatile("cp.async.wait_group 0;" ::: "memory");
    } else {
      uint4 now[R::kChunks];
      for (int count = 0; alive; ++count) {
        const int n = next_item(count);
        if (n < 0) break;
        const Item it = ms.items[count % kItems];
        free_item(count);
        if (n == 0) continue;
        auto load = [&](uint4 (&v)[R::kChunks]) {
#pragma unroll
          for (int k = 0; k < R::kChunks; ++k) {
            const uint8_t* from = R::row(mine, row0 + k * R::kStep);
            v[k] = load16_if(from + chunk * 16, from != nullptr);
          }
        };
        find(it, it.s0 * 128 + w * 32 + lane);
        load(now);
        for (int i = 0; i < n && alive; ++i, ++tiles) {
          const bool there = mine != nullptr;
          const int e = exponent;
          if (i + 1 < n) find(it, (it.s0 + i + 1) * 128 + w * 32 + lane);
          alive = wait_all(&ms.k_empty[st], ph ^ 1);
          if (!alive) break;
          uint8_t* const tile = ring + st * C::kTile;
          describe(there, e);
#pragma unroll
          for (int k = 0; k < R::kChunks; ++k) {
            const int row = w * 32 + row0 + k * R::kStep;
            uint4 lo, hi;
            bytes_to_halves<CODE>(now[k].x, lo.x, lo.y);
            bytes_to_halves<CODE>(now[k].y, lo.z, lo.w);
            bytes_to_halves<CODE>(now[k].z, hi.x, hi.y);
            bytes_to_halves<CODE>(now[k].w, hi.z, hi.w);
            *reinterpret_cast<uint4*>(tile + (chunk >> 2) * 16384 + swz128(row, 2 * chunk & 7)) = lo;
            *reinterpret_cast<uint4*>(tile + (chunk >> 2) * 16384 + swz128(row, (2 * chunk + 1) & 7)) = hi;
          }
          if (i + 1 < n) load(now);
          fence_async_smem();
          mbar_arrive(&ms.k_full[st]);
          if (++st == NS) st = 0, ph ^= 1;
        }
      }
    }
  } else if (warp < 12) {
    set_regs<kRegsLaunch, kRegsForm>();
    // ------------------------------------------------------------------ Q
    const int w = warp & 3, chunk = lane % R::kChunks, row0 = lane / R::kChunks;
    constexpr int kEach = CODE == TRITT_CODE_F16 ? 8 : 16, kAtOnce = R::kChunks < 8 ? R::kChunks : 8;   // elements of a chunk; chunks on their way together
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
      const int field = (int)(__reduce_max_sync(0xffffffffu, top) >> 23), largest = uniform(byte == 255 ? 0 : byte);
      const float up = to_operand(field) * (1.f / (1 << kDown<CODE>));
#pragma unroll
      for (int e = 0; e < kEach; ++e) q[e] = field == 255 ? 0.f : q[e] * up;
      const uint32_t there = __ballot_sync(0xffffffffu, mine != nullptr);
      alive = wait_all(&ms.q_free[buf], ((pieces >> 1) & 1) ^ 1);
      if (!alive) break;
      Columns& col = ms.columns[buf];
      col.scale[w * 32 + lane] = mine == nullptr ? 0.f : byte == 255 ? __uint_as_float(0x7fffffffu) : power_of_two(byte - largest);
      if (lane == 0) {
        col.there[w] = there;
        col.largest[w] = largest;
        col.field = field;   // (all four warps the same)
      }
      uint8_t* const hi_tile = smem + C::kOffQ + buf * 2 * C::kTile;
      uint8_t* const lo_tile = hi_tile + C::kTile;
      auto put = [&](int row, int at16, const uint32_t (&h)[4], int e0) {   // eight elements, 16 bytes of either number
        uint32_t hi[4], lo[4];
#pragma unroll
        for (int x = 0; x < 4; ++x) {
          const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h[x]));
          const float va = q[e0 + 2 * x] * f.x, vb = q[e0 + 2 * x + 1] * f.y;
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
          if constexpr (CODE == TRITT_CODE_F16) {
            const uint32_t h[4] = {v[x].x, v[x].y, v[x].z, v[x].w};
            put(row, chunk, h, 0);
          } else {
            uint32_t h[4];
            bytes_to_halves<CODE>(v[x].x, h[0], h[1]);
            bytes_to_halves<CODE>(v[x].y, h[2], h[3]);
            put(row, 2 * chunk, h, 0);
            bytes_to_halves<CODE>(v[x].z, h[0], h[1]);
            bytes_to_halves<CODE>(v[x].w, h[2], h[3]);
            put(row, 2 * chunk + 1, h, kEach / 2);
          }
        }
      }
      fence_async_smem();
      mbar_arrive(&ms.q_full[buf]);
      ++pieces;
    }
  } else {
    set_regs<kRegsLaunch, kRegsSum>();
    // ------------------------------------------------------------------ sums: a row a thread, 64 columns
    const int wg = (warp - 12) / 4, wq = warp & 3, row = wq * 32 + lane;
    const uint32_t t_lane = (uint32_t)(wq * 32) << 16;
    int pieces = 0;
    uint32_t tiles = 0;
    bool alive = true;
    for (int count = 0; alive; ++count) {
      const int n = next_item(count);
      if (n < 0) break;
      const Item& it = ms.items[count % kItems];
      const int pos = it.pos, base = it.base, s0 = it.s0, k0 = it.kg * 128 + wg * 64, k_lo = it.k_lo, j_lo = it.j_lo;
      const float minus = -it.minus;
      float* const slot = weigh_slot(p, it.b, it.head);
      float* const row_sums = slot + (size_t)wg * p.span;   // (each thread's own rows, here and where they are cleared)
      float* const col_sums = slot + (size_t)2 * p.span;
      if (it.fresh) {
        for (int x = row; x <= it.last - base; x += 128) row_sums[x] = 0.f;
        if (row < 64)
          for (int x = wg * 64 + row; x <= it.last - base; x += 128) col_sums[x] = 0.f;
      }
      const int last = it.last;
      free_item(count);
      if (n == 0) continue;
      const int buf = pieces & 1;
      alive = wait_all(&ms.q_full[buf], (pieces >> 1) & 1);
      if (!alive) break;
      const Columns& col = ms.columns[buf];
      const uint32_t there0 = col.there[2 * wg], there1 = col.there[2 * wg + 1];
      const int field = col.field, power0 = col.largest[2 * wg] + field - 382 + kDown<CODE>, power1 = col.largest[2 * wg + 1] + field - 382 + kDown<CODE>;
      const bool all_there = (there0 & there1) == 0xffffffffu;
      float2 column[32];
#pragma unroll
      for (int c = 0; c < 32; ++c) column[c] = make_float2(0.f, 0.f);
      for (int i = 0; i < n; ++i, ++tiles) {
        const uint32_t sb = tiles % kScores, mt = tiles % kMetas;
        const int j = (s0 + i) * 128 + row;
        float* const mine = row_sums + (j - base);
        const float before = j <= last ? *mine : 0.f;
        alive = wait_all(&ms.meta_full[mt], (tiles / kMetas) & 1);
        if (!alive) break;
        const int e = ms.meta[mt].exponent[row];
        const bool on = (ms.meta[mt].there[wq] >> lane & 1) && j >= j_lo && j <= pos;
        // the row's power of two with that of the columns, q and Q (beyond fp32's range scores have no use for)
        auto factor = [&](int power) {
          power += e;
          power = power < -126 ? -126 : power > 127 ? 127 : power;
          return e == 255 || field == 255 ? __uint_as_float(0x7fffffffu) : field == 0 ? 0.f : p.scale2 * power_of_two(power);
        };
        const float f0 = factor(power0), f1 = factor(power1);
        const int c_lo = (k_lo > j - p.kkr ? k_lo : j - p.kkr) - k0, c_hi = on ? (p.kkl < pos - j ? j + p.kkl : pos) - k0 : -1;
        const bool plain = __all_sync(0xffffffffu, all_there && c_lo <= 0 && c_hi >= 63);
        alive = wait_all(&ms.s_full[sb], (tiles / kScores) & 1);
        if (!alive) break;
        tc_fence_after();
        float2 sum0 = make_float2(0.f, 0.f), sum1 = sum0;
        auto half = [&](int h, float f, auto masked) {
          uint32_t s[32];
          tmem_ld32(tmem + sb * 128 + wg * 64 + h * 32 + t_lane, s);
          // bits of the columns that the row has pairs with
          uint32_t seen = 0xffffffffu;
          if constexpr (masked.value) {
            const int lo = c_lo - h * 32, hi = c_hi - h * 32;
            seen = h ? there1 : there0;
            if (lo > 0) seen &= lo > 31 ? 0u : 0xffffffffu << lo;
            if (hi < 31) seen &= hi < 0 ? 0u : 0xffffffffu >> (31 - hi);
          }
          tmem_wait_ld(s);
          if (h) {
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&ms.s_free[sb]);
          }
          const float4* by = reinterpret_cast<const float4*>(col.scale + wg * 64 + h * 32);
#pragma unroll
          for (int c = 0; c < 32; c += 4) {
            const float4 g = by[c / 4];
            float2 x = fma_pair(mul_pair(make_float2(__uint_as_float(s[c]), __uint_as_float(s[c + 1])), make_float2(g.x, g.y)), f, minus);
            float2 y = fma_pair(mul_pair(make_float2(__uint_as_float(s[c + 2]), __uint_as_float(s[c + 3])), make_float2(g.z, g.w)), f, minus);
            x.x = exp2f(x.x), x.y = exp2f(x.y), y.x = exp2f(y.x), y.y = exp2f(y.y);
            if constexpr (masked.value) {
              x.x = seen >> c & 1 ? x.x : 0.f, x.y = seen >> (c + 1) & 1 ? x.y : 0.f;
              y.x = seen >> (c + 2) & 1 ? y.x : 0.f, y.y = seen >> (c + 3) & 1 ? y.y : 0.f;
            }
            sum0 = add_pair(sum0, x);
            sum1 = add_pair(sum1, y);
            column[h * 16 + c / 2] = add_pair(column[h * 16 + c / 2], x);
            column[h * 16 + c / 2 + 1] = add_pair(column[h * 16 + c / 2 + 1], y);
          }
        };
        if (plain) {
          half(0, f0, std::false_type{});
          half(1, f1, std::false_type{});
        } else {
          half(0, f0, std::true_type{});
          half(1, f1, std::true_type{});
        }
        if (j <= last) *mine = before + ((sum0.x + sum0.y) + (sum1.x + sum1.y));
      }
      if (!alive) break;
      __syncwarp();
      if (lane == 0) mbar_arrive(&ms.q_free[buf]);
      // the columns' sums over the rows: halves change hands within the warp until a lane has columns 2 lane and the next; then over the four warps
      float* v = reinterpret_cast<float*>(column);
#pragma unroll
      for (int h = 16; h > 0; h >>= 1) {
        const bool upper = lane & h;
#pragma unroll
        for (int x = 0; x < 2 * h; ++x) {
          const float give = upper ? v[x] : v[x + 2 * h], keep = upper ? v[x + 2 * h] : v[x];
          v[x] = keep + __shfl_xor_sync(0xffffffffu, give, h);
        }
      }
      float(&sums)[4][64] = ms.sums[wg][buf];
      *reinterpret_cast<float2*>(&sums[wq][2 * lane]) = make_float2(v[0], v[1]);
      named_bar_sync(1 + wg, 128);   // (the other parity's numbers have been read by then)
      if (row < 64 && k0 + row <= last) col_sums[k0 + row - base] += (sums[0][row] + sums[1][row]) + (sums[2][row] + sums[3][row]);
      ++pieces;
    }
  }

  // ------------------------------------------------------------------ teardown
  tc_fence_before();
  __syncthreads();
  if (warp == 0) tmem_dealloc(tmem, 512);
  if (tid == 0 && ms.abort_flag && a.status) atomicOr(a.status, kStatusTdpDecode);
}

template <typename T, int D, int CODE> int launch(const TdpWeighArgs& p, cudaStream_t stream) {
  TRITT_CUDA_OK(cudaFuncSetAttribute(tdp_weigh_sm100_kernel<T, D, CODE>, cudaFuncAttributeMaxDynamicSharedMemorySize, Cfg<D>::kSmem));
  tdp_weigh_sm100_kernel<T, D, CODE><<<p.ctas, kThreads, Cfg<D>::kSmem, stream>>>(p);
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
