// One soft-max attention of new tokens over two parts of the quantised cache, 16-bit queries, head dimension 64 or 128: either leg of the
// dot-product-sum form (append: rows k2 over K1, SiLU(V1) within a window;  decode: rows q over K2, W with a bias for each token).
//
// Bound by HBM: a cached row is read once for up to 8 NT new tokens, 2 flops a byte and token.  Each warp has a ring of its own in
// shared memory, filled by bulk copies (16 rows each, whole pages' neighbours) and 4-byte asynchronous ones (exponents, biases): no registers
// wait for memory and nearly no instructions address it (a first form with loads to registers executed 1046 instructions for 32
// tokens, more than HBM leaves time for: 253 us for a token of 32 sequences of up to 8191, 16 heads of 64, e4m3; now 90, 4.8 TB/s).  Rows then go, as fp16, into warp-level matrix
// instructions with the cached rows as the 16-row operand:
//   S^T[16 tokens x 8 queries] = K Q^T,   O^T[D x 8 queries] += V^T P^T
// (one token is an eighth of a tile instead of a sixteenth, and a query's statistics lie in the threads that hold its results).  The contraction of S
// runs over the head dimension in any order, so a thread takes 16 contiguous bytes of a row for the elements that it needs; the rows of
// V^T are columns of V in any order, so a thread takes D / 8 contiguous elements of four tokens and pairs them by byte permutes.  P^T is
// the transpose of S^T's fragments (movmatrix).
//
// The line of all (sequence, head, group of new tokens, tile) steps is cut in equal parts, one for each block that the chip holds at
// once: sequences differ in length, and nothing of it is known to the host.  A block's warps take its tiles in turn; each piece of a group
// leaves maximum, sum and result, which a second kernel joins in a fixed order.
//
// Codes are exact as fp16, the scores' powers of two are applied in fp32; P is formed times 2^(its row's exponent - the largest so far + 13),
// so that values of any size meet in one accumulator, and its sum is taken before that.  Queries are brought to [1, 2) by a power of two.
// Where rows are few or new tokens many, the way to the first tile and each piece's end count as much as the bytes: 24 tokens over 3001, 4 x 16
// heads of 128, fp16: 38 us, of which a tile of 16 rows takes 2.5 thousand cycles (two warps a scheduler, a chain of two products and a soft-max)
// and a piece 10 (first rows, queries, joining of the warps).
// A tile's rows may be hidden from some or all of its queries (another branch of a tree, before a window).  Where one could be so much larger than what
// the queries attend to that their P would leave fp16's range (2^12), each query goes on with an exponent of its own, the largest of the rows
// that it attends to (looking for it costs 1 to 3 %).
// Append forms P as the sum of two fp16 numbers (22 bits): its result is rounded again, to codes, and each element that a less exact one moves over
// a border is off by a whole step (e4m3: 0.13 % of W's norm with one fp16 number, 2e-5 with two).
#include "tritt_cache.cuh"
#include "tritt_sm100.cuh"
#include "tritt_sm100_tdp.cuh"

namespace tritt {
namespace {
using namespace sm100;

constexpr int kWarps = 4;
constexpr int kLift = 5;        // P is formed times 2^5; the reference is raised when a score is 2^8 above it: at most 2^13
constexpr float kGap = 8.f;
constexpr int kHidden = 12;     // see above
constexpr int kLeastSteps = 8;  // of a block: two tiles a warp

// What the line of steps has of one sequence.
struct Line {
  int ctx, cnt;          // tokens before the new ones, new ones
  int groups, tiles;     // groups of new tokens; tiles of a group (the most of any)
};
struct LineEntry {       // in the workspace, for the kernel that joins
  long long base, group_base;
  Line line;
};

struct Params {
  DpsDecodeArgs a;
  LineEntry* table;      // [B]
  float* part;           // [pieces][Q][D + 2]
  int ctas;
  bool early;
};

__device__ __forceinline__ void mma_16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transposed(uint32_t v) {   // an 8 x 8 fragment of 16-bit elements
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}
__device__ __forceinline__ uint32_t pack_half(float lo, float hi) {
  const __half2 v = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ float power(int e) { return e > -127 ? __uint_as_float((uint32_t)(e + 127) << 23) : 0.f; }

template <int D, int CODE> struct Shape {
  static constexpr bool kWide = CODE == TRITT_CODE_F16;
  static constexpr int kRowBytes = D * (kWide ? 2 : 1);
  static constexpr int kTokens = 4096 / kRowBytes;              // of a tile, 64 to 16: 8 KB of keys and values
  static constexpr int kBlocks = kTokens / 16;                  // of 16 tokens, each in one page
  static constexpr int kKeyLoads = kRowBytes / 64;              // of 16 bytes, of a lane's row
  static constexpr int kValueWords = kRowBytes / 32;            // 32-bit words of a lane's eighth of a row
  // a stage of the ring: keys, values, then biases, exponents of keys and values, and which blocks are there
  static constexpr int kOffV = 4096, kOffBias = 8192, kOffEk = kOffBias + 256, kOffEv = kOffEk + 64, kOffThere = kOffEv + 64;
  static constexpr int kStage = 8704;
};
template <int NT> constexpr int kBlocksPerSm = NT == 1 ? 3 : 2;   // by registers
// Stages of a warp's ring: of three blocks an SM each warp has one in flight and one that it works on.
template <int NT> constexpr int kStages = kBlocksPerSm<NT> == 3 ? 2 : 3;
// The ring's memory takes the warps' results at the end of a piece: [warps][Q][D + 4] fp32.
template <int D, int CODE, int NT> constexpr int smem_bytes() {
  constexpr int ring = kWarps * kStages<NT> * Shape<D, CODE>::kStage, out = kWarps * 8 * NT * (D + 4) * 4;
  return ring > out ? ring : out;
}

// Asynchronous copies of 16 bytes, and their arrival at a barrier.
__device__ __forceinline__ void copy16(void* dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(dst)), "l"(src) : "memory");
}
__device__ __forceinline__ void copies_arrive(uint64_t* bar) {
  asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}

// Which row of a block of 16 is row r of the fragments: with rows of 64 bytes, so that the four that a quarter of the lanes' value loads
// touch lie in both halves of the banks.
template <int ROW_BYTES> __device__ __forceinline__ int actual_row(int r) { return ROW_BYTES == 64 ? r ^ (r >> 1 & 1) : r; }

template <int TK, int Q> __device__ __forceinline__ Line line_of(const DpsDecodeArgs& a, int b) {
  Line l;
  l.ctx = context_of(a.cache, b);
  l.cnt = new_tokens(a.cache, b);
  l.groups = (l.cnt + Q - 1) / Q;
  l.tiles = l.cnt ? (min(l.ctx, a.window) + l.cnt + 15 + TK - 1) / TK : 0;   // (a group's first tile starts at a multiple of 16)
  return l;
}
// CTAs that the line is cut for.
__host__ __device__ __forceinline__ int parts_of(long long total, int ctas) {
  const long long n = total / kLeastSteps;
  return n < 1 ? 1 : n < ctas ? (int)n : ctas;
}

// ONE: a single new token (a query's column of the fragments; the others are not worked on).
template <int D, int CODE, int NT, bool ONE, bool EXACT>
__global__ void __launch_bounds__(kWarps * 32, kBlocksPerSm<NT>) dps_decode_kernel(const __grid_constant__ Params p) {
  using S = Shape<D, CODE>;
  constexpr int NB = S::kBlocks, TK = S::kTokens, KL = S::kKeyLoads, VW = S::kValueWords, NS = kStages<NT>, RB = S::kRowBytes;
  constexpr int Q = 8 * NT, NQ = ONE ? 1 : 2;
  extern __shared__ __align__(128) uint8_t ring_all[];
  __shared__ uint64_t s_full[kWarps][NS];
  __shared__ int s_abort, s_first;
  __shared__ long long s_total, s_base, s_groups;
  __shared__ float4 s_side[kWarps][TK];   // of a tile's tokens: scale of scores, bias, scale of P
  __shared__ unsigned long long s_word[Q];
  __shared__ int s_lo[Q], s_pos[Q];
  __shared__ float s_scale[Q], s_m[kWarps][Q], s_l[kWarps][Q];
  __shared__ int s_own[kWarps][Q];   // queries' exponents, where they differ
  const DpsDecodeArgs& a = p.a;
  const CacheArgs& ca = a.cache;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  uint8_t* ring = ring_all + warp * NS * S::kStage;
  uint64_t* full = s_full[warp];
  let_next_start();
  if (lane == 0) {
    for (int i = 0; i < NS; ++i) mbar_init(&full[i], 33);   // one arrival with the bulk copies' bytes, one of each lane
    fence_barrier_init();
  }
  if (warp == 0) {
    // the whole line's length, 32 sequences at a time, and the sequence of this block's first step (a walk from sequence to sequence took 200
    // cycles each)
    long long total = 0, groups = 0, behind = 0, here = 0, groups_before = 0;   // steps, groups; of the lane's sequence: up to its end, its own
    auto sums = [&](int b0, bool write) {
      const int b = b0 + lane;
      Line l{};
      if (b < ca.c.B) l = line_of<TK, Q>(a, b);
      const long long ng = (long long)l.groups * ca.c.N;
      here = ng * l.tiles;
      long long s = here, q = ng;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const long long s2 = __shfl_up_sync(0xffffffffu, s, o), q2 = __shfl_up_sync(0xffffffffu, q, o);
        if (lane >= o) s += s2, q += q2;
      }
      behind = total + s;
      groups_before = groups + q - ng;
      if (write && blockIdx.x == 0 && b < ca.c.B) p.table[b] = LineEntry{behind - here, groups_before, l};
      total = __shfl_sync(0xffffffffu, behind, 31);
      groups = __shfl_sync(0xffffffffu, groups + q, 31);
    };
    for (int b0 = 0; b0 < ca.c.B; b0 += 32) sums(b0, true);
    if (lane == 0) s_total = total, s_abort = 0;
    const long long x = (long long)blockIdx.x * total / parts_of(total, p.ctas);
    int b0 = 0;
    if (ca.c.B > 32) {
      total = groups = 0;
      for (; b0 < ca.c.B; b0 += 32) {
        sums(b0, false);
        if (x < total) break;
      }
    }
    const uint32_t found = __ballot_sync(0xffffffffu, x < behind);
    if (found && lane == __ffs(found) - 1) s_first = b0 + lane, s_base = behind - here, s_groups = groups_before;
  }
  __syncthreads();
  const long long total = s_total;
  const int parts = parts_of(total, p.ctas);
  if ((int)blockIdx.x >= parts) return wait_for_previous();   // (a kernel that ended without one would let the next start beside the previous)
  long long x = (long long)blockIdx.x * total / parts, base = s_base, group_base = s_groups;
  const long long x_end = ((long long)blockIdx.x + 1) * total / parts;
  if (x >= x_end) return wait_for_previous();
  const size_t part_rows = (size_t)ca.c.N << ca.page_log2;   // rows of one part of a page
  const size_t page_bytes = 4 * part_rows * RB;
  const int row_mask = ca.c.page_size - 1;
  int st = 0, phase = 0;   // the ring's next stage
  int b = s_first;
  Line line = line_of<TK, Q>(a, b);
  bool alive = true, waited = false;

  while (x < x_end && alive) {
    // --- the next piece: tiles s0 .. s1 - 1 of one group of new tokens
    while (x >= base + (long long)line.groups * line.tiles * ca.c.N) {
      base += (long long)line.groups * line.tiles * ca.c.N;
      group_base += (long long)line.groups * ca.c.N;
      if (++b >= ca.c.B) return wait_for_previous();   // (contexts that changed under the kernel)
      line = line_of<TK, Q>(a, b);
    }
    const long long rel = x - base, grp = rel / line.tiles;
    const int s0 = (int)(rel % line.tiles), s1 = (int)(line.tiles - s0 < x_end - x ? line.tiles : s0 + (x_end - x));
    const int head = (int)(grp / line.groups), i0 = (int)(grp % line.groups) * Q;
    float* part = p.part + (size_t)(group_base + grp + blockIdx.x) * Q * (D + 2);
    x += s1 - s0;
    const int ctx = line.ctx, nq = min(Q, line.cnt - i0);
    // tokens that any of these queries attends to: first .. end - 1
    const int first = max(0, ctx + (ca.c.ancestors ? 0 : i0) - a.window) & ~15, end = ctx + i0 + nq;
    const int tile1 = min(s1, (end - first + TK - 1) / TK);
    if (s0 >= tile1) {
      for (int i = tid; i < nq; i += kWarps * 32) part[i * (D + 2)] = -INFINITY, part[i * (D + 2) + 1] = 0.f;
      continue;
    }

    // --- the queries' rows, on their way while the ring is filled (those past the last: its own, not looked at)
    uint4 raw[NT][D / 32];
    constexpr int EPL = S::kWide ? 8 : 16;   // elements of 16 bytes of codes
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const uint16_t* q = (const uint16_t*)a.q.p + rows_at(a.q, b, head, i0 + min(nt * 8 + g, nq - 1)) + t * EPL;
#pragma unroll
      for (int k = 0; k < D / 32; ++k) raw[nt][k] = __ldg(reinterpret_cast<const uint4*>(q + k / (EPL / 8) * 4 * EPL + k % (EPL / 8) * 8));
    }

    unsigned long long words[NT];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) words[nt] = warp == 0 && ca.c.ancestors && nt * 8 + g < nq ? seen_word(ca, b, i0 + nt * 8 + g) : 0;

    // --- the ring: this warp takes tiles s0 + warp, + kWarps, ...
    const uint8_t* key_rows = (const uint8_t*)ca.c.codes + (a.key_part * part_rows + ((size_t)head << ca.page_log2)) * RB;
    const long long to_values = (long long)(a.value_part - a.key_part) * (long long)part_rows;
    const unsigned char* key_exp = ca.c.exponents + a.key_part * part_rows + ((size_t)head << ca.page_log2);
    const float* biases = ca.c.lse + ((size_t)head << ca.page_log2);
    // the page of a tile's block of 16 tokens lane % NB, -1: none, or no such tokens
    auto find_page = [&](int tile) {
      const int token = first + tile * TK + lane % NB * 16;
      return tile < tile1 && token < end ? place_of(ca, b, token).page : -1;
    };
    // (what a page has behind the last token comes along and is not looked at)
    auto fill = [&](int tile, int stage, int page) {
      uint8_t* to = ring + stage * S::kStage;
      const uint32_t there = __ballot_sync(0xffffffffu, page >= 0) & ((1u << NB) - 1);
      if (lane == 0) {
        *reinterpret_cast<uint32_t*>(to + S::kOffThere) = there;
        mbar_arrive_expect_tx(&full[stage], (uint32_t)__popc(there) * 2 * 16 * RB);
      }
      __syncwarp();
      if (page >= 0) {
        // lanes NB k .. NB k + NB - 1: keys, values, their exponents, and four times the quarters of the biases
        const int blk = lane % NB, kind = lane / NB, row = (first + tile * TK + blk * 16) & row_mask;
        if (kind < 2)
          bulk_load(to + kind * S::kOffV + blk * 16 * RB, key_rows + page * page_bytes + (size_t)row * RB + (kind ? to_values * RB : 0), 16 * RB,
                    &full[stage]);
        else if (kind < 4)
          copy16(to + (kind == 2 ? S::kOffEk : S::kOffEv) + blk * 16, key_exp + page * (4 * part_rows) + row + (kind == 2 ? 0 : to_values));
        else if (kind < 8 && a.biased)
          copy16(to + S::kOffBias + blk * 64 + (kind - 4) * 16, biases + page * part_rows + row + (kind - 4) * 4);
      }
      copies_arrive(&full[stage]);
    };
    int next_page;   // of the tile that is filled next
    {
      int pg[NS + 1];
#pragma unroll
      for (int i = 0; i <= NS; ++i) pg[i] = find_page(s0 + warp + i * kWarps);
      // (what is read above, no kernel that may still run has written)
      if (!waited) wait_for_previous();
      waited = true;
      int f = st;
#pragma unroll
      for (int i = 0; i < NS; ++i) {
        if (s0 + warp + i * kWarps < tile1) fill(s0 + warp + i * kWarps, f, pg[i]);
        f = f + 1 == NS ? 0 : f + 1;
      }
      next_page = pg[NS];
    }

    // --- queries: fragments of Q^T, and what masks them
    uint32_t qf[NT][D / 16][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int i = i0 + nt * 8 + g;
      const bool on = nt * 8 + g < nq;
      float f[D / 4];   // elements of this thread's positions, in the order of its fragments
      uint32_t big = 0;
#pragma unroll
      for (int k = 0; k < D / 32; ++k) {
        const uint32_t w[4] = {raw[nt][k].x, raw[nt][k].y, raw[nt][k].z, raw[nt][k].w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float2 v = a.dtype == TRITT_F16 ? unpack2<__half>(w[e]) : unpack2<__nv_bfloat16>(w[e]);
          f[k * 8 + 2 * e] = on ? v.x : 0.f;
          f[k * 8 + 2 * e + 1] = on ? v.y : 0.f;
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) big = max(big, __float_as_uint(f[k * 8 + e]) & 0x7fffffffu);
      }
      big = max(big, __shfl_xor_sync(0xffffffffu, big, 1));
      big = max(big, __shfl_xor_sync(0xffffffffu, big, 2));
      const int up = max(min(254 - (int)(big >> 23), 253), 1);
      const float mul = __uint_as_float((uint32_t)up << 23);
#pragma unroll
      for (int s = 0; s < D / 16; ++s) {
        qf[nt][s][0] = pack_half(f[s * 4] * mul, f[s * 4 + 1] * mul);
        qf[nt][s][1] = pack_half(f[s * 4 + 2] * mul, f[s * 4 + 3] * mul);
      }
      if (warp == 0 && t == 0) {
        const unsigned long long word = words[nt];
        const int pos = ctx + (ca.c.ancestors ? __popcll(word) - 1 : i);
        s_word[nt * 8 + g] = word;
        s_pos[nt * 8 + g] = on ? pos : -1;
        s_lo[nt * 8 + g] = on ? max(0, pos - a.window) : 0x7fffffff;
        s_scale[nt * 8 + g] = a.scale2 * __uint_as_float((uint32_t)(254 - up) << 23);
      }
    }
    __syncthreads();
    // from lo_all on every query attends to all of the context (those that are not there take no part in this: their results are not looked at)
    const int lo_all = __reduce_max_sync(0xffffffffu, lane < nq ? s_lo[lane] : 0);
    float qs[NT][NQ];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int q = 0; q < NQ; ++q) qs[nt][q] = s_scale[nt * 8 + 2 * t + q];

    float acc[NT][D / 16][4], m[NT][NQ], l[NT][NQ];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
      for (int mb = 0; mb < D / 16; ++mb)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[nt][mb][e] = 0.f;
#pragma unroll
      for (int q = 0; q < NQ; ++q) m[nt][q] = -INFINITY, l[nt][q] = 0.f;
    }
    int v_exp = 0;   // largest exponent byte of the values so far
    int low = 255;   // least one that may have to be told from it: of the tiles with rows that some query does not attend to, and before them
    bool own = false;
    for (int tile = s0 + warp; tile < tile1; tile += kWarps) {
      if (!__all_sync(0xffffffffu, mbar_wait(&full[st], phase, (volatile int*)&s_abort))) {
        // give copies still in flight a bounded chance to land before the block ends
        for (int i = 0; i < NS; ++i) {
          const long long t0 = clock64();
          while (!mbar_try_wait(&full[i], i < st ? phase ^ 1 : phase) && clock64() - t0 < kWaitTicks / 8) {
          }
        }
        if (lane == 0 && ca.status) atomicOr(ca.status, 16);
        break;
      }
      const uint8_t* from = ring + st * S::kStage;
      const int token0 = first + tile * TK;
      // one lane a token or two: scales, and whether all of the tile counts for every query
      const uint32_t there = *reinterpret_cast<const uint32_t*>(from + S::kOffThere);
      bool plain = token0 >= lo_all && token0 + TK <= ctx && there == (1u << NB) - 1;
      {
        constexpr int PER = (TK + 31) / 32;
        int ek[PER], ev[PER], most = 0, fewest = 255;
        bool bad = false;
#pragma unroll
        for (int k = 0; k < PER; ++k) {
          const int token = k * 32 + lane;
          const bool on = token < TK && token0 + token < end && (there >> (token >> 4) & 1);
          ek[k] = on ? from[S::kOffEk + token] : 0;
          ev[k] = on ? from[S::kOffEv + token] : 0;
          bad = bad || ek[k] == 255 || ev[k] == 255;
          most = max(most, ev[k] == 255 ? 0 : ev[k]);
          fewest = min(fewest, least_byte(ev[k]));
        }
        plain = !__any_sync(0xffffffffu, bad) && plain;
        most = __reduce_max_sync(0xffffffffu, most);
        bool apart;
        if (plain) {
          apart = most > 1 && v_exp - most > kHidden;
        } else {
          low = min(min(low, least_byte(v_exp)), (int)__reduce_min_sync(0xffffffffu, fewest));
          apart = max(v_exp, most) - low > kHidden;
        }
        most = max(v_exp, most);
        if (apart && !own) {
          own = true;
          if (lane < Q) s_own[warp][lane] = v_exp;
        }
        // (the products lie in the accumulator times 2^(largest exponent))
        if (most > v_exp && !own) {
          const float grown = v_exp ? power(v_exp - most) : 1.f;
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int mb = 0; mb < D / 16; ++mb)
#pragma unroll
              for (int e = 0; e < 4; ++e) acc[nt][mb][e] *= grown;
          v_exp = most;
        }
#pragma unroll
        for (int k = 0; k < PER; ++k) {
          const int token = k * 32 + lane;
          if (TK >= 32 || token < TK)
            s_side[warp][token] = make_float4(
                power(ek[k] - 127), a.biased ? *reinterpret_cast<const float*>(from + S::kOffBias + token * 4) * kLog2e : 0.f,
                ev[k] == 255 || ev[k] == 0 ? 0.f : power(ev[k] - most + kLift), ek[k] == 255 || ev[k] == 255 ? 1.f : 0.f);
        }
      }
      __syncwarp();
      // S^T
      float s[NT][NB][4];
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int e = 0; e < 4; ++e) s[nt][nb][e] = 0.f;
        const uint8_t* row = from + (nb * 16 + actual_row<RB>(g)) * RB + t * 16;
#pragma unroll
        for (int j = 0; j < KL; ++j) {
          const uint4 r0 = *reinterpret_cast<const uint4*>(row + j * 64), r1 = *reinterpret_cast<const uint4*>(row + 8 * RB + j * 64);
          const uint32_t lo[4] = {r0.x, r0.y, r0.z, r0.w}, hi[4] = {r1.x, r1.y, r1.z, r1.w};
          constexpr int STEPS = S::kWide ? 2 : 4;   // contraction steps of 16 bytes
#pragma unroll
          for (int k = 0; k < STEPS; ++k) {
            uint32_t f[4];
            if constexpr (S::kWide) {
              f[0] = lo[2 * k], f[1] = hi[2 * k], f[2] = lo[2 * k + 1], f[3] = hi[2 * k + 1];
            } else {
              bytes_to_halves<CODE>(lo[k], f[0], f[2]);
              bytes_to_halves<CODE>(hi[k], f[1], f[3]);
            }
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) mma_16816(s[nt][nb], f, qf[nt][j * STEPS + k][0], qf[nt][j * STEPS + k][1]);
          }
        }
      }
      // scores in log2 units
      float vf[NB][2];
#pragma unroll
      for (int nb = 0; nb < NB; ++nb)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int k = nb * 16 + h * 8 + actual_row<RB>(g);
          const float4 side = s_side[warp][k];
          vf[nb][h] = side.z;
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int q = 0; q < NQ; ++q) s[nt][nb][2 * h + q] = fmaf(s[nt][nb][2 * h + q] * side.x, qs[nt][q], side.y);
          if (!plain) {
            const int token = token0 + k;
            const bool here = there >> (k >> 4) & 1;
            bool missing = false;
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
              for (int q = 0; q < NQ; ++q) {
                const int i = nt * 8 + 2 * t + q;
                bool seen = token >= s_lo[i] && token < end;
                if (token >= ctx && token < end) {
                  const int n = token - ctx;
                  if (ca.c.ancestors) {
                    const unsigned long long word = s_word[i];
                    seen = (word >> n & 1) && ctx + __popcll(word & ((1ull << n) - 1)) >= s_lo[i];
                  } else {
                    seen = seen && token <= s_pos[i];
                  }
                }
                missing = missing || (seen && !here);
                float& v = s[nt][nb][2 * h + q];
                v = seen && here ? (side.w != 0.f ? __uint_as_float(0x7fffffffu) : v) : -INFINITY;
              }
            if (missing && ca.status) atomicOr(ca.status, kStatusPlace);
          }
        }
      auto raise_reference = [&](int nt, const float (&mx)[NQ]) {
        float corr[NQ];
#pragma unroll
        for (int q = 0; q < NQ; ++q) {
          float v = fmaxf(mx[q], m[nt][q]);
          v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 4));
          v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 8));
          v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 16));
          corr[q] = v == -INFINITY ? 1.f : exp2f(m[nt][q] - v);
          m[nt][q] = v;
          l[nt][q] *= corr[q];
        }
#pragma unroll
        for (int mb = 0; mb < D / 16; ++mb)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if ((e & 1) < NQ) acc[nt][mb][e] *= corr[e & 1 ? NQ - 1 : 0];
      };
      // Queries with exponents of their own: these, and the rows' powers of two in the scores, from which P is formed; the sum is told beforehand of
      // what that takes away
      if (own) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          float mx[NQ];
#pragma unroll
          for (int q = 0; q < NQ; ++q) {
            int& mine = s_own[warp][nt * 8 + 2 * t + q];
            const int old = m[nt][q] == -INFINITY ? 0 : mine;   // (0: nothing attended so far)
            int now = old;
            mx[q] = -INFINITY;
#pragma unroll
            for (int nb = 0; nb < NB; ++nb)
#pragma unroll
              for (int h = 0; h < 2; ++h) {
                const int byte = from[S::kOffEv + nb * 16 + h * 8 + actual_row<RB>(g)];
                if (s[nt][nb][2 * h + q] != -INFINITY && byte != 255) now = max(now, byte);
                mx[q] = fmaxf(mx[q], s[nt][nb][2 * h + q]);
              }
            now = max(now, __shfl_xor_sync(0xffffffffu, now, 4));
            now = max(now, __shfl_xor_sync(0xffffffffu, now, 8));
            now = max(now, __shfl_xor_sync(0xffffffffu, now, 16));
            const float grown = power_of_two(old - now);
#pragma unroll
            for (int mb = 0; mb < D / 16; ++mb) acc[nt][mb][q] *= grown, acc[nt][mb][2 + q] *= grown;
            __syncwarp();
            if (g == 0) mine = now;
            __syncwarp();
          }
          raise_reference(nt, mx);
#pragma unroll
          for (int q = 0; q < NQ; ++q) {
            const float base = m[nt][q] == -INFINITY ? 0.f : m[nt][q];
            const int mine = s_own[warp][nt * 8 + 2 * t + q];
            float whole = 0.f, rest = 0.f;
#pragma unroll
            for (int nb = 0; nb < NB; ++nb)
#pragma unroll
              for (int h = 0; h < 2; ++h) {
                float& v = s[nt][nb][2 * h + q];
                whole += exp2f(v - base);
                // (a row that the query does not attend to has -infinity, and may have any exponent)
                v += (float)min(0, from[S::kOffEv + nb * 16 + h * 8 + actual_row<RB>(g)] - mine);
                rest += exp2f(v - base);
              }
            l[nt][q] += whole - rest;
          }
        }
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) vf[nb][0] = vf[nb][1] = 1 << kLift;
      }
      // the reference (raised where a score is 2^8 above it), P
      uint32_t pf[NT][NB][2], pl[EXACT ? NT : 1][NB][2];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        float mx[NQ], base2[NQ];
        bool raise = false;
#pragma unroll
        for (int q = 0; q < NQ; ++q) {
          mx[q] = fmaxf(s[nt][0][q], s[nt][0][2 + q]);
#pragma unroll
          for (int nb = 1; nb < NB; ++nb) mx[q] = fmaxf(mx[q], fmaxf(s[nt][nb][q], s[nt][nb][2 + q]));
          raise = raise || mx[q] > m[nt][q] + kGap;
        }
        if (__any_sync(0xffffffffu, raise)) raise_reference(nt, mx);
#pragma unroll
        for (int q = 0; q < NQ; ++q) base2[q] = m[nt][q] == -INFINITY ? 0.f : m[nt][q];   // (nothing attended so far: all P are 0)
#pragma unroll
        for (int nb = 0; nb < NB; ++nb)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            float v[2] = {0.f, 0.f};
#pragma unroll
            for (int q = 0; q < NQ; ++q) {
              const float e = exp2f(s[nt][nb][2 * h + q] - base2[q]);
              l[nt][q] += e;
              v[q] = e * vf[nb][h];
            }
            const uint32_t high = pack_half(v[0], v[1]);
            pf[nt][nb][h] = transposed(high);
            if constexpr (EXACT) {
              const float2 r = __half22float2(*reinterpret_cast<const __half2*>(&high));
              pl[nt][nb][h] = transposed(pack_half(v[0] - r.x, v[1] - r.y));
            }
          }
      }
      // O^T += V^T P^T
#pragma unroll
      for (int nb = 0; nb < NB; ++nb) {
        // of tokens 2t, 2t + 1, 2t + 8, 2t + 9 of the block (as the fragments count), the g-th eighth of the row
        uint32_t v[4][VW];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const int row = nb * 16 + (k >> 1) * 8 + actual_row<RB>(2 * t + (k & 1));
          const uint8_t* r = from + S::kOffV + row * RB + g * (VW * 4);
          if constexpr (VW == 2) {
            const uint2 w = *reinterpret_cast<const uint2*>(r);
            v[k][0] = w.x, v[k][1] = w.y;
          } else {
#pragma unroll
            for (int j = 0; j < VW / 4; ++j) {
              const uint4 w = *(reinterpret_cast<const uint4*>(r) + j);
              v[k][4 * j] = w.x, v[k][4 * j + 1] = w.y, v[k][4 * j + 2] = w.z, v[k][4 * j + 3] = w.w;
            }
          }
          if (!plain && !(token0 + row < end && (there >> (row >> 4) & 1))) {   // (what lies there is of another tile, or no number)
#pragma unroll
            for (int w = 0; w < VW; ++w) v[k][w] = 0u;
          }
        }
#pragma unroll
        for (int w = 0; w < VW; ++w) {
          if constexpr (S::kWide) {
            // two elements of four tokens: one block of 16 rows of V^T
            uint32_t f[4];
            f[0] = __byte_perm(v[0][w], v[1][w], 0x5410);
            f[1] = __byte_perm(v[0][w], v[1][w], 0x7632);
            f[2] = __byte_perm(v[2][w], v[3][w], 0x5410);
            f[3] = __byte_perm(v[2][w], v[3][w], 0x7632);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
              mma_16816(acc[nt][w], f, pf[nt][nb][0], pf[nt][nb][1]);
              if constexpr (EXACT) mma_16816(acc[nt][w], f, pl[nt][nb][0], pl[nt][nb][1]);
            }
          } else {
            // four elements: two blocks
#pragma unroll
            for (int half = 0; half < 2; ++half) {
              const uint32_t lo = __byte_perm(v[0][w], v[1][w], half ? 0x7362 : 0x5140);
              const uint32_t hi = __byte_perm(v[2][w], v[3][w], half ? 0x7362 : 0x5140);
              uint32_t f[4];
              bytes_to_halves<CODE>(lo, f[0], f[1]);
              bytes_to_halves<CODE>(hi, f[2], f[3]);
#pragma unroll
              for (int nt = 0; nt < NT; ++nt) {
                mma_16816(acc[nt][2 * w + half], f, pf[nt][nb][0], pf[nt][nb][1]);
                if constexpr (EXACT) mma_16816(acc[nt][2 * w + half], f, pl[nt][nb][0], pl[nt][nb][1]);
              }
            }
          }
        }
      }
      __syncwarp();   // every lane has read this stage
      if (tile + NS * kWarps < tile1) fill(tile + NS * kWarps, st, next_page);
      next_page = find_page(tile + (NS + 1) * kWarps);
      if (++st == NS) st = 0, phase ^= 1;
    }

    // --- the warps' results on their common maximum, added up in order
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int q = 0; q < NQ; ++q) {
        float sum = l[nt][q];
        sum += __shfl_xor_sync(0xffffffffu, sum, 4);
        sum += __shfl_xor_sync(0xffffffffu, sum, 8);
        sum += __shfl_xor_sync(0xffffffffu, sum, 16);
        if (g == 0) {
          s_m[warp][nt * 8 + 2 * t + q] = m[nt][q];
          s_l[warp][nt * 8 + 2 * t + q] = sum;
        }
      }
    __syncthreads();   // (and every warp is done with its ring)
    alive = s_abort == 0;
    float(*out)[Q][D + 4] = reinterpret_cast<float(*)[Q][D + 4]>(ring_all);
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int q = 0; q < NQ; ++q) {
        const int i = nt * 8 + 2 * t + q;
        if (i >= nq) continue;
        float top = -INFINITY;
#pragma unroll
        for (int k = 0; k < kWarps; ++k) top = fmaxf(top, s_m[k][i]);
        // (a warp without a value has exponent 0 and adds nothing)
        const int e = own ? s_own[warp][i] : v_exp;
        const float f = m[nt][q] == -INFINITY || e == 0 ? 0.f : exp2f(m[nt][q] - top) * power(e - 127) * (1.f / (1 << kLift));
#pragma unroll
        for (int mb = 0; mb < D / 16; ++mb)
          *reinterpret_cast<float2*>(&out[warp][i][g * (D / 8) + 2 * mb]) =
              f == 0.f ? make_float2(0.f, 0.f) : make_float2(acc[nt][mb][q] * f, acc[nt][mb][2 + q] * f);
      }
    __syncthreads();
    if (tid < nq) {
      float top = -INFINITY, sum = 0.f;
#pragma unroll
      for (int k = 0; k < kWarps; ++k) top = fmaxf(top, s_m[k][tid]);
#pragma unroll
      for (int k = 0; k < kWarps; ++k)
        sum += s_m[k][tid] == -INFINITY ? (s_l[k][tid] != s_l[k][tid] ? s_l[k][tid] : 0.f) : s_l[k][tid] * exp2f(s_m[k][tid] - top);
      *reinterpret_cast<float2*>(part + tid * (D + 2)) = make_float2(top, sum);
    }
#pragma unroll 2
    for (int x = tid; x < nq * (D / 4); x += kWarps * 32) {
      const int i = x / (D / 4), c = x % (D / 4) * 4;
      float4 v = *reinterpret_cast<const float4*>(&out[0][i][c]);
#pragma unroll
      for (int k = 1; k < kWarps; ++k) {
        const float4 o = *reinterpret_cast<const float4*>(&out[k][i][c]);
        v.x += o.x, v.y += o.y, v.z += o.z, v.w += o.w;
      }
      float2* to = reinterpret_cast<float2*>(part + i * (D + 2) + 2 + c);
      to[0] = make_float2(v.x, v.y);
      to[1] = make_float2(v.z, v.w);
    }
    fence_async_smem();   // (the next piece's copies come into the same memory)
    __syncthreads();
  }
  if (!waited) wait_for_previous();
}

struct DpsJoinParams {
  DpsDecodeArgs a;
  const LineEntry* table;
  const float* part;
  int ctas, queries;     // of the first kernel; new tokens of a group
  void* o;               // [B, N, n, D], or null: append
  float* lse;            // [B, N, n]
  tritt_rows_t v2;       // append: W = result * v2 goes to the cache, and the log-sum-exp
};

// The CTA of a step.
__device__ __forceinline__ int cta_of(long long x, long long total, int parts) {
  if (total < 1 << 20) return (int)(((uint32_t)(x + 1) * (uint32_t)parts - 1) / (uint32_t)total);   // (a division of 64 bits is long)
  return (int)(((x + 1) * parts - 1) / total);
}

// One warp a row where a row has few pieces, else four that take its pieces in turn; D / 8 of a warp's lanes hold eight elements each.
template <typename T, int CODE, int W>
__global__ void __launch_bounds__(128) dps_join_kernel(const __grid_constant__ DpsJoinParams j) {
  wait_for_previous();
  __shared__ float sm[4], sl[4], so[4][256];
  const CacheArgs& ca = j.a.cache;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, col = lane * 8, D = ca.c.D;
  const long long row = W == 1 ? (long long)blockIdx.x * 4 + warp : blockIdx.x;
  if (row >= (long long)ca.c.B * ca.c.N * ca.c.n) return;
  const int i = (int)(row % ca.c.n), head = (int)(row / ca.c.n % ca.c.N), b = (int)(row / ca.c.n / ca.c.N);
  const LineEntry e = j.table[b], end = j.table[ca.c.B - 1];
  const long long total = end.base + (long long)end.line.groups * end.line.tiles * ca.c.N;
  const int parts = parts_of(total, j.ctas);
  float m = -INFINITY, l = 0.f, f[8];
#pragma unroll
  for (int k = 0; k < 8; ++k) f[k] = 0.f;
  if (i < e.line.cnt) {
    const long long grp = (long long)head * e.line.groups + i / j.queries, first = e.base + grp * e.line.tiles;
    // CTA c has the steps from c total / parts to the next one's.  A lane looks at a piece's maximum and sum; then the results are added
    // up, four pieces' loads in flight
    const int c0 = cta_of(first, total, parts), count = cta_of(first + e.line.tiles - 1, total, parts) - c0 + 1;
    const float* part = j.part + ((size_t)(e.group_base + grp + c0) * j.queries + i % j.queries) * (D + 2);
    const size_t pitch = (size_t)j.queries * (D + 2);
    for (int k0 = W == 1 ? 0 : warp * 32; k0 < count; k0 += 32 * W) {
      const int mine = k0 + lane, here = count - k0 < 32 ? count - k0 : 32;
      float mp = -INFINITY, lp = 0.f;
      if (mine < count) mp = part[mine * pitch], lp = part[mine * pitch + 1];
      float mn = fmaxf(m, mp);
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) mn = fmaxf(mn, __shfl_xor_sync(0xffffffffu, mn, o));
      const float w0 = m == -INFINITY ? 0.f : exp2f(m - mn);
      // (a piece that has seen nothing has written no result; a maximum of -infinity with a sum of NaN is of a row that reads as NaN)
      const float w1 = mp == -INFINITY ? 0.f : exp2f(mp - mn);
      float add = mp == -INFINITY ? (lp != lp ? lp : 0.f) : lp * w1;
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) add += __shfl_xor_sync(0xffffffffu, add, o);
      l = (m == -INFINITY && l == 0.f ? 0.f : l * w0) + add;
#pragma unroll
      for (int k = 0; k < 8; ++k) f[k] *= w0;
#pragma unroll 1
      for (int q = 0; q < here; q += 4) {
        float2 v[4][4];
#pragma unroll
        for (int u = 0; u < 4; ++u)
#pragma unroll
          for (int k = 0; k < 4; ++k)
            v[u][k] = q + u < here && col < D ? *reinterpret_cast<const float2*>(part + (k0 + q + u) * pitch + 2 + col + 2 * k) : make_float2(0.f, 0.f);
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          const float w = __shfl_sync(0xffffffffu, w1, (q + u) & 31);
          if (q + u >= here || w == 0.f) continue;
#pragma unroll
          for (int k = 0; k < 4; ++k) f[2 * k] = fmaf(v[u][k].x, w, f[2 * k]), f[2 * k + 1] = fmaf(v[u][k].y, w, f[2 * k + 1]);
        }
      }
      m = mn;
    }
  }
  if constexpr (W > 1) {
    if (lane == 0) sm[warp] = m, sl[warp] = l;
#pragma unroll
    for (int k = 0; k < 8; ++k)
      if (col < D) so[warp][col + k] = f[k];
    __syncthreads();
    if (warp) return;
    m = -INFINITY, l = 0.f;
#pragma unroll
    for (int w = 0; w < 4; ++w) m = fmaxf(m, sm[w]);
#pragma unroll
    for (int k = 0; k < 8; ++k) f[k] = 0.f;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const float x = sm[w] == -INFINITY ? (sl[w] != sl[w] ? 1.f : 0.f) : exp2f(sm[w] - m);
      l += x == 0.f ? 0.f : sl[w] * x;
#pragma unroll
      for (int k = 0; k < 8; ++k)
        if (col < D && x != 0.f) f[k] = fmaf(so[w][col + k], x, f[k]);
    }
  }
  const bool none = m == -INFINITY && l == 0.f;
  const float inv = none ? 0.f : 1.f / l, lse = none ? -INFINITY : l != l ? l : (m + log2f(l)) * kLn2;
#pragma unroll
  for (int k = 0; k < 8; ++k) f[k] = none ? 0.f : f[k] * inv;
  if (j.o) {
    if (col < D) store8((T*)j.o + (size_t)row * D + col, f);
    if (j.lse && lane == 0) j.lse[row] = lse;
    return;
  }
  join_into_cache<T, CODE>(ca, b, head, i, col, f, lse, j.v2);
}

constexpr int most_tiles(int D) { return D == 64 ? 4 : 3; }   // of 8 queries, by registers

struct Plan {
  int groups, tiles;
};
Plan plan_of(int n, int D) {
  const int all = (n + 7) / 8, groups = (all + most_tiles(D) - 1) / most_tiles(D);
  return Plan{groups, (all + groups - 1) / groups};
}
size_t table_bytes(const tritt_cache_t& c) { return align_up((size_t)c.B * sizeof(LineEntry), 256); }

template <int D, int CODE, int NT, bool ONE, bool EXACT> int launch_kernel(Params p, cudaStream_t stream, int& ctas) {
  auto kern = dps_decode_kernel<D, CODE, NT, ONE, EXACT>;
  constexpr int kSmem = smem_bytes<D, CODE, NT>();
  TRITT_CUDA_OK(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem));
  p.ctas = ctas = num_sms() * kBlocksPerSm<NT>;
  return launch_kernel_after(kern, dim3(ctas), kWarps * 32, kSmem, stream, p.early, p);
}
template <int D, int CODE, int NT> int launch(const Params& p, cudaStream_t stream, int& ctas) {
  if constexpr (NT == 1) {
    if (p.a.cache.c.n == 1)
      return p.a.exact ? launch_kernel<D, CODE, 1, true, true>(p, stream, ctas) : launch_kernel<D, CODE, 1, true, false>(p, stream, ctas);
  }
  return p.a.exact ? launch_kernel<D, CODE, NT, false, true>(p, stream, ctas) : launch_kernel<D, CODE, NT, false, false>(p, stream, ctas);
}
template <int D, int CODE> int by_tiles(const Params& p, int tiles, cudaStream_t stream, int& ctas) {
  switch (tiles) {
    case 1: return launch<D, CODE, 1>(p, stream, ctas);
    case 2: return launch<D, CODE, 2>(p, stream, ctas);
    case 3: return launch<D, CODE, 3>(p, stream, ctas);
    default:
      if constexpr (most_tiles(D) >= 4) return launch<D, CODE, 4>(p, stream, ctas);
      return -1;
  }
}
template <int D> int by_code(const Params& p, int tiles, cudaStream_t stream, int& ctas) {
  if (p.a.cache.c.code == TRITT_CODE_F16) return by_tiles<D, TRITT_CODE_F16>(p, tiles, stream, ctas);
  return p.a.cache.c.code == TRITT_CODE_E4M3 ? by_tiles<D, TRITT_CODE_E4M3>(p, tiles, stream, ctas) : by_tiles<D, TRITT_CODE_INT8>(p, tiles, stream, ctas);
}

template <typename T, int CODE> int launch_dps_join(const DpsJoinParams& j, cudaStream_t stream) {
  const long long rows = (long long)j.a.cache.c.B * j.a.cache.c.N * j.a.cache.c.n;
  // (a row has about ctas / groups of new tokens pieces and one more; four warps share more than 64 of them)
  if (rows / j.a.cache.c.n * 64 < j.ctas)
    return launch_kernel_after(dps_join_kernel<T, CODE, 4>, dim3((unsigned)rows), 128, 0, stream, true, j);
  return launch_kernel_after(dps_join_kernel<T, CODE, 1>, dim3((unsigned)((rows + 3) / 4)), 128, 0, stream, true, j);
}
template <typename T> int join_by_code(const DpsJoinParams& j, cudaStream_t s) {
  const int code = j.a.cache.c.code;
  if (code == TRITT_CODE_F16) return launch_dps_join<T, TRITT_CODE_F16>(j, s);
  return code == TRITT_CODE_E4M3 ? launch_dps_join<T, TRITT_CODE_E4M3>(j, s) : launch_dps_join<T, TRITT_CODE_INT8>(j, s);
}

}  // namespace

bool mma_dps_decode_supported(int D, int dtype) { return (D == 64 || D == 128) && (dtype == TRITT_F16 || dtype == TRITT_BF16); }

size_t mma_dps_decode_workspace(const tritt_cache_t& c) {
  const Plan plan = plan_of(c.n, c.D);
  return table_bytes(c) + align_up((size_t)((long long)c.B * c.N * plan.groups + 4 * num_sms()) * 8 * plan.tiles * (c.D + 2) * 4, 256);
}

int mma_dps_decode(const DpsDecodeArgs& a, void* workspace, void* o, float* lse, const tritt_rows_t* v2, bool early, cudaStream_t stream) {
  const tritt_cache_t& c = a.cache.c;
  const Plan plan = plan_of(c.n, c.D);
  const Params p{a, (LineEntry*)workspace, (float*)((char*)workspace + table_bytes(c)), 0, early};
  int ctas = 0;
  if (int rc = c.D == 64 ? by_code<64>(p, plan.tiles, stream, ctas) : by_code<128>(p, plan.tiles, stream, ctas)) return rc;
  const DpsJoinParams j{a, p.table, p.part, ctas, 8 * plan.tiles, o, lse, v2 ? *v2 : tritt_rows_t{}};
  return a.dtype == TRITT_F16 ? join_by_code<__half>(j, stream) : join_by_code<__nv_bfloat16>(j, stream);
}

}  // namespace tritt
