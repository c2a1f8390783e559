// One soft-max attention of new tokens over two parts of the quantised cache, 16-bit queries, head dimension 64 or 128: either leg of the
// dot-product-sum form (append: rows k2 over K1, SiLU(V1) within a window;  decode: rows q over K2, W with a bias for each token).
//
// Bound by HBM: a cached row is read once for up to 8 NT new tokens, 2 flops a byte and token.  Each warp has a ring of its own in
// shared memory, filled by bulk copies (16 rows each, whole pages' neighbours) and 4-byte asynchronous ones (exponents, biases): no registers
// wait for memory and nearly no instructions address it (a first form with loads to registers executed 1046 instructions for 32
// tokens, more than HBM leaves time for: 253 us for a token of 32 x 8191).  Rows then go, as fp16, into warp-level matrix
// instructions with the cached rows as the 16-row operand:
//   S^T[16 tokens x 8 queries] = K Q^T,   O^T[D x 8 queries] += V^T P^T
// (one token is an eighth of a tile instead of a sixteenth, and a query's statistics lie in the threads that hold its results).  The contraction of S
// runs over the head dimension in any order, so a thread takes 16 contiguous bytes of a row for the elements that it needs; the rows of
// V^T are columns of V in any order, so a thread takes D / 8 contiguous elements of four tokens and pairs them by byte permutes.  P^T is
// the transpose of S^T's fragments (movmatrix).  A warp walks its tiles of tokens with the next keys and values in flight.
//
// Codes are exact as fp16, the scores' powers of two are applied in fp32; P is formed times 2^(its row's exponent - the largest so far + 13),
// so that values of any size meet in one accumulator, and its sum is taken before that.  Queries are brought to [1, 2) by a power of two.
// Append forms P as the sum of two fp16 numbers (22 bits): its result is rounded again, to codes, and each element that a less exact one moves over
// a border is off by a whole step (e4m3: 0.13 % of W's norm with one fp16 number, 2e-5 with two).
#include "tritt_cache.cuh"
#include "tritt_sm100.cuh"

namespace tritt {
namespace {
using namespace sm100;

constexpr int kWarps = 4;
constexpr int kLift = 13;

struct Params {
  DpsDecodeArgs a;
  int query_groups;   // of 8 NT new tokens
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
  static constexpr int kTokens = kRowBytes == 256 ? 16 : 32;    // of a tile: 4 or 8 KB of keys and values
  static constexpr int kBlocks = kTokens / 16;
  static constexpr int kKeyLoads = kRowBytes / 64;              // of 16 bytes, of a lane's row
  static constexpr int kValueWords = kRowBytes / 32;            // 32-bit words of a lane's eighth of a row
  // a stage of the ring: keys, values, then biases, exponents of keys and values, and which tokens are there
  static constexpr int kOffV = kTokens * kRowBytes, kOffBias = 2 * kOffV, kOffEk = kOffBias + 128, kOffEv = kOffEk + 32, kOffThere = kOffEv + 32;
  static constexpr int kStage = kOffBias + 256;
  static constexpr int kStages = 3;
  static constexpr int kSmem = kWarps * kStages * kStage;
};

// Copies of four bytes, and their arrival at a barrier.
__device__ __forceinline__ void copy4(void* dst, const void* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(smem_u32(dst)), "l"(src) : "memory");
}
__device__ __forceinline__ void copies_arrive(uint64_t* bar) {
  asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}

template <int D, int CODE, int NT> constexpr int blocks_per_sm() {   // by registers and shared memory
  return Shape<D, CODE>::kRowBytes == 64 ? (NT == 1 ? 4 : NT == 2 ? 3 : 2) : 2;
}

template <int D, int CODE, int NT, bool EXACT>
__global__ void __launch_bounds__(kWarps * 32, blocks_per_sm<D, CODE, NT>()) dps_decode_kernel(const __grid_constant__ Params p) {
  using S = Shape<D, CODE>;
  constexpr int NB = S::kBlocks, TK = S::kTokens, KL = S::kKeyLoads, VW = S::kValueWords, NS = S::kStages;
  constexpr int Q = 8 * NT;
  extern __shared__ __align__(128) uint8_t ring_all[];
  __shared__ uint64_t s_full[kWarps][NS];
  __shared__ int s_abort;
  __shared__ float4 s_side[kWarps][TK];   // of a tile's tokens: scale of scores, bias, scale of P
  __shared__ unsigned long long s_word[Q];
  __shared__ int s_lo[Q], s_pos[Q];
  __shared__ float s_scale[Q], s_m[kWarps][Q], s_l[kWarps][Q], s_out[Q][D + 4];
  const DpsDecodeArgs& a = p.a;
  const CacheArgs& ca = a.cache;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  const int head = blockIdx.y % ca.c.N, b = blockIdx.y / ca.c.N, split = blockIdx.x, i0 = blockIdx.z * Q;
  const int ctx = context_of(ca, b), cnt = new_tokens(ca, b), nq = min(Q, cnt - i0);
  const int rows = min(Q, ca.c.n - i0);   // rows of the result
  float* part = a.part + (((size_t)blockIdx.y * ca.c.n + i0) * a.splits + split) * (D + 2);
  const size_t pitch = (size_t)a.splits * (D + 2);

  // tokens that any of these queries attends to: first .. end - 1, in tiles from a multiple of 16 on
  const int first = nq > 0 ? max(0, min(ctx, ctx + (ca.c.ancestors ? 0 : i0) - a.window)) & ~15 : 0, end = nq > 0 ? ctx + i0 + nq : 0;
  const int tiles = (end - first + TK - 1) / TK, each = (tiles + a.splits - 1) / a.splits;
  const int tile0 = split * each, tile1 = min(tiles, tile0 + each);
  if (tile0 >= tile1) {
    for (int i = tid; i < rows; i += kWarps * 32) part[i * pitch] = -INFINITY, part[i * pitch + 1] = 0.f;
    return;
  }

  // --- the ring: this warp takes tiles tile0 + warp, + kWarps, ...
  uint8_t* ring = ring_all + warp * NS * S::kStage;
  uint64_t* full = s_full[warp];
  if (lane == 0) {
    for (int i = 0; i < NS; ++i) mbar_init(&full[i], 33);   // one arrival with the bulk copies' bytes, one of each lane
    fence_barrier_init();
  }
  if (tid == 0) s_abort = 0;
  const size_t part_rows = (size_t)ca.c.N << ca.page_log2;   // rows of one part of a page
  const int row_mask = ca.c.page_size - 1;
  // the page of this lane's token of a tile, -1: none, or no such token
  auto find_page = [&](int tile) {
    const int token = first + tile * TK + lane;
    return lane < TK && tile < tile1 && token < end ? place_of(ca, b, token).page : -1;
  };
  auto fill = [&](int tile, int st, int page) {
    uint8_t* to = ring + st * S::kStage;
    const uint32_t there = __ballot_sync(0xffffffffu, page >= 0);
    // (a group of 16 tokens lies in one page; its first token is there if any is)
    if (lane == 0) {
      *reinterpret_cast<uint32_t*>(to + S::kOffThere) = there;
      mbar_arrive_expect_tx(&full[st], (uint32_t)(((there & 1u) + (there >> 16 & 1u)) * 2 * 16 * S::kRowBytes));
    }
    __syncwarp();
    if (page >= 0) {
      const int r = (first + tile * TK + lane) & row_mask;
      const size_t at = (size_t)page * 4 * part_rows + ((size_t)head << ca.page_log2) + r;   // of part 0
      // lanes 0, 16 copy a group's keys, lanes 1, 17 its values (lane 1's token may be behind the last: then lane 0 copies both)
      const bool second = there >> (lane | 1) & 1;
      if ((lane & 15) == 0) {
        bulk_load(to + lane * S::kRowBytes, (const uint8_t*)ca.c.codes + (at + a.key_part * part_rows) * S::kRowBytes, 16 * S::kRowBytes, &full[st]);
        if (!second)
          bulk_load(to + S::kOffV + lane * S::kRowBytes, (const uint8_t*)ca.c.codes + (at + a.value_part * part_rows) * S::kRowBytes,
                    16 * S::kRowBytes, &full[st]);
      } else if ((lane & 15) == 1) {
        bulk_load(to + S::kOffV + (lane - 1) * S::kRowBytes,
                  (const uint8_t*)ca.c.codes + (at - 1 + a.value_part * part_rows) * S::kRowBytes, 16 * S::kRowBytes, &full[st]);
      }
      if (a.biased) copy4(to + S::kOffBias + lane * 4, ca.c.lse + (((size_t)page * ca.c.N + head) << ca.page_log2) + r);
      if ((lane & 3) == 0) {
        copy4(to + S::kOffEk + lane, ca.c.exponents + at + a.key_part * part_rows);
        copy4(to + S::kOffEv + lane, ca.c.exponents + at + a.value_part * part_rows);
      }
    }
    copies_arrive(&full[st]);
  };
  __syncwarp();
  int next_page;   // of the tile that is filled next
  {
    int pg[NS + 1];
#pragma unroll
    for (int i = 0; i <= NS; ++i) pg[i] = find_page(tile0 + warp + i * kWarps);
#pragma unroll
    for (int i = 0; i < NS; ++i)
      if (tile0 + warp + i * kWarps < tile1) fill(tile0 + warp + i * kWarps, i, pg[i]);
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
    const size_t off = on ? rows_at(a.q, b, head, i) : 0;
    constexpr int EPL = S::kWide ? 8 : 16;   // elements of 16 bytes of codes
#pragma unroll
    for (int j = 0; j < D / (4 * EPL); ++j)
#pragma unroll
      for (int c = 0; c < EPL / 8; ++c) {
        float x[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = 0.f;
        const size_t at = off + j * 4 * EPL + t * EPL + c * 8;
        if (on) {
          if (a.dtype == TRITT_F16)
            load8((const __half*)a.q.p + at, x);
          else
            load8((const __nv_bfloat16*)a.q.p + at, x);
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          f[j * EPL + c * 8 + e] = x[e];
          big = max(big, __float_as_uint(x[e]) & 0x7fffffffu);
        }
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
      const unsigned long long word = on && ca.c.ancestors ? seen_word(ca, b, i) : 0;
      const int pos = ctx + (ca.c.ancestors ? __popcll(word) - 1 : i);
      s_word[nt * 8 + g] = word;
      s_pos[nt * 8 + g] = on ? pos : -1;
      s_lo[nt * 8 + g] = on ? max(0, pos - a.window) : 0x7fffffff;
      s_scale[nt * 8 + g] = a.scale2 * __uint_as_float((uint32_t)(254 - up) << 23);
    }
  }
  __syncthreads();
  // from lo_all on every query attends to all of the context (those that are not there take no part in this: their results are not looked at)
  int lo_all = 0;
  for (int i = 0; i < nq; ++i) lo_all = max(lo_all, s_lo[i]);
  float qs[NT][2];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    qs[nt][0] = s_scale[nt * 8 + 2 * t];
    qs[nt][1] = s_scale[nt * 8 + 2 * t + 1];
  }

  float acc[NT][D / 16][4], m[NT][2], l[NT][2];
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
    for (int mb = 0; mb < D / 16; ++mb)
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[nt][mb][e] = 0.f;
    m[nt][0] = m[nt][1] = -INFINITY;
    l[nt][0] = l[nt][1] = 0.f;
  }
  int v_exp = 0;   // largest exponent byte of the values so far
  int st = 0, phase = 0;
  for (int tile = tile0 + warp; tile < tile1; tile += kWarps) {
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
    // one lane a token: scales, and whether all of the tile counts for every query
    const uint32_t there = *reinterpret_cast<const uint32_t*>(from + S::kOffThere);
    bool plain = token0 >= lo_all && token0 + TK <= ctx;
    uint32_t bad;
    {
      const bool on = lane < TK && (there >> lane & 1);
      const int ek = on ? from[S::kOffEk + lane] : 0, ev = on ? from[S::kOffEv + lane] : 0;
      const float bias = on && a.biased ? *reinterpret_cast<const float*>(from + S::kOffBias + lane * 4) * kLog2e : 0.f;
      bad = __ballot_sync(0xffffffffu, ek == 255 || ev == 255);
      const int most = max(v_exp, (int)__reduce_max_sync(0xffffffffu, ev == 255 ? 0 : ev));
      plain = plain && there == (TK == 32 ? 0xffffffffu : 0xffffu) && bad == 0u;
      // (the products lie in the accumulator times 2^(largest exponent))
      if (most > v_exp) {
        const float grown = v_exp ? power(v_exp - most) : 1.f;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int mb = 0; mb < D / 16; ++mb)
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[nt][mb][e] *= grown;
        v_exp = most;
      }
      if (lane < TK) s_side[warp][lane] = make_float4(power(ek - 127), bias, ev == 255 || !on ? 0.f : power(ev - most + kLift), 0.f);
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
#pragma unroll
      for (int j = 0; j < KL; ++j) {
        const uint4 r0 = *reinterpret_cast<const uint4*>(from + (nb * 16 + g) * S::kRowBytes + j * 64 + t * 16);
        const uint4 r1 = *reinterpret_cast<const uint4*>(from + (nb * 16 + 8 + g) * S::kRowBytes + j * 64 + t * 16);
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
        const int k = nb * 16 + h * 8 + g;
        const float4 side = s_side[warp][k];
        vf[nb][h] = side.z;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int q = 0; q < 2; ++q) s[nt][nb][2 * h + q] = fmaf(s[nt][nb][2 * h + q] * side.x, qs[nt][q], side.y);
        if (!plain) {
          const int token = token0 + k;
          bool missing = false;
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int q = 0; q < 2; ++q) {
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
              missing = missing || (seen && !(there >> k & 1));
              float& x = s[nt][nb][2 * h + q];
              x = seen && (there >> k & 1) ? (bad >> k & 1 ? __uint_as_float(0x7fffffffu) : x) : -INFINITY;
            }
          if (missing && ca.status) atomicOr(ca.status, kStatusPlace);
        }
      }
    // running maximum, P
    uint32_t pf[NT][NB][2], pl[EXACT ? NT : 1][NB][2];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      float base[2], corr[2];
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        float mx = m[nt][q];
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) mx = fmaxf(mx, fmaxf(s[nt][nb][q], s[nt][nb][2 + q]));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
        base[q] = mx == -INFINITY ? 0.f : mx;   // (nothing attended so far: all P are 0)
        corr[q] = exp2f(m[nt][q] - base[q]);
        m[nt][q] = mx;
        l[nt][q] *= corr[q];
      }
      if (__any_sync(0xffffffffu, corr[0] != 1.f || corr[1] != 1.f)) {
#pragma unroll
        for (int mb = 0; mb < D / 16; ++mb)
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[nt][mb][e] *= corr[e & 1];
      }
#pragma unroll
      for (int nb = 0; nb < NB; ++nb)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const float p0 = exp2f(s[nt][nb][2 * h] - base[0]), p1 = exp2f(s[nt][nb][2 * h + 1] - base[1]);
          l[nt][0] += p0;
          l[nt][1] += p1;
          const float x0 = p0 * vf[nb][h], x1 = p1 * vf[nb][h];
          const uint32_t high = pack_half(x0, x1);
          pf[nt][nb][h] = transposed(high);
          if constexpr (EXACT) {
            const float2 r = __half22float2(*reinterpret_cast<const __half2*>(&high));
            pl[nt][nb][h] = transposed(pack_half(x0 - r.x, x1 - r.y));
          }
        }
    }
    // O^T += V^T P^T
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
      // of tokens 2t, 2t + 1, 2t + 8, 2t + 9 of the block, the g-th eighth of the row
      uint32_t v[4][VW];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int row = nb * 16 + (k >> 1) * 8 + 2 * t + (k & 1);
        const uint8_t* r = from + S::kOffV + row * S::kRowBytes + g * (VW * 4);
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
        if (!plain && !(there >> row & 1)) {   // (what lies there is of another tile, or no number)
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
    for (int q = 0; q < 2; ++q) {
      l[nt][q] += __shfl_xor_sync(0xffffffffu, l[nt][q], 4);
      l[nt][q] += __shfl_xor_sync(0xffffffffu, l[nt][q], 8);
      l[nt][q] += __shfl_xor_sync(0xffffffffu, l[nt][q], 16);
      if (g == 0) {
        s_m[warp][nt * 8 + 2 * t + q] = m[nt][q];
        s_l[warp][nt * 8 + 2 * t + q] = l[nt][q];
      }
    }
  for (int i = tid; i < Q * (D + 4); i += kWarps * 32) (&s_out[0][0])[i] = 0.f;
  __syncthreads();
  for (int w = 0; w < kWarps; ++w) {
    if (warp == w && v_exp > 0) {
      // (exponents of values only scale the accumulator; a warp without a value has v_exp 0 and nothing to add)
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int q = 0; q < 2; ++q) {
          const int i = nt * 8 + 2 * t + q;
          float top = -INFINITY;
          for (int k = 0; k < kWarps; ++k) top = fmaxf(top, s_m[k][i]);
          const float f = m[nt][q] == -INFINITY ? 0.f : exp2f(m[nt][q] - top) * power(v_exp - 127) * (1.f / (1 << kLift));
#pragma unroll
          for (int mb = 0; mb < D / 16; ++mb) {
            s_out[i][g * (D / 8) + 2 * mb] += f == 0.f ? 0.f : acc[nt][mb][q] * f;
            s_out[i][g * (D / 8) + 2 * mb + 1] += f == 0.f ? 0.f : acc[nt][mb][2 + q] * f;
          }
        }
    }
    __syncthreads();
  }
  for (int i = warp; i < rows; i += kWarps) {
    float top = -INFINITY, sum = 0.f;
    for (int k = 0; k < kWarps; ++k) top = fmaxf(top, s_m[k][i]);
    for (int k = 0; k < kWarps; ++k)
      sum += s_m[k][i] == -INFINITY ? (s_l[k][i] != s_l[k][i] ? s_l[k][i] : 0.f) : s_l[k][i] * exp2f(s_m[k][i] - top);
    float* out = part + i * pitch;
    if (i >= nq) top = -INFINITY, sum = 0.f;   // (behind the sequence's last new token)
    if (lane == 0) out[0] = top, out[1] = sum;
    for (int c = lane; c < D; c += 32) out[2 + c] = s_out[i][c];
  }
}

constexpr int most_tiles(int D) { return D == 64 ? 4 : 3; }   // of 8 queries, by registers

struct Plan {
  int groups, tiles;
};
Plan plan_of(int n, int D) {
  const int all = (n + 7) / 8, groups = (all + most_tiles(D) - 1) / most_tiles(D);
  return Plan{groups, (all + groups - 1) / groups};
}

template <int D, int CODE, int NT> int launch(const Params& p, cudaStream_t stream) {
  auto kern = p.a.exact ? dps_decode_kernel<D, CODE, NT, true> : dps_decode_kernel<D, CODE, NT, false>;
  TRITT_CUDA_OK(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, Shape<D, CODE>::kSmem));
  kern<<<dim3(p.a.splits, p.a.cache.c.B * p.a.cache.c.N, p.query_groups), kWarps * 32, Shape<D, CODE>::kSmem, stream>>>(p);
  count_launch();
  TRITT_CUDA_OK(cudaGetLastError());
  return 0;
}
template <int D, int CODE> int by_tiles(const Params& p, int tiles, cudaStream_t stream) {
  switch (tiles) {
    case 1: return launch<D, CODE, 1>(p, stream);
    case 2: return launch<D, CODE, 2>(p, stream);
    case 3: return launch<D, CODE, 3>(p, stream);
    default:
      if constexpr (most_tiles(D) >= 4) return launch<D, CODE, 4>(p, stream);
      return -1;
  }
}
template <int D> int by_code(const Params& p, int tiles, cudaStream_t stream) {
  if (p.a.cache.c.code == TRITT_CODE_F16) return by_tiles<D, TRITT_CODE_F16>(p, tiles, stream);
  return p.a.cache.c.code == TRITT_CODE_E4M3 ? by_tiles<D, TRITT_CODE_E4M3>(p, tiles, stream) : by_tiles<D, TRITT_CODE_INT8>(p, tiles, stream);
}

}  // namespace

bool mma_dps_decode_supported(int D, int dtype) { return (D == 64 || D == 128) && (dtype == TRITT_F16 || dtype == TRITT_BF16); }

// Blocks for the chip four times over (three or four blocks an SM), so that sequences of unequal length even out; a split has at least 256 tokens.
int mma_dps_decode_splits(const tritt_cache_t& c) {
  const long long rows = (long long)c.B * c.N * plan_of(c.n, c.D).groups, want = (4 * 4 * 148 + rows - 1) / rows;
  const long long most = ((long long)c.page_size * c.table_pages + 255) / 256;
  const long long s = want < most ? want : most;
  return (int)(s < 1 ? 1 : s > 64 ? 64 : s);
}

int mma_dps_decode(const DpsDecodeArgs& a, cudaStream_t stream) {
  const Plan plan = plan_of(a.cache.c.n, a.cache.c.D);
  const Params p{a, plan.groups};
  return a.cache.c.D == 64 ? by_code<64>(p, plan.tiles, stream) : by_code<128>(p, plan.tiles, stream);
}

}  // namespace tritt
