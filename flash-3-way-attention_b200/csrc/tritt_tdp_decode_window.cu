// Triple-dot-product attention of new tokens over the cache where all that they attend to fits in shared memory: narrow windows, or
// short tables.
//
// A block takes some new tokens of one sequence and head.  The tokens of a tree or chain see almost the same window, so their rows of
// the cache are read and converted once: K1 and SiLU(V1) as fp16 with one power of two for each part, K2 and V2 as fp16 codes.  A warp takes 16
// rows k of one new token at a time (m16n8k16 products, A = alpha q*K2 formed in registers), walks the 32-column blocks j that any of them
// attends to, and sums its rows times V2; the sums of a new token meet in shared memory, in order, and leave as the result: one launch.
//
// Bound by instruction issue (2000 a unit of 16 rows under a window of 129 and a band of 65, staging included: 54 % of the issue slots) and, for few rows, by the
// chain load, convert, product, exponential.  Trees of 16 under windows 128/128/32/32, 8 sequences of 16 heads, D=64, int8, fp16
// queries: 68 us (61 with bfloat16's); the kernel with tcgen05 tiles of 128 x 128 cells, which such a window fills to a half: 120.
#include "tritt_cache.cuh"
#include "tritt_sm100.cuh"
#include "tritt_sm100_tdp.cuh"

#include <type_traits>

namespace tritt {
namespace {
using namespace sm100;

constexpr int kWarps = 8;
constexpr float kGap = 8.f, kLift = 7.f;   // as in the other kernel: P times 2^7, the reference raised where a score is 2^8 above it
constexpr int kMostSmem = 200 * 1024;
constexpr int kPartBytes = 40 * 1024;      // of the sums of a block's units

struct WindowParams {
  TdpDecodeArgs a;
  void* o;
  float* lse;
  int tokens;        // new tokens of a block
  int cols, rows;    // places for staged tokens: columns j, rows k
  int tiles;         // of 16 rows, of a new token (the most)
};

template <int CODE> constexpr int kUp = CODE == TRITT_CODE_F16 ? 0 : CODE == TRITT_CODE_E4M3 ? 5 : 7;
template <int CODE> constexpr int kDown = CODE == TRITT_CODE_F16 ? 7 : 0;

__device__ __forceinline__ void mma_16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t mul_half2(uint32_t a, uint32_t b) {
  const __half2 r = __hmul2(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&b));
  return *reinterpret_cast<const uint32_t*>(&r);
}
// What the rounded product of `a` and `b` leaves of it (fp16 has it exactly)
__device__ __forceinline__ uint32_t rest_half2(uint32_t a, uint32_t b, uint32_t product) {
  const __half2 r = __hfma2(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&b), __hneg2(*reinterpret_cast<const __half2*>(&product)));
  return *reinterpret_cast<const uint32_t*>(&r);
}
__device__ __forceinline__ uint32_t half_power(int e) {   // 2^e as a pair of fp16 (0 below its range; e <= 15)
  const uint32_t h = e >= -14 ? (uint32_t)(e + 15) << 10 : e >= -24 ? 1u << (e + 24) : 0u;
  return h | h << 16;
}
// Byte offset of 16-byte chunk `chunk` of a staged row of D fp16 numbers.  Chunks change places with the row's number, so that both two rows' four
// chunks (the fragments of K1 and K2) and eight rows' one (ldmatrix of V1) lie in different banks.
template <int D> __device__ __forceinline__ int staged(int row, int chunk) {
  return row * (2 * D) + ((chunk ^ ((row & 1) << 2 | (row >> 1 & 3))) << 4);
}

template <typename T16, int D, int CODE>
__global__ void __launch_bounds__(kWarps * 32, D == 64 ? 2 : 1) tdp_decode_window_kernel(const __grid_constant__ WindowParams p) {
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ int s_most[2], s_least[2];   // exponents of the staged rows of K1 and of V1
  const TdpDecodeArgs& a = p.a;
  const CacheArgs& ca = a.cache;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
  const int head = blockIdx.x % ca.c.N, b = blockIdx.x / ca.c.N, i0 = blockIdx.y * p.tokens;
  const int ctx = context_of(ca, b), cnt = new_tokens(ca, b), ni = min(p.tokens, cnt - i0), want = min(p.tokens, ca.c.n - i0);
  // staged: K1, V1 [cols], K2, V2 [rows], then the exponent bytes of the rows' K2 and V2 and of the columns (0: not there, 255: NaN), queries,
  // their words, of each 32 columns those that are there and those that read as NaN, sums
  uint8_t* const sK1 = smem;
  uint8_t* const sV1 = sK1 + p.cols * 2 * D;
  uint8_t* const sK2 = sV1 + p.cols * 2 * D;
  uint8_t* const sV2 = sK2 + p.rows * 2 * D;
  uint8_t* const sEk2 = sV2 + p.rows * 2 * D;
  uint8_t* const sEv2 = sEk2 + p.rows;
  uint8_t* const sEk1 = sEv2 + p.rows;
  uint8_t* const sEv1 = sEk1 + p.cols;
  __half* const sQ = reinterpret_cast<__half*>(sEv1 + p.cols);          // [tokens][D]
  float* const sScale = reinterpret_cast<float*>(sQ + p.tokens * D);    // [tokens]
  unsigned long long* const sWord = reinterpret_cast<unsigned long long*>(sScale + (p.tokens + 1) / 2 * 2);   // [tokens]
  uint32_t* const sThere = reinterpret_cast<uint32_t*>(sWord + p.tokens);   // [cols / 32]
  uint32_t* const sNan = sThere + p.cols / 32;
  uint8_t* const sTree = reinterpret_cast<uint8_t*>(sNan + p.cols / 32);   // [tokens][64]: which new token is the d-th that a new token attends to
  float* const sPart = reinterpret_cast<float*>(sTree + (ca.c.ancestors ? p.tokens * 64 : 0));   // [tokens][tiles][D + 2]
  if (tid < 2) s_most[tid] = 0, s_least[tid] = 255;
  __syncthreads();

  // --- what these tokens attend to, by numbers in the sequence: columns lo_j .. end - 1, rows lo_k .. end - 1
  const int first_pos = ctx + (ca.c.ancestors ? 0 : i0);
  const int end = ni > 0 ? ctx + i0 + ni : 0, lo_j = max(0, min(ctx, first_pos - a.k1w)), lo_k = max(0, min(ctx, first_pos - a.k2w));
  const int nj = ni > 0 ? end - lo_j : 0, nk = ni > 0 ? end - lo_k : 0;
  constexpr int L = D / 8;   // lanes of a row
  // two parts of the same tokens; four rows of a thread at a time, whose loads overlap
  auto stage = [&](int part, int part2, int lo, int n, int places, uint8_t* to, uint8_t* to2, uint8_t* exps, uint8_t* exps2, bool columns) {
    constexpr int kStep = kWarps * 32 / L, kBatch = 4;
    const int ch = tid % L;
    for (int r0 = tid / L; r0 < (n + 31) / 32 * 32; r0 += kStep * kBatch) {
      int page[kBatch], e1[kBatch], e2[kBatch];
      Codes8<CODE> c1[kBatch], c2[kBatch];
#pragma unroll
      for (int k = 0; k < kBatch; ++k) {
        const int r = r0 + k * kStep;
        page[k] = r < n ? place_of(ca, b, lo + r).page : -1;
      }
#pragma unroll
      for (int k = 0; k < kBatch; ++k) {
        const size_t at = row_of(ca, Place{max(page[k], 0), (lo + r0 + k * kStep) & (ca.c.page_size - 1)}, part, head);
        const size_t at2 = at + (size_t)(part2 - part) * ((size_t)ca.c.N << ca.page_log2);
        constexpr int kBytes = D * (CODE == TRITT_CODE_F16 ? 2 : 1);
        c1[k].load((const uint8_t*)ca.c.codes + at * kBytes, ch * 8);
        c2[k].load((const uint8_t*)ca.c.codes + at2 * kBytes, ch * 8);
        e1[k] = __ldg(ca.c.exponents + at);
        e2[k] = __ldg(ca.c.exponents + at2);
      }
      int m1 = 0, m2 = 0, n1 = 255, n2 = 255;
#pragma unroll
      for (int k = 0; k < kBatch; ++k) {
        const int r = r0 + k * kStep;
        if (r >= places) break;
        uint32_t w1[4], w2[4];
        c1[k].halves(w1);
        c2[k].halves(w2);
        const uint32_t on = page[k] >= 0 ? 0xffffffffu : 0u;
        *reinterpret_cast<uint4*>(to + staged<D>(r, ch)) = make_uint4(w1[0] & on, w1[1] & on, w1[2] & on, w1[3] & on);
        *reinterpret_cast<uint4*>(to2 + staged<D>(r, ch)) = make_uint4(w2[0] & on, w2[1] & on, w2[2] & on, w2[3] & on);
        e1[k] = on ? max(e1[k], 1) : 0;   // (a row that nobody has written is one of zeros)
        e2[k] = on ? max(e2[k], 1) : 0;
        if (ch == 0) exps[r] = (uint8_t)e1[k], exps2[r] = (uint8_t)e2[k];
        m1 = max(m1, e1[k] == 255 ? 0 : e1[k]);
        m2 = max(m2, e2[k] == 255 ? 0 : e2[k]);
        n1 = min(n1, least_byte(e1[k]));
        n2 = min(n2, least_byte(e2[k]));
      }
      if (columns && ch == 0) atomicMax(&s_most[0], m1), atomicMax(&s_most[1], m2), atomicMin(&s_least[0], n1), atomicMin(&s_least[1], n2);
    }
  };
  stage(kPartK1, kPartV1, lo_j, nj, p.cols, sK1, sV1, sEk1, sEv1, true);
  stage(kPartK2, kPartV2, lo_k, nk, p.rows, sK2, sV2, sEk2, sEv2, false);
  // queries, brought to [1, 2)
  for (int i = warp; i < ni; i += kWarps) {
    constexpr int E = D / 32;
    const T16* q = (const T16*)a.q.p + rows_at(a.q, b, head, i0 + i) + lane * E;
    float f[E];
    uint32_t big = 0;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      f[e] = to_f(q[e]);
      big = max(big, __float_as_uint(f[e]) & 0x7fffffffu);
    }
    big = __reduce_max_sync(0xffffffffu, big);
    const int power = max(min(254 - (int)(big >> 23), 253), 1);
    const float up = __uint_as_float((uint32_t)power << 23) * (a.scale2 < 0.f ? -1.f : 1.f);
#pragma unroll
    for (int e = 0; e < E; e += 2) *reinterpret_cast<uint32_t*>(sQ + i * D + lane * E + e) = pack2<__half>(f[e] * up, f[e + 1] * up);
    const unsigned long long word = ca.c.ancestors ? seen_word(ca, b, i0 + i) : 0;
    if (lane == 0) sWord[i] = word;
    if (ca.c.ancestors) {
#pragma unroll
      for (int m = lane; m < 64; m += 32)
        if (word >> m & 1) sTree[i * 64 + __popcll(word & ((1ull << m) - 1))] = (uint8_t)m;
    }
    if (lane == 0) sScale[i] = fabsf(a.scale2) * __uint_as_float((uint32_t)(254 - power) << 23) * (float)(1 << kDown<CODE>);
  }
  __syncthreads();
  // K1 and V1 to the largest exponent of all staged rows, where they are near enough to each other (else, trees of 16 as above with one row 2^40 larger: 92 us,
  // not 68)
  const int ek1 = s_most[0], ev1 = s_most[1];
  const bool wide_k = ek1 - s_least[0] > kSpread<CODE>, wide_v = ev1 - s_least[1] > kSpread<CODE>;
  {
    auto bring = [&](uint8_t* at, const uint8_t* exps, int most, bool wide) {
      for (int x = tid; x < nj * L; x += kWarps * 32) {
        const int r = x / L, byte = exps[r];
        const uint32_t f = half_power(wide ? kUp<CODE> : kUp<CODE> + (byte == 255 ? 0 : byte) - most);
        uint4& v = *reinterpret_cast<uint4*>(at + staged<D>(r, x % L));
        v = make_uint4(mul_half2(v.x, f), mul_half2(v.y, f), mul_half2(v.z, f), mul_half2(v.w, f));
      }
    };
    bring(sK1, sEk1, ek1, wide_k);
    bring(sV1, sEv1, ev1, wide_v);
    for (int w = warp; w < (nj + 31) / 32; w += kWarps) {
      const int e1 = sEk1[w * 32 + lane], e2 = sEv1[w * 32 + lane];
      const uint32_t there = __ballot_sync(0xffffffffu, e1 && e2), nan = __ballot_sync(0xffffffffu, e1 == 255 || e2 == 255);
      if (lane == 0) sThere[w] = there, sNan[w] = nan;
    }
  }
  __syncthreads();
  const float k1_scale = wide_k ? 1.f : ek1 > kUp<CODE> ? __uint_as_float((uint32_t)(ek1 - kUp<CODE>) << 23) : 0.f;

  // (staged rows from a multiple of 8 on: where a thread's chunks lie does not change)
  const uint8_t* key_at[D / 32];
  uint32_t value_at[D / 16];
#pragma unroll
  for (int j = 0; j < D / 32; ++j) key_at[j] = sK1 + staged<D>(g, j * 4 + t);
#pragma unroll
  for (int d = 0; d < D / 16; ++d) value_at[d] = smem_u32(sV1 + staged<D>(lane & 15, d * 2 + (lane >> 4)));

  // --- units: 16 rows of one new token
  for (int u = warp; u < ni * p.tiles; u += kWarps) {
    const int i = u / p.tiles, row0 = u % p.tiles * 16;
    float* const out = sPart + (size_t)u * (D + 2);
    const unsigned long long word = sWord[i];
    const int pos_q = ctx + (ca.c.ancestors ? __popcll(word) - 1 : i0 + i), klo = max(0, pos_q - a.k2w);
    if (klo + row0 > pos_q) {   // (fewer rows than the most)
      if (lane == 0) out[0] = -INFINITY, out[1] = 0.f;
      continue;
    }
    // this thread's rows g and g + 8: staged place, scale, and columns that they attend to
    int place[2], c_lo[2], c_hi[2];
    float scale[2], vweight[2];
    unsigned long long tree[2];
    bool nan[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int pk = klo + row0 + g + h * 8;
      int token = pk;
      if (ca.c.ancestors && pk >= ctx && pk <= pos_q) token = ctx + sTree[i * 64 + pk - ctx];
      bool on = pk <= pos_q;
      place[h] = on ? token - lo_k : 0;
      const int e1 = sEk2[place[h]], e2 = sEv2[place[h]];
      if (on && (e1 == 0 || e2 == 0)) {
        on = false;
        if (ca.status) atomicOr(ca.status, kStatusPlace);
      }
      nan[h] = e1 == 255 || e2 == 255;   // (or, below, of a column that the row attends to)
      scale[h] = on && e1 != 255 ? sScale[i] * __uint_as_float((uint32_t)e1 << 23) * k1_scale : 0.f;
      vweight[h] = on && e2 != 255 ? exp2f((float)(e2 - 127)) : 0.f;
      const int last = pk < (1 << 30) - a.kkr ? min(pos_q, pk + a.kkr) : pos_q;
      c_lo[h] = on ? max(max(0, pos_q - a.k1w), pk - min(pk, a.kkl)) : 1 << 30;
      c_hi[h] = !on ? -1 : ca.c.ancestors ? min(ctx - 1, last) : last;
      tree[h] = 0;
      if (on && ca.c.ancestors && last >= ctx && last >= c_lo[h])   // (its tokens between the first and the last of the window)
        tree[h] = word & (~0ull << sTree[i * 64 + max(c_lo[h] - ctx, 0)]) & (~0ull >> (63 - sTree[i * 64 + last - ctx]));
    }
    const bool large = wide_k || __any_sync(0xffffffffu, scale[0] > kLargeFactor || scale[1] > kLargeFactor);
    // (not 0: masked columns' -infinity stays one)
    const float factor[2] = {large ? 1.f : fmaxf(scale[0], 1e-37f), large ? 1.f : fmaxf(scale[1], 1e-37f)};
    // A's fragments: elements 32 j + 8 t + 4 s + {0, 1 | 2, 3} of rows g, g + 8 in steps s = 0, 1.  For fp16 each as its upper 11 bits and what
    // they leave: under a narrow window a result has few terms whose errors could cancel.  (With the upper bits alone trees of 16 under a band of 65
    // were off by 3.1e-4, 58 us; so by 2.3e-4, 66 us then, where fp16's own rounding of the result is 2.1e-4; with P in two parts instead 2.9e-4, 68 us.
    // bfloat16 rounds results by 1.7e-3.)
    constexpr bool kRest = std::is_same<T16, __half>::value;
    uint32_t af[D / 16][4], al[kRest ? D / 16 : 1][4];
#pragma unroll
    for (int j = 0; j < D / 32; ++j) {
      const uint4 q = *reinterpret_cast<const uint4*>(sQ + i * D + j * 32 + t * 8);
      const uint4 r0 = *reinterpret_cast<const uint4*>(sK2 + staged<D>(place[0], j * 4 + t));
      const uint4 r1 = *reinterpret_cast<const uint4*>(sK2 + staged<D>(place[1], j * 4 + t));
      const uint32_t qw[4] = {q.x, q.y, q.z, q.w}, w0[4] = {r0.x, r0.y, r0.z, r0.w}, w1[4] = {r1.x, r1.y, r1.z, r1.w};
      const uint32_t down = half_power(-kDown<CODE>);
#pragma unroll
      for (int s = 0; s < 2; ++s)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const uint32_t c0 = kDown<CODE> ? mul_half2(w0[2 * s + e], down) : w0[2 * s + e], c1 = kDown<CODE> ? mul_half2(w1[2 * s + e], down) : w1[2 * s + e];
          af[2 * j + s][2 * e] = mul_half2(c0, qw[2 * s + e]);
          af[2 * j + s][2 * e + 1] = mul_half2(c1, qw[2 * s + e]);
          if constexpr (kRest) {
            al[2 * j + s][2 * e] = rest_half2(c0, qw[2 * s + e], af[2 * j + s][2 * e]);
            al[2 * j + s][2 * e + 1] = rest_half2(c1, qw[2 * s + e], af[2 * j + s][2 * e + 1]);
          }
        }
    }
    // columns that any of the warp's rows attends to
    int from = min(c_lo[0], c_lo[1]), to = max(c_hi[0], c_hi[1]);
    if (tree[0] | tree[1]) to = max(to, ctx + 63 - __clzll(tree[0] | tree[1])), from = min(from, ctx);
    from = __reduce_min_sync(0xffffffffu, from);
    to = __reduce_max_sync(0xffffffffu, to);
    float acc[D / 8][4], m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
    int v_exp[2] = {wide_v ? 0 : ev1, wide_v ? 0 : ev1};   // the exponent that a row's results count in
#pragma unroll
    for (int n = 0; n < D / 8; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[n][e] = 0.f;
#pragma unroll 1
    for (int c0 = (from - lo_j) & ~31; from <= to && c0 <= to - lo_j; c0 += 32) {
      // columns that the thread's two rows attend to, as bits, and those of them that are there
      uint32_t mask[2];
      const uint32_t there = sThere[c0 >> 5], poison = sNan[c0 >> 5];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int c1 = lo_j + c0, lo = max(c_lo[h] - c1, 0), hi = min(c_hi[h] - c1, 31), off = ctx - c1;
        uint32_t w = lo > 31 || hi < lo ? 0u : (0xffffffffu << lo) & (0xffffffffu >> (31 - hi));
        if (tree[h] && off < 32 && off > -64) w |= (uint32_t)(off >= 0 ? tree[h] << off : tree[h] >> -off);
        if ((w & ~there) && ca.status) atomicOr(ca.status, kStatusPlace);
        mask[h] = w & there;
        if (mask[h] & poison) nan[h] = true;
      }
      if (!__any_sync(0xffffffffu, mask[0] | mask[1])) continue;
      float s[4][4];
#pragma unroll
      for (int n = 0; n < 4; ++n) {
#pragma unroll
        for (int e = 0; e < 4; ++e) s[n][e] = 0.f;
#pragma unroll
        for (int j = 0; j < D / 32; ++j) {
          const uint4 k = *reinterpret_cast<const uint4*>(key_at[j] + (c0 + n * 8) * (2 * D));
          mma_16816(s[n], af[2 * j], k.x, k.y);
          mma_16816(s[n], af[2 * j + 1], k.z, k.w);
          if constexpr (kRest) {
            mma_16816(s[n], al[2 * j], k.x, k.y);
            mma_16816(s[n], al[2 * j + 1], k.z, k.w);
          }
        }
      }
      if (large) {
#pragma unroll
        for (int n = 0; n < 4; ++n)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const float f = wide_k ? power_of_two(sEk1[c0 + n * 8 + 2 * t + e] - 127 - kUp<CODE>) : 1.f;
            s[n][e] *= f * scale[0];
            s[n][2 + e] *= f * scale[1];
          }
      }
      if (wide_v) {   // the largest exponent of the rows that each of the two attends to
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          int top = v_exp[h];
#pragma unroll
          for (int n = 0; n < 4; ++n)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const int byte = sEv1[c0 + n * 8 + 2 * t + e];
              if ((mask[h] >> (n * 8 + 2 * t + e) & 1) && byte != 255) top = max(top, byte);
            }
          top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
          top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
          const float grown = power_of_two(v_exp[h] - top);
          v_exp[h] = top;
#pragma unroll
          for (int n = 0; n < D / 8; ++n) acc[n][2 * h] *= grown, acc[n][2 * h + 1] *= grown;
        }
      }
      if (__any_sync(0xffffffffu, (mask[0] & mask[1]) != 0xffffffffu)) {
        const uint32_t b0 = mask[0] >> (2 * t), b1 = mask[1] >> (2 * t);
#pragma unroll
        for (int n = 0; n < 4; ++n)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            s[n][e] = b0 >> (n * 8 + e) & 1 ? s[n][e] : -INFINITY;
            s[n][2 + e] = b1 >> (n * 8 + e) & 1 ? s[n][2 + e] : -INFINITY;
          }
      }
      float mx[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        mx[h] = fmaxf(s[0][2 * h], s[0][2 * h + 1]);
#pragma unroll
        for (int n = 1; n < 4; ++n) mx[h] = fmaxf(mx[h], fmaxf(s[n][2 * h], s[n][2 * h + 1]));
        mx[h] *= factor[h];
      }
      if (__any_sync(0xffffffffu, mx[0] > m[0] + kGap || mx[1] > m[1] + kGap)) {
        float corr[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          float v = fmaxf(mx[h], m[h]);
          v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 1));
          v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 2));
          corr[h] = v == -INFINITY ? 1.f : exp2f(m[h] - v);
          m[h] = v;
          l[h] *= corr[h];
        }
#pragma unroll
        for (int n = 0; n < D / 8; ++n)
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[n][e] *= corr[e >> 1];
      }
      uint32_t pf[2][4];   // P as the next product's operand: columns c0 + 16 k2 ..
      const float shift[2] = {kLift - (m[0] == -INFINITY ? 0.f : m[0]), kLift - (m[1] == -INFINITY ? 0.f : m[1])};
#pragma unroll
      for (int n = 0; n < 4; ++n)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          float p0 = exp2f(fmaf(s[n][2 * h], factor[h], shift[h])), p1 = exp2f(fmaf(s[n][2 * h + 1], factor[h], shift[h]));
          l[h] += p0 + p1;
          if (wide_v) {   // (a column that does not count has P = 0, and may have any exponent)
            p0 *= power_of_two(min(0, sEv1[c0 + n * 8 + 2 * t] - v_exp[h]));
            p1 *= power_of_two(min(0, sEv1[c0 + n * 8 + 2 * t + 1] - v_exp[h]));
          }
          pf[n >> 1][(n & 1) * 2 + h] = pack2<__half>(p0, p1);
        }
#pragma unroll
      for (int k2 = 0; k2 < 2; ++k2)
#pragma unroll
        for (int d = 0; d < D / 16; ++d) {
          // V1 of 16 tokens x 16 columns: four 8 x 8 blocks, transposed
          uint32_t v[4];
          ldmatrix_x4_trans(v, value_at[d] + (c0 + k2 * 16) * (2 * D));
          mma_16816(acc[2 * d], pf[k2], v[0], v[1]);
          mma_16816(acc[2 * d + 1], pf[k2], v[2], v[3]);
        }
    }
    // --- the unit's sum: rows' sums over the four lanes, then over the 16 rows
    float top = -INFINITY, sum = 0.f, w[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      l[h] += __shfl_xor_sync(0xffffffffu, l[h], 1);
      l[h] += __shfl_xor_sync(0xffffffffu, l[h], 2);
      if (nan[h] && l[h] > 0.f) l[h] = __uint_as_float(0x7fffffffu);
      top = fmaxf(top, m[h]);
    }
#pragma unroll
    for (int o = 4; o < 32; o <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      w[h] = m[h] == -INFINITY ? 0.f : exp2f(m[h] - top - kLift);
      sum += m[h] == -INFINITY ? (l[h] != l[h] ? l[h] : 0.f) : l[h] * w[h];
      w[h] *= vweight[h];
    }
#pragma unroll
    for (int o = 4; o < 32; o <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    const float v1_scale[2] = {power_of_two(v_exp[0] - 127 - kUp<CODE>), power_of_two(v_exp[1] - 127 - kUp<CODE>)};
    float v[D / 4];   // columns 8 n + 2 t + e at 2 n + e
#pragma unroll
    for (int n = 0; n < D / 8; ++n) {
      v[2 * n] = v[2 * n + 1] = 0.f;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const float2 c = unpack2<__half>(*reinterpret_cast<const uint32_t*>(sV2 + staged<D>(place[h], n) + t * 4));
        if (w[h] != 0.f) v[2 * n] = fmaf(c.x * w[h], acc[n][2 * h] * v1_scale[h], v[2 * n]), v[2 * n + 1] = fmaf(c.y * w[h], acc[n][2 * h + 1] * v1_scale[h], v[2 * n + 1]);
      }
    }
    // over the eight lanes of a column: halves change hands until each has D / 32 columns
    int col = 0;   // of the first: n of the pair v[0], v[1]
#pragma unroll
    for (int o = 16, count = D / 4; o >= 4; o >>= 1, count >>= 1) {
      const bool upper = lane & o;
      if (upper) col += count / 4;
#pragma unroll
      for (int e = 0; e < count / 2; ++e) {
        const float give = upper ? v[e] : v[e + count / 2], keep = upper ? v[e + count / 2] : v[e];
        v[e] = keep + __shfl_xor_sync(0xffffffffu, give, o);
      }
    }
#pragma unroll
    for (int e = 0; e < D / 32; e += 2) out[2 + (col + e / 2) * 8 + 2 * t] = v[e], out[2 + (col + e / 2) * 8 + 2 * t + 1] = v[e + 1];
    if (lane == 0) out[0] = top, out[1] = sum;
  }
  __syncthreads();

  // --- each new token's units, in order
  for (int i = warp; i < want; i += kWarps) {
    const size_t row = ((size_t)blockIdx.x) * ca.c.n + i0 + i;
    float top = -INFINITY, sum = 0.f, v[D / 32];
#pragma unroll
    for (int k = 0; k < D / 32; ++k) v[k] = 0.f;
    if (i < ni) {
      const float* in = sPart + (size_t)i * p.tiles * (D + 2);
      for (int u = 0; u < p.tiles; ++u) top = fmaxf(top, in[u * (D + 2)]);
      for (int u = 0; u < p.tiles; ++u) {
        const float* x = in + u * (D + 2);
        const float w = x[0] == -INFINITY ? 0.f : exp2f(x[0] - top);
        sum += x[0] == -INFINITY ? (x[1] != x[1] ? x[1] : 0.f) : x[1] * w;
#pragma unroll
        for (int k = 0; k < D / 32; ++k) v[k] += w == 0.f ? 0.f : x[2 + k * 32 + lane] * w;
      }
    }
    const bool none = top == -INFINITY && sum == 0.f;
#pragma unroll
    for (int k = 0; k < D / 32; ++k)
      ((T16*)p.o)[row * D + k * 32 + lane] = from_f<T16>(none ? 0.f : sum != sum ? sum : v[k] * (1.f / sum));
    if (p.lse && lane == 0) p.lse[row] = none ? -INFINITY : sum != sum ? sum : (top + log2f(sum)) * kLn2;
  }
}

size_t smem_of(const WindowParams& p, int D) {
  return (size_t)(p.cols + p.rows) * (4 * D + 2) + (size_t)p.tokens * (2 * D + 12 + 64) + 4 + (size_t)p.cols / 4 + (size_t)p.tokens * p.tiles * (D + 2) * 4 + 16;
}

// Of the two kernels this one is the faster up to so many cells (rows by columns) a new token; beyond, the one with tcgen05 tiles.  That one's time goes by
// slabs of 128 columns: at D=128, windows of 100, it takes half of what those of 128 do, so the border lies lower where one slab holds all columns, but
// for calls that leave most SMs idle.  us, this kernel / that one, int8 codes; windows (band) of
//                       one token, 4 x 8      one token, 32 x 16    trees of 16, 8 x 16   trees of 4, 2 x 16
//   D=64  bf16  128     19 / 20               41 / 60               79 / 122              25 / 25
//               160     21 / 20               49 / 60               137 / 143             27 / 25
//               200     23 / 21               86 / 59               176 / 148             35 / 27
//               300 (65) 23 / 25              85 / 110              -                     25 / 35
//   D=64  fp16  128     21 / 21               47 / 60               94 / 122              27 / 25
//               160     23 / 21               55 / 60               172 / 144             33 / 26
//               300 (65) 25 / 25              93 / 109              -                     28 / 35
//   D=128 bf16  80      14 / 21               50 / 49               73 / 82               23 / 25
//               100     17 / 21               58 / 47               93 / 94               27 / 25
//               128     25 / 25               90 / 95               133 / 188             31 / 35
//               160     27 / 25               105 / 93              -                     -
//   D=128 fp16  80      14 / 21               53 / 49               82 / 82               25 / 25
//               100     17 / 21               62 / 47               109 / 93              31 / 25
//               128     27 / 25               99 / 96               159 / 189             35 / 35
//               160     31 / 25               115 / 93              -                     -
// (fp16 queries cost more here: A in two parts.)
long long most_cells(const tritt_cache_t& c, int dtype, long long columns) {
  if (c.D == 64) return dtype == TRITT_F16 ? 25000 : 28000;
  return columns <= 128 && (long long)c.B * c.N * c.n > num_sms() / 2 ? 7000 : 25000;
}
// What a call's blocks stage, and how many new tokens each takes: as few as fill the chip, for the more, the more read a row once.  False: not a call
// for this kernel, or too much for shared memory.
bool plan(const tritt_cache_t& c, int dtype, int k1w, int k2w, int kkl, int kkr, WindowParams& p) {
  const long long tokens = (long long)c.page_size * c.table_pages + c.n;   // a sequence's most
  const long long rows = tokens < (long long)k2w + 1 ? tokens : (long long)k2w + 1;
  if (rows > 1024) return false;
  const long long band = (long long)kkl + kkr + 16;   // of a unit's 16 rows
  long long seen = tokens < (long long)k1w + 1 ? tokens : (long long)k1w + 1;
  if (band < seen) seen = band;
  const long long old = (long long)c.page_size * c.table_pages;
  if (rows * seen > most_cells(c, dtype, (old < k1w ? old : k1w) + c.n)) return false;
  p.tiles = (int)(rows + 15) / 16;
  const int pairs = c.B * c.N, most = kPartBytes / (p.tiles * (c.D + 2) * 4);
  // one wave of two blocks an SM where there are not more sequences and heads (a second one of a third as many costs as much as the
  // first: trees of 16 under windows of 129, 128 of them: 3 blocks each 84 us, 2 each 58), but at least two units a warp
  const int blocks = 2 * num_sms() / pairs;
  int per = blocks < 1 ? c.n : (c.n + blocks - 1) / blocks;
  const int least = (2 * kWarps + p.tiles - 1) / p.tiles;
  per = per > least ? per : least;
  per = per < most ? per : most;
  per = per < c.n ? per : c.n;
  if (per < 1) return false;
  p.tokens = per;
  // (a tree's tokens lie at depths up to their numbers: the windows of all of them)
  auto places = [&](int w) {
    const long long n = tokens < (long long)w + c.n + 1 ? tokens : (long long)w + c.n + 1;
    return (n + 31) / 32 * 32;
  };
  const long long cols = places(k1w), rws = places(k2w);
  if (cols + rws > 4096) return false;
  p.cols = (int)cols;
  p.rows = (int)rws;
  return smem_of(p, c.D) <= (size_t)kMostSmem;
}

template <typename T16, int D, int CODE> int launch(const WindowParams& p, cudaStream_t stream) {
  auto kern = tdp_decode_window_kernel<T16, D, CODE>;
  const size_t bytes = smem_of(p, D);
  TRITT_CUDA_OK(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kMostSmem));
  const tritt_cache_t& c = p.a.cache.c;
  kern<<<dim3(c.B * c.N, (c.n + p.tokens - 1) / p.tokens), kWarps * 32, bytes, stream>>>(p);
  count_launch();
  TRITT_CUDA_OK(cudaGetLastError());
  return 0;
}
template <typename T16, int D> int by_code(const WindowParams& p, cudaStream_t s) {
  const int code = p.a.cache.c.code;
  if (code == TRITT_CODE_F16) return launch<T16, D, TRITT_CODE_F16>(p, s);
  return code == TRITT_CODE_E4M3 ? launch<T16, D, TRITT_CODE_E4M3>(p, s) : launch<T16, D, TRITT_CODE_INT8>(p, s);
}

}  // namespace

bool window_tdp_decode_applies(const tritt_cache_t& c, int dtype, int k1w, int k2w, int kkl, int kkr) {
  WindowParams p{};
  return plan(c, dtype, k1w, k2w, kkl, kkr, p);
}

int window_tdp_decode(const TdpDecodeArgs& a, void* o, float* lse, cudaStream_t stream) {
  WindowParams p{};
  p.a = a;
  p.o = o;
  p.lse = lse;
  plan(a.cache.c, a.dtype, a.k1w, a.k2w, a.kkl, a.kkr, p);
  if (a.dtype == TRITT_F16) return a.cache.c.D == 64 ? by_code<__half, 64>(p, stream) : by_code<__half, 128>(p, stream);
  return a.cache.c.D == 64 ? by_code<__nv_bfloat16, 64>(p, stream) : by_code<__nv_bfloat16, 128>(p, stream);
}

}  // namespace tritt
