// One soft-max attention of new tokens over two parts of the quantised cache, 16-bit queries, head dimension 64 or 128: either leg of the
// dot-product-sum form (append: rows k2 over K1, SiLU(V1) within a window;  decode: rows q over K2, W with a bias for each token).
//
// Bound by HBM: a cached row is read once for up to 8 NT new tokens, 2 flops a byte and token.  There is no reuse to stage for, so
// rows go from memory to registers and, as fp16, into warp-level matrix instructions with the cached rows as the 16-row operand:
//   S^T[16 tokens x 8 queries] = K Q^T,   O^T[D x 8 queries] += V^T P^T
// (one token is an eighth of a tile instead of a sixteenth, and a query's statistics lie in the threads that hold its results).  The contraction of S
// runs over the head dimension in any order, so a thread takes 16 contiguous bytes of a row for the elements that it needs; the rows of
// V^T are columns of V in any order, so a thread takes D / 8 contiguous elements of four tokens and pairs them by byte permutes.  P^T is
// the transpose of S^T's fragments (movmatrix).  A warp walks its tiles of tokens with the next keys and values in flight.
//
// Codes are exact as fp16, the scores' powers of two are applied in fp32; P is formed times 2^(its row's exponent - the largest so far + 13),
// so that values of any size meet in one accumulator, and its sum is taken before that.  Queries are brought to [1, 2) by a power of two.
#include "tritt_cache.cuh"

namespace tritt {
namespace {

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
  static constexpr int kTokens = kRowBytes == 256 ? 16 : 32;    // of a tile: 2 to 4 KB of keys
  static constexpr int kBlocks = kTokens / 16;
  static constexpr int kKeyLoads = kRowBytes / 64;              // of 16 bytes, of a lane's row
  static constexpr int kValueWords = kRowBytes / 32;            // 32-bit words of a lane's eighth of a row
};

// A tile's keys: rows g and g + 8 of each block of 16 tokens; chunk t + 4 j of a row.
template <int D, int CODE> struct Keys {
  using S = Shape<D, CODE>;
  uint4 v[S::kBlocks][2][S::kKeyLoads];
};
// Values: of tokens 2t, 2t + 1, 2t + 8, 2t + 9 of each block, the g-th eighth of the row.
template <int D, int CODE> struct Values {
  using S = Shape<D, CODE>;
  uint32_t v[S::kBlocks][4][S::kValueWords];
};

template <int D, int CODE, int NT>
__global__ void __launch_bounds__(kWarps * 32) dps_decode_kernel(const __grid_constant__ Params p) {
  using S = Shape<D, CODE>;
  constexpr int NB = S::kBlocks, TK = S::kTokens, KL = S::kKeyLoads, VW = S::kValueWords;
  constexpr int Q = 8 * NT;
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

  // --- tiles
  const size_t part_rows = (size_t)ca.c.N << ca.page_log2;   // rows of one part of a page
  auto row_base = [&](int page, int part_) { return ((size_t)page * 4 + part_) * part_rows + ((size_t)head << ca.page_log2); };
  // pages of a tile's groups of eight tokens (one page each), in the first lanes
  auto find_pages = [&](int tile) {
    const int token = first + tile * TK + lane * 8;
    return lane < TK / 8 && tile < tile1 && token < end ? place_of(ca, b, token).page : -1;
  };
  Keys<D, CODE> keys;
  Values<D, CODE> values;
  struct Side {                  // of this thread's tokens g, g + 8 of each block: exponents and biases
    int ek[NB][2], ev[NB][2];
    float bias[NB][2];
  } side;
  auto load_keys = [&](int tile, int pages) {
#pragma unroll
    for (int nb = 0; nb < NB; ++nb)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int found = __shfl_sync(0xffffffffu, pages, nb * 2 + h), token = first + tile * TK + nb * 16 + h * 8 + g;
        const int r = token & (ca.c.page_size - 1), page = token < end ? found : -1;
        const size_t at = page >= 0 ? row_base(page, a.key_part) + r : 0;
        const uint8_t* row = (const uint8_t*)ca.c.codes + at * S::kRowBytes + t * 16;
#pragma unroll
        for (int j = 0; j < KL; ++j)
          keys.v[nb][h][j] = page >= 0 ? __ldg(reinterpret_cast<const uint4*>(row + j * 64)) : make_uint4(0u, 0u, 0u, 0u);
        side.ek[nb][h] = page >= 0 ? __ldg(ca.c.exponents + at) : -1;
        side.ev[nb][h] = page >= 0 ? __ldg(ca.c.exponents + row_base(page, a.value_part) + r) : -1;
        side.bias[nb][h] = page >= 0 && a.biased ? __ldg(ca.c.lse + (((size_t)page * ca.c.N + head) << ca.page_log2) + r) : 0.f;
      }
  };
  auto load_values = [&](int tile, int pages) {
#pragma unroll
    for (int nb = 0; nb < NB; ++nb)
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int found = __shfl_sync(0xffffffffu, pages, nb * 2 + (k >> 1));
        const int token = first + tile * TK + nb * 16 + (k >> 1) * 8 + 2 * t + (k & 1);
        const int r = token & (ca.c.page_size - 1), page = token < end ? found : -1;   // (what lies behind the last token is not looked at)
        const uint8_t* row = (const uint8_t*)ca.c.codes + (page >= 0 ? row_base(page, a.value_part) + r : 0) * S::kRowBytes + g * (VW * 4);
        uint32_t(&v)[VW] = values.v[nb][k];
        if constexpr (VW == 2) {
          const uint2 w = page >= 0 ? __ldg(reinterpret_cast<const uint2*>(row)) : make_uint2(0u, 0u);
          v[0] = w.x, v[1] = w.y;
        } else {
#pragma unroll
          for (int j = 0; j < VW / 4; ++j) {
            const uint4 w = page >= 0 ? __ldg(reinterpret_cast<const uint4*>(row) + j) : make_uint4(0u, 0u, 0u, 0u);
            v[4 * j] = w.x, v[4 * j + 1] = w.y, v[4 * j + 2] = w.z, v[4 * j + 3] = w.w;
          }
        }
      }
  };

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
  int tile = tile0 + warp;
  int pages = find_pages(tile), pages_next = find_pages(tile + kWarps);
  if (tile < tile1) {
    load_keys(tile, pages);
    load_values(tile, pages);
  }
  for (; tile < tile1; tile += kWarps) {
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
        const uint32_t lo[4] = {keys.v[nb][0][j].x, keys.v[nb][0][j].y, keys.v[nb][0][j].z, keys.v[nb][0][j].w};
        const uint32_t hi[4] = {keys.v[nb][1][j].x, keys.v[nb][1][j].y, keys.v[nb][1][j].z, keys.v[nb][1][j].w};
        constexpr int STEPS = S::kWide ? 2 : 4;   // contraction steps of 16 bytes
#pragma unroll
        for (int st = 0; st < STEPS; ++st) {
          uint32_t f[4];
          if constexpr (S::kWide) {
            f[0] = lo[2 * st], f[1] = hi[2 * st], f[2] = lo[2 * st + 1], f[3] = hi[2 * st + 1];
          } else {
            bytes_to_halves<CODE>(lo[st], f[0], f[2]);
            bytes_to_halves<CODE>(hi[st], f[1], f[3]);
          }
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) mma_16816(s[nt][nb], f, qf[nt][j * STEPS + st][0], qf[nt][j * STEPS + st][1]);
        }
      }
    }
    const Side now = side;
    if (tile + kWarps < tile1) load_keys(tile + kWarps, pages_next);
    const int pages_after = find_pages(tile + 2 * kWarps);
    // largest exponent of the values, and whether every token of the tile counts for every query
    const int token0 = first + tile * TK;
    bool plain = token0 >= lo_all && token0 + TK <= ctx;
    int ev_most = 0;
#pragma unroll
    for (int nb = 0; nb < NB; ++nb)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        plain = plain && now.ek[nb][h] >= 0 && now.ek[nb][h] != 255 && now.ev[nb][h] != 255;
        ev_most = max(ev_most, now.ev[nb][h] == 255 ? 0 : now.ev[nb][h]);
      }
    plain = __all_sync(0xffffffffu, plain);
    ev_most = max(v_exp, __reduce_max_sync(0xffffffffu, ev_most));
    // scores in log2 units
#pragma unroll
    for (int nb = 0; nb < NB; ++nb)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const float kf = power(now.ek[nb][h] - 127), bias = now.bias[nb][h] * kLog2e;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int q = 0; q < 2; ++q) s[nt][nb][2 * h + q] = fmaf(s[nt][nb][2 * h + q] * kf, qs[nt][q], bias);
        if (!plain) {
          const int token = token0 + nb * 16 + h * 8 + g;
          const bool there = now.ek[nb][h] >= 0, bad = now.ek[nb][h] == 255 || now.ev[nb][h] == 255;
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
              missing = missing || (seen && !there);
              float& x = s[nt][nb][2 * h + q];
              x = seen && there ? (bad ? __uint_as_float(0x7fffffffu) : x) : -INFINITY;
            }
          if (missing && ca.status) atomicOr(ca.status, kStatusPlace);
        }
      }
    // running maximum, P
    uint32_t pf[NT][NB][2];
    const float grown = power(v_exp - ev_most);
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      float corr[2], base[2];
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
        corr[q] *= grown;
      }
#pragma unroll
      for (int mb = 0; mb < D / 16; ++mb)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[nt][mb][e] *= corr[e & 1];
#pragma unroll
      for (int nb = 0; nb < NB; ++nb)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const float vf = now.ev[nb][h] == 255 ? 0.f : power(now.ev[nb][h] - ev_most + kLift);
          const float p0 = exp2f(s[nt][nb][2 * h] - base[0]), p1 = exp2f(s[nt][nb][2 * h + 1] - base[1]);
          l[nt][0] += p0;
          l[nt][1] += p1;
          pf[nt][nb][h] = transposed(pack_half(p0 * vf, p1 * vf));
        }
    }
    v_exp = ev_most;
    // O^T += V^T P^T
#pragma unroll
    for (int nb = 0; nb < NB; ++nb)
#pragma unroll
      for (int w = 0; w < VW; ++w) {
        if constexpr (S::kWide) {
          // two elements of four tokens: one block of 16 rows of V^T
          uint32_t f[4];
          f[0] = __byte_perm(values.v[nb][0][w], values.v[nb][1][w], 0x5410);
          f[1] = __byte_perm(values.v[nb][0][w], values.v[nb][1][w], 0x7632);
          f[2] = __byte_perm(values.v[nb][2][w], values.v[nb][3][w], 0x5410);
          f[3] = __byte_perm(values.v[nb][2][w], values.v[nb][3][w], 0x7632);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) mma_16816(acc[nt][w], f, pf[nt][nb][0], pf[nt][nb][1]);
        } else {
          // four elements: two blocks
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            const uint32_t lo = __byte_perm(values.v[nb][0][w], values.v[nb][1][w], half ? 0x7362 : 0x5140);
            const uint32_t hi = __byte_perm(values.v[nb][2][w], values.v[nb][3][w], half ? 0x7362 : 0x5140);
            uint32_t f[4];
            bytes_to_halves<CODE>(lo, f[0], f[1]);
            bytes_to_halves<CODE>(hi, f[2], f[3]);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) mma_16816(acc[nt][2 * w + half], f, pf[nt][nb][0], pf[nt][nb][1]);
          }
        }
      }
    if (tile + kWarps < tile1) load_values(tile + kWarps, pages_next);
    pages_next = pages_after;
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
  dps_decode_kernel<D, CODE, NT><<<dim3(p.a.splits, p.a.cache.c.B * p.a.cache.c.N, p.query_groups), kWarps * 32, 0, stream>>>(p);
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
