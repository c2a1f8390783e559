// A paged cache of quantised rows: places, codes, and which tokens a new one attends to.
#pragma once

#include <cuda_fp8.h>

#include "tritt_common.cuh"

#include <type_traits>

namespace tritt {

enum { kPartK1 = 0, kPartK2 = 1, kPartV1 = 2, kPartV2 = 3 };
enum { kStatusPosition = 256, kStatusPlace = 512, kStatusTdpDecode = 1024 };

// The cache as kernels see it.
struct CacheArgs {
  tritt_cache_t c;
  int page_log2;
  int* status;
};

inline int code_bytes(int code) { return code == TRITT_CODE_F16 ? 2 : 1; }

// 0, or the error code of what is wrong with a cache's description (host).
int check_cache(const tritt_cache_t* c);
int check_rows(const tritt_rows_t* rows, int count, int dtype);
CacheArgs cache_args(const tritt_cache_t& c, int* status);

// A token's place in the cache: its page and row, page -1 where the table or the cache have none.
struct Place {
  int page, row;
};
__device__ __forceinline__ Place place_of(const CacheArgs& a, int b, int token) {
  const int i = token >> a.page_log2;
  Place at{-1, token & (a.c.page_size - 1)};
  if (token >= 0 && i < a.c.table_pages) {
    const int page = __ldg(a.c.table + b * a.c.table_stride + i);
    if (page >= 0 && page < a.c.pages) at.page = page;
  }
  return at;
}
// Number of a part's row among all rows of the cache (rows of D codes, one exponent each), and of a token's log-sum-exp.
__device__ __forceinline__ size_t row_of(const CacheArgs& a, Place at, int part, int head) {
  return ((((size_t)at.page * 4 + part) * a.c.N + head) << a.page_log2) + at.row;
}
__device__ __forceinline__ size_t lse_of(const CacheArgs& a, Place at, int head) {
  return (((size_t)at.page * a.c.N + head) << a.page_log2) + at.row;
}

// New tokens that sequence b has in this call.
__device__ __forceinline__ int new_tokens(const CacheArgs& a, int b) {
  if (__ldg(a.c.context + b) < 0) return 0;
  const int n = a.c.counts ? __ldg(a.c.counts + b) : a.c.n;
  return n < 0 ? 0 : n > a.c.n ? a.c.n : n;
}
// Tokens of sequence b before the new ones, at most what its table has places for (more is an error of a sequence that
// has new ones, and the bound is one of every loop over them).
__device__ __forceinline__ int context_of(const CacheArgs& a, int b) {
  const int c = __ldg(a.c.context + b), most = a.c.table_pages << a.page_log2;
  if (c > most && a.status && new_tokens(a, b) > 0) atomicOr(a.status, kStatusPlace);
  return c < most ? c : most;
}

// Bit m: new token i attends to new token m (only with ancestors).
__device__ __forceinline__ unsigned long long seen_word(const CacheArgs& a, int b, int i) {
  const unsigned long long own = 1ull << i;
  return ((unsigned long long)__ldg(a.c.ancestors + (size_t)b * a.c.n + i) & (own - 1)) | own;
}
// Position of new token i of sequence b, counted from its context.
__device__ __forceinline__ int depth_of(const CacheArgs& a, int b, int i) {
  return a.c.ancestors ? __popcll(seen_word(a, b, i)) - 1 : i;
}

// ---------------------------------------------------------------- codes
// The exponent byte of a row whose largest |element| has these bits (those of a NaN are larger than any).
template <int CODE> __device__ __forceinline__ int exponent_byte(uint32_t largest) {
  const int field = (int)(largest >> 23);
  const uint32_t mantissa = largest & 0x7fffffu;
  if (field == 255) return 255;
  const int e = CODE == TRITT_CODE_F16    ? field - 14                             // below 2^15
                : CODE == TRITT_CODE_E4M3 ? field - 8 + (mantissa > 0x600000u)     // at most 448 = 1.75 * 2^8
                                          : field - 6 + (mantissa > 0x7e0000u);    // at most 127 = 1.984375 * 2^6
  return e < 1 ? 1 : e;
}
// What a row's elements are multiplied by before they are rounded to codes, and what codes stand for.
__device__ __forceinline__ float to_code_scale(int byte) { return byte == 255 ? 0.f : __uint_as_float((uint32_t)(254 - byte) << 23); }
__device__ __forceinline__ float code_scale(int byte) {
  return byte == 255 ? __uint_as_float(0x7fffffffu) : __uint_as_float((uint32_t)byte << 23);
}

// Rows of a tile are brought to one exponent as fp16 numbers (the products' operands): exactly for 8-bit codes and for the elements of fp16 codes down
// to 2^-14 of their row's largest one, as long as exponents lie no further apart than this.  The largest row may be one that nobody attends to, so beyond each row keeps
// its own, and scores and P are multiplied by it column by column (slower, and rare: rows of zeros do not count).
template <int CODE> constexpr int kSpread = CODE == TRITT_CODE_F16 ? 14 : CODE == TRITT_CODE_E4M3 ? 20 : 24;
// An exponent byte, where it counts towards the least one of several: rows of zeros or next to it, NaN and those that are not there do not.
__device__ __forceinline__ int least_byte(int byte) { return byte > 1 ? byte : 255; }
// From this on a score's factor (its sum of products may be 2^30) is multiplied in, and rounded, before the maximum is subtracted: as one multiplication and
// addition, scores from 2^25 on would be off from the rounded maximum by enough to leave the range of P.
constexpr float kLargeFactor = 1.f / 64;
__device__ __forceinline__ float power_of_two(int e) { return exp2f((float)e); }   // any e

// Eight codes of neighbouring elements: 16 bytes of fp16, 8 of the others.  A row that is not finite has zeros.
template <int CODE> struct Codes8;
template <> struct Codes8<TRITT_CODE_F16> {
  uint4 v;
  __device__ __forceinline__ void load(const void* row, int col) { v = *reinterpret_cast<const uint4*>((const __half*)row + col); }
  __device__ __forceinline__ void store(void* row, int col) const { *reinterpret_cast<uint4*>((__half*)row + col) = v; }
  __device__ __forceinline__ void encode(const float (&f)[8]) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const __half2 h = __floats2half2_rn(f[2 * i], f[2 * i + 1]);
      w[i] = *reinterpret_cast<const uint32_t*>(&h);
    }
    v = make_uint4(w[0], w[1], w[2], w[3]);
  }
  __device__ __forceinline__ void halves(uint32_t (&w)[4]) const { w[0] = v.x, w[1] = v.y, w[2] = v.z, w[3] = v.w; }
};
// Four bytes as two pairs of fp16.
template <int CODE> __device__ __forceinline__ void bytes_to_halves(uint32_t v, uint32_t& lo, uint32_t& hi) {
  if constexpr (CODE == TRITT_CODE_E4M3) {
    asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, a;\n\tcvt.rn.f16x2.e4m3x2 %1, b;\n\t}" : "=r"(lo), "=r"(hi) : "r"(v));
  } else {
    // 0x64bb is 1024 + bb in fp16; with the sign bit turned over bb is the element + 128
    const uint32_t u = v ^ 0x80808080u;
    const __half2 off = __halves2half2(__ushort_as_half(0x6480), __ushort_as_half(0x6480));   // 1152
    uint32_t l = __byte_perm(u, 0x64646464u, 0x4140), h = __byte_perm(u, 0x64646464u, 0x4342);
    const __half2 a = __hsub2(*reinterpret_cast<__half2*>(&l), off), b = __hsub2(*reinterpret_cast<__half2*>(&h), off);
    lo = *reinterpret_cast<const uint32_t*>(&a);
    hi = *reinterpret_cast<const uint32_t*>(&b);
  }
}
template <int CODE> struct Codes8 {
  uint2 v;
  __device__ __forceinline__ void load(const void* row, int col) { v = *reinterpret_cast<const uint2*>((const uint8_t*)row + col); }
  __device__ __forceinline__ void store(void* row, int col) const { *reinterpret_cast<uint2*>((uint8_t*)row + col) = v; }
  __device__ __forceinline__ void encode(const float (&f)[8]) {
    uint32_t w[2] = {0u, 0u};
#pragma unroll
    for (int i = 0; i < 8; i += 2) {
      uint32_t pair;
      if constexpr (CODE == TRITT_CODE_E4M3)
        pair = __nv_cvt_float2_to_fp8x2(make_float2(f[i], f[i + 1]), __NV_SATFINITE, __NV_E4M3);
      else
        // (1.5 * 2^23 more leaves the rounded integer in the lowest bits; conversions are slow)
        pair = __byte_perm(__float_as_uint(f[i] + 12582912.f), __float_as_uint(f[i + 1] + 12582912.f), 0x0040) & 0xffffu;
      w[i / 4] |= pair << (8 * (i % 4));
    }
    v = make_uint2(w[0], w[1]);
  }
  __device__ __forceinline__ void halves(uint32_t (&w)[4]) const {
    bytes_to_halves<CODE>(v.x, w[0], w[1]);
    bytes_to_halves<CODE>(v.y, w[2], w[3]);
  }
};
template <int CODE> __device__ __forceinline__ void code_values(const Codes8<CODE>& c, float scale, float (&f)[8]) {
  uint32_t w[4];
  c.halves(w);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 v = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
    f[2 * i] = v.x * scale;
    f[2 * i + 1] = v.y * scale;
  }
}

// Eight neighbouring elements of a row of any type.
template <typename T> __device__ __forceinline__ void load8(const T* p, float (&f)[8]) {
  const uint4 v = __ldg(reinterpret_cast<const uint4*>(p));
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    T lo, hi;
    *reinterpret_cast<uint16_t*>(&lo) = (uint16_t)w[i];
    *reinterpret_cast<uint16_t*>(&hi) = (uint16_t)(w[i] >> 16);
    f[2 * i] = to_f(lo);
    f[2 * i + 1] = to_f(hi);
  }
}
template <> __device__ __forceinline__ void load8<float>(const float* p, float (&f)[8]) {
  const float4 a = __ldg(reinterpret_cast<const float4*>(p)), b = __ldg(reinterpret_cast<const float4*>(p) + 1);
  f[0] = a.x, f[1] = a.y, f[2] = a.z, f[3] = a.w, f[4] = b.x, f[5] = b.y, f[6] = b.z, f[7] = b.w;
}
template <typename T> __device__ __forceinline__ void store8(T* p, const float (&f)[8]) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const T lo = from_f<T>(f[2 * i]), hi = from_f<T>(f[2 * i + 1]);
    w[i] = (uint32_t)*reinterpret_cast<const uint16_t*>(&lo) | (uint32_t)*reinterpret_cast<const uint16_t*>(&hi) << 16;
  }
  *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
}
template <> __device__ __forceinline__ void store8<float>(float* p, const float (&f)[8]) {
  reinterpret_cast<float4*>(p)[0] = make_float4(f[0], f[1], f[2], f[3]);
  reinterpret_cast<float4*>(p)[1] = make_float4(f[4], f[5], f[6], f[7]);
}

__device__ __forceinline__ size_t rows_at(const tritt_rows_t& r, int b, int n, int t) {
  return (size_t)(b * r.stride_b + n * r.stride_n + t * r.stride_t);
}

// Largest |element| of eight, as bits; then over the L neighbouring lanes of a row.
__device__ __forceinline__ uint32_t largest8(const float (&f)[8]) {
  uint32_t m = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e) m = max(m, __float_as_uint(f[e]) & 0x7fffffffu);
  return m;
}
template <int L> __device__ __forceinline__ uint32_t largest_of_row(uint32_t m) {
#pragma unroll
  for (int o = L / 2; o > 0; o >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
  return m;
}
// Two 16-bit maxima at a time: of eight elements' magnitudes, in either half of the word, and as fp32 bits.
__device__ __forceinline__ uint32_t largest_halves(uint4 v) {
  const uint32_t m = 0x7fff7fffu;
  const uint32_t w = __vmaxu2(__vmaxu2(v.x & m, v.y & m), __vmaxu2(v.z & m, v.w & m));
  return max(w & 0xffffu, w >> 16);
}
template <int L> __device__ __forceinline__ uint32_t largest_of_two_rows(uint32_t m) {
#pragma unroll
  for (int o = L / 2; o > 0; o >>= 1) m = __vmaxu2(m, __shfl_xor_sync(0xffffffffu, m, o));
  return m;
}
template <typename T> __device__ __forceinline__ uint32_t bits_of_half(uint32_t h) {
  T x;
  *reinterpret_cast<uint16_t*>(&x) = (uint16_t)h;
  return __float_as_uint(to_f(x));
}
// A row's eight elements of this lane as codes for the exponent `byte`.
template <int CODE> __device__ __forceinline__ Codes8<CODE> codes_of(int byte, const float (&f)[8]) {
  const float scale = to_code_scale(byte);
  float y[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) y[e] = f[e] * scale;
  Codes8<CODE> codes;
  codes.encode(y);
  if (byte == 255) codes.v = {};   // (a row that is not finite)
  return codes;
}

// Append: a warp's row (eight elements from column `col` on of its first lanes) times v2 becomes W in the cache, with its log-sum-exp.  All
// lanes call it; a token that is not there has no place.
template <typename T, int CODE>
__device__ __forceinline__ void join_into_cache(const CacheArgs& a, int b, int head, int i, int col, float (&f)[8], float lse, const tritt_rows_t& v2) {
  const int D = a.c.D;
  bool on = i < new_tokens(a, b);
  Place at{-1, 0};
  if (on) {
    at = place_of(a, b, context_of(a, b) + i);
    on = at.page >= 0;
  }
  if (on && col < D) {
    float v[8];
    load8((const T*)v2.p + rows_at(v2, b, head, i) + col, v);
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] *= v[e];
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] = 0.f;
  }
  // (lanes past the row have zeros, which change no maximum)
  const int byte = exponent_byte<CODE>(largest_of_row<32>(largest8(f)));
  if (!on) return;
  const size_t to = row_of(a, at, kPartV2, head);
  if (col == 0) {
    a.c.exponents[to] = (unsigned char)byte;
    a.c.lse[lse_of(a, at, head)] = lse;
  }
  if (col < D) {
    codes_of<CODE>(byte, f).store((uint8_t*)a.c.codes + to * (size_t)(D * (CODE == TRITT_CODE_F16 ? 2 : 1)), col);
  }
}

// ---------------------------------------------------------------- kernels one behind the other
// A kernel that may be launched before the one ahead of it in the stream has ended (`early`): it calls wait_for_previous() before it reads or
// writes anything; the one ahead calls let_next_start() as soon as all its blocks are on the chip.  (The launch and the start of the blocks, 2 to 3 us,
// then lie beside the kernel ahead.)
__device__ __forceinline__ void wait_for_previous() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void let_next_start() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
template <typename K, typename P> int launch_kernel_after(K kern, dim3 grid, int threads, size_t smem, cudaStream_t stream, bool early, const P& p) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = early ? 1 : 0;
  TRITT_CUDA_OK(cudaLaunchKernelEx(&cfg, kern, p));
  count_launch();
  return 0;
}

// ---------------------------------------------------------------- parts of a row's soft-max, and what becomes of them
// Each split of a new token's attended tokens leaves its maximum (log2 units), sum and unnormalised result in the workspace,
// [rows][splits][D + 2] fp32 (rows = (b * N + head) * n + i), and a second kernel joins them.
struct JoinArgs {
  CacheArgs cache;
  const float* part;
  int splits, dtype;
  void* o;            // [B, N, n, D], or null: append
  float* lse;         // [B, N, n] or null
  tritt_rows_t v2;    // append: W = result * v2 goes to the cache, and the log-sum-exp
};
int launch_join(const JoinArgs& j, cudaStream_t stream);
int launch_write(const CacheArgs& a, const tritt_rows_t* rows, int dtype, int parts, cudaStream_t stream);

// The CUDA cores' kernels (any type, fp32 arithmetic): triple dot product, and one soft-max attention over two parts of the cache.
struct TdpDecodeArgs {
  CacheArgs cache;
  tritt_rows_t q;
  int dtype, k1w, k2w, kkl, kkr;
  float scale2;       // alpha * log2(e)
  float* part;
  int splits;
};
struct DpsDecodeArgs {
  CacheArgs cache;
  tritt_rows_t q;     // the rows that attend
  int dtype, key_part, value_part, biased, window, exact;   // exact: P in 22 bits (its result is quantised)
  float scale2;
  float* part;
  int splits;
};
// ... on the tensor cores (16-bit queries, head dimension 64 or 128), both kernels of it
bool sm100_tdp_decode_supported(int D, int dtype);
size_t sm100_tdp_decode_workspace(const tritt_cache_t& c);
int sm100_tdp_decode(const TdpDecodeArgs& a, void* workspace, void* o, float* lse, cudaStream_t stream);

// ... with all of the windows in shared memory, where they fit (the same types; one kernel, no workspace)
bool window_tdp_decode_applies(const tritt_cache_t& c, int dtype, int k1w, int k2w, int kkl, int kkr);
int window_tdp_decode(const TdpDecodeArgs& a, void* o, float* lse, cudaStream_t stream);
// ... the soft-max attention with warp-level matrix instructions (the same)
bool mma_dps_decode_supported(int D, int dtype);
size_t mma_dps_decode_workspace(const tritt_cache_t& c);
// (early: the kernel ahead in the stream is launch_write's)
int mma_dps_decode(const DpsDecodeArgs& a, void* workspace, void* o, float* lse, const tritt_rows_t* v2, bool early, cudaStream_t stream);

int simt_decode_splits(const tritt_cache_t& c);
int simt_tdp_decode(const TdpDecodeArgs& a, cudaStream_t stream);
int simt_dps_decode(const DpsDecodeArgs& a, cudaStream_t stream);

}  // namespace tritt
