// Attention of new tokens over the cache on the CUDA cores, in fp32, for every type and head dimension: what the tensor-core kernels
// do not take (fp32 tensors, other head dimensions), and what they are compared with.
//
// A warp takes a token k (triple dot product: and then each j) of the attended ones, a lane D / 32 elements; scores are warp sums, the
// soft-max is the running one.  The warps of a block and the splits of a row meet in the parts that the join kernel adds up.
// Bound by the warp sums: about 40 instructions a pair, 0.2 us for a thousand pairs of a row.
#include "tritt_cache.cuh"

namespace tritt {
namespace {

constexpr int kWarps = 4;

template <int CODE> __device__ __forceinline__ float element(const CacheArgs& a, size_t row, int i) {
  const size_t at = row * a.c.D + i;
  if constexpr (CODE == TRITT_CODE_F16) {
    return __half2float(((const __half*)a.c.codes)[at]);
  } else if constexpr (CODE == TRITT_CODE_E4M3) {
    const __half_raw h = __nv_cvt_fp8_to_halfraw(((const uint8_t*)a.c.codes)[at], __NV_E4M3);
    return __half2float(*reinterpret_cast<const __half*>(&h));
  } else {
    return (float)((const int8_t*)a.c.codes)[at];
  }
}

// A lane's E elements of a cached row; false: the row reads as NaN.
template <int CODE, int E>
__device__ __forceinline__ bool load_row(const CacheArgs& a, Place at, int part, int head, int lane, float (&f)[E]) {
  const size_t row = row_of(a, at, part, head);
  const int byte = a.c.exponents[row];
  const float scale = code_scale(byte);
#pragma unroll
  for (int e = 0; e < E; ++e) f[e] = lane * E + e < a.c.D ? element<CODE>(a, row, lane * E + e) * scale : 0.f;
  return byte != 255;
}

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// Running soft-max of a warp: maximum (log2 units), sum, result.
template <int E> struct Running {
  float m = -INFINITY, l = 0.f, acc[E];
  __device__ __forceinline__ Running() {
#pragma unroll
    for (int e = 0; e < E; ++e) acc[e] = 0.f;
  }
  // one more score and value (a NaN score leaves the maximum and makes sum and result NaN)
  __device__ __forceinline__ void add(float s, const float (&v)[E]) {
    if (s > m) {
      const float c = exp2f(m - s);
      l *= c;
#pragma unroll
      for (int e = 0; e < E; ++e) acc[e] *= c;
      m = s;
    }
    const float p = s == -INFINITY ? 0.f : exp2f(s - m);
    l += p;
#pragma unroll
    for (int e = 0; e < E; ++e) acc[e] = fmaf(p, v[e], acc[e]);
  }
};

// The block's warps to one part.
template <int E> __device__ __forceinline__ void write_part(const Running<E>& r, float* part, int D, int warp, int lane) {
  __shared__ float ms[kWarps], ls[kWarps], acc[kWarps][32 * E];
  if (lane == 0) ms[warp] = r.m, ls[warp] = r.l;
#pragma unroll
  for (int e = 0; e < E; ++e) acc[warp][lane * E + e] = r.acc[e];
  __syncthreads();
  float m = -INFINITY, l = 0.f;
#pragma unroll
  for (int w = 0; w < kWarps; ++w) m = fmaxf(m, ms[w]);
  float c[kWarps];
#pragma unroll
  for (int w = 0; w < kWarps; ++w) {
    c[w] = ms[w] == -INFINITY ? (ls[w] == 0.f ? 0.f : ls[w]) : exp2f(ms[w] - m);   // (a sum of NaN alone stays NaN)
    l += ms[w] == -INFINITY ? c[w] : ls[w] * c[w];
  }
  for (int i = threadIdx.x; i < D; i += kWarps * 32) {
    float v = 0.f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) v += c[w] == 0.f ? 0.f : acc[w][i] * c[w];
    part[2 + i] = v;
  }
  if (threadIdx.x == 0) part[0] = m, part[1] = l;
}

struct Row {
  int b, head, i, ctx;
  long long row;
  bool on;
  int pos;
  unsigned long long seen;
};
__device__ __forceinline__ Row row_of_block(const CacheArgs& a, long long row) {
  Row r;
  r.row = row;
  r.i = (int)(r.row % a.c.n);
  r.head = (int)(r.row / a.c.n % a.c.N);
  r.b = (int)(r.row / a.c.n / a.c.N);
  r.ctx = context_of(a, r.b);
  r.on = r.i < new_tokens(a, r.b);
  r.seen = a.c.ancestors ? seen_word(a, r.b, r.i) : 0;
  r.pos = r.ctx + depth_of(a, r.b, r.i);
  return r;
}
// Position of token t (a number of the sequence, at most ctx + i) if the row attends to it, else -1.
__device__ __forceinline__ int attended(const CacheArgs& a, const Row& r, int t) {
  if (t < r.ctx) return t;
  const int m = t - r.ctx;
  if (!a.c.ancestors) return t;
  return (r.seen >> m & 1) ? r.ctx + __popcll(r.seen & ((1ull << m) - 1)) : -1;
}
__device__ __forceinline__ Place find(const CacheArgs& a, int b, int t) {
  const Place at = place_of(a, b, t);
  if (at.page < 0 && a.status && (threadIdx.x & 31) == 0) atomicOr(a.status, kStatusPlace);
  return at;
}

template <typename T, int E>
__device__ __forceinline__ void load_query(const tritt_rows_t& q, const Row& r, int D, int lane, float scale, float (&f)[E]) {
  const T* p = (const T*)q.p + rows_at(q, r.b, r.head, r.i);
#pragma unroll
  for (int e = 0; e < E; ++e) f[e] = lane * E + e < D ? to_f(p[lane * E + e]) * scale : 0.f;
}

template <typename T, int CODE, int E>
__global__ void __launch_bounds__(kWarps * 32) simt_tdp_decode_kernel(const __grid_constant__ TdpDecodeArgs a) {
  const CacheArgs& ca = a.cache;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, D = ca.c.D;
  const long long rows = (long long)ca.c.B * ca.c.N * ca.c.n;
  for (long long row = blockIdx.x; row < rows; row += gridDim.x) {
  const Row r = row_of_block(ca, row);
  Running<E> run;
  if (r.on) {
    float q[E];
    load_query<T, E>(a.q, r, D, lane, a.scale2, q);
    const int end = r.ctx + r.i + 1;
    const int k0 = r.pos - a.k2w > 0 ? min(r.pos - a.k2w, r.ctx) : 0, j0 = r.pos - a.k1w > 0 ? min(r.pos - a.k1w, r.ctx) : 0;
    for (int k = k0 + blockIdx.y * kWarps + warp; k < end; k += gridDim.y * kWarps) {
      const int pk = attended(ca, r, k);
      if (pk < 0 || r.pos - pk > a.k2w) continue;
      const Place at = find(ca, r.b, k);
      if (at.page < 0) continue;
      float x[E], v2[E];
      bool fine = load_row<CODE, E>(ca, at, kPartK2, r.head, lane, x);
      fine = load_row<CODE, E>(ca, at, kPartV2, r.head, lane, v2) && fine;
#pragma unroll
      for (int e = 0; e < E; ++e) x[e] *= q[e];
      for (int j = max(j0, min(r.ctx, pk - min(a.kkl, pk))); j < end; ++j) {
        const int pj = attended(ca, r, j);
        if (pj >= 0 && pj < r.ctx && pj - pk > a.kkr) {   // (the rest of the context is further on)
          j = r.ctx - 1;
          continue;
        }
        if (pj < 0 || r.pos - pj > a.k1w || pk - pj > a.kkl || pj - pk > a.kkr) continue;
        const Place aj = find(ca, r.b, j);
        if (aj.page < 0) continue;
        float y[E], v[E], s = 0.f;
        bool good = load_row<CODE, E>(ca, aj, kPartK1, r.head, lane, y) && fine;
        good = load_row<CODE, E>(ca, aj, kPartV1, r.head, lane, v) && good;
#pragma unroll
        for (int e = 0; e < E; ++e) s = fmaf(x[e], y[e], s), v[e] *= v2[e];
        s = warp_sum(s);
        run.add(good ? s : __uint_as_float(0x7fffffffu), v);
      }
    }
  }
  __syncthreads();
  write_part<E>(run, a.part + ((size_t)r.row * a.splits + blockIdx.y) * (D + 2), D, warp, lane);
  __syncthreads();
  }
}

template <typename T, int CODE, int E>
__global__ void __launch_bounds__(kWarps * 32) simt_dps_decode_kernel(const __grid_constant__ DpsDecodeArgs a) {
  const CacheArgs& ca = a.cache;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, D = ca.c.D;
  const long long rows = (long long)ca.c.B * ca.c.N * ca.c.n;
  for (long long row = blockIdx.x; row < rows; row += gridDim.x) {
  const Row r = row_of_block(ca, row);
  Running<E> run;
  if (r.on) {
    float q[E];
    load_query<T, E>(a.q, r, D, lane, a.scale2, q);
    const int first = r.pos - a.window > 0 ? min(r.pos - a.window, r.ctx) : 0;
    for (int t = first + blockIdx.y * kWarps + warp; t < r.ctx + r.i + 1; t += gridDim.y * kWarps) {
      const int pt = attended(ca, r, t);
      if (pt < 0 || r.pos - pt > a.window) continue;
      const Place at = find(ca, r.b, t);
      if (at.page < 0) continue;
      float x[E], v[E], s = 0.f;
      bool good = load_row<CODE, E>(ca, at, a.key_part, r.head, lane, x);
      good = load_row<CODE, E>(ca, at, a.value_part, r.head, lane, v) && good;
#pragma unroll
      for (int e = 0; e < E; ++e) s = fmaf(x[e], q[e], s);
      s = warp_sum(s);
      if (a.biased) s = fmaf(ca.c.lse[lse_of(ca, at, r.head)], kLog2e, s);
      run.add(good ? s : __uint_as_float(0x7fffffffu), v);
    }
  }
  __syncthreads();
  write_part<E>(run, a.part + ((size_t)r.row * a.splits + blockIdx.y) * (D + 2), D, warp, lane);
  __syncthreads();
  }
}

template <typename A, typename T, int CODE, int E> int launch(const A& a, cudaStream_t stream) {
  const long long rows = (long long)a.cache.c.B * a.cache.c.N * a.cache.c.n;
  const dim3 grid((unsigned)(rows < 1 << 20 ? rows : 1 << 20), a.splits);
  if constexpr (std::is_same<A, TdpDecodeArgs>::value)
    simt_tdp_decode_kernel<T, CODE, E><<<grid, kWarps * 32, 0, stream>>>(a);
  else
    simt_dps_decode_kernel<T, CODE, E><<<grid, kWarps * 32, 0, stream>>>(a);
  count_launch();
  TRITT_CUDA_OK(cudaGetLastError());
  return 0;
}
template <typename A, typename T, int CODE> int by_size(const A& a, cudaStream_t stream) {
  switch (a.cache.c.D) {
    case 64: return launch<A, T, CODE, 2>(a, stream);
    case 128: return launch<A, T, CODE, 4>(a, stream);
    case 256: return launch<A, T, CODE, 8>(a, stream);
    default: return launch<A, T, CODE, 1>(a, stream);
  }
}
template <typename A, typename T> int by_code(const A& a, cudaStream_t stream) {
  if (a.cache.c.code == TRITT_CODE_F16) return by_size<A, T, TRITT_CODE_F16>(a, stream);
  return a.cache.c.code == TRITT_CODE_E4M3 ? by_size<A, T, TRITT_CODE_E4M3>(a, stream) : by_size<A, T, TRITT_CODE_INT8>(a, stream);
}
template <typename A> int by_type(const A& a, cudaStream_t stream) {
  if (a.dtype == TRITT_F32) return by_code<A, float>(a, stream);
  return a.dtype == TRITT_F16 ? by_code<A, __half>(a, stream) : by_code<A, __nv_bfloat16>(a, stream);
}

}  // namespace

// Blocks for eight an SM, at most 64 a row.
int simt_decode_splits(const tritt_cache_t& c) {
  const long long rows = (long long)c.B * c.N * c.n, want = 8 * 148 / rows;
  return (int)(want < 1 ? 1 : want > 64 ? 64 : want);
}
int simt_tdp_decode(const TdpDecodeArgs& a, cudaStream_t stream) { return by_type(a, stream); }
int simt_dps_decode(const DpsDecodeArgs& a, cudaStream_t stream) { return by_type(a, stream); }

}  // namespace tritt
