// Norms of queries and keys for each head with the position rotation in the same pass, forward and backward.
//
// A row x of D elements (q, k1 or k2; one token and head):  r = 1 / sqrt(mean x^2 + eps),  h = x r,  u = h w,  and of the first R
// elements each pair (a, b) is turned by its position's angle.  With du = the turned-back gradient and g = du w:
//   dw = sum over rows of du h,   dx = r (g - h mean(g h)).
// Everything between the load of a row and its store is fp32.
//
// Bound by HBM: forward one read and one write of the rows, backward two reads and one write.  A thread holds eight neighbouring
// elements, D / 8 lanes a row; the two sums and the other half of a rotated pair cross lanes by shuffles.  The tables (a cosine and a sine, 8
// bytes, for two elements) would be twice the traffic of 16-bit rows, so a thread keeps its position's values for four heads and,
// where there are blocks enough, all three tensors.
#include "tritt_common.cuh"

namespace tritt {
namespace {

constexpr int kNormThreads = 256;
constexpr int kSms = 148;   // of a B200
constexpr int kHeads = 4;   // heads of a token that a group of lanes takes at a time, loads of all in flight together

struct NormParams {
  tritt_norm_rotary_t a;
  int chunks;          // of kHeads heads
  float* partial;      // backward: [3][N][gridDim.x][D]
  int* status;
};

template <typename T> struct Eight;   // eight elements, 16-byte accesses
template <> struct Eight<float> {
  float4 v[2];
  __device__ __forceinline__ void load(const float* p) {
    v[0] = __ldg(reinterpret_cast<const float4*>(p));
    v[1] = __ldg(reinterpret_cast<const float4*>(p) + 1);
  }
  __device__ __forceinline__ void get(float (&f)[8]) const {
    f[0] = v[0].x, f[1] = v[0].y, f[2] = v[0].z, f[3] = v[0].w, f[4] = v[1].x, f[5] = v[1].y, f[6] = v[1].z, f[7] = v[1].w;
  }
  static __device__ __forceinline__ void store(float* p, const float (&f)[8]) {
    reinterpret_cast<float4*>(p)[0] = make_float4(f[0], f[1], f[2], f[3]);
    reinterpret_cast<float4*>(p)[1] = make_float4(f[4], f[5], f[6], f[7]);
  }
};
template <typename T> struct Eight16 {
  uint4 v;
  __device__ __forceinline__ void load(const T* p) { v = __ldg(reinterpret_cast<const uint4*>(p)); }
  __device__ __forceinline__ void get(float (&f)[8]) const {
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
  static __device__ __forceinline__ void store(T* p, const float (&f)[8]) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const T lo = from_f<T>(f[2 * i]), hi = from_f<T>(f[2 * i + 1]);
      w[i] = (uint32_t)*reinterpret_cast<const uint16_t*>(&lo) | (uint32_t)*reinterpret_cast<const uint16_t*>(&hi) << 16;
    }
    *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
  }
};
template <> struct Eight<__half> : Eight16<__half> {};
template <> struct Eight<__nv_bfloat16> : Eight16<__nv_bfloat16> {};

// Sum over the lanes of a row (a power of two of neighbouring lanes).
template <int L> __device__ __forceinline__ float row_sum(float v) {
#pragma unroll
  for (int o = L / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// The eight weights of a thread's columns (1 where there are none).
template <typename T> __device__ __forceinline__ void load_weights(const NormParams& p, int which, int head, int col, float (&w)[8]) {
  const void* base = p.a.w[which];
  const size_t off = (p.a.weight_heads ? (size_t)head * p.a.D : 0) + col;
  if (base == nullptr) {
#pragma unroll
    for (int e = 0; e < 8; ++e) w[e] = 1.f;
  } else if (p.a.weight_dtype == TRITT_F32) {
    Eight<float> v;
    v.load((const float*)base + off);
    v.get(w);
  } else {
    Eight<T> v;
    v.load((const T*)base + off);
    v.get(w);
  }
}

// Cosines and sines of a thread's eight columns: of each column of a half (halves), or of four pairs (interleaved).
struct Turn {
  float c[8], s[8];
};
__device__ __forceinline__ void load_turn(const NormParams& p, int b, int t, int col, Turn& turn) {
  const int R = p.a.rot;
  if (col >= R) return;
  long long at = t;
  if (p.a.positions) {
    const long long i = b * p.a.position_stride_b + t * p.a.position_stride_t;
    at = p.a.positions64 ? ((const long long*)p.a.positions)[i] : ((const int*)p.a.positions)[i];
  }
  if (at < 0 || at >= p.a.table) {
    if (p.status) atomicOr(p.status, 256);
    at = at < 0 ? 0 : p.a.table - 1;
  }
  const size_t row = (size_t)at * (R / 2);
  if (p.a.interleaved) {
    const float4 c = __ldg(reinterpret_cast<const float4*>(p.a.cos + row + col / 2));
    const float4 s = __ldg(reinterpret_cast<const float4*>(p.a.sin + row + col / 2));
    turn.c[0] = c.x, turn.c[1] = c.y, turn.c[2] = c.z, turn.c[3] = c.w;
    turn.s[0] = s.x, turn.s[1] = s.y, turn.s[2] = s.z, turn.s[3] = s.w;
  } else {
    const size_t i = row + (col < R / 2 ? col : col - R / 2);
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      const float4 c = __ldg(reinterpret_cast<const float4*>(p.a.cos + i) + q);
      const float4 s = __ldg(reinterpret_cast<const float4*>(p.a.sin + i) + q);
      turn.c[4 * q] = c.x, turn.c[4 * q + 1] = c.y, turn.c[4 * q + 2] = c.z, turn.c[4 * q + 3] = c.w;
      turn.s[4 * q] = s.x, turn.s[4 * q + 1] = s.y, turn.s[4 * q + 2] = s.z, turn.s[4 * q + 3] = s.w;
    }
  }
}

// Turns a row's eight elements (sign 1), or turns them back (-1).  All lanes of the row call it.
__device__ __forceinline__ void rotate(const NormParams& p, const Turn& turn, float sign, int col, float (&u)[8]) {
  const int R = p.a.rot;
  if (R == 0) return;
  if (p.a.interleaved) {
    if (col < R) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float x = u[2 * i], y = u[2 * i + 1], s = sign * turn.s[i];
        u[2 * i] = x * turn.c[i] - y * s;
        u[2 * i + 1] = y * turn.c[i] + x * s;
      }
    }
    return;
  }
  // the pair's other element is R / 2 columns on or back, R / 16 lanes
  const bool first = col < R / 2;
  const int lane = threadIdx.x & 31, other = col >= R ? lane : first ? lane + R / 16 : lane - R / 16;
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const float o = __shfl_sync(0xffffffffu, u[e], other);
    if (col < R) u[e] = u[e] * turn.c[e] + (first ? -o : o) * (sign * turn.s[e]);
  }
}

__device__ __forceinline__ size_t row_offset(const tritt_rows_t& r, int b, int n, int t) {
  return (size_t)(b * r.stride_b + n * r.stride_n + t * r.stride_t);
}

template <typename T, int D>
__global__ void __launch_bounds__(kNormThreads) norm_rotary_fwd_kernel(const __grid_constant__ NormParams p) {
  constexpr int L = D / 8, kSlots = kNormThreads / L;
  const int col = threadIdx.x % L * 8;
  const long long tokens = (long long)p.a.B * p.a.T;
  // (lanes without a row of their own stay for the shuffles)
  const long long slot = (long long)blockIdx.x * kSlots + threadIdx.x / L;
  const long long token = slot / p.chunks;
  const bool live = token < tokens;
  const int h0 = (int)(slot % p.chunks) * kHeads;
  const int b = live ? (int)(token / p.a.T) : 0, t = live ? (int)(token % p.a.T) : 0;
  Turn turn;
  if (live && p.a.rot) load_turn(p, b, t, col, turn);
  for (int which = blockIdx.y; which < 3; which += gridDim.y) {
    Eight<T> in[kHeads];
#pragma unroll
    for (int i = 0; i < kHeads; ++i)
      if (live && h0 + i < p.a.N) in[i].load((const T*)p.a.x[which].p + row_offset(p.a.x[which], b, h0 + i, t) + col);
    float w[8];
    if (!p.a.weight_heads) load_weights<T>(p, which, 0, col, w);
#pragma unroll
    for (int i = 0; i < kHeads; ++i) {
      const bool on = live && h0 + i < p.a.N;
      float u[8], sq = 0.f;
      if (on) {
        in[i].get(u);
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) u[e] = 0.f;
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) sq = fmaf(u[e], u[e], sq);
      const float r = rsqrtf(row_sum<L>(sq) * (1.f / D) + p.a.eps);
      if (p.a.weight_heads && on) load_weights<T>(p, which, h0 + i, col, w);
#pragma unroll
      for (int e = 0; e < 8; ++e) u[e] = u[e] * r * w[e];
      rotate(p, turn, 1.f, col, u);
      if (on) Eight<T>::store((T*)p.a.y[which].p + row_offset(p.a.y[which], b, h0 + i, t) + col, u);
    }
  }
}

// A block takes kHeads heads of one tensor and tokens blockIdx.x, + gridDim.x, ... in groups, so that the weights' gradients add up
// in registers: then over the block's rows, and by the kernel below over the blocks, always in the same order.
template <typename T, int D>
__global__ void __launch_bounds__(kNormThreads) norm_rotary_bwd_kernel(const __grid_constant__ NormParams p) {
  constexpr int L = D / 8, kSlots = kNormThreads / L;
  __shared__ float sums[kSlots][D];
  const int col = threadIdx.x % L * 8, slot = threadIdx.x / L;
  const int which = blockIdx.y / p.chunks, h0 = blockIdx.y % p.chunks * kHeads;
  const long long tokens = (long long)p.a.B * p.a.T;
  const bool weights = p.partial != nullptr && p.a.dw[which] != nullptr;
  float dw[kHeads][8];
#pragma unroll
  for (int i = 0; i < kHeads; ++i)
#pragma unroll
    for (int e = 0; e < 8; ++e) dw[i][e] = 0.f;
  float w[8];
  if (!p.a.weight_heads) load_weights<T>(p, which, 0, col, w);
  for (long long first = (long long)blockIdx.x * kSlots; first < tokens; first += (long long)gridDim.x * kSlots) {
    const long long token = first + slot;
    const bool live = token < tokens;
    const int b = live ? (int)(token / p.a.T) : 0, t = live ? (int)(token % p.a.T) : 0;
    Eight<T> in[kHeads], up[kHeads];
#pragma unroll
    for (int i = 0; i < kHeads; ++i)
      if (live && h0 + i < p.a.N) {
        in[i].load((const T*)p.a.x[which].p + row_offset(p.a.x[which], b, h0 + i, t) + col);
        up[i].load((const T*)p.a.y[which].p + row_offset(p.a.y[which], b, h0 + i, t) + col);
      }
    Turn turn;
    if (live && p.a.rot) load_turn(p, b, t, col, turn);
#pragma unroll
    for (int i = 0; i < kHeads; ++i) {
      const bool on = live && h0 + i < p.a.N;
      float x[8], g[8], sq = 0.f, dot = 0.f;
      if (on) {
        in[i].get(x);
        up[i].get(g);
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = g[e] = 0.f;
      }
      rotate(p, turn, -1.f, col, g);
#pragma unroll
      for (int e = 0; e < 8; ++e) sq = fmaf(x[e], x[e], sq);
      const float r = rsqrtf(row_sum<L>(sq) * (1.f / D) + p.a.eps);
      if (p.a.weight_heads && on) load_weights<T>(p, which, h0 + i, col, w);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        x[e] *= r;
        if (on) dw[i][e] = fmaf(g[e], x[e], dw[i][e]);
        g[e] *= w[e];
        dot = fmaf(g[e], x[e], dot);
      }
      const float mean = row_sum<L>(dot) * (1.f / D);
#pragma unroll
      for (int e = 0; e < 8; ++e) g[e] = r * (g[e] - x[e] * mean);
      if (on) Eight<T>::store((T*)p.a.dx[which].p + row_offset(p.a.dx[which], b, h0 + i, t) + col, g);
    }
  }
  if (!weights) return;
  for (int i = 0; i < kHeads && h0 + i < p.a.N; ++i) {
    __syncthreads();
#pragma unroll
    for (int e = 0; e < 8; ++e) sums[slot][col + e] = dw[i][e];
    __syncthreads();
    for (int c = threadIdx.x; c < D; c += kNormThreads) {
      float total = 0.f;
      for (int s = 0; s < kSlots; ++s) total += sums[s][c];
      p.partial[(((size_t)which * p.a.N + h0 + i) * gridDim.x + blockIdx.x) * D + c] = total;
    }
  }
}

// Adds up `rows` partial sums of each column: those of a head, or of all heads.  One block a (tensor, head or all), 32 columns a warp-row.
template <typename T>
__global__ void __launch_bounds__(1024) norm_rotary_weights_kernel(const __grid_constant__ NormParams p, int blocks) {
  __shared__ float sums[32][33];
  const int which = blockIdx.z, head = blockIdx.y, D = p.a.D;
  const int c = blockIdx.x * 32 + threadIdx.x % 32, group = threadIdx.x / 32;
  if (p.a.dw[which] == nullptr) return;
  const int rows = p.a.weight_heads ? blocks : blocks * p.a.N;
  const float* base = p.partial + ((size_t)which * p.a.N + head) * blocks * D;
  float total = 0.f;
  if (c < D)
    for (int i = group; i < rows; i += 32) total += base[(size_t)i * D + c];
  sums[group][threadIdx.x % 32] = total;
  __syncthreads();
  if (group == 0 && c < D) {
    total = 0.f;
    for (int s = 0; s < 32; ++s) total += sums[s][threadIdx.x % 32];
    const size_t at = (p.a.weight_heads ? (size_t)head * D : 0) + c;
    if (p.a.weight_dtype == TRITT_F32)
      ((float*)p.a.dw[which])[at] = total;
    else
      ((T*)p.a.dw[which])[at] = from_f<T>(total);
  }
}

// Blocks of the backward along the tokens: as many as the chip holds at once (three of 256 threads an SM) over the heads' and tensors' groups.
int bwd_blocks(const tritt_norm_rotary_t& a) {
  const int chunks = (a.N + kHeads - 1) / kHeads, slots = kNormThreads / (a.D / 8);
  const long long tokens = (long long)a.B * a.T, most = (tokens + slots - 1) / slots;
  const long long fill = (3LL * kSms + 3 * chunks - 1) / (3 * chunks);
  return (int)(most < fill ? most : fill);
}

int check(const tritt_norm_rotary_t* a, bool backward) {
  if (!a || a->B <= 0 || a->N <= 0 || a->T <= 0) {
    set_error("B, N and T must be positive");
    return -1;
  }
  if (a->D != 16 && a->D != 32 && a->D != 64 && a->D != 128 && a->D != 256) {
    set_error("head_dim must be 16, 32, 64, 128 or 256, got %d", a->D);
    return -2;
  }
  if (a->dtype != TRITT_F32 && a->dtype != TRITT_F16 && a->dtype != TRITT_BF16) {
    set_error("unknown dtype code %d", a->dtype);
    return -3;
  }
  if (a->weight_dtype != TRITT_F32 && a->weight_dtype != a->dtype) {
    set_error("weights must be of the rows' type or fp32");
    return -3;
  }
  for (int i = 0; i < 3; ++i)
    if (((uintptr_t)a->w[i] | (uintptr_t)a->dw[i]) & 15) {
      set_error("weights must start on 16-byte boundaries");
      return -5;
    }
  const long long unit = a->dtype == TRITT_F32 ? 4 : 8;
  for (int i = 0; i < 3; ++i) {
    const tritt_rows_t* rows[3] = {&a->x[i], &a->y[i], &a->dx[i]};
    for (int k = 0; k < (backward ? 3 : 2); ++k) {
      if (!rows[k]->p) {
        set_error("null tensor pointer");
        return -4;
      }
      if (((uintptr_t)rows[k]->p & 15) || rows[k]->stride_b % unit || rows[k]->stride_n % unit || rows[k]->stride_t % unit) {
        set_error("rows must start on 16-byte boundaries");
        return -5;
      }
    }
  }
  if (a->rot < 0 || a->rot > a->D || a->rot % 16) {
    set_error("the rotated part must be a multiple of 16 elements of the head dimension, got %d", a->rot);
    return -13;
  }
  if (a->rot && (!a->cos || !a->sin || ((uintptr_t)a->cos & 15) || ((uintptr_t)a->sin & 15) || a->table < 1)) {
    set_error("a rotation needs tables of cosines and sines on 16-byte boundaries");
    return -13;
  }
  if (a->rot && !a->positions && a->T > a->table) {
    set_error("the tables have %d positions, the sequence %d", a->table, a->T);
    return -13;
  }
  return 0;
}

template <typename T, int D> int launch_fwd(const NormParams& p, cudaStream_t stream) {
  constexpr int kSlots = kNormThreads / (D / 8);
  const long long slots = (long long)p.a.B * p.a.T * p.chunks, blocks = (slots + kSlots - 1) / kSlots;
  if (blocks > 0x7fffffff) {
    set_error("too many rows for one call");
    return -11;
  }
  // one tensor a block until the chip is full several times over
  const dim3 grid((unsigned)blocks, blocks >= 8LL * kSms ? 1 : 3);
  norm_rotary_fwd_kernel<T, D><<<grid, kNormThreads, 0, stream>>>(p);
  count_launch();
  TRITT_CUDA_OK(cudaGetLastError());
  return 0;
}

template <typename T, int D> int launch_bwd(const NormParams& p, cudaStream_t stream) {
  const int blocks = bwd_blocks(p.a);
  norm_rotary_bwd_kernel<T, D><<<dim3(blocks, 3 * p.chunks), kNormThreads, 0, stream>>>(p);
  count_launch();
  TRITT_CUDA_OK(cudaGetLastError());
  if (!p.partial) return 0;
  norm_rotary_weights_kernel<T><<<dim3((D + 31) / 32, p.a.weight_heads ? p.a.N : 1, 3), 1024, 0, stream>>>(p, blocks);
  count_launch();
  TRITT_CUDA_OK(cudaGetLastError());
  return 0;
}

template <typename T> int by_size(const NormParams& p, bool backward, cudaStream_t stream) {
  switch (p.a.D) {
    case 16: return backward ? launch_bwd<T, 16>(p, stream) : launch_fwd<T, 16>(p, stream);
    case 32: return backward ? launch_bwd<T, 32>(p, stream) : launch_fwd<T, 32>(p, stream);
    case 64: return backward ? launch_bwd<T, 64>(p, stream) : launch_fwd<T, 64>(p, stream);
    case 128: return backward ? launch_bwd<T, 128>(p, stream) : launch_fwd<T, 128>(p, stream);
    default: return backward ? launch_bwd<T, 256>(p, stream) : launch_fwd<T, 256>(p, stream);
  }
}
int by_type(const NormParams& p, bool backward, cudaStream_t stream) {
  if (p.a.dtype == TRITT_F32) return by_size<float>(p, backward, stream);
  return p.a.dtype == TRITT_F16 ? by_size<__half>(p, backward, stream) : by_size<__nv_bfloat16>(p, backward, stream);
}

bool wants_weights(const tritt_norm_rotary_t& a) { return a.dw[0] || a.dw[1] || a.dw[2]; }

}  // namespace
}  // namespace tritt

using namespace tritt;

extern "C" {

int tritt_qk_norm_rotary_fwd(const tritt_norm_rotary_t* a, int* status_word, tritt_stream_t stream) {
  if (int rc = check(a, false)) return rc;
  NormParams p{*a, (a->N + kHeads - 1) / kHeads, nullptr, status_word};
  return by_type(p, false, (cudaStream_t)stream);
}

size_t tritt_qk_norm_rotary_workspace(const tritt_norm_rotary_t* a) {
  if (!a || a->B <= 0 || a->N <= 0 || a->T <= 0 || a->D < 16 || a->D > 256 || !wants_weights(*a)) return 0;
  return align_up((size_t)3 * a->N * bwd_blocks(*a) * a->D * 4, 256);
}

int tritt_qk_norm_rotary_bwd(const tritt_norm_rotary_t* a, void* workspace, size_t workspace_bytes, int* status_word,
                             tritt_stream_t stream) {
  if (int rc = check(a, true)) return rc;
  const size_t need = tritt_qk_norm_rotary_workspace(a);
  if (need && (!workspace || workspace_bytes < need || ((uintptr_t)workspace & 15))) {
    set_error("workspace too small or misaligned: need %zu bytes, got %zu", need, workspace ? workspace_bytes : (size_t)0);
    return -6;
  }
  if (((long long)a->N + kHeads - 1) / kHeads * 3 > 65535) {
    set_error("too many heads");
    return -11;
  }
  NormParams p{*a, (a->N + kHeads - 1) / kHeads, need ? (float*)workspace : nullptr, status_word};
  return by_type(p, true, (cudaStream_t)stream);
}

}  // extern "C"
