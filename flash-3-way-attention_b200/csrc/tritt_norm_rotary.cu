// Norms of queries and keys for each head with the position rotation in the same pass, forward and backward.
//
// A row x of D elements (q, k1 or k2; one token and head):  r = 1 / sqrt(mean x^2 + eps),  h = x r,  u = h w,  and of the first R
// elements each pair (a, b) is turned by its position's angle.  With du = the turned-back gradient and g = du w:
//   dw = sum over rows of du h,   dx = r (g - h mean(g h)).
// Everything between the load of a row and its store is fp32.
//
// Bound by HBM: forward one read and one write of the rows, backward two reads and one write.  D / 8 lanes take a row, eight elements each:
// two groups of four that lie R / 2 apart, so that a thread holds both of each rotated pair (neighbours where there is no rotation or
// neighbours are rotated).  With eight neighbours a lane and the other half by shuffles the forward executed 202 instructions for eight
// elements, and instruction issue bounded it (4 x 16 heads x 2048 x 128 bf16: 53 us, the backward 121).  Two fp32 numbers an instruction: 38 us without rotation
// (5.3 TB/s), 41 with positions 0, 1, 2, ... and 43 with an array of them, whose load comes before that of the tables; the backward, whose chains of two sums over a row's lanes leave half of the issue slots, 69, 72 and 74
// (4.1 to 4.4 TB/s) and 4 to 5 for the weights' last sums.  (Kernels by themselves.)
// The tables (a cosine and a sine, 8 bytes, for two elements) would be twice the traffic of 16-bit rows, so a thread keeps its position's
// values for four heads and, where there are blocks enough, all three tensors.
// Positions of several axes are kernels of their own (AXES): the same, but that a lane whose four pairs are not all of one axis takes their values one
// by one.  4 x 16 heads x 2048 x 128 bf16, three axes: calls of the forward 45.6 us one axis after the other and 46.3 in turn, 45.1 with one axis; forward and backward
// 134 to 136 in turn (132 with one).
#include "tritt_cache.cuh"
#include "tritt_common.cuh"

#include <type_traits>

namespace tritt {
namespace {

constexpr int kNormThreads = 256;
constexpr int kSms = 148;   // of a B200
constexpr int kHeads = 4;   // heads of a token that a group of lanes takes at a time, loads of all in flight together

struct NormParams {
  tritt_norm_rotary_t a;
  tritt_axes_t axes;   // of kernels with AXES
  int chunks;          // of kHeads heads
  int blocks, groups;  // backward: its grid
  float* partial;      // backward: [3][heads, or groups of heads][blocks][D]
  int* status;
};

__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  float2 r;
  asm("{\n\t.reg .b64 x, y;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tmul.rn.ftz.f32x2 x, x, y;\n\tmov.b64 {%0, %1}, x;\n\t}"
      : "=f"(r.x), "=f"(r.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return r;
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 r;
  asm("{\n\t.reg .b64 x, y, z;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tmov.b64 z, {%6, %7};\n\tfma.rn.ftz.f32x2 x, x, y, z;\n\tmov.b64 {%0, %1}, x;\n\t}"
      : "=f"(r.x), "=f"(r.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return r;
}
__device__ __forceinline__ float2 both(float v) { return make_float2(v, v); }

// A lane's eight elements as four pairs of neighbours: pairs 0, 1 from column a on, 2, 3 from column b on.
struct Cols {
  int a, b;
};
// With the halves rotated, lane i of the first R / 8 takes columns 4 i .. and R / 2 + 4 i ..; any other lane eight neighbours.
__device__ __forceinline__ Cols cols_of(int lane, int rot, int interleaved) {
  if (!interleaved && lane * 8 < rot) return Cols{lane * 4, rot / 2 + lane * 4};
  return Cols{lane * 8, lane * 8 + 4};
}

template <typename T> struct Eight {   // of a 16-bit type
  uint2 v[2];
  __device__ __forceinline__ void load(const T* p, Cols c) {
    v[0] = __ldg(reinterpret_cast<const uint2*>(p + c.a));
    v[1] = __ldg(reinterpret_cast<const uint2*>(p + c.b));
  }
  __device__ __forceinline__ void get(float2 (&f)[4]) const {
    const uint32_t w[4] = {v[0].x, v[0].y, v[1].x, v[1].y};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (std::is_same<T, __half>::value)
        f[i] = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
      else
        f[i] = make_float2(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xffff0000u));
    }
  }
  static __device__ __forceinline__ void store(T* p, Cols c, const float2 (&f)[4]) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (std::is_same<T, __half>::value) {
        const __half2 h = __floats2half2_rn(f[i].x, f[i].y);
        w[i] = *reinterpret_cast<const uint32_t*>(&h);
      } else {
        const __nv_bfloat162 h = __floats2bfloat162_rn(f[i].x, f[i].y);
        w[i] = *reinterpret_cast<const uint32_t*>(&h);
      }
    }
    *reinterpret_cast<uint2*>(p + c.a) = make_uint2(w[0], w[1]);
    *reinterpret_cast<uint2*>(p + c.b) = make_uint2(w[2], w[3]);
  }
};
template <> struct Eight<float> {
  float4 v[2];
  __device__ __forceinline__ void load(const float* p, Cols c) {
    v[0] = __ldg(reinterpret_cast<const float4*>(p + c.a));
    v[1] = __ldg(reinterpret_cast<const float4*>(p + c.b));
  }
  __device__ __forceinline__ void get(float2 (&f)[4]) const {
    f[0] = make_float2(v[0].x, v[0].y), f[1] = make_float2(v[0].z, v[0].w), f[2] = make_float2(v[1].x, v[1].y), f[3] = make_float2(v[1].z, v[1].w);
  }
  static __device__ __forceinline__ void store(float* p, Cols c, const float2 (&f)[4]) {
    *reinterpret_cast<float4*>(p + c.a) = make_float4(f[0].x, f[0].y, f[1].x, f[1].y);
    *reinterpret_cast<float4*>(p + c.b) = make_float4(f[2].x, f[2].y, f[3].x, f[3].y);
  }
};

// Sum over the lanes of a row (a power of two of neighbouring lanes).
template <int L> __device__ __forceinline__ float row_sum(float v) {
#pragma unroll
  for (int o = L / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
__device__ __forceinline__ float dot(const float2 (&a)[4], const float2 (&b)[4]) {
  float2 s = mul2(a[0], b[0]);
#pragma unroll
  for (int i = 1; i < 4; ++i) s = fma2(a[i], b[i], s);
  return s.x + s.y;
}

// The weights of a thread's columns (1 where there are none).
template <typename T> __device__ __forceinline__ void load_weights(const NormParams& p, int which, int head, Cols c, float2 (&w)[4]) {
  const void* base = p.a.w[which];
  const size_t off = p.a.weight_heads ? (size_t)head * p.a.D : 0;
  if (base == nullptr) {
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = both(1.f);
  } else if (p.a.weight_dtype == TRITT_F32) {
    Eight<float> v;
    v.load((const float*)base + off, c);
    v.get(w);
  } else {
    Eight<T> v;
    v.load((const T*)base + off, c);
    v.get(w);
  }
}

// Cosines and sines of a thread's four rotated pairs: (1, 0) where its columns are not rotated.
struct Turn {
  float c[4], s[4];
};
// A position from the given place of its array, as the tables have it.
__device__ __forceinline__ long long position_at(const NormParams& p, long long i) {
  return p.a.positions64 ? ((const long long*)p.a.positions)[i] : ((const int*)p.a.positions)[i];
}
__device__ __forceinline__ long long table_row(const NormParams& p, long long at) {
  if (at < 0 || at >= p.a.table) {
    if (p.status) atomicOr(p.status, 256);
    at = at < 0 ? 0 : p.a.table - 1;
  }
  return at;
}
template <bool AXES> __device__ __forceinline__ Turn load_turn(const NormParams& p, int b, int t, int lane) {
  Turn turn{{1.f, 1.f, 1.f, 1.f}, {0.f, 0.f, 0.f, 0.f}};
  if (lane * 8 >= p.a.rot) return turn;
  long long at = t;
  if constexpr (AXES) {
    const long long i = b * p.a.position_stride_b + t * p.a.position_stride_t;
    const int of = p.axes.of[lane];   // two bits for each of the lane's four pairs
    const long long first = table_row(p, position_at(p, i + (of & 3) * p.axes.position_stride));
    if (of != (of & 3) * 0x55) {   // pairs of several axes: element by element (the rows are in L1, for the block's other heads)
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int axis = of >> 2 * k & 3;
        const long long row = axis == (of & 3) ? first : table_row(p, position_at(p, i + axis * p.axes.position_stride));
        turn.c[k] = __ldg(p.a.cos + row * (p.a.rot / 2) + lane * 4 + k);
        turn.s[k] = __ldg(p.a.sin + row * (p.a.rot / 2) + lane * 4 + k);
      }
      return turn;
    }
    at = first;
  } else {
    if (p.a.positions) at = position_at(p, b * p.a.position_stride_b + t * p.a.position_stride_t);
    at = table_row(p, at);
  }
  const size_t i = (size_t)at * (p.a.rot / 2) + lane * 4;   // (either way of pairing: lane i has pairs 4 i .. 4 i + 3)
  const float4 c = __ldg(reinterpret_cast<const float4*>(p.a.cos + i)), s = __ldg(reinterpret_cast<const float4*>(p.a.sin + i));
  turn.c[0] = c.x, turn.c[1] = c.y, turn.c[2] = c.z, turn.c[3] = c.w;
  turn.s[0] = s.x, turn.s[1] = s.y, turn.s[2] = s.z, turn.s[3] = s.w;
  return turn;
}

// Turns a lane's eight elements (sign 1), or turns them back (-1).
__device__ __forceinline__ void rotate(bool interleaved, const Turn& turn, float sign, float2 (&u)[4]) {
  if (interleaved) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      u[i] = fma2(make_float2(-u[i].y, u[i].x), both(sign * turn.s[i]), mul2(u[i], both(turn.c[i])));
    return;
  }
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const float2 c = make_float2(turn.c[2 * i], turn.c[2 * i + 1]), s = make_float2(sign * turn.s[2 * i], sign * turn.s[2 * i + 1]);
    const float2 x = u[i], y = u[2 + i];
    u[i] = fma2(y, make_float2(-s.x, -s.y), mul2(x, c));
    u[2 + i] = fma2(x, s, mul2(y, c));
  }
}

__device__ __forceinline__ size_t row_offset(const tritt_rows_t& r, int b, int n, int t) {
  return (size_t)(b * r.stride_b + n * r.stride_n + t * r.stride_t);
}

template <typename T, int D, bool AXES>
__global__ void __launch_bounds__(kNormThreads) norm_rotary_fwd_kernel(const __grid_constant__ NormParams p) {
  constexpr int L = D / 8, kSlots = kNormThreads / L;
  const int lane = threadIdx.x % L;
  const Cols cols = cols_of(lane, p.a.rot, p.a.interleaved);
  const bool interleaved = p.a.interleaved;
  // (32 bits, which the host has seen to; lanes without a row of their own stay for the sums)
  const uint32_t tokens = (uint32_t)p.a.B * p.a.T, slot = blockIdx.x * kSlots + threadIdx.x / L, token = slot / p.chunks;
  const bool live = token < tokens;
  const int h0 = (int)(slot - token * p.chunks) * kHeads;
  const int b = live ? token / p.a.T : 0, t = live ? token - (uint32_t)b * p.a.T : 0;
  Turn turn;
  if (p.a.rot) turn = load_turn<AXES>(p, b, t, lane);
  for (int which = blockIdx.y; which < 3; which += gridDim.y) {
    Eight<T> in[kHeads];
    const T* from = (const T*)p.a.x[which].p + row_offset(p.a.x[which], b, h0, t);
    T* to = (T*)p.a.y[which].p + row_offset(p.a.y[which], b, h0, t);
#pragma unroll
    for (int i = 0; i < kHeads; ++i)
      if (live && h0 + i < p.a.N) in[i].load(from + i * p.a.x[which].stride_n, cols);
    float2 w[4];
    if (!p.a.weight_heads) load_weights<T>(p, which, 0, cols, w);
#pragma unroll
    for (int i = 0; i < kHeads; ++i) {
      const bool on = live && h0 + i < p.a.N;
      float2 u[4] = {both(0.f), both(0.f), both(0.f), both(0.f)};
      if (on) in[i].get(u);
      const float2 r = both(rsqrtf(row_sum<L>(dot(u, u)) * (1.f / D) + p.a.eps));
      if (p.a.weight_heads && on) load_weights<T>(p, which, h0 + i, cols, w);
#pragma unroll
      for (int k = 0; k < 4; ++k) u[k] = mul2(mul2(u[k], r), w[k]);
      if (p.a.rot) rotate(interleaved, turn, 1.f, u);
      if (on) Eight<T>::store(to + i * p.a.y[which].stride_n, cols, u);
    }
  }
}

// A block takes one tensor's rows of tokens blockIdx.x, + gridDim.x, ... in groups: neighbouring slots (D / 8 lanes) kHeads heads each of a
// token, whose rows are neighbours where the tensors come out of one projection (a block for each four heads read 1 KB here and
// there: 98 us instead of 86, then, for 4 x 16 heads x 2048 x 128 bf16).  A slot's heads stay the same, so the weights' gradients add up
// in registers: then over the block's slots, and by the kernel below over the blocks, always in the same order.
//
// Rows of 16-bit types come by asynchronous copies, one or two tokens ahead, each thread's into places of its own: loads to
// registers, of which there are no more, waited for one token's rows while nothing else was on its way (86 us then, 77 with the copies).  SHARED: one
// weight for all heads, so one sum, and registers for three blocks an SM (73 us); tokens found by counting instead of division (70).
template <typename T, bool SHARED> constexpr int kPerSm = SHARED && sizeof(T) == 2 ? 3 : 2;
template <bool SHARED> constexpr int kStages = SHARED ? 2 : 3;
constexpr int kStageBytes = kHeads * 4 * kNormThreads * 8;
template <typename T, bool SHARED> constexpr int kBwdSmem = sizeof(T) == 2 ? kStages<SHARED> * kStageBytes : 0;
__device__ __forceinline__ void copy8(void* dst, const void* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"((uint32_t)__cvta_generic_to_shared(dst)), "l"(src) : "memory");
}

template <typename T, int D, bool SHARED, bool AXES>
__global__ void __launch_bounds__(kNormThreads, kPerSm<T, SHARED>) norm_rotary_bwd_kernel(const __grid_constant__ NormParams p) {
  constexpr int L = D / 8, kSlots = kNormThreads / L, kSums = SHARED ? 1 : kHeads, NS = kStages<SHARED>;
  constexpr bool kAsync = sizeof(T) == 2;
  extern __shared__ __align__(16) uint8_t staged[];
  __shared__ float sums[kSlots][D];
  const int lane = threadIdx.x % L, slot = threadIdx.x / L;
  const Cols cols = cols_of(lane, p.a.rot, p.a.interleaved);
  const bool interleaved = p.a.interleaved;
  const int here = p.chunks < kSlots ? p.chunks : kSlots, at_once = kSlots / here;   // heads' groups of a token, tokens
  const int groups = (p.chunks + here - 1) / here, which = blockIdx.y / groups, chunk0 = blockIdx.y % groups * here;
  const int chunk = chunk0 + slot % here, h0 = chunk * kHeads;
  const bool used = slot < at_once * here && chunk < p.chunks;
  const uint32_t tokens = (uint32_t)p.a.B * p.a.T;
  const bool weights = p.partial != nullptr && p.a.dw[which] != nullptr;
  const tritt_rows_t rx = p.a.x[which], ry = p.a.y[which], rd = p.a.dx[which];
  float2 dw[kSums][4];
#pragma unroll
  for (int i = 0; i < kSums; ++i)
#pragma unroll
    for (int k = 0; k < 4; ++k) dw[i][k] = both(0.f);
  float2 w[4];
  if (SHARED) load_weights<T>(p, which, 0, cols, w);
  const uint32_t step = gridDim.x * at_once;
  uint2* const mine = reinterpret_cast<uint2*>(staged) + threadIdx.x;   // [stage][head][x, x, dy, dy][thread]
  // a thread's token as batch and position, found by division once, then step by step
  struct Token {
    uint32_t n;
    int b, t;
  };
  const int step_b = (int)(step / (uint32_t)p.a.T), step_t = (int)(step - (uint32_t)step_b * p.a.T);
  auto next = [&](Token k) {
    k.n += step;
    k.b += step_b;
    k.t += step_t;
    if (k.t >= p.a.T) k.t -= p.a.T, ++k.b;
    return k;
  };
  auto send = [&](Token k, int stage) {
    if constexpr (kAsync) {
      if (used && k.n < tokens) {
        const int b = k.b, t = k.t;
        const T *x0 = (const T*)rx.p + row_offset(rx, b, h0, t), *y0 = (const T*)ry.p + row_offset(ry, b, h0, t);
        uint2* to = mine + stage * (kStageBytes / 8);
#pragma unroll
        for (int i = 0; i < kHeads; ++i)
          if (h0 + i < p.a.N) {
            const T *x = x0 + i * rx.stride_n, *y = y0 + i * ry.stride_n;
            copy8(to + (i * 4 + 0) * kNormThreads, x + cols.a);
            copy8(to + (i * 4 + 1) * kNormThreads, x + cols.b);
            copy8(to + (i * 4 + 2) * kNormThreads, y + cols.a);
            copy8(to + (i * 4 + 3) * kNormThreads, y + cols.b);
          }
      }
      asm volatile("cp.async.commit_group;" ::: "memory");
    }
  };
  int stage = 0;
  Token now{blockIdx.x * at_once + slot / here, 0, 0};
  now.b = (int)(now.n / (uint32_t)p.a.T), now.t = (int)(now.n - (uint32_t)now.b * p.a.T);
  Token ahead = now;
#pragma unroll
  for (int s = 0; s < NS - 1; ++s, ahead = next(ahead)) send(ahead, s);
  for (uint32_t first = blockIdx.x * at_once; first < tokens; first += step, now = next(now), ahead = next(ahead)) {
    const bool live = used && now.n < tokens;
    const int b = live ? now.b : 0, t = live ? now.t : 0;
    send(ahead, stage == 0 ? NS - 1 : stage - 1);
    Eight<T> in[kAsync ? 1 : kHeads], up[kAsync ? 1 : kHeads];
    T* d0 = (T*)rd.p + row_offset(rd, b, h0, t);
    if constexpr (!kAsync) {
      const T *x0 = (const T*)rx.p + row_offset(rx, b, h0, t), *y0 = (const T*)ry.p + row_offset(ry, b, h0, t);
#pragma unroll
      for (int i = 0; i < kHeads; ++i)
        if (live && h0 + i < p.a.N) {
          in[i].load(x0 + i * rx.stride_n, cols);
          up[i].load(y0 + i * ry.stride_n, cols);
        }
    }
    Turn turn;
    if (p.a.rot) turn = load_turn<AXES>(p, b, t, lane);
    if constexpr (kAsync) asm volatile("cp.async.wait_group %0;" ::"n"(NS - 1) : "memory");
    const uint2* from = mine + stage * (kStageBytes / 8);
#pragma unroll
    for (int i = 0; i < kHeads; ++i) {
      // (what a row that is not there leaves in its lanes is not looked at: its sums cross no other row's)
      const bool on = live && h0 + i < p.a.N;
      float2 x[4], g[4];
      if constexpr (kAsync) {
        in[0].v[0] = from[(i * 4 + 0) * kNormThreads], in[0].v[1] = from[(i * 4 + 1) * kNormThreads];
        up[0].v[0] = from[(i * 4 + 2) * kNormThreads], up[0].v[1] = from[(i * 4 + 3) * kNormThreads];
      } else if (!on) {
        in[i] = up[i] = {};
      }
      in[kAsync ? 0 : i].get(x);
      up[kAsync ? 0 : i].get(g);
      if (p.a.rot) rotate(interleaved, turn, -1.f, g);
      const float r = rsqrtf(row_sum<L>(dot(x, x)) * (1.f / D) + p.a.eps);
      if (!SHARED && on) load_weights<T>(p, which, h0 + i, cols, w);
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        x[k] = mul2(x[k], both(r));
        if (on) dw[SHARED ? 0 : i][k] = fma2(g[k], x[k], dw[SHARED ? 0 : i][k]);
        g[k] = mul2(g[k], w[k]);
      }
      const float mean = row_sum<L>(dot(g, x)) * (-1.f / D);
#pragma unroll
      for (int k = 0; k < 4; ++k) g[k] = mul2(fma2(x[k], both(mean), g[k]), both(r));
      if (on) Eight<T>::store(d0 + i * rd.stride_n, cols, g);
    }
    if (++stage == NS) stage = 0;
  }
  let_next_start();
  if (!weights) return;
  if (SHARED) {   // (a sum for all of the block's heads)
#pragma unroll
    for (int k = 0; k < 4; ++k) *reinterpret_cast<float2*>(&sums[slot][(k < 2 ? cols.a : cols.b) + 2 * (k & 1)]) = dw[0][k];
    __syncthreads();
    for (int c = threadIdx.x; c < D; c += kNormThreads) {
      float total = 0.f;
      for (int s = 0; s < at_once * here; ++s) total += sums[s][c];
      p.partial[(((size_t)which * groups + blockIdx.y % groups) * gridDim.x + blockIdx.x) * D + c] = total;
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < kSums; ++i) {
    __syncthreads();
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      *reinterpret_cast<float2*>(&sums[slot][cols.a + 2 * k]) = dw[i][k];
      *reinterpret_cast<float2*>(&sums[slot][cols.b + 2 * k]) = dw[i][2 + k];
    }
    __syncthreads();
    for (int x = threadIdx.x; x < here * D; x += kNormThreads) {
      const int c = x % D, q = x / D, head = (chunk0 + q) * kHeads + i;
      if (head >= p.a.N) continue;
      float total = 0.f;
      for (int s = q; s < at_once * here; s += here) total += sums[s][c];
      p.partial[(((size_t)which * p.a.N + head) * gridDim.x + blockIdx.x) * D + c] = total;
    }
  }
}

// Adds up the blocks' sums of each column: those of a head, or of all heads' groups.  One block a (tensor, head or all), 32 columns a warp-row.
template <typename T>
__global__ void __launch_bounds__(1024) norm_rotary_weights_kernel(const __grid_constant__ NormParams p) {
  wait_for_previous();
  __shared__ float sums[32][33];
  const int which = blockIdx.z, head = blockIdx.y, D = p.a.D, blocks = p.blocks;
  const int c = blockIdx.x * 32 + threadIdx.x % 32, group = threadIdx.x / 32;
  if (p.a.dw[which] == nullptr) return;
  const int sets = p.a.weight_heads ? p.a.N : p.groups, rows = p.a.weight_heads ? blocks : blocks * p.groups;
  const float* base = p.partial + ((size_t)which * sets + head) * blocks * D;
  float total = 0.f;
  if (c < D)
#pragma unroll 8
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

// The backward's grid: blocks along the tokens, as many as the chip holds at once, and groups of a token's heads.
struct Grid {
  int blocks, groups;
};
Grid bwd_grid(const tritt_norm_rotary_t& a) {
  const int chunks = (int)(((long long)a.N + kHeads - 1) / kHeads), slots = kNormThreads / (a.D / 8);
  const int here = chunks < slots ? chunks : slots, groups = (chunks + here - 1) / here, at_once = slots / here;
  const long long per_sm = a.dtype == TRITT_F32 ? kPerSm<float, true> : a.weight_heads ? kPerSm<__half, false> : kPerSm<__half, true>;
  const long long most = ((long long)a.B * a.T + at_once - 1) / at_once, fill = per_sm * kSms / (3 * groups);
  return Grid{(int)(most < fill ? most : fill < 1 ? 1 : fill), groups};
}

bool wants_weights(const tritt_norm_rotary_t& a) { return a.dw[0] || a.dw[1] || a.dw[2]; }

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
  const long long tokens = (long long)a->B * a->T, chunks = ((long long)a->N + kHeads - 1) / kHeads;
  if (tokens > (1LL << 30) || tokens * chunks > (1LL << 31)) {
    set_error("too many rows for one call (B*T = %lld, N = %d); split the batch", tokens, a->N);
    return -11;
  }
  // (the backward's grids have three times the groups of heads, and the heads, in a dimension that ends at 65535)
  if (backward && (chunks * 3 > 65535 || (a->weight_heads && wants_weights(*a) && a->N > 65535))) {
    set_error("too many heads for a backward call, N = %d", a->N);
    return -11;
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
  if (a->rot && ((uintptr_t)a->positions & (a->positions64 ? 7 : 3))) {
    set_error("the positions' pointer is not aligned");
    return -5;
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
  // one tensor a block until the chip is full several times over
  const dim3 grid((unsigned)blocks, blocks >= 8LL * kSms ? 1 : 3);
  if (p.axes.count)
    norm_rotary_fwd_kernel<T, D, true><<<grid, kNormThreads, 0, stream>>>(p);
  else
    norm_rotary_fwd_kernel<T, D, false><<<grid, kNormThreads, 0, stream>>>(p);
  count_launch();
  TRITT_CUDA_OK(cudaGetLastError());
  return 0;
}

template <typename T, int D> int launch_bwd(NormParams p, cudaStream_t stream) {
  const Grid grid = bwd_grid(p.a);
  p.blocks = grid.blocks;
  p.groups = grid.groups;
  auto run = [&](auto kern, int bytes) -> int {
    if (bytes) TRITT_CUDA_OK(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
    return launch_kernel_after(kern, dim3(p.blocks, 3 * p.groups), kNormThreads, bytes, stream, false, p);
  };
  auto choose = [&](auto axes) -> int {
    return p.a.weight_heads ? run(norm_rotary_bwd_kernel<T, D, false, axes.value>, kBwdSmem<T, false>)
                            : run(norm_rotary_bwd_kernel<T, D, true, axes.value>, kBwdSmem<T, true>);
  };
  if (int rc = p.axes.count ? choose(std::true_type{}) : choose(std::false_type{})) return rc;
  if (!p.partial) return 0;
  return launch_kernel_after(norm_rotary_weights_kernel<T>, dim3((D + 31) / 32, p.a.weight_heads ? p.a.N : 1, 3), 1024, 0, stream, true, p);
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

int check_axes(const tritt_norm_rotary_t* a, const tritt_axes_t* x) {
  if (!x || x->count < 1 || x->count > TRITT_MAX_AXES || !a->rot || !a->positions) {
    set_error("positions of several axes: expected 1 to %d axes, tables and positions", TRITT_MAX_AXES);
    return -13;
  }
  for (int i = 0; i < a->rot / 2; ++i)
    if ((x->of[i / 4] >> 2 * (i % 4) & 3) >= x->count) {
      set_error("rotated pair %d is of axis %d, there are %d", i, x->of[i / 4] >> 2 * (i % 4) & 3, x->count);
      return -13;
    }
  return 0;
}

int forward(const tritt_norm_rotary_t* a, const tritt_axes_t& axes, int* status_word, tritt_stream_t stream) {
  NormParams p{*a, axes, (a->N + kHeads - 1) / kHeads, 0, 0, nullptr, status_word};
  return by_type(p, false, (cudaStream_t)stream);
}
int backward(const tritt_norm_rotary_t* a, const tritt_axes_t& axes, void* workspace, size_t workspace_bytes, int* status_word,
             tritt_stream_t stream) {
  const size_t need = tritt_qk_norm_rotary_workspace(a);
  if (need && (!workspace || workspace_bytes < need || ((uintptr_t)workspace & 15))) {
    set_error("workspace too small or misaligned: need %zu bytes, got %zu", need, workspace ? workspace_bytes : (size_t)0);
    return -6;
  }
  NormParams p{*a, axes, (a->N + kHeads - 1) / kHeads, 0, 0, need ? (float*)workspace : nullptr, status_word};
  return by_type(p, true, (cudaStream_t)stream);
}

}  // namespace
}  // namespace tritt

using namespace tritt;

extern "C" {

int tritt_qk_norm_rotary_fwd(const tritt_norm_rotary_t* a, int* status_word, tritt_stream_t stream) {
  if (int rc = check(a, false)) return rc;
  return forward(a, tritt_axes_t{}, status_word, stream);
}
int tritt_qk_norm_rotary_axes_fwd(const tritt_norm_rotary_t* a, const tritt_axes_t* axes, int* status_word, tritt_stream_t stream) {
  if (int rc = check(a, false)) return rc;
  if (int rc = check_axes(a, axes)) return rc;
  return forward(a, *axes, status_word, stream);
}

size_t tritt_qk_norm_rotary_workspace(const tritt_norm_rotary_t* a) {
  if (!a || a->B <= 0 || a->N <= 0 || a->T <= 0 || a->D < 16 || a->D > 256 || !wants_weights(*a)) return 0;
  return align_up((size_t)3 * a->N * bwd_grid(*a).blocks * a->D * 4, 256);
}

int tritt_qk_norm_rotary_bwd(const tritt_norm_rotary_t* a, void* workspace, size_t workspace_bytes, int* status_word,
                             tritt_stream_t stream) {
  if (int rc = check(a, true)) return rc;
  return backward(a, tritt_axes_t{}, workspace, workspace_bytes, status_word, stream);
}
int tritt_qk_norm_rotary_axes_bwd(const tritt_norm_rotary_t* a, const tritt_axes_t* axes, void* workspace, size_t workspace_bytes, int* status_word,
                                  tritt_stream_t stream) {
  if (int rc = check(a, true)) return rc;
  if (int rc = check_axes(a, axes)) return rc;
  return backward(a, *axes, workspace, workspace_bytes, status_word, stream);
}

}  // extern "C"
