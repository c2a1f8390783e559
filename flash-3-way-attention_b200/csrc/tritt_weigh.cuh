// The attention weight of cached tokens: what the kernels that add it up share.
#pragma once

#include "tritt_cache.cuh"

namespace tritt {

// host: 0 or an error code
int check_weights(const tritt_cache_t* c, const tritt_weights_t* w);
int check_weigh_scores(const float* lse, float alpha);

// What a token's weight of before counts for.
__device__ __forceinline__ float faded(const tritt_weights_t& w, int b, int head, int x) {
  return w.decay == 0.f ? 0.f : w.decay * w.before[b * w.before_stride_b + head * w.before_stride_n + x];
}
__device__ __forceinline__ float* weight_of(const tritt_weights_t& w, int b, int head, int x) {
  return w.after + b * w.after_stride_b + head * w.after_stride_n + x;
}
// Tokens of a sequence that have places for their weights: all, or the call reports.
__device__ __forceinline__ int weighed_tokens(const CacheArgs& a, const tritt_weights_t& w, int tokens) {
  const int most = w.after_length < w.before_length ? w.after_length : w.before_length;
  if (tokens > most && a.status) atomicOr(a.status, kStatusPlace);
  return tokens < most ? tokens : most;
}

// A row that is to be a matrix operand: its largest element's exponent field, 0 of a row of zeros (or next to it), 255 of one that is not finite.  The elements are multiplied by
// to_operand(field), which brings the largest to [2, 4), and the products by from_operand(field).
__device__ __forceinline__ float to_operand(int field) { return field == 0 || field == 255 ? 0.f : __uint_as_float((uint32_t)(255 - field) << 23); }
__device__ __forceinline__ float from_operand(int field) {
  return field == 255 ? __uint_as_float(0x7fffffffu) : field <= 1 ? 0.f : __uint_as_float((uint32_t)(field - 1) << 23);
}
// Where rows of one operand have powers of two of their own, a score is multiplied by its row's, relative to that of this exponent byte (largest: the largest byte of a row that is finite), and that one joins the other
// row's.  Rows may be as far apart as fp32 has numbers, the largest one is often one that the token does not attend to, and the score of the smallest has to be right beside it: so the factors reach from 2^-149, below fp32's
// normal numbers, to 2^kMostPower, which brings no sum of products (below 2^38, 2^27.7, 2^24 with 256 elements) to infinity.
template <int CODE> constexpr int kMostPower = CODE == TRITT_CODE_F16 ? 90 : CODE == TRITT_CODE_E4M3 ? 100 : 103;
template <int CODE> __device__ __forceinline__ int middle_byte(int largest) {
  return largest <= 127 ? largest : largest - kMostPower<CODE> > 127 ? largest - kMostPower<CODE> : 127;
}
__device__ __forceinline__ float relative_power(int e) {   // 2^e, e <= 127; 0 below 2^-149
  return __uint_as_float(e >= -126 ? (uint32_t)(e + 127) << 23 : e >= -149 ? 1u << (e + 149) : 0u);
}
// sum * column * row - minus with numbers below fp32's normal ones (which the compiler's own arithmetic takes for zeros here)
__device__ __forceinline__ float scaled_score(float sum, float column, float row, float minus) {
  float x;
  asm("{\n\t.reg .f32 t;\n\tmul.rn.f32 t, %1, %2;\n\tfma.rn.f32 %0, t, %3, %4;\n\t}" : "=f"(x) : "f"(sum), "f"(column), "f"(row), "f"(-minus));
  return x;
}
__device__ __forceinline__ uint32_t pack_halves(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
// What is left of two numbers when they have been rounded to fp16.
__device__ __forceinline__ uint32_t pack_rests(float a, float b, uint32_t rounded) {
  const float2 r = __half22float2(*reinterpret_cast<const __half2*>(&rounded));
  return pack_halves(a - r.x, b - r.y);
}
// Four neighbouring elements of a row.
template <typename T> __device__ __forceinline__ float4 load4(const T* p) {
  const uint2 v = __ldg(reinterpret_cast<const uint2*>(p));
  T e[4];
  *reinterpret_cast<uint2*>(e) = v;
  return make_float4(to_f(e[0]), to_f(e[1]), to_f(e[2]), to_f(e[3]));
}
template <> __device__ __forceinline__ float4 load4<float>(const float* p) { return __ldg(reinterpret_cast<const float4*>(p)); }
__device__ __forceinline__ uint32_t largest4(float4 f) {
  const uint32_t m = 0x7fffffffu;
  return max(max(__float_as_uint(f.x) & m, __float_as_uint(f.y) & m), max(__float_as_uint(f.z) & m, __float_as_uint(f.w) & m));
}

// The products of 16 rows of the cache, read by a warp straight into the fragments of a 16 x 8 x 16 matrix instruction: lane 4 g + c has of rows g and g + 8 a quarter of the
// elements, as chunks c, c + 4, ... of up to 16 bytes, and each four elements of a chunk are one instruction's (the order of a sum's terms is free; the other operand's
// fragments follow the same order).
template <int D, int CODE> struct RowFragments {
  static constexpr int kSize = CODE == TRITT_CODE_F16 ? 2 : 1;
  static constexpr int kLane = D * kSize / 4;                     // bytes of a row that a lane has
  static constexpr int kChunk = kLane < 16 ? kLane : 16, kChunks = kLane / kChunk;
  static constexpr int kSteps = D / 16, kStepsOfChunk = kSteps / kChunks;
  static constexpr int kWords = kLane / 4;
  uint32_t v[2][kWords];
  // row: the first of the 16 (they follow one another)
  __device__ __forceinline__ void load(const uint8_t* row, int lane) { load_by(row, lane, [](const auto* p) { return __ldg(p); }); }
  // ... of a copy of the rows in shared memory
  __device__ __forceinline__ void load_copy(const uint8_t* row, int lane) { load_by(row, lane, [](const auto* p) { return *p; }); }
  template <typename F> __device__ __forceinline__ void load_by(const uint8_t* row, int lane, F&& get) {
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      const uint8_t* p = row + (size_t)(lane / 4 + 8 * r) * (D * kSize) + lane % 4 * kChunk;
#pragma unroll
      for (int i = 0; i < kChunks; ++i) {
        uint32_t* to = v[r] + i * (kChunk / 4);
        if constexpr (kChunk == 16) {
          const uint4 x = get(reinterpret_cast<const uint4*>(p + i * 64));
          to[0] = x.x, to[1] = x.y, to[2] = x.z, to[3] = x.w;
        } else if constexpr (kChunk == 8) {
          const uint2 x = get(reinterpret_cast<const uint2*>(p));
          to[0] = x.x, to[1] = x.y;
        } else {
          to[0] = get(reinterpret_cast<const uint32_t*>(p));
        }
      }
    }
  }
  // fragments of one instruction
  __device__ __forceinline__ void step(int s, uint32_t (&a)[4]) const {
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      if constexpr (CODE == TRITT_CODE_F16) {
        a[r] = v[r][2 * s], a[2 + r] = v[r][2 * s + 1];
      } else {
        bytes_to_halves<CODE>(v[r][s], a[r], a[2 + r]);
      }
    }
  }
  // where a row's four elements from `column` on go among the other operand's fragments: instruction, and lane's part of it
  struct Slot {
    int step, c;
  };
  static __device__ __forceinline__ Slot slot_of(int column) {
    const int chunk = column / (kChunk / kSize), within = column % (kChunk / kSize);
    return Slot{chunk / 4 * kStepsOfChunk + within / 4, chunk % 4};
  }
};
__device__ __forceinline__ void mma_16816(float (&d)[4], const uint32_t (&a)[4], uint2 b) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b.x), "r"(b.y));
}

// ---------------------------------------------------------------- triple dot product
struct TdpWeighArgs {
  CacheArgs cache;
  tritt_weights_t w;
  tritt_rows_t q;
  const float* lse;
  int dtype, k1w, k2w, kkl, kkr;
  float scale2;          // alpha * log2(e)
  long long* table;      // the workspace: steps before each sequence, and of all ...
  float* part;           // ... and slots, see below
  int ctas, span, sums;  // sums of a slot
};

// Tokens come in tiles of 128 by their numbers.  The line of all (sequence, head, new token, tile of k, tile of j) steps is cut in equal parts, one for each CTA.  What a CTA adds up of a
// head stands in a slot of the workspace, [sums][span] fp32 by the tokens' numbers from the head's base on; the CTAs that share a head and the heads that share a CTA follow one another, so
// (CTA + head) numbers the slots.  Another kernel adds each token's slots up, in order.
constexpr long long kMostWeighSteps = 1ll << 39;   // of a sequence's head: those of 65535 heads times the CTAs stay below 2^63
struct WeighLine {
  int ctx, cnt;
  int base, last;        // numbers of the slots' first token (a multiple of 128) and of the last token that there is
  int k0, j0;            // first tiles
  int groups, slabs;     // tiles of k and of j that a new token may attend to: the same count for all
  long long unit;        // steps of a head
};
__device__ __forceinline__ WeighLine weigh_line(const TdpWeighArgs& a, int b) {
  WeighLine l;
  l.cnt = new_tokens(a.cache, b);
  l.ctx = context_of(a.cache, b);
  if (l.cnt == 0 || l.ctx < 0) {
    l.cnt = l.groups = l.slabs = 0;
    l.unit = 0;
    return l;
  }
  const int lo_j = l.ctx - (a.k1w < l.ctx ? a.k1w : l.ctx), lo_k = l.ctx - (a.k2w < l.ctx ? a.k2w : l.ctx);
  const int places = a.cache.c.table_pages << a.cache.page_log2;   // (tokens behind the table's end are not there, and the slots have no room for them: reported)
  if (l.cnt > places - l.ctx && a.cache.status) atomicOr(a.cache.status, kStatusPlace);
  l.last = (l.cnt < places - l.ctx ? l.ctx + l.cnt : places) - 1;
  l.j0 = lo_j / 128;
  l.k0 = lo_k / 128;
  l.base = (lo_j < lo_k ? l.j0 : l.k0) * 128;
  l.slabs = l.last / 128 - l.j0 + 1;
  l.groups = l.last / 128 - l.k0 + 1;
  const long long of_token = (long long)l.groups * l.slabs;
  const bool much = l.slabs > 0 && l.groups > 0 && l.cnt > kMostWeighSteps / of_token;   // reported, and left out
  if (much && a.cache.status) atomicOr(a.cache.status, kStatusTdpDecode);
  if (l.slabs <= 0 || l.groups <= 0 || much) l.cnt = l.groups = l.slabs = 0;
  l.unit = l.cnt * of_token;
  return l;
}
// 128-token tiles that a slot has room for: what the windows and the new tokens can touch, at most the table (or the weights)
inline int weigh_span(const tritt_cache_t& c, int k1w, int k2w) {
  long long tokens = (long long)c.table_pages * c.page_size;
  const long long reach = (long long)(k1w > k2w ? k1w : k2w) + c.n + 127;   // (the base is rounded down)
  if (reach < tokens) tokens = reach;
  return (int)((tokens + 127) / 128 * 128);
}
constexpr int kWeighCtas = 148;

// (a division of 64 bits is long, and few are needed)
__device__ __forceinline__ long long quotient(long long a, long long b) {
  return ((unsigned long long)(a | b) >> 32) == 0 ? (long long)((uint32_t)a / (uint32_t)b) : a / b;
}
// CTAs that the line is cut among: each has a step at least.  Part i begins with step i * total / parts.
__device__ __forceinline__ int weigh_parts(const TdpWeighArgs& a, long long total) { return total < a.ctas ? (int)total : a.ctas; }
// The line's length, where this CTA's part begins, and the sequence that the step is of, with the number of the steps before its first.  A warp calls it together; that of the first CTA leaves the steps before each
// sequence, and of all, in the workspace for the kernel that joins.
struct WeighPart {
  long long total, first, before;
  int b;
};
__device__ __forceinline__ WeighPart weigh_part(const TdpWeighArgs& a) {
  const int lane = threadIdx.x % 32;
  WeighPart w{0, 0, 0, 0};
  long long own = 0, behind = 0;   // steps of the lane's sequence, and of those up to it
  auto sums = [&](int b0) {
    const int b = b0 + lane;
    own = b < a.cache.c.B ? weigh_line(a, b).unit * a.cache.c.N : 0;
    long long s = own;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long u = __shfl_up_sync(0xffffffffu, s, o);
      if (lane >= o) s += u;
    }
    behind = w.before + s;
  };
  for (int b0 = 0; b0 < a.cache.c.B; b0 += 32) {
    sums(b0);
    if (blockIdx.x == 0 && b0 + lane < a.cache.c.B) a.table[b0 + lane] = behind - own;
    w.before = __shfl_sync(0xffffffffu, behind, 31);
  }
  w.total = w.before;
  if (blockIdx.x == 0 && lane == 0) a.table[a.cache.c.B] = w.total;
  const int parts = weigh_parts(a, w.total);
  if ((int)blockIdx.x >= parts) return w;
  w.first = quotient((long long)blockIdx.x * w.total, parts);
  int b0 = 0;
  if (a.cache.c.B > 32) {
    w.before = 0;
    for (;; b0 += 32) {
      sums(b0);
      const long long next = __shfl_sync(0xffffffffu, behind, 31);
      if (w.first < next) break;
      w.before = next;
    }
  }
  const int at = __ffs(__ballot_sync(0xffffffffu, w.first < behind)) - 1;
  w.b = b0 + at;
  w.before = __shfl_sync(0xffffffffu, behind - own, at);
  return w;
}
// The i-th new token in the order of the line.  Later ones attend to more: in steps that are prime to their number and near its golden section, every stretch of the line has early
// and late ones alike.
__device__ __forceinline__ int weigh_step(int cnt) {
  if (cnt < 3) return 1;
  int step = (int)(cnt * 0.618f);
  if (step < 1) step = 1;
  for (;; ++step) {
    int x = cnt, y = step;
    while (y) {
      const int r = x % y;
      x = y;
      y = r;
    }
    if (x == 1) return step;   // (cnt - 1 is prime to cnt)
  }
}

// A CTA's way along its part of the line.
struct WeighPiece {
  int b, head, i, kg, s0, s1;   // token, tile of k, tiles of j (absolute)
  WeighLine l;
  bool fresh;                   // the first piece of its head
};
struct WeighWalk {
  long long left;
  int b, head, slab, group, n, token, step;   // n: how many of the head's tokens are behind
  WeighLine l;
  bool fresh;
};
__device__ __forceinline__ WeighWalk weigh_start(const TdpWeighArgs& a, const WeighPart& part) {
  WeighWalk w{0, part.b, 0, 0, 0, 0, 0, 1, {}, true};
  const int parts = weigh_parts(a, part.total);
  if ((int)blockIdx.x >= parts) return w;
  long long x = part.first - part.before;
  w.left = quotient(((long long)blockIdx.x + 1) * part.total, parts) - part.first;
  w.l = weigh_line(a, part.b);
  w.head = (int)quotient(x, w.l.unit);
  x -= w.head * w.l.unit;
  const long long of_token = (long long)w.l.groups * w.l.slabs;
  w.n = (int)quotient(x, of_token);
  x -= w.n * of_token;
  w.group = (int)quotient(x, w.l.slabs);
  w.slab = (int)(x - (long long)w.group * w.l.slabs);
  w.step = weigh_step(w.l.cnt);
  w.token = (int)((long long)w.n * w.step - quotient((long long)w.n * w.step, w.l.cnt) * w.l.cnt);
  return w;
}
__device__ __forceinline__ bool weigh_next(const TdpWeighArgs& a, WeighWalk& w, WeighPiece& s) {
  while (w.left > 0) {
    if (w.slab == w.l.slabs) {
      w.slab = 0;
      if (++w.group == w.l.groups) {
        w.group = 0;
        w.token += w.step;
        if (w.token >= w.l.cnt) w.token -= w.l.cnt;
        if (++w.n == w.l.cnt) {
          w.n = w.token = 0;
          w.fresh = true;
          if (++w.head == a.cache.c.N) {
            w.head = 0;
            do {
              if (++w.b >= a.cache.c.B) return false;
              w.l = weigh_line(a, w.b);
            } while (w.l.cnt == 0);
            w.step = weigh_step(w.l.cnt);
          }
        }
      }
    }
    const int take = w.l.slabs - w.slab < w.left ? w.l.slabs - w.slab : (int)w.left;
    s = WeighPiece{w.b, w.head, w.token, w.l.k0 + w.group, w.l.j0 + w.slab, w.l.j0 + w.slab + take, w.l, w.fresh};
    w.left -= take;
    w.slab += take;
    // the tiles of j that the token and the tile of k have pairs in
    const int pos = w.l.ctx + w.token, k_lo = s.kg * 128, k_hi = k_lo + 127 < pos ? k_lo + 127 : pos;
    int lo = pos - (a.k1w < pos ? a.k1w : pos), hi = pos;
    if (k_lo - a.kkl > lo) lo = k_lo - a.kkl;
    if (a.kkr < pos && k_hi + a.kkr < hi) hi = k_hi + a.kkr;
    if (k_lo <= pos && k_hi >= pos - a.k2w && lo <= hi) {
      if (s.s0 < lo / 128) s.s0 = lo / 128;
      if (s.s1 > hi / 128 + 1) s.s1 = hi / 128 + 1;
      if (s.s0 < s.s1) {
        w.fresh = false;
        return true;
      }
    }
    if (w.fresh) {   // (a slot is cleared even if all of the CTA's part of a head is empty)
      s.s1 = s.s0;
      w.fresh = false;
      return true;
    }
  }
  return false;
}
__device__ __forceinline__ float* weigh_slot(const TdpWeighArgs& a, int b, int head) {
  return a.part + ((size_t)blockIdx.x + (size_t)b * a.cache.c.N + head) * a.sums * a.span;
}

// on the tensor cores (head dimension 64 or 128; five sums a slot), and with warp-level matrix instructions (two)
bool sm100_tdp_weigh_supported(int D);
int sm100_tdp_weigh(const TdpWeighArgs& a, cudaStream_t stream);
int mma_tdp_weigh(const TdpWeighArgs& a, cudaStream_t stream);
// where the rows fit in shared memory: one launch, which writes the new weights, too
bool window_tdp_weigh_applies(const TdpWeighArgs& a);
int window_tdp_weigh(const TdpWeighArgs& a, cudaStream_t stream);
int launch_tdp_weigh_join(const TdpWeighArgs& a, cudaStream_t stream);

}  // namespace tritt
