// The attention weight of cached tokens in the dot-product sum: what new tokens' queries give them through K2, and what the new tokens' own k2 give them through K1.
//
//   w[x] = decay w[x] + sum_i exp(alpha q_i.K2[x] + lse[x] - m_i) + sum_i [p_i - x <= k_diff] exp(alpha k2_i.K1[x] - lse[p_i]),   x <= p_i = context + i
// The soft-maxes' sums are known (m, lse), so a cached row is read once, each token's sum has one owner, and nothing is joined.  Bound by the bytes of K1 and K2.
//
// A warp takes 16 tokens: their rows go from memory straight into the fragments of warp-level matrix instructions (eight new tokens the other side, in shared memory in the order of
// the fragments), exact as fp16 codes; each row's exponent, and the new row's, multiply the sums.  fp32 rows are two fp16 numbers (22 bits), as the products are
// summed in fp32 all the same.
// Measured: a token of 32 x 16 heads of 64 over up to 8191, e4m3, 73 us (278 MB, 3.8 TB/s; 70 % of the issue slots); 24 tokens over 3001, 4 x 16 heads of 128, fp16 codes 27 to 31 us (78 MB; a block's way to its first
// tile, and one tile behind the other).  One token of 32 x 16 heads over up to 8191 otherwise: head dimension 16, int8 57 us (floor by bytes 15), 32, fp16 codes 70 (43), 128, e4m3 117 (79), 128, fp16 codes 205 (151; rows of
// 256 bytes, by the kernel for several tokens); over up to 4095 head dimension 256, fp16 codes 257 (166), int8 403 (85: fragments of 16 steps beside the rows of both parts, of which 570 to 660 bytes a thread are spilled).
#include "tritt_weigh.cuh"

#include <type_traits>

namespace tritt {
namespace {

constexpr int kThreads = 256, kTokens = 128;   // of a block at a time
constexpr int kSms = 148;

struct Params {
  CacheArgs cache;
  tritt_weights_t w;
  tritt_rows_t rows[2];   // q, k2
  const float* m;
  int k_diff, repeat;     // repeat: times that a block takes kTokens
  int chunk;              // new tokens at a time (a multiple of 8)
  float scale2;
};

struct __align__(16) Query {
  float scale, minus;     // of its scores (log2 units); what is subtracted (natural units)
  int last, pad;          // the last token that it attends to; -1: none
};

// Bytes of a chunk's fragments for each new token, and how many of them are taken at once.
template <typename T, int D> constexpr int kBytesEach = 2 * D * 2 * (std::is_same<T, float>::value ? 2 : 1);
template <typename T, int D> constexpr int kMostChunk = 32768 / kBytesEach<T, D> < 64 ? 32768 / kBytesEach<T, D> : 64;
static_assert(kMostChunk<float, 256> == 16 && kMostChunk<__half, 64> == 64, "chunks are multiples of 8");

// The rows q and k2 of new tokens q0 .. q0 + here - 1 as fragments, eight tokens a tile, and what their scores need, by all of a block's warps.
template <typename T, int D, int CODE>
__device__ __forceinline__ void form_queries(const Params& p, int b, int head, int ctx, int q0, int here, int tiles, uint2* frags, Query (&queries)[2][64]) {
  using Rows = RowFragments<D, CODE>;
  constexpr bool kWide = std::is_same<T, float>::value;
  constexpr int kSteps = Rows::kSteps, kHalves = kWide ? 2 : 1;
  const CacheArgs& a = p.cache;
  const int lane = threadIdx.x % 32;
  for (int i = threadIdx.x / 32; i < 2 * tiles * 8; i += kThreads / 32) {
    const int part = i >= tiles * 8, n = i - part * tiles * 8;
    const bool on = n < here;
    const T* row = (const T*)p.rows[part].p + (on ? rows_at(p.rows[part], b, head, q0 + n) : 0);
    float4 f[D > 128 ? 2 : 1];
    uint32_t top = 0;
#pragma unroll
    for (int k = 0; k < (D > 128 ? 2 : 1); ++k) {
      f[k] = on && lane + 32 * k < D / 4 ? load4(row + (lane + 32 * k) * 4) : make_float4(0.f, 0.f, 0.f, 0.f);
      top = max(top, largest4(f[k]));
    }
    const int field = (int)(largest_of_row<32>(top) >> 23);
    const float up = to_operand(field);
#pragma unroll
    for (int k = 0; k < (D > 128 ? 2 : 1); ++k) {
      const int col = (lane + 32 * k) * 4;
      if (col >= D) continue;
      float4 v = f[k];
      v.x *= up, v.y *= up, v.z *= up, v.w *= up;
      if (field == 255) v = make_float4(0.f, 0.f, 0.f, 0.f);
      const auto slot = Rows::slot_of(col);
      uint2* to = frags + ((size_t)((part * tiles + n / 8) * kHalves) * kSteps + slot.step) * 32 + n % 8 * 4 + slot.c;
      const uint2 hi = make_uint2(pack_halves(v.x, v.y), pack_halves(v.z, v.w));
      to[0] = hi;
      if constexpr (kWide) to[kSteps * 32] = make_uint2(pack_rests(v.x, v.y, hi.x), pack_rests(v.z, v.w, hi.y));
    }
    if (lane == 0) {
      Query q{p.scale2 * from_operand(field), 0.f, -1, 0};
      if (on) {
        q.last = ctx + q0 + n;
        if (part == 0) {
          q.minus = __ldg(p.m + ((size_t)b * a.c.N + head) * a.c.n + q0 + n);
        } else {
          const Place own = place_of(a, b, ctx + q0 + n);
          if (own.page >= 0)
            q.minus = __ldg(a.c.lse + lse_of(a, own, head));
          else
            q.last = -1;
        }
        if (q.minus == -INFINITY) q.last = -1;
      }
      queries[part][n] = q;
    }
  }
}

// A few new tokens, rows of up to 128 bytes: 32 tokens a warp at a time, in two products' fragments, whose scores then change lanes so that each lane has one token, its row's exponent, its
// log-sum-exp and its weight (with two tokens a lane of four and eight columns for one new token the kernel below executed four times the instructions: 178 us for 32 x 16 heads over
// 8191, e4m3).  A warp's rows, K2's and then, where a new token's k2 attends to them, K1's, come by asynchronous copies into places of its own, two steps ahead (a step ahead in
// registers: 105 us; so 75, and 84 with three steps ahead for two blocks an SM).
constexpr int kFew = 4, kFewTokens = 256;   // new tokens at most; of a block at a time
template <int D, int CODE> constexpr bool kFewApplies = RowFragments<D, CODE>::kWords <= 8;
template <int D, int CODE> struct FewStage {   // of a warp
  uint8_t codes[32 * D * RowFragments<D, CODE>::kSize];
  float lse[32], before[32];
  uint8_t exponent[32];
};
constexpr int kFewStages = 3;
template <int D, int CODE> constexpr int kFewSmem = kThreads / 32 * kFewStages * (int)sizeof(FewStage<D, CODE>);

__device__ __forceinline__ void copy_if(void* dst, const void* src, bool on) {   // 16 bytes, zeros where not (src: an address that can be read)
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"((uint32_t)__cvta_generic_to_shared(dst)), "l"(src), "r"(on ? 16 : 0) : "memory");
}
__device__ __forceinline__ void copy4_if(void* dst, const void* src, bool on) {   // four bytes
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"((uint32_t)__cvta_generic_to_shared(dst)), "l"(src), "r"(on ? 4 : 0) : "memory");
}

template <typename T, int D, int CODE> __global__ void __launch_bounds__(kThreads, RowFragments<D, CODE>::kWords <= 4 ? 3 : 2) dps_weigh_few_kernel(const __grid_constant__ Params p) {
  using Rows = RowFragments<D, CODE>;
  using Stage = FewStage<D, CODE>;
  constexpr bool kWide = std::is_same<T, float>::value;
  constexpr int kSteps = Rows::kSteps, kHalves = kWide ? 2 : 1, NS = kFewStages;
  constexpr int kRow = D * Rows::kSize, kChunks = kRow / 16;
  extern __shared__ __align__(16) uint8_t smem[];   // stages of the warps, then fragments [part][hi, lo][step][lane]
  __shared__ Query queries[2][64];
  const CacheArgs& a = p.cache;
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
  Stage* const stages = reinterpret_cast<Stage*>(smem) + warp * NS;
  uint2* const frags = reinterpret_cast<uint2*>(smem + kFewSmem<D, CODE>);
  const int bh = blockIdx.y, b = bh / a.c.N, head = bh - b * a.c.N;
  if (__ldg(a.c.context + b) < 0) return;
  const int ctx = context_of(a, b), cnt = new_tokens(a, b), end = weighed_tokens(a, p.w, ctx + cnt);
  const int first = blockIdx.x * p.repeat * kFewTokens + warp * 32;
  if ((int)blockIdx.x * p.repeat * kFewTokens >= end) return;
  const int behind = ctx - (p.k_diff < ctx ? p.k_diff : ctx);   // the first token that any new one's k2 attends to
  const uint8_t* const codes = (const uint8_t*)a.c.codes;
  const size_t part_rows = (size_t)a.c.N << a.page_log2;
  int steps = end > first ? (end - first + kFewTokens - 1) / kFewTokens : 0;   // of this warp, 32 tokens each
  if (steps > p.repeat) steps = p.repeat;
  auto inner = [&](int r) { return cnt > 0 && first + r * kFewTokens + 31 >= behind; };

  // the page of the lane's token, as the table has it (a step before it is needed, and not looked at here, so that nothing waits for it); -1: the token is not there, or the table has none
  auto page_of = [&](int r) {
    const int x = first + r * kFewTokens + lane, i = x >> a.page_log2;
    int page = -1;
    if (r < steps && x < end && i < a.c.table_pages) page = __ldg(a.c.table + b * a.c.table_stride + i);
    return page;
  };
  // What is sent next: K2's rows of step `ahead`, or its K1's; one group of copies each, empty ones at the end.
  int ahead = 0, slot = 0, page = page_of(0);
  bool second = false;
  size_t row = 0;             // number of the lane's K2 row
  bool on = false;
  auto send = [&]() {
    if (ahead < steps) {
      Stage& to = stages[slot];
      const int x = first + ahead * kFewTokens + lane;
      if (!second) {
        on = page >= 0 && page < a.c.pages;
        if (x < end && !on && a.status) atomicOr(a.status, kStatusPlace);
        const Place at{page, x & (a.c.page_size - 1)};
        row = on ? row_of(a, at, kPartK2, head) : 0;
        copy4_if(&to.lse[lane], on ? a.c.lse + lse_of(a, at, head) : a.c.lse, on);
        page = page_of(ahead + 1);
        const bool old = x < end && x < ctx && p.w.decay != 0.f;
        copy4_if(&to.before[lane], old ? p.w.before + b * p.w.before_stride_b + head * p.w.before_stride_n + x : p.w.before, old);
      }
      const size_t mine = second ? row - part_rows : row;   // (K1's rows lie a part ahead)
      if (lane % 4 == 0) copy4_if(&to.exponent[lane], on ? a.c.exponents + mine : a.c.exponents, on);
#pragma unroll
      for (int k = 0; k < kChunks; ++k) {
        const int at = k * 32 + lane, from = at / (16 * kChunks) * 16;   // (16 tokens' rows follow one another)
        const size_t base = (size_t)__shfl_sync(0xffffffffu, (uint32_t)(mine >> 32), from) << 32 | __shfl_sync(0xffffffffu, (uint32_t)mine, from);
        const bool there = __shfl_sync(0xffffffffu, (int)on, from);
        copy_if(to.codes + at * 16, there ? codes + base * kRow + at % (16 * kChunks) * 16 : codes, there);
      }
      if (!second && inner(ahead)) {
        second = true;
      } else {
        second = false;
        ++ahead;
      }
      if (++slot == NS) slot = 0;
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  // the scores of the 32 tokens of a stage, and what they add to them
  auto gain = [&](const Stage& from, int part, int x, float lse) {
    float d[2][4];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      Rows rows;
      rows.load_copy(from.codes + h * 16 * kRow, lane);
#pragma unroll
      for (int k = 0; k < 4; ++k) d[h][k] = 0.f;
#pragma unroll
      for (int s = 0; s < kSteps; ++s) {
        uint32_t frag[4];
        rows.step(s, frag);
        const uint2* f = frags + (size_t)(part * kHalves * kSteps + s) * 32 + lane;
        mma_16816(d[h], frag, f[0]);
        if constexpr (kWide) mma_16816(d[h], frag, f[kSteps * 32]);
      }
    }
    const float scale = code_scale(from.exponent[lane]);
    float sum = 0.f;
#pragma unroll
    for (int n = 0; n < kFew; ++n) {
      if (n >= cnt) break;
      // the score of this lane's token: row lane % 16 of half lane / 16
      const int at = lane % 8 * 4 + n / 2;
      const float s0 = __shfl_sync(0xffffffffu, d[0][n % 2], at), s1 = __shfl_sync(0xffffffffu, d[0][2 + n % 2], at);
      const float s2 = __shfl_sync(0xffffffffu, d[1][n % 2], at), s3 = __shfl_sync(0xffffffffu, d[1][2 + n % 2], at);
      const float score = lane < 16 ? (lane < 8 ? s0 : s1) : (lane < 24 ? s2 : s3);
      const Query q = queries[part][n];
      const bool seen = x <= q.last && (part == 0 || q.last - x <= p.k_diff);
      const float less = part == 0 ? lse - q.minus : -q.minus;
      sum += seen ? exp2f(fmaf(score * scale, q.scale, less * kLog2e)) : 0.f;
    }
    return sum;
  };
  for (int k = 0; k < NS - 1; ++k) send();
  if (cnt > 0) form_queries<T, D, CODE>(p, b, head, ctx, 0, cnt, 1, frags, queries);
  __syncthreads();
  int use = 0;
  int there_page = page_of(0);   // (whether the step's tokens have places, for what they get)
  for (int r = 0; r < steps; ++r) {
    const int x = first + r * kFewTokens + lane;
    const bool there = there_page >= 0 && there_page < a.c.pages;
    there_page = page_of(r + 1);
    float sum = 0.f;
#pragma unroll
    for (int part = 0; part < 2; ++part) {
      if (part && !inner(r)) break;
      asm volatile("cp.async.wait_group %0;" ::"n"(NS - 2) : "memory");
      __syncwarp();
      const Stage& from = stages[use];
      if (part == 0 && p.w.decay != 0.f) sum = p.w.decay * from.before[lane];
      if (cnt > 0) {
        const float more = gain(from, part, x, part == 0 ? from.lse[lane] : 0.f);
        if (there) sum += more;
      }
      __syncwarp();   // (the stage has been read)
      if (++use == NS) use = 0;
      send();
    }
    if (x < end) *weight_of(p.w, b, head, x) = sum;
  }
}

// Blocks an SM: registers for the bytes of rows that are to be in flight.
template <int D, int CODE> constexpr int kPerSm = RowFragments<D, CODE>::kWords <= 4 ? 3 : RowFragments<D, CODE>::kWords <= 16 ? 2 : 1;

template <typename T, int D, int CODE> __global__ void __launch_bounds__(kThreads, kPerSm<D, CODE>) dps_weigh_kernel(const __grid_constant__ Params p) {
  using Rows = RowFragments<D, CODE>;
  constexpr bool kWide = std::is_same<T, float>::value;
  constexpr int kSteps = Rows::kSteps, kHalves = kWide ? 2 : 1;
  constexpr bool kBoth = Rows::kWords <= 16;   // rows of both parts on their way together
  constexpr bool kAhead = Rows::kWords <= 8;   // ... and two tiles' (registers)
  extern __shared__ __align__(16) uint2 frags[];   // [part][8 new tokens][hi, lo][step][lane]
  __shared__ Query queries[2][64];
  const CacheArgs& a = p.cache;
  const int lane = threadIdx.x % 32, warp = threadIdx.x / 32, g = lane / 4, c = lane % 4;
  const int bh = blockIdx.y, b = bh / a.c.N, head = bh - b * a.c.N;
  if (__ldg(a.c.context + b) < 0) return;
  const int ctx = context_of(a, b), cnt = new_tokens(a, b), end = weighed_tokens(a, p.w, ctx + cnt);
  const int first = blockIdx.x * p.repeat * kTokens;
  const int behind = ctx - (p.k_diff < ctx ? p.k_diff : ctx);   // the first token that any new one's k2 attends to
  const int chunks = (cnt + p.chunk - 1) / p.chunk;
  const uint8_t* codes = (const uint8_t*)a.c.codes;
  constexpr size_t kRow = D * Rows::kSize;

  // a tile of 128 tokens, 16 a warp: the warp's rows, on their way from `fetch` on
  struct Tile {
    Rows rows[kBoth ? 2 : 1];
    size_t row_k2, row_k1;
    uint8_t byte[2][2];
    float lse[2], before;
    bool there, inner;
  };
  auto fetch = [&](int r, Tile& t) {
    const int x0 = first + r * kTokens + warp * 16;
    Place at{-1, 0};
    if (x0 < end) {
      at = place_of(a, b, x0);   // (16 tokens lie in one page)
      if (at.page < 0 && a.status) atomicOr(a.status, kStatusPlace);
    }
    t.there = at.page >= 0;
    t.inner = t.there && x0 + 15 >= behind;
    t.row_k2 = t.there ? row_of(a, at, kPartK2, head) : 0;
    t.row_k1 = t.there ? row_of(a, at, kPartK1, head) : 0;
    if (t.there) {
      t.rows[0].load(codes + t.row_k2 * kRow, lane);
      if (kBoth && t.inner) t.rows[kBoth].load(codes + t.row_k1 * kRow, lane);
      const float* lse_row = a.c.lse + lse_of(a, at, head);
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        t.byte[0][h] = __ldg(a.c.exponents + t.row_k2 + g + 8 * h);
        t.byte[1][h] = t.inner ? __ldg(a.c.exponents + t.row_k1 + g + 8 * h) : 0;
        t.lse[h] = __ldg(lse_row + g + 8 * h);
      }
    }
    const int mine = x0 + g + (c == 1 ? 8 : 0);   // the token whose weight this lane writes
    t.before = 0.f;
    if (c < 2 && mine < end && mine < ctx) t.before = faded(p.w, b, head, mine);
  };
  auto work = [&](int r, Tile& t) {
    const int x0 = first + r * kTokens + warp * 16, mine = x0 + g + (c == 1 ? 8 : 0);
    float gain[2] = {0.f, 0.f};
    for (int q0 = 0, chunk = 0; chunk < chunks; ++chunk, q0 += p.chunk) {
      const int here = cnt - q0 < p.chunk ? cnt - q0 : p.chunk, tiles = (here + 7) / 8;
      if (r == 0 || chunks > 1) {   // the new tokens' rows as fragments
        if (r || chunk) __syncthreads();
        form_queries<T, D, CODE>(p, b, head, ctx, q0, here, tiles, frags, queries);
        __syncthreads();
      }
      if (!t.there) continue;
#pragma unroll
      for (int part = 0; part < 2; ++part) {
        if (part && !t.inner) break;
        Rows& now = t.rows[kBoth ? part : 0];
        if (!kBoth && (part || chunk)) now.load(codes + (part ? t.row_k1 : t.row_k2) * kRow, lane);
        const float scale[2] = {code_scale(t.byte[part][0]), code_scale(t.byte[part][1])};
        uint32_t frag[kSteps][4];
#pragma unroll
        for (int s = 0; s < kSteps; ++s) now.step(s, frag[s]);
        for (int i = 0; i < tiles; ++i) {
          float d[4] = {0.f, 0.f, 0.f, 0.f};
          const uint2* from = frags + (size_t)((part * tiles + i) * kHalves) * kSteps * 32 + lane;
#pragma unroll
          for (int s = 0; s < kSteps; ++s) {
            mma_16816(d, frag[s], from[s * 32]);
            if constexpr (kWide) mma_16816(d, frag[s], from[(kSteps + s) * 32]);
          }
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            const Query q = queries[part][i * 8 + 2 * c + k];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              const int x = x0 + g + 8 * h;
              const bool on = x <= q.last && (part == 0 || q.last - x <= p.k_diff);
              const float less = part == 0 ? t.lse[h] - q.minus : -q.minus;
              gain[h] += on ? exp2f(fmaf(d[2 * h + k] * scale[h], q.scale, less * kLog2e)) : 0.f;
            }
          }
        }
      }
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      gain[h] += __shfl_xor_sync(0xffffffffu, gain[h], 1);
      gain[h] += __shfl_xor_sync(0xffffffffu, gain[h], 2);
    }
    if (c < 2 && mine < end) *weight_of(p.w, b, head, mine) = t.before + (c ? gain[1] : gain[0]);
  };
  int tiles_here = end > first ? (end - first + kTokens - 1) / kTokens : 0;
  if (tiles_here > p.repeat) tiles_here = p.repeat;
  if constexpr (kAhead) {   // the next tile's rows are on their way while one is worked on
    Tile even, odd;
    if (tiles_here > 0) fetch(0, even);
    for (int r = 0; r < tiles_here; r += 2) {
      if (r + 1 < tiles_here) fetch(r + 1, odd);
      work(r, even);
      if (r + 1 >= tiles_here) break;
      if (r + 2 < tiles_here) fetch(r + 2, even);
      work(r + 1, odd);
    }
  } else {
    Tile tile;
    for (int r = 0; r < tiles_here; ++r) {
      fetch(r, tile);
      work(r, tile);
    }
  }
}

template <typename T, int D, int CODE> int launch(Params p, cudaStream_t stream) {
  const tritt_cache_t& c = p.cache.c;
  long long tokens = (long long)c.table_pages * c.page_size + c.n;   // (weights of tokens behind the table's end are written, and the tokens reported)
  const int length = p.w.after_length < p.w.before_length ? p.w.after_length : p.w.before_length;
  if (length < tokens) tokens = length;
  if constexpr (kFewApplies<D, CODE>) {
    if (c.n <= kFew) {
      const long long blocks = (tokens + kFewTokens - 1) / kFewTokens, repeat = blocks * c.B * c.N / (kSms * 12);
      p.repeat = (int)(repeat < 1 ? 1 : repeat > 8 ? 8 : repeat);
      const int bytes = kFewSmem<D, CODE> + 8 * kBytesEach<T, D>;
      TRITT_CUDA_OK(cudaFuncSetAttribute(dps_weigh_few_kernel<T, D, CODE>, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
      dps_weigh_few_kernel<T, D, CODE><<<dim3((unsigned)((blocks + p.repeat - 1) / p.repeat), c.B * c.N), kThreads, bytes, stream>>>(p);
      count_launch();
      TRITT_CUDA_OK(cudaGetLastError());
      return 0;
    }
  }
  const int most = kMostChunk<T, D>, n8 = (c.n + 7) / 8 * 8;
  p.chunk = n8 < most ? n8 : most;
  const int bytes = p.chunk * kBytesEach<T, D>;
  const long long blocks = (tokens + kTokens - 1) / kTokens;
  // the new rows are formed once a block: as many blocks as the chip holds at once (two an SM), each for as many times kTokens as that leaves
  // (24 tokens over 3001, 4 x 16 heads of 128, fp16 codes: 29 us, with half as many tokens a block 36)
  long long repeat = blocks * c.B * c.N / (kSms * 2);
  p.repeat = (int)(repeat < 1 ? 1 : repeat > 8 ? 8 : repeat);
  const dim3 grid((unsigned)((blocks + p.repeat - 1) / p.repeat), c.B * c.N);
  dps_weigh_kernel<T, D, CODE><<<grid, kThreads, bytes, stream>>>(p);
  count_launch();
  TRITT_CUDA_OK(cudaGetLastError());
  return 0;
}

template <typename T, int CODE> int by_size(const Params& p, cudaStream_t stream) {
  switch (p.cache.c.D) {
    case 16: return launch<T, 16, CODE>(p, stream);
    case 32: return launch<T, 32, CODE>(p, stream);
    case 64: return launch<T, 64, CODE>(p, stream);
    case 128: return launch<T, 128, CODE>(p, stream);
    default: return launch<T, 256, CODE>(p, stream);
  }
}
template <typename T> int by_code(const Params& p, cudaStream_t stream) {
  switch (p.cache.c.code) {
    case TRITT_CODE_F16: return by_size<T, TRITT_CODE_F16>(p, stream);
    case TRITT_CODE_E4M3: return by_size<T, TRITT_CODE_E4M3>(p, stream);
    default: return by_size<T, TRITT_CODE_INT8>(p, stream);
  }
}

}  // namespace
}  // namespace tritt

using namespace tritt;

extern "C" int tritt_dps_weigh(const tritt_cache_t* c, const tritt_weights_t* w, const tritt_rows_t* q, const tritt_rows_t* k2, const float* m, int dtype,
                               float alpha, int k_diff, int* status_word, tritt_stream_t stream) {
  if (int rc = check_cache(c)) return rc;
  if (int rc = check_weights(c, w)) return rc;
  if (int rc = check_rows(q, 1, dtype)) return rc;
  if (int rc = check_rows(k2, 1, dtype)) return rc;
  if (int rc = check_weigh_scores(m, alpha)) return rc;
  if (!c->lse) {
    set_error("the cache has no log-sum-exps: it is not one of the dot-product-sum form");
    return -16;
  }
  if (k_diff < 0) {
    set_error("k_diff must be >= 0, got %d", k_diff);
    return -10;
  }
  Params p{cache_args(*c, status_word), *w, {*q, *k2}, m, k_diff, 0, 0, alpha * kLog2e};
  if (dtype == TRITT_F32) return by_code<float>(p, (cudaStream_t)stream);
  return dtype == TRITT_F16 ? by_code<__half>(p, (cudaStream_t)stream) : by_code<__nv_bfloat16>(p, (cudaStream_t)stream);
}
