// The attention weight of cached tokens in the triple dot product, with warp-level matrix instructions: head dimensions
// 16, 32 and 256 (64 and 128 run on tcgen05, or where their rows fit in shared memory as the windows' kernel).
//
//   P[j, k] = exp(alpha sum_h q[h] K1[j, h] K2[k, h] - lse),   w[x] = decay w[x] + sum_i (sum_k P_i[x, k] + sum_j P_i[j, x])
// For one new token and a tile of 128 tokens k the operand A[k] = q * K2[k] is formed once, as two fp16 numbers an element (22 bits: 16-bit queries times any code are exact), in the order of the
// fragments; each warp takes 16 rows j of K1 straight from memory, and its scores' exponentials add up along both sides: over k in the warp's registers to one number a row, over j in as many as it
// has columns, which leave at the end of the tile.  Sums go to slots of the CTA (see the line in tritt_weigh.cuh), each number by one thread, and a second kernel adds the slots up.
// Measured: one token of 2 x 16 heads over 2047 and 1050 tokens, int8 codes 82 us at head dimension 16, 97 at 32, 397 at 256 (430 with float16 codes); of 4 x 8 heads of 32 over up to 700, e4m3 28; 8 tokens over 2040,
// 16 heads of 32, float16 codes 500.  Bound by instructions: a product of 16 x 8 x 16 is one for each warp and step, twice, and an exponential, its mask and its two sums follow for each pair.
#include "tritt_weigh.cuh"

#include <cmath>

namespace tritt {
namespace {

constexpr int kThreads = 256;
constexpr int kUnlimited = 1 << 30;

// q times a code times 2^-kDown fits fp16: q is below 4, the codes below 2^15, 448, 127
template <int CODE> constexpr int kDown = CODE == TRITT_CODE_F16 ? 2 : 0;

template <int D> struct Shared {
  uint2 frags[16][2][D / 16][32];   // [8 tokens k][hi, lo][step][lane]
  float columns[8][128];            // of each warp
  float scale[128];                 // of the scores with each token k
  float q[D];
  uint32_t there[4];                // tokens k that have a place
  int field;                        // q's exponent
  int largest;                      // of their exponent bytes
};

template <typename T, int D, int CODE> __global__ void __launch_bounds__(kThreads) tdp_weigh_kernel(const __grid_constant__ TdpWeighArgs p) {
  using Rows = RowFragments<D, CODE>;
  constexpr int kSteps = Rows::kSteps;
  constexpr size_t kRow = D * Rows::kSize;
  extern __shared__ __align__(16) uint8_t smem[];
  Shared<D>& sh = *reinterpret_cast<Shared<D>*>(smem);
  const CacheArgs& a = p.cache;
  const uint8_t* codes = (const uint8_t*)a.c.codes;
  const int tid = threadIdx.x, lane = tid % 32, warp = tid / 32, g = lane / 4, c = lane % 4;
  WeighWalk walk = weigh_start(p, weigh_part(p));   // (each warp for itself)
  WeighPiece s;
  while (weigh_next(p, walk, s)) {
    float* const rows_sum = weigh_slot(p, s.b, s.head);
    float* const cols_sum = rows_sum + p.span;
    if (s.fresh)
      for (int x = tid % 128; x <= s.l.last - s.l.base; x += 128) (tid < 128 ? rows_sum : cols_sum)[x] = 0.f;
    const float lse = __ldg(p.lse + ((size_t)s.b * a.c.N + s.head) * a.c.n + s.i);
    __syncthreads();   // (the slot, and what the tile before has read)
    if (s.s0 == s.s1 || lse == -INFINITY) continue;
    const int pos = s.l.ctx + s.i, k_lo = pos - (p.k2w < pos ? p.k2w : pos), j_lo = pos - (p.k1w < pos ? p.k1w : pos);
    // q, the tokens k and their exponents
    if (warp == 0) {
      const T* row = (const T*)p.q.p + rows_at(p.q, s.b, s.head, s.i);
      float4 f[D > 128 ? 2 : 1];
      uint32_t top = 0;
#pragma unroll
      for (int k = 0; k < (D > 128 ? 2 : 1); ++k) {
        f[k] = lane + 32 * k < D / 4 ? load4(row + (lane + 32 * k) * 4) : make_float4(0.f, 0.f, 0.f, 0.f);
        top = max(top, largest4(f[k]));
      }
      const int field = (int)(largest_of_row<32>(top) >> 23);
      const float up = to_operand(field);
#pragma unroll
      for (int k = 0; k < (D > 128 ? 2 : 1); ++k)
        if (lane + 32 * k < D / 4)
          *reinterpret_cast<float4*>(sh.q + (lane + 32 * k) * 4) =
              field == 255 ? make_float4(0.f, 0.f, 0.f, 0.f) : make_float4(f[k].x * up, f[k].y * up, f[k].z * up, f[k].w * up);
      if (lane == 0) sh.field = field, sh.largest = 0;
    }
    const int k = s.kg * 128 + tid;   // (of the first four warps)
    int byte = 0;
    Place own{-1, 0};
    if (tid < 128) {
      const bool seen = k >= k_lo && k <= pos;
      if (seen) {
        own = place_of(a, s.b, k);
        if (own.page < 0 && a.status) atomicOr(a.status, kStatusPlace);
      }
      if (own.page >= 0) byte = __ldg(a.c.exponents + row_of(a, own, kPartK2, s.head));
      const uint32_t word = __ballot_sync(0xffffffffu, own.page >= 0);
      if (lane == 0) sh.there[warp] = word;
    }
    __syncthreads();
    if (tid < 128 && own.page >= 0 && byte != 255) atomicMax(&sh.largest, byte);
    __syncthreads();
    const int field = sh.field, middle = middle_byte<CODE>(sh.largest);
    if (tid < 128) sh.scale[tid] = own.page < 0 ? 0.f : byte == 255 ? __uint_as_float(0x7fffffffu) : relative_power(byte - middle);
    // A
    for (int x = tid; x < 128 * (D / 4); x += kThreads) {
      const int col = x / (D / 4), h = x % (D / 4) * 4, kk = s.kg * 128 + col;
      float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
      if (sh.there[col / 32] >> col % 32 & 1) {
        const Place at = place_of(a, s.b, kk);
        const uint8_t* from = codes + row_of(a, at, kPartK2, s.head) * kRow + h * Rows::kSize;
        uint32_t w[2];
        if constexpr (CODE == TRITT_CODE_F16) {
          const uint2 t = __ldg(reinterpret_cast<const uint2*>(from));
          w[0] = t.x, w[1] = t.y;
        } else {
          bytes_to_halves<CODE>(__ldg(reinterpret_cast<const uint32_t*>(from)), w[0], w[1]);
        }
        const float2 lo = __half22float2(*reinterpret_cast<const __half2*>(&w[0])), hi = __half22float2(*reinterpret_cast<const __half2*>(&w[1]));
        constexpr float kScale = 1.f / (1 << kDown<CODE>);
        v = make_float4(sh.q[h] * lo.x * kScale, sh.q[h + 1] * lo.y * kScale, sh.q[h + 2] * hi.x * kScale, sh.q[h + 3] * hi.y * kScale);
      }
      const auto slot = Rows::slot_of(h);
      const uint2 top = make_uint2(pack_halves(v.x, v.y), pack_halves(v.z, v.w));
      sh.frags[col / 8][0][slot.step][col % 8 * 4 + slot.c] = top;
      sh.frags[col / 8][1][slot.step][col % 8 * 4 + slot.c] = make_uint2(pack_rests(v.x, v.y, top.x), pack_rests(v.z, v.w, top.y));
    }
    __syncthreads();
    float column[16][2];
#pragma unroll
    for (int t = 0; t < 16; ++t) column[t][0] = column[t][1] = 0.f;
    const float lse2 = lse * kLog2e;
    for (int jt = s.s0; jt < s.s1; ++jt) {
      const int x0 = jt * 128 + warp * 16;
      if (x0 > pos || x0 + 15 < j_lo) continue;
      const Place at = place_of(a, s.b, x0);
      if (at.page < 0) {
        if (a.status) atomicOr(a.status, kStatusPlace);
        continue;
      }
      const size_t row = row_of(a, at, kPartK1, s.head);
      Rows rows;
      rows.load(codes + row * kRow, lane);
      float scale[2], sum[2] = {0.f, 0.f};
      int c_lo[2], c_hi[2];   // columns that the row has pairs with
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int e = __ldg(a.c.exponents + row + g + 8 * h), j = x0 + g + 8 * h;
        // 2^e of the row, that of the columns' in the middle, q and A
        int power = e + middle - 254 + field - 128 + kDown<CODE>;
        power = power < -126 ? -126 : power > 127 ? 127 : power;
        scale[h] = e == 255 || field == 255 ? __uint_as_float(0x7fffffffu) : field == 0 ? 0.f : p.scale2 * power_of_two(power);
        const bool on = j >= j_lo && j <= pos;
        c_lo[h] = (k_lo > j - p.kkr ? k_lo : j - p.kkr) - s.kg * 128;
        c_hi[h] = on ? (p.kkl < pos - j ? j + p.kkl : pos) - s.kg * 128 : -1;
      }
#pragma unroll
      for (int t = 0; t < 16; ++t) {
        float d[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int st = 0; st < kSteps; ++st) {
          uint32_t frag[4];
          rows.step(st, frag);
          mma_16816(d, frag, sh.frags[t][0][st][lane]);
          mma_16816(d, frag, sh.frags[t][1][st][lane]);
        }
        const int col = t * 8 + 2 * c;
        const float2 by = *reinterpret_cast<const float2*>(&sh.scale[col]);
        const uint32_t there = sh.there[t / 4] >> (col % 32);
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const bool on = col + e >= c_lo[h] && col + e <= c_hi[h] && (there >> e & 1);
            const float prob = on ? exp2f(scaled_score(d[2 * h + e], e ? by.y : by.x, scale[h], lse2)) : 0.f;
            sum[h] += prob;
            column[t][e] += prob;
          }
      }
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        sum[h] += __shfl_xor_sync(0xffffffffu, sum[h], 1);
        sum[h] += __shfl_xor_sync(0xffffffffu, sum[h], 2);
      }
      if (c < 2) rows_sum[x0 + g + 8 * c - s.l.base] += c ? sum[1] : sum[0];
    }
#pragma unroll
    for (int t = 0; t < 16; ++t)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float v = column[t][e];
        v += __shfl_xor_sync(0xffffffffu, v, 4);
        v += __shfl_xor_sync(0xffffffffu, v, 8);
        v += __shfl_xor_sync(0xffffffffu, v, 16);
        if (g == 0) sh.columns[warp][t * 8 + 2 * c + e] = v;
      }
    __syncthreads();
    if (tid < 128 && k <= s.l.last) {
      float v = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) v += sh.columns[i][tid];
      cols_sum[k - s.l.base] += v;
    }
  }
}

// Adds up a head's slots, and the weights of before.
__global__ void __launch_bounds__(256) tdp_weigh_join_kernel(const __grid_constant__ TdpWeighArgs p) {
  const CacheArgs& a = p.cache;
  const int bh = blockIdx.y, b = bh / a.c.N, head = bh - b * a.c.N;
  // (a kernel that ended without a wait would let the next one, and who uses the scratch after it, start beside the previous: of blocks that have nothing to do the first waits all the same)
  const bool first = blockIdx.x == 0 && blockIdx.y == 0;
  if (__ldg(a.c.context + b) < 0) {
    if (first) wait_for_previous();
    return;
  }
  const int ctx = context_of(a, b), end = weighed_tokens(a, p.w, ctx + new_tokens(a, b)), x = blockIdx.x * 256 + threadIdx.x;
  if ((int)blockIdx.x * 256 >= end) {
    if (first) wait_for_previous();
    return;
  }
  const WeighLine l = weigh_line(p, b);
  float v = x < ctx && x < end ? faded(p.w, b, head, x) : 0.f, sum = 0.f;
  const bool any = l.unit > 0 && x >= l.base && x <= l.last;
  wait_for_previous();   // (what is above depends on the call's arguments alone)
  int c0 = 0, c1 = -1;   // CTAs that have steps of this head
  if (any) {
    const long long total = __ldcg(p.table + a.c.B), s0 = __ldcg(p.table + b) + head * l.unit, s1 = s0 + l.unit;
    const int parts = weigh_parts(p, total);
    c0 = (int)quotient((s0 + 1) * parts - 1, total);   // (the largest part that begins no later than step s0)
    c1 = (int)quotient(s1 * parts - 1, total);
  }
  const float* slot = p.part + ((size_t)c0 + bh) * p.sums * p.span + (any ? x - l.base : 0);
  const int terms = (c1 - c0 + 1) * p.sums;
  for (int i0 = 0; i0 < terms; i0 += 16) {   // (sixteen on their way together, the last ones too)
    float some[16];
#pragma unroll
    for (int k = 0; k < 16; ++k) some[k] = i0 + k < terms ? __ldcg(slot + (size_t)(i0 + k) * p.span) : 0.f;
#pragma unroll
    for (int k = 0; k < 16; ++k) sum += some[k];
  }
  if (x < end) *weight_of(p.w, b, head, x) = v + sum;
}

template <typename T, int D, int CODE> int launch(const TdpWeighArgs& p, cudaStream_t stream) {
  const int bytes = (int)sizeof(Shared<D>);
  TRITT_CUDA_OK(cudaFuncSetAttribute(tdp_weigh_kernel<T, D, CODE>, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes));
  tdp_weigh_kernel<T, D, CODE><<<p.ctas, kThreads, bytes, stream>>>(p);
  count_launch();
  TRITT_CUDA_OK(cudaGetLastError());
  return 0;
}
template <typename T, int CODE> int by_size(const TdpWeighArgs& p, cudaStream_t stream) {
  switch (p.cache.c.D) {
    case 16: return launch<T, 16, CODE>(p, stream);
    case 32: return launch<T, 32, CODE>(p, stream);
    default: return launch<T, 256, CODE>(p, stream);
  }
}
template <typename T> int by_code(const TdpWeighArgs& p, cudaStream_t stream) {
  switch (p.cache.c.code) {
    case TRITT_CODE_F16: return by_size<T, TRITT_CODE_F16>(p, stream);
    case TRITT_CODE_E4M3: return by_size<T, TRITT_CODE_E4M3>(p, stream);
    default: return by_size<T, TRITT_CODE_INT8>(p, stream);
  }
}

// Slots take a number for each token that a table has room for, whatever the contexts, and heads may be many: a call takes as many sequences at a time as keep them below this, but one at least, and has a slot for each CTA
// (fewer CTAs would be that much slower, whatever the contexts are).
constexpr long long kMostSlots = 1ll << 30;
int sums_of(const tritt_cache_t& c) { return sm100_tdp_weigh_supported(c.D) ? 5 : 2; }   // (on tcgen05 four of the rows and one of the columns)
int sequences_at_once(const tritt_cache_t& c, int span) {
  const long long heads = kMostSlots / (sums_of(c) * 4ll * span) - kWeighCtas, n = heads / c.N;
  return (int)(n < 1 ? 1 : n < c.B ? n : c.B);
}
size_t table_bytes(const tritt_cache_t& c) { return align_up(((size_t)c.B + 1) * 8, 256); }
size_t slots_bytes(const tritt_cache_t& c, int span) { return (size_t)(kWeighCtas + (long long)sequences_at_once(c, span) * c.N) * sums_of(c) * span * 4; }

}  // namespace

int mma_tdp_weigh(const TdpWeighArgs& p, cudaStream_t stream) {
  if (p.dtype == TRITT_F32) return by_code<float>(p, stream);
  return p.dtype == TRITT_F16 ? by_code<__half>(p, stream) : by_code<__nv_bfloat16>(p, stream);
}

int launch_tdp_weigh_join(const TdpWeighArgs& p, cudaStream_t stream) {
  const tritt_cache_t& c = p.cache.c;
  long long tokens = (long long)c.table_pages * c.page_size + c.n;   // (weights of tokens behind the table's end fade all the same)
  const int length = p.w.after_length < p.w.before_length ? p.w.after_length : p.w.before_length;
  if (length < tokens) tokens = length;
  return launch_kernel_after(tdp_weigh_join_kernel, dim3((unsigned)((tokens + 255) / 256), c.B * c.N), 256, 0, stream, true, p);
}

int check_weights(const tritt_cache_t* c, const tritt_weights_t* w) {
  if (!w || !w->before || !w->after) {
    set_error("null pointer to weights");
    return -4;
  }
  if (((uintptr_t)w->before | (uintptr_t)w->after) & 3) {
    set_error("the weights' pointer is not aligned");
    return -5;
  }
  if (w->before_length < 1 || w->after_length < 1) {
    set_error("weights of %d and %d tokens", w->before_length, w->after_length);
    return -1;
  }
  if (!std::isfinite(w->decay) || w->decay < 0.f) {
    set_error("decay must be a finite number >= 0, got %g", w->decay);
    return -14;
  }
  if (c->ancestors) {
    set_error("tokens are weighed without ancestors, once they are accepted");
    return -15;
  }
  return 0;
}
int check_weigh_scores(const float* lse, float alpha) {
  if (!lse) {
    set_error("null tensor pointer");
    return -4;
  }
  if ((uintptr_t)lse & 3) {
    set_error("the log-sum-exps' pointer is not aligned");
    return -5;
  }
  if (!std::isfinite(alpha)) {
    set_error("the scale of the scores must be finite, got %g", alpha);
    return -14;
  }
  return 0;
}

}  // namespace tritt

using namespace tritt;

extern "C" {

size_t tritt_tdp_weigh_workspace(const tritt_cache_t* c, int k1_window, int k2_window) {
  if (check_cache(c) || k1_window < 0 || k2_window < 0) return 0;
  return table_bytes(*c) + slots_bytes(*c, weigh_span(*c, k1_window < kUnlimited ? k1_window : kUnlimited, k2_window < kUnlimited ? k2_window : kUnlimited));
}

int tritt_tdp_weigh(const tritt_cache_t* c, const tritt_weights_t* w, const tritt_rows_t* q, const float* lse, int dtype, float alpha, int k1_window,
                    int k2_window, int kk_left, int kk_right, void* workspace, size_t workspace_bytes, int* status_word, tritt_stream_t stream) {
  if (int rc = check_cache(c)) return rc;
  if (int rc = check_weights(c, w)) return rc;
  if (int rc = check_rows(q, 1, dtype)) return rc;
  if (int rc = check_weigh_scores(lse, alpha)) return rc;
  if (k1_window < 0 || k2_window < 0 || kk_left < 0 || kk_right < 0) {
    set_error("window arguments must be >= 0 (got %d, %d, %d, %d)", k1_window, k2_window, kk_left, kk_right);
    return -10;
  }
  const size_t need = tritt_tdp_weigh_workspace(c, k1_window, k2_window);
  if (!workspace || workspace_bytes < need || ((uintptr_t)workspace & 15)) {
    set_error("workspace too small or misaligned: need %zu bytes, got %zu", need, workspace ? workspace_bytes : (size_t)0);
    return -6;
  }
  auto window = [](int v) { return v < kUnlimited ? v : kUnlimited; };
  TdpWeighArgs p{cache_args(*c, status_word), *w, *q, lse, dtype, window(k1_window), window(k2_window), window(kk_left), window(kk_right), alpha * kLog2e,
                 (long long*)workspace, (float*)((uint8_t*)workspace + table_bytes(*c)), kWeighCtas, weigh_span(*c, window(k1_window), window(k2_window)), 0};
  if (window_tdp_weigh_applies(p)) return window_tdp_weigh(p, (cudaStream_t)stream);
  const bool fast = sm100_tdp_weigh_supported(c->D);
  p.sums = sums_of(*c);
  const int most = sequences_at_once(*c, p.span), size = dtype == TRITT_F32 ? 4 : 2;
  for (int b0 = 0; b0 < c->B; b0 += most) {
    TdpWeighArgs s = p;   // of sequences b0 and on
    tritt_cache_t& some = s.cache.c;
    some.B = c->B - b0 < most ? c->B - b0 : most;
    some.table += b0 * c->table_stride;
    some.context += b0;
    if (some.counts) some.counts += b0;
    s.q.p = (const uint8_t*)q->p + b0 * q->stride_b * size;
    s.lse += (size_t)b0 * c->N * c->n;
    s.w.before += b0 * w->before_stride_b;
    s.w.after += b0 * w->after_stride_b;
    if (int rc = fast ? sm100_tdp_weigh(s, (cudaStream_t)stream) : mma_tdp_weigh(s, (cudaStream_t)stream)) return rc;
    if (int rc = launch_tdp_weigh_join(s, (cudaStream_t)stream)) return rc;
  }
  return 0;
}

}  // extern "C"
