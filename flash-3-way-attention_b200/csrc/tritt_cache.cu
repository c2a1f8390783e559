// The paged cache: rows quantised as they are written, read back, and the entry points of the attention over it.
//
// Writing and reading are bound by HBM (16-bit rows in, codes out).  D / 8 lanes take a row of one token and head, eight elements
// a lane, and the token's four parts, their loads in flight together; a row's largest element crosses its lanes by shuffles, so
// the row is read once.  The magnitudes of 16-bit elements order as integers: their maxima are taken two at a time.  A prompt of 8 x 16 x 2048
// rows of 64, bfloat16 to e4m3: written in 39 us (5.2 TB/s; with maxima in fp32, a choice for each element of rows that are not finite,
// and rows that waited for their places 634 instructions a warp: 61 us), read in 31 (6.5 TB/s).
#include "tritt_cache.cuh"
#include "tritt_sm100_tdp.cuh"

namespace tritt {
namespace {

constexpr int kThreads = 256;

struct WriteArgs {
  CacheArgs cache;
  tritt_rows_t rows[4];   // k1, k2, raw v1, v2
  int parts;              // the first 3 or all 4
};

template <typename T, int CODE, int D>
__global__ void __launch_bounds__(kThreads) cache_write_kernel(const __grid_constant__ WriteArgs w) {
  let_next_start();
  constexpr int L = D / 8, kSlots = kThreads / L;
  const CacheArgs& a = w.cache;
  const int col = threadIdx.x % L * 8;
  // neighbouring slots: heads of a token, whose rows are neighbours in the tensors (with four tokens of a head, neighbours in the cache, in
  // turn it took a tenth longer).  32 bits do: the host refuses more rows
  const uint32_t slot = blockIdx.x * kSlots + threadIdx.x / L, token = slot / (uint32_t)a.c.N;
  const int head = (int)(slot - token * a.c.N), b = (int)(token / (uint32_t)a.c.n), i = (int)(token - (uint32_t)b * a.c.n);
  bool on = b < a.c.B;
  // k1, k2, raw v1, v2 in the order of the parts; a padded token's rows too: they need not wait for the counts and the table
  constexpr int kWords = sizeof(T) / 2;   // of 16 bytes
  uint4 raw[4][kWords];
#pragma unroll
  for (int part = 0; part < 4; ++part) {
    const uint4* p = reinterpret_cast<const uint4*>((const T*)w.rows[part].p + rows_at(w.rows[part], b, head, i) + col);
#pragma unroll
    for (int k = 0; k < kWords; ++k) raw[part][k] = on && part < w.parts ? __ldg(p + k) : make_uint4(0u, 0u, 0u, 0u);
  }
  on = on && i < new_tokens(a, b);
  Place at{-1, 0};
  if (on) {
    at = place_of(a, b, context_of(a, b) + i);
    if (at.page < 0) {
      on = false;
      if (a.status) atomicOr(a.status, kStatusPlace);
    }
  }
  auto elements = [&](int part, float (&f)[8]) {
    if constexpr (kWords == 2) {
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const uint4 v = raw[part][k];
        f[4 * k] = __uint_as_float(v.x), f[4 * k + 1] = __uint_as_float(v.y), f[4 * k + 2] = __uint_as_float(v.z), f[4 * k + 3] = __uint_as_float(v.w);
      }
    } else {
      const uint32_t h[4] = {raw[part][0].x, raw[part][0].y, raw[part][0].z, raw[part][0].w};
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const float2 v = unpack2<T>(h[k]);
        f[2 * k] = v.x, f[2 * k + 1] = v.y;
      }
    }
  };
  // the rows' largest elements: of 16-bit tensors K1's and K2's in one word
  uint32_t most[4];
  float gated[8];
  elements(kPartV1, gated);
#pragma unroll
  for (int e = 0; e < 8; ++e) gated[e] = silu_f(gated[e]);
  most[kPartV1] = largest_of_row<L>(largest8(gated));
  if constexpr (kWords == 1) {
    const uint32_t keys = largest_of_two_rows<L>(largest_halves(raw[kPartK1][0]) | largest_halves(raw[kPartK2][0]) << 16);
    most[kPartK1] = bits_of_half<T>(keys & 0xffffu);
    most[kPartK2] = bits_of_half<T>(keys >> 16);
    most[kPartV2] = bits_of_half<T>(largest_of_row<L>(largest_halves(raw[kPartV2][0])));
  } else {
#pragma unroll
    for (int part = 0; part < 4; ++part) {
      if (part == kPartV1) continue;
      float f[8];
      elements(part, f);
      most[part] = largest_of_row<L>(largest8(f));
    }
  }
  if (!on) return;
  constexpr int kRowBytes = D * (CODE == TRITT_CODE_F16 ? 2 : 1);
  const size_t row = row_of(a, at, 0, head), part_rows = (size_t)a.c.N << a.page_log2;
  uint8_t* codes = (uint8_t*)a.c.codes + row * kRowBytes;
  unsigned char* exponent = a.c.exponents + row;
#pragma unroll
  for (int part = 0; part < 4; ++part) {
    if (part < w.parts) {
      const int byte = exponent_byte<CODE>(most[part]);
      float f[8];
      if (part != kPartV1) elements(part, f);
      codes_of<CODE>(byte, part == kPartV1 ? gated : f).store(codes, col);
      if (col == 0) *exponent = (unsigned char)byte;
    }
    codes += part_rows * kRowBytes;
    exponent += part_rows;
  }
}

struct ReadArgs {
  CacheArgs cache;
  void* parts[4];
  float* lse;
};

template <typename T, int CODE, int D>
__global__ void __launch_bounds__(kThreads) cache_read_kernel(const __grid_constant__ ReadArgs r) {
  constexpr int L = D / 8, kSlots = kThreads / L;
  const CacheArgs& a = r.cache;
  const int col = threadIdx.x % L * 8;
  // neighbouring slots: tokens of a head, whose rows are neighbours in a page and in the result
  const uint32_t slot = blockIdx.x * kSlots + threadIdx.x / L, bh = slot / (uint32_t)a.c.n;
  const int i = (int)(slot - bh * a.c.n), b = (int)(bh / (uint32_t)a.c.N), head = (int)(bh - (uint32_t)b * a.c.N);
  if (b >= a.c.B) return;
  Place at{-1, 0};
  if (i < new_tokens(a, b)) {
    at = place_of(a, b, context_of(a, b) + i);
    if (at.page < 0 && a.status) atomicOr(a.status, kStatusPlace);
  }
  Codes8<CODE> codes[4];
  int byte[4];
#pragma unroll
  for (int part = 0; part < 4; ++part) {
    if (at.page < 0) continue;
    const size_t row = row_of(a, at, part, head);
    codes[part].load((const uint8_t*)a.c.codes + row * (size_t)(D * (CODE == TRITT_CODE_F16 ? 2 : 1)), col);
    byte[part] = a.c.exponents[row];
  }
#pragma unroll
  for (int part = 0; part < 4; ++part) {
    float f[8];
    if (at.page < 0) {
#pragma unroll
      for (int e = 0; e < 8; ++e) f[e] = 0.f;
    } else {
      code_values<CODE>(codes[part], code_scale(byte[part]), f);
    }
    store8((T*)r.parts[part] + (size_t)slot * D + col, f);
  }
  if (r.lse && col == 0) r.lse[slot] = at.page < 0 ? 0.f : a.c.lse[lse_of(a, at, head)];
}

// One warp a row: D / 8 of its lanes hold eight elements each.  The splits' maxima and sums are looked at twice, their results once.
template <typename T, int CODE>
__global__ void __launch_bounds__(128) join_kernel(const __grid_constant__ JoinArgs j) {
  const CacheArgs& a = j.cache;
  const int lane = threadIdx.x & 31, col = lane * 8, D = a.c.D;
  const long long row = (long long)blockIdx.x * 4 + (threadIdx.x >> 5);
  if (row >= (long long)a.c.B * a.c.N * a.c.n) return;
  const int i = (int)(row % a.c.n), head = (int)(row / a.c.n % a.c.N), b = (int)(row / a.c.n / a.c.N);
  const float* part = j.part + (size_t)row * j.splits * (D + 2);
  // a maximum of -infinity: a split that has seen nothing; of NaN (which the comparisons below let through): a row of the cache that reads as NaN
  float m = -INFINITY;
  for (int s = lane; s < j.splits; s += 32) m = fmaxf(m, part[(size_t)s * (D + 2)]);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  float l = 0.f, f[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) f[e] = 0.f;
  for (int s = 0; s < j.splits; ++s) {
    const float* p = part + (size_t)s * (D + 2);
    const float ms = p[0], ls = p[1];
    if (ms == -INFINITY && ls == 0.f) continue;   // (its result is not written)
    const float weight = exp2f(ms - m);
    l = fmaf(ls, weight, l);
    if (col < D) {
#pragma unroll
      for (int e = 0; e < 8; ++e) f[e] = fmaf(p[2 + col + e], weight, f[e]);
    }
  }
  const bool none = m == -INFINITY && l == 0.f;
  const float inv = none ? 0.f : 1.f / l, lse = none ? -INFINITY : l != l ? l : (m + log2f(l)) * kLn2;
#pragma unroll
  for (int e = 0; e < 8; ++e) f[e] *= inv;
  if (j.o) {
    if (col < D) store8((T*)j.o + (size_t)row * D + col, f);
    if (j.lse && lane == 0) j.lse[row] = lse;
    return;
  }
  join_into_cache<T, CODE>(a, b, head, i, col, f, lse, j.v2);
}

template <typename T, int CODE, int D> int write_for(const WriteArgs& w, cudaStream_t stream) {
  const long long slots = (long long)w.cache.c.B * w.cache.c.n * w.cache.c.N;
  constexpr int kSlots = kThreads / (D / 8);
  cache_write_kernel<T, CODE, D><<<(unsigned)((slots + kSlots - 1) / kSlots), kThreads, 0, stream>>>(w);
  count_launch();
  TRITT_CUDA_OK(cudaGetLastError());
  return 0;
}
template <typename T, int CODE, int D> int read_for(const ReadArgs& r, cudaStream_t stream) {
  const long long slots = (long long)r.cache.c.B * r.cache.c.n * r.cache.c.N;
  constexpr int kSlots = kThreads / (D / 8);
  cache_read_kernel<T, CODE, D><<<(unsigned)((slots + kSlots - 1) / kSlots), kThreads, 0, stream>>>(r);
  count_launch();
  TRITT_CUDA_OK(cudaGetLastError());
  return 0;
}

template <typename T, int CODE> int write_d(const WriteArgs& w, cudaStream_t s) {
  switch (w.cache.c.D) {
    case 16: return write_for<T, CODE, 16>(w, s);
    case 32: return write_for<T, CODE, 32>(w, s);
    case 64: return write_for<T, CODE, 64>(w, s);
    case 128: return write_for<T, CODE, 128>(w, s);
    default: return write_for<T, CODE, 256>(w, s);
  }
}
template <typename T, int CODE> int read_d(const ReadArgs& r, cudaStream_t s) {
  switch (r.cache.c.D) {
    case 16: return read_for<T, CODE, 16>(r, s);
    case 32: return read_for<T, CODE, 32>(r, s);
    case 64: return read_for<T, CODE, 64>(r, s);
    case 128: return read_for<T, CODE, 128>(r, s);
    default: return read_for<T, CODE, 256>(r, s);
  }
}
template <typename T, int CODE> int join_for(const JoinArgs& j, cudaStream_t stream) {
  const long long rows = (long long)j.cache.c.B * j.cache.c.N * j.cache.c.n;
  join_kernel<T, CODE><<<(unsigned)((rows + 3) / 4), 128, 0, stream>>>(j);
  count_launch();
  TRITT_CUDA_OK(cudaGetLastError());
  return 0;
}

// f(type, code) with the types of a call
template <typename F> int by_type(int dtype, int code, F f) {
  auto with = [&](auto t) {
    using T = decltype(t);
    if (code == TRITT_CODE_F16) return f(T{}, std::integral_constant<int, TRITT_CODE_F16>{});
    if (code == TRITT_CODE_E4M3) return f(T{}, std::integral_constant<int, TRITT_CODE_E4M3>{});
    return f(T{}, std::integral_constant<int, TRITT_CODE_INT8>{});
  };
  if (dtype == TRITT_F32) return with(float{});
  return dtype == TRITT_F16 ? with(__half{}) : with(__nv_bfloat16{});
}

int check_scratch(size_t need, const void* ws, size_t have) {
  if (need && (!ws || have < need || ((uintptr_t)ws & 255))) {
    set_error("workspace too small or not 256-byte aligned: need %zu bytes, got %zu", need, ws ? have : (size_t)0);
    return -6;
  }
  return 0;
}

int check_lse(const float* lse) {   // (null: not wanted)
  if ((uintptr_t)lse & 3) {
    set_error("the log-sum-exps' pointer is not aligned");
    return -5;
  }
  return 0;
}

int check_out(const void* p, const float* lse) {
  if (!p) {
    set_error("null tensor pointer");
    return -4;
  }
  if ((uintptr_t)p & 15) {
    set_error("tensor pointer is not 16-byte aligned");
    return -5;
  }
  return check_lse(lse);
}

// (a scale that is not a number would come out of the kernels' maxima as one next to 0)
int check_scale(float alpha) {
  if (alpha - alpha != 0.f) {
    set_error("the soft-max scale must be finite, got %f", alpha);
    return -10;
  }
  return 0;
}

bool fast(int op, int D, int dtype, int flags) {
  if (flags & TRITT_FLAG_FORCE_SIMT) return false;
  return op == TRITT_OP_TDP_DECODE ? sm100_tdp_decode_supported(D, dtype) : mma_dps_decode_supported(D, dtype);
}

size_t part_bytes(const tritt_cache_t& c, int splits) {
  return align_up((size_t)c.B * c.N * c.n * splits * (c.D + 2) * 4, 256);
}

int window(int w) { return w < 0 ? 0 : w < 1 << 30 ? w : 1 << 30; }

}  // namespace

CacheArgs cache_args(const tritt_cache_t& c, int* status) {
  CacheArgs a{c, 0, status};
  while ((1 << a.page_log2) < c.page_size) ++a.page_log2;
  return a;
}

int check_cache(const tritt_cache_t* c) {
  if (!c || c->B <= 0 || c->N <= 0 || c->n <= 0 || c->pages <= 0 || c->table_pages <= 0) {
    set_error("sequences, heads, tokens and pages must be positive");
    return -1;
  }
  if (c->D != 16 && c->D != 32 && c->D != 64 && c->D != 128 && c->D != 256) {
    set_error("head_dim must be 16, 32, 64, 128 or 256, got %d", c->D);
    return -2;
  }
  if (c->code != TRITT_CODE_F16 && c->code != TRITT_CODE_E4M3 && c->code != TRITT_CODE_INT8) {
    set_error("unknown code type %d", c->code);
    return -3;
  }
  if (c->page_size < 16 || (c->page_size & (c->page_size - 1)) || (long long)c->page_size * c->table_pages > (1LL << 28)) {
    set_error("a page must have a power of two from 16 tokens on, a table at most 2^28 in all (page_size %d, %d pages)", c->page_size,
              c->table_pages);
    return -14;
  }
  if (!c->codes || !c->exponents || !c->table || !c->context) {
    set_error("null cache pointer");
    return -4;
  }
  if ((((uintptr_t)c->codes | (uintptr_t)c->exponents | (uintptr_t)c->lse) & 15) ||
      (((uintptr_t)c->table | (uintptr_t)c->context | (uintptr_t)c->counts) & 3) || ((uintptr_t)c->ancestors & 7)) {
    set_error("cache pointer is not aligned");
    return -5;
  }
  if (c->ancestors && c->n > TRITT_MAX_ANCESTORS) {
    set_error("at most %d new tokens with ancestors, got %d", TRITT_MAX_ANCESTORS, c->n);
    return -15;
  }
  if ((long long)c->B * c->N > 65535 || (long long)c->B * c->N * c->n > (1LL << 30)) {
    set_error("B*N = %lld, or with n = %d new tokens, is too much for one call; split the batch", (long long)c->B * c->N, c->n);
    return -11;
  }
  return 0;
}

int check_rows(const tritt_rows_t* rows, int count, int dtype) {
  if (dtype != TRITT_F32 && dtype != TRITT_F16 && dtype != TRITT_BF16) {
    set_error("unknown dtype code %d", dtype);
    return -3;
  }
  const long long unit = dtype == TRITT_F32 ? 4 : 8;
  for (int i = 0; i < count; ++i) {
    if (!rows || !rows[i].p) {
      set_error("null tensor pointer");
      return -4;
    }
    if (((uintptr_t)rows[i].p & 15) || rows[i].stride_b % unit || rows[i].stride_n % unit || rows[i].stride_t % unit) {
      set_error("rows must start on 16-byte boundaries");
      return -5;
    }
  }
  return 0;
}

int launch_write(const CacheArgs& a, const tritt_rows_t* rows, int dtype, int parts, cudaStream_t stream) {
  WriteArgs w{a, {rows[0], rows[1], rows[2], rows[3]}, parts};
  return by_type(dtype, a.c.code, [&](auto t, auto code) { return write_d<decltype(t), decltype(code)::value>(w, stream); });
}

int launch_join(const JoinArgs& j, cudaStream_t stream) {
  return by_type(j.dtype, j.cache.c.code, [&](auto t, auto code) { return join_for<decltype(t), decltype(code)::value>(j, stream); });
}

}  // namespace tritt

using namespace tritt;

extern "C" {

int tritt_cache_write(const tritt_cache_t* c, const tritt_rows_t* rows, int dtype, int* status_word, tritt_stream_t stream) {
  if (int rc = check_cache(c)) return rc;
  if (int rc = check_rows(rows, 4, dtype)) return rc;
  return launch_write(cache_args(*c, status_word), rows, dtype, 4, (cudaStream_t)stream);
}

int tritt_cache_read(const tritt_cache_t* c, void* const* parts, float* lse, int dtype, int* status_word, tritt_stream_t stream) {
  if (int rc = check_cache(c)) return rc;
  if (!parts) {
    set_error("null tensor pointer");
    return -4;
  }
  if (int rc = check_lse(lse)) return rc;
  ReadArgs r{cache_args(*c, status_word), {parts[0], parts[1], parts[2], parts[3]}, c->lse ? lse : nullptr};
  for (int i = 0; i < 4; ++i) {
    const tritt_rows_t row{parts[i], 0, 0, 0};
    if (int rc = check_rows(&row, 1, dtype)) return rc;
  }
  return by_type(dtype, c->code, [&](auto t, auto code) { return read_d<decltype(t), decltype(code)::value>(r, (cudaStream_t)stream); });
}

int tritt_decode_path(int op, int D, int dtype, int flags) { return fast(op, D, dtype, flags) ? TRITT_PATH_TCGEN05 : TRITT_PATH_SIMT; }

size_t tritt_decode_workspace(int op, const tritt_cache_t* c, int dtype, int k1_window, int k2_window, int flags) {
  if (check_cache(c)) return 0;
  if (op == TRITT_OP_TDP_DECODE && fast(op, c->D, dtype, flags))
    return window_tdp_decode_applies(*c, dtype, window(k1_window), window(k2_window), 1 << 30, 1 << 30) ? 0 : sm100_tdp_decode_workspace(*c);
  if (fast(op, c->D, dtype, flags)) return mma_dps_decode_workspace(*c);
  return part_bytes(*c, simt_decode_splits(*c));
}

int tritt_tdp_decode(const tritt_cache_t* c, const tritt_rows_t* q, void* o, float* lse, int dtype, float alpha, int k1_window,
                     int k2_window, int kk_left, int kk_right, void* workspace, size_t workspace_bytes, int* status_word, int flags,
                     tritt_stream_t stream) {
  if (int rc = check_cache(c)) return rc;
  if (int rc = check_rows(q, 1, dtype)) return rc;
  if (int rc = check_out(o, lse)) return rc;
  if (int rc = check_scale(alpha)) return rc;
  if (k1_window < 0 || k2_window < 0 || kk_left < 0 || kk_right < 0) {
    set_error("window arguments must be >= 0 (got %d, %d, %d, %d)", k1_window, k2_window, kk_left, kk_right);
    return -10;
  }
  const size_t need = tritt_decode_workspace(TRITT_OP_TDP_DECODE, c, dtype, k1_window, k2_window, flags);
  if (int rc = check_scratch(need, workspace, workspace_bytes)) return rc;
  TdpDecodeArgs a{cache_args(*c, status_word), *q, dtype, window(k1_window), window(k2_window), window(kk_left), window(kk_right), alpha * kLog2e, (float*)workspace, 0};
  if (fast(TRITT_OP_TDP_DECODE, c->D, dtype, flags) && window_tdp_decode_applies(*c, dtype, a.k1w, a.k2w, a.kkl, a.kkr))
    return window_tdp_decode(a, o, lse, (cudaStream_t)stream);
  if (fast(TRITT_OP_TDP_DECODE, c->D, dtype, flags)) return sm100_tdp_decode(a, workspace, o, lse, (cudaStream_t)stream);
  JoinArgs j{a.cache, a.part, 0, dtype, o, lse, {}};
  j.splits = a.splits = simt_decode_splits(*c);
  if (int rc = simt_tdp_decode(a, (cudaStream_t)stream)) return rc;
  return launch_join(j, (cudaStream_t)stream);
}

int tritt_dps_append(const tritt_cache_t* c, const tritt_rows_t* rows, int dtype, float alpha, int k_diff, void* workspace,
                     size_t workspace_bytes, int* status_word, int flags, tritt_stream_t stream) {
  if (int rc = check_cache(c)) return rc;
  if (int rc = check_rows(rows, 4, dtype)) return rc;
  if (!c->lse) {
    set_error("the cache has no log-sum-exps: it is not one of the dot-product-sum form");
    return -16;
  }
  if (int rc = check_scale(alpha)) return rc;
  if (k_diff < 0) {
    set_error("k_diff must be >= 0, got %d", k_diff);
    return -10;
  }
  const size_t need = tritt_decode_workspace(TRITT_OP_DPS_APPEND, c, dtype, 0, 0, flags);
  if (int rc = check_scratch(need, workspace, workspace_bytes)) return rc;
  const CacheArgs cache = cache_args(*c, status_word);
  if (int rc = launch_write(cache, rows, dtype, 3, (cudaStream_t)stream)) return rc;
  DpsDecodeArgs a{cache, rows[1], dtype, kPartK1, kPartV1, 0, window(k_diff), 1, alpha * kLog2e, (float*)workspace, 0};
  if (fast(TRITT_OP_DPS_APPEND, c->D, dtype, flags)) return mma_dps_decode(a, workspace, nullptr, nullptr, &rows[3], true, (cudaStream_t)stream);
  JoinArgs j{cache, a.part, 0, dtype, nullptr, nullptr, rows[3]};
  j.splits = a.splits = simt_decode_splits(*c);
  if (int rc = simt_dps_decode(a, (cudaStream_t)stream)) return rc;
  return launch_join(j, (cudaStream_t)stream);
}

int tritt_dps_decode(const tritt_cache_t* c, const tritt_rows_t* q, void* o, float* m, int dtype, float alpha, void* workspace,
                     size_t workspace_bytes, int* status_word, int flags, tritt_stream_t stream) {
  if (int rc = check_cache(c)) return rc;
  if (int rc = check_rows(q, 1, dtype)) return rc;
  if (int rc = check_out(o, m)) return rc;
  if (int rc = check_scale(alpha)) return rc;
  if (!c->lse) {
    set_error("the cache has no log-sum-exps: it is not one of the dot-product-sum form");
    return -16;
  }
  const size_t need = tritt_decode_workspace(TRITT_OP_DPS_DECODE, c, dtype, 0, 0, flags);
  if (int rc = check_scratch(need, workspace, workspace_bytes)) return rc;
  const CacheArgs cache = cache_args(*c, status_word);
  DpsDecodeArgs a{cache, *q, dtype, kPartK2, kPartV2, 1, 1 << 30, 0, alpha * kLog2e, (float*)workspace, 0};
  if (fast(TRITT_OP_DPS_DECODE, c->D, dtype, flags)) return mma_dps_decode(a, workspace, o, m, nullptr, false, (cudaStream_t)stream);
  JoinArgs j{cache, a.part, 0, dtype, o, m, {}};
  j.splits = a.splits = simt_decode_splits(*c);
  if (int rc = simt_dps_decode(a, (cudaStream_t)stream)) return rc;
  return launch_join(j, (cudaStream_t)stream);
}

}  // extern "C"
