// Rotary embedding at each token's own position, and the append of new keys and values to a paged cache.
//
//   theta = position * f_i,  (a, b) -> amplitude * (a cos theta - b sin theta, a sin theta + b cos theta),  i < rotary_dim / 2
// on the pairs (2i, 2i + 1) of the interleaved layout or (i, i + rotary_dim / 2) of the half layout; the rest of the head is
// copied.  The backward pass is the transpose: theta negated.  Extends the dense form of cpp/src/Positional.cpp:120-147.
//
// Bound by memory: every element is read once and written once.  One CTA takes up to four tokens; it evaluates each (token, pair) angle
// once into shared memory and uses it for all heads, so the angles can be exact: the product with the 64-bit frequency and the
// reduction to one turn are done in 64 bits (a 32-bit product is off by 6e-3 rad at position 10^5), the sine and cosine of the
// reduced angle in 32.  Vectors of 16 bytes when alignment and layout allow, else element by element.  What hides the memory's
// latency is the number of threads: eight CTAs of 256 per SM with one vector each in flight take 33.2 us for the gradients of 16384
// tokens of 16 + 4 heads of 128 in bf16 (5.1 TB/s); two or four vectors a thread at four to six CTAs took 41 to 51 where this took 37, a form with the
// angles in registers that walks over the heads (less contiguous) 40 to 47.
// Appending k and v with the rotation of q and k is one launch: rows go from the projection's output straight to their pages
// (8892 tokens of 32 + 8 + 8 heads of 128 in bf16: 41.8 us, 5.2 TB/s).
#include "paged_common.cuh"
#include <algorithm>
#include <cmath>

namespace {

constexpr int THREADS = 256, MAX_PAIRS = 512, MAX_TOKENS = 8, TOKENS = 4;      // MAX_PAIRS: (token, pair) angles in shared memory per CTA

struct RopeArgs {
  const double *freqs;
  const int *positions;                  // null: positions are those of the paged batch
  const void *q, *k, *v;
  void *q_out, *k_out, *v_out;           // k_out / v_out: linear rows, or the pages when `paged`
  long long ld_q, ld_k, ld_v, ld_qo, ld_ko;
  int tokens, qh, kvh, hd, rd, per_cta;
  float amplitude, sign;
  int paged;
};

// Two bf16 values at a time where the type allows.
template <class T> __device__ __forceinline__ void unpack16(const Vec16<T> &v, float *f) {
  if constexpr (sizeof(T) == 2) {
    const uint32_t w[4] = {v.raw.x, v.raw.y, v.raw.z, v.raw.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) { f[2 * i] = __uint_as_float(w[i] << 16); f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u); }
  } else v.unpack(f);
}
template <class T> __device__ __forceinline__ void pack16(Vec16<T> &v, const float *f) {
  if constexpr (sizeof(T) == 2) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) { const __nv_bfloat162 h = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]); w[i] = *reinterpret_cast<const uint32_t *>(&h); }
    v.raw = make_uint4(w[0], w[1], w[2], w[3]);
  } else v.pack(f);
}

// A rotated vector of a head: its 16 bytes (interleaved layout, or the copied rest), or the two that pair (half layout).  The sines and cosines
// of an item are float4 (two pairs each) `stride` apart, so that the items of a warp read neighbouring ones.
template <class T, bool HALF>
struct Piece {
  static constexpr int N = Vec16<T>::N, PAIRS = HALF ? N : N / 2, QUADS = PAIRS / 2;
  Vec16<T> x, y;
  __device__ __forceinline__ void load(const T *src, int item, int turned) {
    if constexpr (HALF) {
      if (item < turned) { x.load(src + item * N); y.load(src + (item + turned) * N); }
      else x.load(src + (item + turned) * N);
    } else x.load(src + item * N);
  }
  __device__ __forceinline__ void turn_store(T *dst, int item, int turned, const float4 *cs, int stride) {
    if (item >= turned) { x.store(dst + (HALF ? item + turned : item) * N); return; }
    float a[N], b[N];
    unpack16(x, a);
    if constexpr (HALF) unpack16(y, b);
#pragma unroll
    for (int k = 0; k < QUADS; ++k) {
      const float4 q = cs[k * stride];
      const float2 c[2] = {make_float2(q.x, q.y), make_float2(q.z, q.w)};
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int p = 2 * k + j;
        float &u = HALF ? a[p] : a[2 * p], &w = HALF ? b[p] : a[2 * p + 1];
        const float u0 = u, w0 = w;
        u = u0 * c[j].x - w0 * c[j].y; w = u0 * c[j].y + w0 * c[j].x;
      }
    }
    pack16(x, a); x.store(dst + item * N);
    if constexpr (HALF) { pack16(y, b); y.store(dst + (item + turned) * N); }
  }
};
// element by element: a pair, then the copied rest
template <class T, bool HALF>
__device__ __forceinline__ void turn_one(const T *src, T *dst, int item, int rd, const float2 *cs) {
  if (item >= rd / 2) { dst[item + rd / 2] = src[item + rd / 2]; return; }
  const int i = HALF ? item : 2 * item, j = HALF ? item + rd / 2 : 2 * item + 1;
  const float a = to_f(src[i]), b = to_f(src[j]);
  const float2 c = cs[item];
  dst[i] = from_f<T>(a * c.x - b * c.y); dst[j] = from_f<T>(a * c.y + b * c.x);
}

// Off: the type of element offsets into q and k, 32 bits where the arrays are that small (a fifth of the instructions is address arithmetic otherwise).
template <class T, bool HALF, bool VEC, class Off>
__global__ void __launch_bounds__(THREADS, 8)
rope_positions_kernel(RopeArgs r, PagedArgs a) {
  pdl_launch_dependents();
  pdl_wait();
  typedef Piece<T, HALF> P;
  constexpr int N = P::N;
  __shared__ float4 cs4[MAX_PAIRS / 2];
  __shared__ int pos_s[MAX_TOKENS];
  __shared__ long long slot_s[MAX_TOKENS];             // element offset of the row's slot in the pages; -1: no slot, -2: no sequence
  float2 *cs = reinterpret_cast<float2 *>(cs4);
  const int t0 = blockIdx.x * r.per_cta, nt = min(r.per_cta, r.tokens - t0), pairs = r.rd / 2, tid = threadIdx.x;
  const int H = r.qh + r.kvh, rows = nt * H, turned = VEC ? pairs / P::PAIRS : pairs;      // rows to rotate: a token's query heads, then its key heads
  if (r.paged) {
    for (int t = tid; t < nt; t += THREADS) slot_s[t] = -2;
    __syncthreads();
    for (int s = tid; s < a.n_seq; s += THREADS) {
      const paged::Seq q = paged::load_seq(a, s);
      const int lo = max(q.q0, t0), hi = min(q.q0 + q.ql, t0 + nt);
      for (int t = lo; t < hi; ++t) {
        const int pos = q.base + (t - q.q0);
        long long slot = -1;                           // rows before the first position are padding
        if (pos >= 0) {
          const int page = paged::page_of(a, s, pos);
          if (page >= 0) slot = (long long)page * a.page_stride + (long long)(pos % a.page_size) * a.token_stride;
        }
        pos_s[t - t0] = pos; slot_s[t - t0] = slot;
      }
    }
    __syncthreads();
  }
  for (int i = tid; i < nt * pairs; i += THREADS) {
    const int t = i / pairs, p = i - t * pairs;
    if (r.paged && slot_s[t] == -2) continue;
    const double turns = (double)(r.paged ? pos_s[t] : r.positions[t0 + t]) * (r.freqs[p] * 0.15915494309189533577);
    float sn, c;
    sincospif(2.0f * (float)(turns - rint(turns)), &sn, &c);
    int at = i;
    if constexpr (VEC) { const int item = p / P::PAIRS, j = p % P::PAIRS; at = ((t * P::QUADS + j / 2) * turned + item) * 2 + (j & 1); }
    cs[at] = make_float2(c * r.amplitude, sn * r.amplitude * r.sign);
  }
  __syncthreads();
  auto source = [&](int t, int h) -> const T * {
    const Off row = (Off)(t0 + t);
    return h < r.qh ? (const T *)r.q + (row * (Off)r.ld_q + (Off)(h * r.hd)) : (const T *)r.k + (row * (Off)r.ld_k + (Off)((h - r.qh) * r.hd));
  };
  auto target = [&](int t, int h) -> T * {             // null: the row is left as it is
    const Off row = (Off)(t0 + t);
    if (h < r.qh) return r.paged && slot_s[t] == -2 ? nullptr : (T *)r.q_out + (row * (Off)r.ld_qo + (Off)(h * r.hd));
    if (r.paged) return slot_s[t] < 0 ? nullptr : (T *)r.k_out + slot_s[t] + (long long)(h - r.qh) * a.head_stride;
    return (T *)r.k_out + (row * (Off)r.ld_ko + (Off)((h - r.qh) * r.hd));
  };
  if constexpr (VEC) {
    // a thread keeps its place in the head and takes rows one pass of the CTA apart
    const int items = HALF ? r.hd / N - turned : r.hd / N, pass = THREADS / items, item = tid % items, first = tid / items;
    if (first < pass) {
      const int dt = pass / H, dh = pass - dt * H;
      int t = first / H, h = first - t * H;
      while (t < nt) {
        T *dst = target(t, h);
        if (dst) {
          P piece;
          piece.load(source(t, h), item, turned);
          piece.turn_store(dst, item, turned, cs4 + t * P::QUADS * turned + item, turned);
        }
        t += dt; h += dh;
        if (h >= H) { h -= H; ++t; }
      }
    }
  } else {
    const int per_row = r.hd - pairs;
    for (int i = tid; i < rows * per_row; i += THREADS) {
      const int x = i / per_row, t = x / H;
      T *dst = target(t, x - t * H);
      if (dst) turn_one<T, HALF>(source(t, x - t * H), dst, i - x * per_row, r.rd, cs + t * pairs);
    }
  }
  if (r.v) {                                           // values are copied to their slots
    const int per_row = VEC ? r.hd / N : r.hd, all = nt * r.kvh * per_row;
    constexpr int U = VEC ? 4 : 1;
    for (int i0 = tid; i0 < all; i0 += U * THREADS) {
      uint4 v[U];
      T one = from_f<T>(0.f);
      long long at[U];
#pragma unroll
      for (int j = 0; j < U; ++j) {
        const int i = i0 + j * THREADS;
        at[j] = -1;
        if (i < all) {
          const int x = i / per_row, d = i - x * per_row, t = x / r.kvh, h = x - t * r.kvh;
          const T *src = (const T *)r.v + ((size_t)t0 + t) * r.ld_v + (size_t)h * r.hd + (VEC ? d * N : d);
          if (slot_s[t] >= 0) at[j] = slot_s[t] + (long long)h * a.head_stride + (VEC ? d * N : d);
          if constexpr (VEC) v[j] = *reinterpret_cast<const uint4 *>(src);
          else one = *src;
        }
      }
#pragma unroll
      for (int j = 0; j < U; ++j)
        if (at[j] >= 0) {
          T *dst = (T *)r.v_out + at[j];
          if constexpr (VEC) *reinterpret_cast<uint4 *>(dst) = v[j];
          else *dst = one;
        }
    }
  }
}

__global__ void rope_frequencies_kernel(double *f, int pairs, b200_rope_config c) {
  pdl_launch_dependents();
  pdl_wait();
  const int i = blockIdx.x * blockDim.x + threadIdx.x;
  if (i >= pairs) return;
  const double two_pi = 6.283185307179586476925, rd = 2.0 * pairs, e = -2.0 * i / rd, base = c.base, s = c.factor, L = c.original_len;
  double v = pow(base, e);
  if (c.scaling == B200_ROPE_LINEAR) v /= s;
  else if (c.scaling == B200_ROPE_NTK) { if (pairs > 1) v = pow(base * pow(s, rd / (rd - 2.0)), e); }
  else if (c.scaling == B200_ROPE_YARN) {
    const double l2 = 2.0 * log(base);
    const double lo = fmax(0.0, floor(rd * log(L / (c.beta_fast * two_pi)) / l2)), hi = fmin(rd - 1.0, ceil(rd * log(L / (c.beta_slow * two_pi)) / l2));
    const double ramp = fmin(1.0, fmax(0.0, (i - lo) / fmax(hi - lo, 0.001)));
    v = v / s * ramp + v * (1.0 - ramp);
  } else if (c.scaling == B200_ROPE_BANDS) {
    const double share = fmin(1.0, fmax(0.0, (L * v / two_pi - c.low_freq_factor) / ((double)c.high_freq_factor - c.low_freq_factor)));
    v = (1.0 - share) * v / s + share * v;
  }
  f[i] = v;
}

int check_config(b200_ctx *ctx, const b200_rope_config *c) {
  B200_REQUIRE(ctx, c, "rope: null configuration");
  B200_REQUIRE(ctx, c->head_dim > 0 && c->head_dim <= 1024 && c->rotary_dim % 2 == 0 && c->rotary_dim <= c->head_dim, "rope: rotary_dim must be even and at most head_dim (at most 1024)");
  B200_REQUIRE(ctx, c->layout == B200_ROPE_INTERLEAVED || c->layout == B200_ROPE_HALF, "rope: unknown layout");
  B200_REQUIRE(ctx, c->scaling >= B200_ROPE_PLAIN && c->scaling <= B200_ROPE_BANDS, "rope: unknown scaling");
  B200_REQUIRE(ctx, std::isfinite(c->amplitude) && c->amplitude >= 0.f, "rope: amplitude must be finite and not negative (0: the scaling's own)");
  return B200_OK;
}

template <class T, bool HALF>
int launch_t(b200_ctx *ctx, const RopeArgs &r, const PagedArgs &a, bool vec) {
  const dim3 grid((unsigned)((r.tokens + r.per_cta - 1) / r.per_cta));
  const unsigned long long most = (unsigned long long)r.tokens * std::max(std::max(r.ld_q, r.ld_qo), std::max(r.ld_k, r.ld_ko));
  const bool small = (unsigned long long)(r.ld_q | r.ld_qo | r.ld_k | r.ld_ko) < (1ull << 31) && most < (1ull << 32);
  if (vec && small) B200_CUDA(ctx, launch_pdl(ctx, rope_positions_kernel<T, HALF, true, unsigned>, grid, dim3(THREADS), 0, 0, r, a));
  else if (vec) B200_CUDA(ctx, launch_pdl(ctx, rope_positions_kernel<T, HALF, true, unsigned long long>, grid, dim3(THREADS), 0, 0, r, a));
  else B200_CUDA(ctx, launch_pdl(ctx, rope_positions_kernel<T, HALF, false, unsigned long long>, grid, dim3(THREADS), 0, 0, r, a));
  B200_LAUNCHED(ctx);
  return B200_OK;
}

int launch(b200_ctx *ctx, RopeArgs &r, const PagedArgs &a, bool half, b200_dtype dt) {
  const size_t es = dtype_size(dt), n = 16 / es;
  const uintptr_t ptrs = (uintptr_t)r.q | (uintptr_t)r.k | (uintptr_t)r.v | (uintptr_t)r.q_out | (uintptr_t)r.k_out | (uintptr_t)r.v_out;
  const unsigned long long lds = (unsigned long long)r.ld_q | r.ld_k | r.ld_v | r.ld_qo | r.ld_ko | (r.paged ? (a.page_stride | a.token_stride | a.head_stride) : 0);
  const bool vec = ptrs % 16 == 0 && lds % n == 0 && (size_t)r.hd % n == 0 && (half ? (size_t)(r.rd / 2) % n == 0 : (size_t)r.rd % n == 0);
  // tokens per CTA: as many as their angles fit, while the grid still covers the SMs several times
  const int fit = r.rd ? std::max(1, MAX_PAIRS / (r.rd / 2)) : 8;
  r.per_cta = std::max(1, std::min(std::min(fit, TOKENS), r.tokens / (4 * ctx->sm_count)));
  if (dt == B200_BF16) return half ? launch_t<bf16, true>(ctx, r, a, vec) : launch_t<bf16, false>(ctx, r, a, vec);
  return half ? launch_t<float, true>(ctx, r, a, vec) : launch_t<float, false>(ctx, r, a, vec);
}

float amplitude_of(const b200_rope_config *c) {
  if (c->amplitude > 0.f) return c->amplitude;
  return c->scaling == B200_ROPE_YARN && c->factor > 1.f ? 0.1f * logf(c->factor) + 1.0f : 1.0f;
}

int rope_linear(b200_ctx *ctx, const b200_rope_config *c, const double *freqs, const int32_t *positions, const void *q, void *q_out, size_t ld_q,
                size_t ld_qo, size_t q_heads, const void *k, void *k_out, size_t ld_k, size_t ld_ko, size_t kv_heads, size_t tokens,
                b200_dtype dt, float sign) {
  if (!ctx) return B200_ERR_INVALID;
  int rc = check_config(ctx, c);
  if (rc) return rc;
  B200_REQUIRE(ctx, dt == B200_F32 || dt == B200_BF16, "rope_positions: unknown dtype");
  if (!k) kv_heads = 0;
  if (!q) q_heads = 0;
  B200_REQUIRE(ctx, q_heads <= 65536 && kv_heads <= 65536, "rope_positions: at most 65536 heads");
  if (tokens == 0 || q_heads + kv_heads == 0) return B200_OK;
  B200_REQUIRE(ctx, tokens <= 0x7fffffff, "rope_positions: at most 2^31 - 1 tokens");
  B200_REQUIRE(ctx, positions && (freqs || c->rotary_dim == 0) && (!q || q_out) && (!k || k_out), "rope_positions: null pointer");
  B200_REQUIRE(ctx, (!q_heads || (ld_q >= q_heads * c->head_dim && ld_qo >= q_heads * c->head_dim)) && (!kv_heads || (ld_k >= kv_heads * c->head_dim && ld_ko >= kv_heads * c->head_dim)),
               "rope_positions: a row stride is shorter than the row");
  DeviceGuard guard(ctx);
  B200_REQUIRE(ctx, guard.ok, "rope_positions: the context's device cannot be selected");
  RopeArgs r = {};
  r.freqs = freqs; r.positions = positions;
  if (q_heads) { r.q = q; r.q_out = q_out; r.ld_q = (long long)ld_q; r.ld_qo = (long long)ld_qo; }
  if (kv_heads) { r.k = k; r.k_out = k_out; r.ld_k = (long long)ld_k; r.ld_ko = (long long)ld_ko; }
  r.tokens = (int)tokens; r.qh = (int)q_heads; r.kvh = (int)kv_heads; r.hd = (int)c->head_dim; r.rd = (int)c->rotary_dim;
  r.amplitude = amplitude_of(c); r.sign = sign;
  return launch(ctx, r, PagedArgs(), c->layout == B200_ROPE_HALF, dt);
}

}  // namespace

extern "C" float b200_rope_amplitude(const b200_rope_config *c) { return c ? amplitude_of(c) : 0.f; }

extern "C" int b200_rope_frequencies(b200_ctx *ctx, const b200_rope_config *c, double *freqs) {
  if (!ctx) return B200_ERR_INVALID;
  int rc = check_config(ctx, c);
  if (rc) return rc;
  if (c->rotary_dim == 0) return B200_OK;
  B200_REQUIRE(ctx, freqs, "rope_frequencies: null pointer");
  B200_REQUIRE(ctx, std::isfinite(c->base) && c->base > 1.f, "rope_frequencies: base must be above 1");
  B200_REQUIRE(ctx, c->scaling == B200_ROPE_PLAIN || (std::isfinite(c->factor) && c->factor >= 1.f), "rope_frequencies: factor must be at least 1");
  B200_REQUIRE(ctx, c->scaling < B200_ROPE_YARN || (std::isfinite(c->original_len) && c->original_len >= 1.f), "rope_frequencies: original_len must be at least 1");
  B200_REQUIRE(ctx, c->scaling != B200_ROPE_YARN || (c->beta_slow > 0.f && c->beta_fast >= c->beta_slow), "rope_frequencies: 0 < beta_slow <= beta_fast");
  B200_REQUIRE(ctx, c->scaling != B200_ROPE_BANDS || (c->low_freq_factor > 0.f && c->high_freq_factor > c->low_freq_factor), "rope_frequencies: 0 < low_freq_factor < high_freq_factor");
  DeviceGuard guard(ctx);
  B200_REQUIRE(ctx, guard.ok, "rope_frequencies: the context's device cannot be selected");
  const int pairs = (int)(c->rotary_dim / 2);
  B200_CUDA(ctx, launch_pdl(ctx, rope_frequencies_kernel, dim3((pairs + 127) / 128), dim3(128), 0, 0, freqs, pairs, *c));
  B200_LAUNCHED(ctx);
  return B200_OK;
}

extern "C" int b200_rope_positions_forward(b200_ctx *ctx, const b200_rope_config *c, const double *freqs, const int32_t *positions, const void *q,
                                           void *q_out, size_t ld_q, size_t ld_q_out, size_t q_heads, const void *k, void *k_out, size_t ld_k,
                                           size_t ld_k_out, size_t kv_heads, size_t tokens, b200_dtype dt) {
  return rope_linear(ctx, c, freqs, positions, q, q_out, ld_q, ld_q_out, q_heads, k, k_out, ld_k, ld_k_out, kv_heads, tokens, dt, 1.0f);
}
extern "C" int b200_rope_positions_backward(b200_ctx *ctx, const b200_rope_config *c, const double *freqs, const int32_t *positions, const void *dq,
                                            void *dq_out, size_t ld_dq, size_t ld_dq_out, size_t q_heads, const void *dk, void *dk_out, size_t ld_dk,
                                            size_t ld_dk_out, size_t kv_heads, size_t tokens, b200_dtype dt) {
  return rope_linear(ctx, c, freqs, positions, dq, dq_out, ld_dq, ld_dq_out, q_heads, dk, dk_out, ld_dk, ld_dk_out, kv_heads, tokens, dt, -1.0f);
}

int paged_args(b200_ctx *ctx, const b200_paged_cache *cache, const b200_paged_batch *batch, PagedArgs *a) {
  B200_REQUIRE(ctx, cache && batch, "paged cache: null descriptor");
  B200_REQUIRE(ctx, cache->dtype == B200_F32 || cache->dtype == B200_BF16, "paged cache: unknown dtype");
  B200_REQUIRE(ctx, cache->k && cache->v && cache->n_pages > 0, "paged cache: null pages");
  B200_REQUIRE(ctx, cache->page_size > 0 && cache->n_kv > 0 && cache->head_dim > 0 && cache->n_pages <= 0x7fffffff && cache->page_size <= 65536 && cache->n_kv <= 65536 && cache->head_dim <= 1024,
               "paged cache: sizes out of range (page_size and n_kv up to 65536, head_dim up to 1024)");
  const size_t big = (size_t)1 << 40;
  B200_REQUIRE(ctx, cache->page_stride < big && cache->token_stride < big && cache->head_stride < big && cache->page_stride > 0 && cache->token_stride > 0 && cache->head_stride >= cache->head_dim,
               "paged cache: strides out of range");
  B200_REQUIRE(ctx, batch->n_seq <= 65536 && batch->rows <= 0x3fffffff, "paged batch: at most 65536 sequences and 2^30 - 1 rows");
  B200_REQUIRE(ctx, batch->n_seq == 0 || (batch->q_start && batch->kv_len && batch->page_table), "paged batch: null pointer");
  B200_REQUIRE(ctx, batch->n_seq == 0 || (batch->table_ld > 0 && batch->table_ld <= 0x7fffffff && batch->table_ld * cache->page_size <= 0x7fffff00), "paged batch: a row of the page table must hold 1 .. 2^31 - 256 positions");
  a->q_start = batch->q_start; a->kv_len = batch->kv_len; a->table = batch->page_table;
  a->n_seq = (int)batch->n_seq; a->table_ld = (int)batch->table_ld; a->rows = (int)batch->rows;
  a->max_q = (int)(batch->max_q ? std::min(batch->max_q, batch->rows) : batch->rows);
  a->page_size = (int)cache->page_size; a->n_pages = (int)cache->n_pages; a->n_kv = (int)cache->n_kv; a->hd = (int)cache->head_dim;
  a->page_stride = (long long)cache->page_stride; a->token_stride = (long long)cache->token_stride; a->head_stride = (long long)cache->head_stride;
  a->status = ctx->dev_status;
  return B200_OK;
}

extern "C" int b200_paged_append(b200_ctx *ctx, const b200_paged_cache *cache, const b200_paged_batch *batch, const void *k, const void *v, size_t ld_k,
                                 size_t ld_v, const b200_rope_config *rope, const double *freqs, const void *q, void *q_out, size_t ld_q,
                                 size_t ld_q_out, size_t q_heads) {
  if (!ctx) return B200_ERR_INVALID;
  PagedArgs a;
  int rc = paged_args(ctx, cache, batch, &a);
  if (rc) return rc;
  if (rope) {
    rc = check_config(ctx, rope);
    if (rc) return rc;
    B200_REQUIRE(ctx, rope->head_dim == cache->head_dim && (freqs || rope->rotary_dim == 0), "paged_append: the rotation needs the cache's head_dim and its frequencies");
  }
  B200_REQUIRE(ctx, (q == nullptr) == (q_out == nullptr), "paged_append: q and q_out come together");
  if (batch->n_seq == 0 || batch->rows == 0) return B200_OK;
  B200_REQUIRE(ctx, k && v, "paged_append: null pointer");
  B200_REQUIRE(ctx, q_heads <= 65536, "paged_append: at most 65536 heads");
  const size_t kv_row = cache->n_kv * cache->head_dim;
  B200_REQUIRE(ctx, ld_k >= kv_row && ld_v >= kv_row && (!q || (ld_q >= q_heads * cache->head_dim && ld_q_out >= q_heads * cache->head_dim)), "paged_append: a row stride is shorter than the row");
  DeviceGuard guard(ctx);
  B200_REQUIRE(ctx, guard.ok, "paged_append: the context's device cannot be selected");
  RopeArgs r = {};
  r.freqs = freqs; r.k = k; r.v = v; r.k_out = cache->k; r.v_out = cache->v;
  r.ld_k = (long long)ld_k; r.ld_v = (long long)ld_v;
  if (q && q_heads) { r.q = q; r.q_out = q_out; r.ld_q = (long long)ld_q; r.ld_qo = (long long)ld_q_out; r.qh = (int)q_heads; }
  r.tokens = a.rows; r.kvh = a.n_kv; r.hd = a.hd; r.rd = rope ? (int)rope->rotary_dim : 0;
  r.amplitude = rope ? amplitude_of(rope) : 1.0f; r.sign = 1.0f; r.paged = 1;
  a.max_q = a.rows;                       // the append has no use for the bound
  return launch(ctx, r, a, rope && rope->layout == B200_ROPE_HALF, cache->dtype);
}
