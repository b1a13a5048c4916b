// Attention of a ragged batch of new tokens over a paged key/value cache: entry point, the CUDA-core kernel that takes
// every type, head size and alignment, and the join of partial results.
//
//   o = sum_j softmax_j(scale q . k_j) v_j over the keys 0 .. p of the row's own sequence, p the row's position;
//   lse = log sum_j exp(scale q . k_j).  Rows that see no key get o = 0 and lse = -inf.
// The single-token and the causal attention of cpp/src/Attention.cpp:236-280, with keys found through a page table.
//
// The CUDA-core kernel: blocks of 32 rows (token, query head of the group) x tiles of 32 keys, one pass with a running
// maximum and sum.  Warp w owns rows w, w + 4, ...; in the scores a lane is a key, in the product with V four dimensions.
// Keys and values pass through shared memory in 32 bits, four vectors of a thread in flight on the way there.  Bound by shared-memory reads (12 per 32
// multiply-adds of a warp with all its rows, fewer instructions with few rows); in small calls by the chain of loads, scores and joins
// (drafts of 14 tokens over seven sequences, 8 query and 2 KV heads of 64 in 32 bits: 22.4 us).
#include "paged_attn.cuh"
#include <algorithm>
#include <atomic>
#include <cmath>

namespace {

constexpr int THREADS = 128, ROWS = 32, TILE = 32, WROWS = ROWS / 4;

// Four elements in 32 bits.
template <class T> __device__ __forceinline__ float4 load4(const T *p);
template <> __device__ __forceinline__ float4 load4<float>(const float *p) { return *reinterpret_cast<const float4 *>(p); }
template <> __device__ __forceinline__ float4 load4<bf16>(const bf16 *p) {
  const uint2 v = *reinterpret_cast<const uint2 *>(p);
  return make_float4(__uint_as_float(v.x << 16), __uint_as_float(v.x & 0xffff0000u), __uint_as_float(v.y << 16), __uint_as_float(v.y & 0xffff0000u));
}
// Copies rows of hd elements at src + off[row] into shared rows `stride` floats apart, zeros where off < 0 and up to the padded size hd4; UNROLL
// vectors of a thread in flight (VEC: rows are four-element aligned), two sources at once.
template <class T, bool VEC, int UNROLL, class A, class B>
__device__ __forceinline__ void copy_rows(const T *src, const T *src2, const long long *off, int rows, int hd, A to, B to2) {
  const int hd4 = (hd + 3) / 4, all = rows * hd4;
  for (int i0 = threadIdx.x; i0 < all; i0 += UNROLL * THREADS) {
    float4 x[UNROLL], y[UNROLL];
#pragma unroll
    for (int j = 0; j < UNROLL; ++j) {
      const int i = i0 + j * THREADS;
      x[j] = y[j] = make_float4(0.f, 0.f, 0.f, 0.f);
      if (i < all) {
        const int r = i / hd4, d = (i - r * hd4) * 4;
        const long long o = off[r];
        if (o >= 0) {
          if constexpr (VEC) { x[j] = load4(src + o + d); if (src2) y[j] = load4(src2 + o + d); }
          else {
            float e[8];
#pragma unroll
            for (int k = 0; k < 4; ++k) { e[k] = d + k < hd ? to_f(src[o + d + k]) : 0.f; e[4 + k] = src2 && d + k < hd ? to_f(src2[o + d + k]) : 0.f; }
            x[j] = make_float4(e[0], e[1], e[2], e[3]); y[j] = make_float4(e[4], e[5], e[6], e[7]);
          }
        }
      }
    }
#pragma unroll
    for (int j = 0; j < UNROLL; ++j) {
      const int i = i0 + j * THREADS;
      if (i < all) { const int r = i / hd4, d = (i - r * hd4) * 4; to(r, d, x[j]); if (src2) to2(r, d, y[j]); }
    }
  }
}

// HJ: 128-dimension slices of the head.
template <class T, int HJ, bool VEC>
__global__ void __launch_bounds__(THREADS)
paged_attn_simt_kernel(PagedAttnArgs a) {
  pdl_wait();
  pdl_launch_dependents();
  extern __shared__ __align__(16) float smem[];
  __shared__ long long red[33];
  __shared__ paged::Place place;
  __shared__ long long off_s[TILE];                    // element offset of a key's row, or of a query's; -1: zeros
  static_assert(TILE >= ROWS, "one table for keys and queries");
  const int hd = a.b.hd, hd4 = (hd + 3) & ~3, kst = hd4 + 4, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  float *sK = smem, *sV = sK + TILE * kst, *sQ = sV + TILE * hd4, *sP = sQ + ROWS * hd4 + warp * WROWS * TILE;
  const int c = blockIdx.x;
  const paged::Run run = paged::line_run<THREADS>(a.b, a.plan, c, a.n_cta, a.min_units, red, &place);
  if (tid == 0) paged_write_head(a, run, place, c);
  if (run.u == run.end) return;
  paged::Walk w;
  const float sl2 = a.scale * PAGED_LOG2E;
  for (w.start(a.plan, place, run.end); w.more; w.next(a.b, a.plan, run.end)) {
    const paged::Place &pl = w.pl;
    // ---- queries of the block, rows that do not exist as zeros
    __syncthreads();
    if (tid < ROWS) {
      int row, head, pos;
      off_s[tid] = paged_row(a, pl, tid, row, head, pos) ? (long long)row * a.ld_q + (long long)head * hd : -1;
    }
    __syncthreads();
    copy_rows<T, VEC, 4>((const T *)a.q, (const T *)nullptr, off_s, ROWS, hd, [&](int r, int d, float4 x) { *reinterpret_cast<float4 *>(sQ + r * hd4 + d) = x; }, [](int, int, float4) {});
    int limit[WROWS], out_row[WROWS], out_head[WROWS], live = 0;      // limit: keys the row sees
    float m[WROWS], l[WROWS];
    float4 acc[WROWS][HJ];
#pragma unroll
    for (int i = 0; i < WROWS; ++i) {
      int pos = 0;
      const bool has = paged_row(a, pl, warp + 4 * i, out_row[i], out_head[i], pos);
      limit[i] = has ? min(max(pos + 1, 0), pl.q.len) : 0;
      if (has) live = i + 1;
      m[i] = -INFINITY; l[i] = 0.f;
#pragma unroll
      for (int j = 0; j < HJ; ++j) acc[i][j] = make_float4(0.f, 0.f, 0.f, 0.f);
    }
    for (int kt = pl.kt; kt < w.k1; ++kt) {
      __syncthreads();
      if (tid < TILE) {                                                // positions never written may hold anything: read as zero
        const int pos = kt * TILE + tid, page = pos < pl.q.len ? paged::page_of(a.b, pl.seq, pos) : -1;
        off_s[tid] = page < 0 ? -1 : (long long)page * a.b.page_stride + (long long)(pos % a.b.page_size) * a.b.token_stride + (long long)pl.kvh * a.b.head_stride;
      }
      __syncthreads();
      copy_rows<T, VEC, 4>((const T *)a.k, (const T *)a.v, off_s, TILE, hd, [&](int r, int d, float4 x) { *reinterpret_cast<float4 *>(sK + r * kst + d) = x; },
                           [&](int r, int d, float4 x) { *reinterpret_cast<float4 *>(sV + r * hd4 + d) = x; });
      __syncthreads();
      if (live == 0) continue;
      float s[WROWS];
#pragma unroll
      for (int i = 0; i < WROWS; ++i) s[i] = 0.f;
      for (int d = 0; d < hd4; d += 4) {
        const float4 k4 = *reinterpret_cast<const float4 *>(sK + lane * kst + d);
#pragma unroll
        for (int i = 0; i < WROWS; ++i)
          if (i < live) {
            const float4 q4 = *reinterpret_cast<const float4 *>(sQ + (warp + 4 * i) * hd4 + d);
            s[i] = fmaf(q4.x, k4.x, fmaf(q4.y, k4.y, fmaf(q4.z, k4.z, fmaf(q4.w, k4.w, s[i]))));
          }
      }
      const int key = kt * TILE + lane;
#pragma unroll
      for (int i = 0; i < WROWS; ++i)
        if (i < live) {
          const float x = key < limit[i] ? s[i] * sl2 : -INFINITY, mn = fmaxf(m[i], warp_max(x));
          const float base = mn == -INFINITY ? 0.f : mn, f = exp2f(m[i] - base), p = exp2f(x - base);
          m[i] = mn;
          l[i] = l[i] * f + warp_sum(p);
#pragma unroll
          for (int j = 0; j < HJ; ++j) { acc[i][j].x *= f; acc[i][j].y *= f; acc[i][j].z *= f; acc[i][j].w *= f; }
          sP[i * TILE + lane] = p;
        }
      __syncwarp();
#pragma unroll 2
      for (int k = 0; k < TILE; k += 4) {
        float4 p4[WROWS];
#pragma unroll
        for (int i = 0; i < WROWS; ++i) p4[i] = i < live ? *reinterpret_cast<const float4 *>(sP + i * TILE + k) : make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int j = 0; j < HJ; ++j) {
          const int d = lane * 4 + 128 * j;
          if (d < hd4) {
#pragma unroll
            for (int kk = 0; kk < 4; ++kk) {
              const float4 v4 = *reinterpret_cast<const float4 *>(sV + (k + kk) * hd4 + d);
#pragma unroll
              for (int i = 0; i < WROWS; ++i)
                if (i < live) {
                  const float p = kk == 0 ? p4[i].x : kk == 1 ? p4[i].y : kk == 2 ? p4[i].z : p4[i].w;
                  acc[i][j].x = fmaf(p, v4.x, acc[i][j].x); acc[i][j].y = fmaf(p, v4.y, acc[i][j].y);
                  acc[i][j].z = fmaf(p, v4.z, acc[i][j].z); acc[i][j].w = fmaf(p, v4.w, acc[i][j].w);
                }
            }
          }
        }
      }
      __syncwarp();
    }
    // ---- the whole block: its rows; a part of it: a partial result
    const bool whole = w.whole();
    float *slot = whole ? nullptr : paged_slot(a, c, pl.kt == 0);
#pragma unroll
    for (int i = 0; i < WROWS; ++i)
      if (i < live) {
        const int r = warp + 4 * i;
        const float inv = whole ? (l[i] > 0.f ? 1.0f / l[i] : 0.f) : 1.0f;
#pragma unroll
        for (int j = 0; j < HJ; ++j) {
          const float e[4] = {acc[i][j].x * inv, acc[i][j].y * inv, acc[i][j].z * inv, acc[i][j].w * inv};
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            const int d = lane * 4 + 128 * j + x;
            if (d < hd) {
              if (whole) ((T *)a.o)[(size_t)out_row[i] * a.ld_o + (size_t)out_head[i] * hd + d] = from_f<T>(e[x]);
              else slot[(size_t)r * hd + d] = e[x];
            }
          }
        }
        if (lane == 0) {
          if (!whole) { slot[(size_t)a.slot_rows * hd + r] = m[i]; slot[(size_t)a.slot_rows * (hd + 1) + r] = l[i]; }
          else if (a.lse) a.lse[(size_t)out_row[i] * a.nH + out_head[i]] = l[i] > 0.f ? (m[i] + log2f(l[i])) / PAGED_LOG2E : -INFINITY;
        }
      }
  }
}

// ---- join: one CTA column per border between runs; it works when the border is the first one inside its block ------------
// A thread owns D dimensions of a row (eight where the head and the alignment allow: the maxima and weights of a row's parts are then looked at half as
// often; with four this kernel was bound by instructions, 23 us of a 127 us mixed batch) and adds its parts in CTA order, two parts in flight at
// once.  With more than eight parts the CTA's eight warps share them out and add their sums.
constexpr int JOIN_THREADS = 256, JOIN_WARPS = JOIN_THREADS / 32;
template <class T, int D>
__global__ void __launch_bounds__(JOIN_THREADS)
paged_join_kernel(PagedAttnArgs a, PagedAttnArgs a2) {
  pdl_wait();
  pdl_launch_dependents();
  int c = blockIdx.x + 1;
  const bool second = c >= a.n_cta;                    // the second kernel's borders follow the first's
  const PagedAttnArgs &p = second ? a2 : a;
  if (second) c -= a.n_cta - 1;
  __shared__ float sh_m[JOIN_WARPS][32], sh_l[JOIN_WARPS][32], sh_e[JOIN_WARPS][D][32];
  const int hd = p.b.hd, tid = threadIdx.x;
  const JoinHead *head_ = paged_head(p, c);
  const int parts = head_->parts;
  if (parts == 0) return;
  const paged::Place pl = head_->pl;
  const float *part0 = paged_slot(p, c - 1, true), *part1 = paged_slot(p, c, false);
  const size_t step = 2 * paged_slot_floats(p.slot_rows, hd);
  const int vecs = (hd + D - 1) / D, items = p.slot_rows * vecs, groups = parts > 8 ? JOIN_WARPS : 1, width = JOIN_THREADS / groups;
  const int group = groups > 1 ? tid >> 5 : 0, k0 = parts * group / groups, k1 = parts * (group + 1) / groups;
  for (int i0 = blockIdx.y * width; i0 < items; i0 += gridDim.y * width) {
    const int i = i0 + (tid & (width - 1)), r = i / vecs, d = (i - r * vecs) * D;
    const size_t at = (size_t)r * hd + d;
    int row = 0, head = 0, pos = 0;
    const bool has = i < items && paged_row(p, pl, r, row, head, pos);
    float mx = -INFINITY, l = 0.f, e[D];
#pragma unroll
    for (int x = 0; x < D; ++x) e[x] = 0.f;
    if (has) {
      const size_t at_m = (size_t)p.slot_rows * hd + r, at_l = at_m + p.slot_rows;
      for (int k = k0; k < k1; k += 2) {
        float m2[2], l2[2], e2[2][D];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const float *q = k + j == 0 ? part0 : part1 + (size_t)(k + j - 1) * step;
          m2[j] = -INFINITY; l2[j] = 0.f;
#pragma unroll
          for (int x = 0; x < D; ++x) e2[j][x] = 0.f;
          if (k + j < k1) {
            m2[j] = q[at_m]; l2[j] = q[at_l];
            if constexpr (D == 8) {
              const float4 u = *reinterpret_cast<const float4 *>(q + at), v = *reinterpret_cast<const float4 *>(q + at + 4);
              e2[j][0] = u.x; e2[j][1] = u.y; e2[j][2] = u.z; e2[j][3] = u.w; e2[j][4] = v.x; e2[j][5] = v.y; e2[j][6] = v.z; e2[j][7] = v.w;
            } else {
#pragma unroll
              for (int x = 0; x < D; ++x) if (d + x < hd) e2[j][x] = q[at + x];
            }
          }
        }
        const float top = fmaxf(mx, fmaxf(m2[0], m2[1])), base = top == -INFINITY ? 0.f : top, f = exp2f(mx - base);
        mx = top;
        l *= f;
#pragma unroll
        for (int x = 0; x < D; ++x) e[x] *= f;
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const float wt = exp2f(m2[j] - base);
          if (wt > 0.f) {                                    // a part that saw no key holds anything
            l = fmaf(wt, l2[j], l);
#pragma unroll
            for (int x = 0; x < D; ++x) e[x] = fmaf(wt, e2[j][x], e[x]);
          }
        }
      }
    }
    if (groups > 1) {
      const int lane = tid & 31;
      __syncthreads();
      sh_m[group][lane] = mx; sh_l[group][lane] = l;
#pragma unroll
      for (int x = 0; x < D; ++x) sh_e[group][x][lane] = e[x];
      __syncthreads();
      if (group == 0) {
        for (int k = 0; k < JOIN_WARPS; ++k) mx = fmaxf(mx, sh_m[k][lane]);
        const float base = mx == -INFINITY ? 0.f : mx;
        l = 0.f;
#pragma unroll
        for (int x = 0; x < D; ++x) e[x] = 0.f;
        for (int k = 0; k < JOIN_WARPS; ++k) {
          const float wt = exp2f(sh_m[k][lane] - base);
          l = fmaf(wt, sh_l[k][lane], l);
#pragma unroll
          for (int x = 0; x < D; ++x) e[x] = fmaf(wt, sh_e[k][x][lane], e[x]);
        }
      }
    }
    if (has && group == 0) {
      const float inv = l > 0.f ? 1.0f / l : 0.f;
      T *dst = (T *)p.o + (size_t)row * p.ld_o + (size_t)head * hd + d;
      if constexpr (D == 8 && sizeof(T) == 2) {
        uint32_t w[4];
#pragma unroll
        for (int x = 0; x < 4; ++x) { const __nv_bfloat162 h = __floats2bfloat162_rn(e[2 * x] * inv, e[2 * x + 1] * inv); w[x] = *reinterpret_cast<const uint32_t *>(&h); }
        *reinterpret_cast<uint4 *>(dst) = make_uint4(w[0], w[1], w[2], w[3]);
      } else {
#pragma unroll
        for (int x = 0; x < D; ++x) if (d + x < hd) dst[x] = from_f<T>(e[x] * inv);
      }
      if (p.lse && d == 0) p.lse[(size_t)row * p.nH + head] = l > 0.f ? (mx + log2f(l)) / PAGED_LOG2E : -INFINITY;
    }
  }
}

template <class T, int HJ, bool VEC>
int simt_launch_t(b200_ctx *ctx, const PagedAttnArgs &a) {
  const int hd4 = (a.b.hd + 3) & ~3;
  const size_t smem = sizeof(float) * (size_t)(TILE * (hd4 + 4) + TILE * hd4 + ROWS * hd4 + ROWS * TILE);
  static std::atomic<unsigned long long> attr{0};
  const unsigned long long bit = 1ull << (ctx->device & 63);
  if (!(attr.load() & bit)) { B200_CUDA(ctx, cudaFuncSetAttribute(paged_attn_simt_kernel<T, HJ, VEC>, cudaFuncAttributeMaxDynamicSharedMemorySize, 112 * 1024)); attr.fetch_or(bit); }
  B200_CUDA(ctx, launch_pdl(ctx, paged_attn_simt_kernel<T, HJ, VEC>, dim3((unsigned)a.n_cta), dim3(THREADS), smem, 0, a));
  B200_LAUNCHED(ctx);
  return B200_OK;
}
template <class T>
int simt_launch(b200_ctx *ctx, const PagedAttnArgs &a) {
  const bool vec = ((uintptr_t)a.k | (uintptr_t)a.v | (uintptr_t)a.q) % (4 * sizeof(T)) == 0 && (a.b.page_stride | a.b.token_stride | a.b.head_stride | a.ld_q | a.b.hd) % 4 == 0;
  if (a.b.hd > 128) return vec ? simt_launch_t<T, 2, true>(ctx, a) : simt_launch_t<T, 2, false>(ctx, a);
  return vec ? simt_launch_t<T, 1, true>(ctx, a) : simt_launch_t<T, 1, false>(ctx, a);
}

constexpr int MIN_UNITS = 1;

}  // namespace

int paged_join_launch(b200_ctx *ctx, const PagedAttnArgs &a, const PagedAttnArgs *b, b200_dtype dt) {
  const int borders = a.n_cta - 1 + (b ? b->n_cta - 1 : 0), rows = std::max(a.slot_rows, b ? b->slot_rows : 0);
  if (borders < 1) return B200_OK;
  const bool eight = a.vec_out && a.b.hd % 8 == 0;      // both kernels of a call have the same head and alignment
  const dim3 grid((unsigned)borders, (unsigned)std::min(16, (rows * (a.b.hd / (eight ? 8 : 4) + (eight ? 0 : 1)) + JOIN_THREADS - 1) / JOIN_THREADS));
  if (dt == B200_F32) B200_CUDA(ctx, launch_pdl(ctx, paged_join_kernel<float, 4>, grid, dim3(JOIN_THREADS), 0, 0, a, b ? *b : a));
  else if (eight) B200_CUDA(ctx, launch_pdl(ctx, paged_join_kernel<bf16, 8>, grid, dim3(JOIN_THREADS), 0, 0, a, b ? *b : a));
  else B200_CUDA(ctx, launch_pdl(ctx, paged_join_kernel<bf16, 4>, grid, dim3(JOIN_THREADS), 0, 0, a, b ? *b : a));
  B200_LAUNCHED(ctx);
  return B200_OK;
}

// Each kernel leaves two partial results per CTA; two kernels of one call may run side by side, so each has its own room.
static size_t partial_bytes(const b200_ctx *ctx, int ctas_per_sm, int slot_rows, size_t hd) {
  return (size_t)ctas_per_sm * ctx->sm_count * (JOIN_HEAD_FLOATS + 2 * paged_slot_floats(slot_rows, (int)hd)) * sizeof(float);
}

extern "C" int b200_paged_attn_workspace(b200_ctx *ctx, const b200_paged_cache *cache, const b200_paged_batch *batch, size_t n_heads, size_t *bytes) {
  if (!ctx) return B200_ERR_INVALID;
  PagedArgs a;
  int rc = paged_args(ctx, cache, batch, &a);
  if (rc) return rc;
  B200_REQUIRE(ctx, bytes, "paged_attn_workspace: null pointer");
  B200_REQUIRE(ctx, n_heads > 0 && n_heads <= 65536 && n_heads % cache->n_kv == 0, "paged_attn: n_heads must be a multiple of the cache's n_kv");
  const size_t hd = cache->head_dim;
  *bytes = partial_bytes(ctx, 2, ROWS, hd) + (cache->dtype == B200_BF16 && hd <= 128 ? partial_bytes(ctx, 1, 256, hd) : 0);
  return B200_OK;
}

extern "C" int b200_paged_attn(b200_ctx *ctx, const b200_paged_cache *cache, const b200_paged_batch *batch, const void *q, size_t ld_q, void *o,
                               size_t ld_o, float *lse, size_t n_heads, float scale, void *workspace, size_t workspace_bytes) {
  if (!ctx) return B200_ERR_INVALID;
  PagedAttnArgs a;
  size_t need = 0;
  int rc = paged_args(ctx, cache, batch, &a.b);
  if (!rc) rc = b200_paged_attn_workspace(ctx, cache, batch, n_heads, &need);
  if (rc) return rc;
  if (cache->head_dim > 256) return b200_fail(ctx, B200_ERR_UNSUPPORTED, "paged_attn: head_dim above 256 has no kernel");
  B200_REQUIRE(ctx, std::isfinite(scale) && scale >= 0.f, "paged_attn: scale must be finite and not negative (0: 1 / sqrt(head_dim))");
  if (batch->n_seq == 0 || batch->rows == 0) return B200_OK;
  B200_REQUIRE(ctx, q && o, "paged_attn: null pointer");
  B200_REQUIRE(ctx, ld_q >= n_heads * cache->head_dim && ld_o >= n_heads * cache->head_dim, "paged_attn: a row stride is shorter than the row");
  B200_REQUIRE(ctx, workspace && workspace_bytes >= need && (uintptr_t)workspace % 16 == 0, "paged_attn: the workspace is smaller than b200_paged_attn_workspace says, or not 16-byte aligned");
  DeviceGuard guard(ctx);
  B200_REQUIRE(ctx, guard.ok, "paged_attn: the context's device cannot be selected");
  a.k = cache->k; a.v = cache->v; a.q = q; a.o = o; a.lse = lse; a.ws = (float *)workspace;
  a.ld_q = (long long)ld_q; a.ld_o = (long long)ld_o; a.nH = (int)n_heads;
  a.scale = scale > 0.f ? scale : 1.0f / sqrtf((float)cache->head_dim);
  const int G = (int)(n_heads / cache->n_kv);
  const bool fast = paged_attn_few_supported(cache, q, ld_q, o, ld_o), tc = fast && paged_attn_tc_supported(cache, n_heads, q, ld_q, o, ld_o);
  // Sequences of up to PAGED_FEW_ROWS rows are the few-row kernel's, the others the chunk kernel's (tcgen05, else CUDA cores).  A lone sequence or
  // two with many rows are not worth a launch that will find nothing (each kernel is right for any row count).
  const long long most = (long long)a.b.max_q * G;
  const bool few = fast && (most <= PAGED_FEW_ROWS || a.b.n_seq > 2), many = !fast || most > PAGED_FEW_ROWS;
  PagedAttnArgs f = a;
  if (many) {
    if (tc) rc = paged_attn_tc_launch(ctx, a, G, few ? PAGED_FEW_ROWS + 1 : 0);
    else {
      a.vec_out = fast; a.beside = 0;                   // (`fast` implies aligned output rows)
      a.plan = paged::Plan{G, 0, ROWS, 5, 1, few ? PAGED_FEW_ROWS + 1 : 0, 0x7fffffff};
      a.n_cta = 2 * ctx->sm_count; a.min_units = MIN_UNITS; a.slot_rows = ROWS;
      rc = cache->dtype == B200_BF16 ? simt_launch<bf16>(ctx, a) : simt_launch<float>(ctx, a);
    }
    if (rc) return rc;
    if (!few) return paged_join_launch(ctx, a, nullptr, cache->dtype);
    f.ws = a.ws + (size_t)a.n_cta * (JOIN_HEAD_FLOATS + 2 * paged_slot_floats(a.slot_rows, a.b.hd));
  }
  rc = paged_attn_few_launch(ctx, f, G, many);
  if (rc) return rc;
  return many ? paged_join_launch(ctx, a, &f, cache->dtype) : paged_join_launch(ctx, f, nullptr, cache->dtype);
}

// Test hooks, on the host, over host arrays: what the kernels' own index code reaches.
// out = {largest row + 1, largest slot + 1, smallest row, smallest slot, status}; slots count page * page_size + offset.
extern "C" int b200_internal_paged_probe(const b200_paged_cache *cache, const b200_paged_batch *batch, long long *out) {
  int status = 0;
  b200_ctx ctx;
  PagedArgs a;
  if (int rc = paged_args(&ctx, cache, batch, &a)) return rc;
  a.status = &status;
  for (int i = 0; i < 4; ++i) out[i] = 0;
  for (int s = 0; s < a.n_seq; ++s) {
    const paged::Seq q = paged::load_seq(a, s);
    if (q.ql > 0) { out[0] = std::max(out[0], (long long)q.q0 + q.ql); out[2] = std::min(out[2], (long long)q.q0); }
    for (int pos = 0; pos < q.len; ++pos) {
      const int page = paged::page_of(a, s, pos);
      if (page < 0) continue;
      const long long slot = (long long)page * a.page_size + pos % a.page_size;
      out[1] = std::max(out[1], slot + 1); out[3] = std::min(out[3], slot);
    }
  }
  out[4] = status;
  return B200_OK;
}
// Steps through the runs of all CTAs; writes (CTA, sequence, KV head, block, tile, whole block, parts to join at the CTA's border) per tile, returns how many.
extern "C" long long b200_internal_paged_cover(const b200_paged_cache *cache, const b200_paged_batch *batch, int G, int tokens, int rows, int tile_log2, int extra,
                                               int lo, int hi, int n_cta, int min_units, int *out, long long room) {
  int status = 0;
  b200_ctx ctx;
  PagedArgs a;
  if (paged_args(&ctx, cache, batch, &a)) return -1;
  a.status = &status;
  const paged::Plan p{G, tokens, rows, tile_log2, extra, lo, hi};
  long long total = 0, n_out = 0;
  for (int s = 0; s < a.n_seq; ++s) total += paged::seq_units(a, p, s);
  if (total == 0) return 0;
  const int n = paged::line_ctas(total, n_cta, min_units);
  for (int c = 0; c < n; ++c) {
    const paged::Run run{paged::line_at(total, n, c), paged::line_at(total, n, c + 1), total, n};
    if (run.u == run.end) continue;
    long long at = 0;
    int s = 0;
    while (true) { const long long m = paged::seq_units(a, p, s); if (run.u < at + m) break; at += m; ++s; }
    paged::Walk w;
    w.start(p, paged::place_in(a, p, s, paged::seq_units(a, p, s), at, run.u), run.end);
    const int parts = paged::parts_at(p, run, w.pl, c);
    for (; w.more; w.next(a, p, run.end))
      for (int t = w.pl.kt; t < w.k1; ++t, ++n_out)
        if (n_out < room) { const int v[7] = {c, w.pl.seq, w.pl.kvh, w.pl.block, t, w.whole(), parts}; std::copy(v, v + 7, out + 7 * n_out); }
  }
  return n_out;
}
