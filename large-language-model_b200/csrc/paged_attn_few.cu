// Attention over a paged cache for sequences with few rows (new tokens x query heads of a group <= 32): single tokens and short
// drafts, bf16, head_dim 64 or 128.
//
// Bound by memory: every key and value is read once, for all rows of its KV head.  A CTA has four warps; each streams its own
// 16-key slices of a 64-key tile through its own ring of shared memory with cp.async (16 bytes a lane, rows past the sequence's end
// filled with zeros), so warps never wait for one another inside a run.  The ring runs ahead over the borders between blocks.
// Scores and the product with V use m16n8k16 tensor instructions: the 16 (or 32) rows are the padded group of query rows, P goes
// from accumulators to operand registers without leaving the warp.  Each warp keeps its own running maximum, sum and output; the
// four are joined through shared memory when a block ends.
// 64 sequences of 100 to 11865 positions, 32 query and 8 KV heads of 128: 117.5 us for 666 MB, 5.7 TB/s (86 % of the copy rate; the CUDA-core
// kernel: 4.1 ms).  Most runs end after the 104 us that the memory needs; those that hold many short sequences set the rest.  Four sequences of
// 200 to 700 positions: 11.5 us with the join, a chain of latencies (division of the work, keys, scores, joins).
#include "paged_attn.cuh"
#include <algorithm>
#include <atomic>

namespace {

constexpr int THREADS = 128, WARPS = 4, SLICE = 16, TILE = WARPS * SLICE, STAGES = 3;

__device__ __forceinline__ uint32_t smem_addr(const void *p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void cp_async16(uint32_t dst, const void *src, bool there) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(there ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void cp_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
__device__ __forceinline__ void ldsm4(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldsm4t(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t *>(&h);
}

// MT: 16-row tiles.
template <int HD, int MT>
__global__ void __launch_bounds__(THREADS, 2)
paged_attn_few_kernel(PagedAttnArgs a) {
  if (!a.beside) pdl_wait();
  pdl_launch_dependents();
  constexpr int CH = HD / 8, KS = HD / 16, NT = HD / 8;        // 16-byte chunks of a row, k steps of the scores, n tiles of the output
  constexpr int ROW = HD * 2, HALF = SLICE * ROW, STAGE = 2 * HALF, OST = HD + 4;
  extern __shared__ __align__(128) uint8_t smem[];
  float *sO = (float *)(smem + WARPS * STAGES * STAGE);        // [16][OST]
  __shared__ long long red[33];
  __shared__ paged::Place place;
  __shared__ float sm_m[WARPS][16 * MT], sm_l[WARPS][16 * MT];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t4 = lane & 3, c = blockIdx.x;
  const paged::Run run = paged::line_run<THREADS>(a.b, a.plan, c, a.n_cta, a.min_units, red, &place);
  if (tid == 0) paged_write_head(a, run, place, c);
  if (run.u == run.end) { if (a.beside) pdl_wait(); return; }
  uint8_t *ring = smem + warp * STAGES * STAGE;
  const float sl2 = a.scale * PAGED_LOG2E;

  // ---- loads: this warp's slice of the walk's tile; the page ids of the next tile are fetched one tile ahead
  paged::Walk ld;
  ld.start(a.plan, place, run.end);
  int ld_kt = ld.pl.kt;
  auto fetch_page = [&]() -> int {                             // lane < 16: page of key `lane` of the slice, -1 past the end
    const int pos = ld_kt * TILE + warp * SLICE + (lane & 15);
    return ld.more && pos < ld.pl.q.len ? paged::page_of(a.b, ld.pl.seq, pos) : -1;
  };
  int page = fetch_page();
  auto load = [&](int stage) {
    if (ld.more) {
      const int pos = ld_kt * TILE + warp * SLICE + (lane & 15);
      const long long off = page < 0 ? -1 : (long long)page * a.b.page_stride + (long long)(pos % a.b.page_size) * a.b.token_stride + (long long)ld.pl.kvh * a.b.head_stride;
      const uint32_t dst = smem_addr(ring + stage * STAGE);
#pragma unroll
      for (int i = 0; i < SLICE * CH / 32; ++i) {
        const int r = i * (32 / CH) + lane / CH, ch = lane % CH;
        const long long o = __shfl_sync(0xffffffffu, off, r);
        const uint32_t d = dst + r * ROW + ((ch ^ (r & 7)) << 4);
        const long long e = (o < 0 ? 0 : o) + ch * 8;
        cp_async16(d, (const bf16 *)a.k + e, o >= 0);
        cp_async16(d + HALF, (const bf16 *)a.v + e, o >= 0);
      }
      if (++ld_kt >= ld.k1) {
        ld.next(a.b, a.plan, run.end); ld_kt = 0;
        // the next block's queries come nearer while the ring still holds keys of this one
        if (ld.more && warp == 0 && lane * 64 < a.plan.G * HD)
          asm volatile("prefetch.global.L1 [%0];" ::"l"((const bf16 *)a.q + (size_t)ld.pl.q.q0 * a.ld_q + (size_t)ld.pl.kvh * a.plan.G * HD + lane * 64));
      }
      page = fetch_page();
    }
    cp_commit();
  };
#pragma unroll
  for (int s = 0; s < STAGES - 1; ++s) load(s);

  paged::Walk w;
  int stage = 0;
  for (w.start(a.plan, place, run.end); w.more; w.next(a.b, a.plan, run.end)) {
    // ---- a block: its queries in registers, rows that do not exist as zeros
    const paged::Place &pl = w.pl;
    uint32_t qf[MT][KS][4];
    int limit[MT][2];
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        int row, head, pos;
        const bool has = paged_row(a, pl, m * 16 + g + 8 * h, row, head, pos);
        limit[m][h] = has ? min(max(pos + 1, 0), pl.q.len) : 0;
        const uint32_t *src = (const uint32_t *)((const bf16 *)a.q + (size_t)row * a.ld_q + (size_t)head * HD) + t4;
#pragma unroll
        for (int k = 0; k < KS; ++k) {
          qf[m][k][h] = has ? src[k * 8] : 0u;
          qf[m][k][2 + h] = has ? src[k * 8 + 4] : 0u;
        }
      }
    const int all_see = min(max(pl.q.base + 1, 0), pl.q.len);    // keys that every row sees
    float o[MT][NT][4], mx[MT][2], l[MT][2];
#pragma unroll
    for (int m = 0; m < MT; ++m) {
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) o[m][n][i] = 0.f;
      mx[m][0] = mx[m][1] = -INFINITY; l[m][0] = l[m][1] = 0.f;
    }
    for (int kt = pl.kt; kt < w.k1; ++kt) {
      cp_wait<STAGES - 2>();
      __syncwarp();
      {
        int next = stage + STAGES - 1;
        if (next >= STAGES) next -= STAGES;
        load(next);
      }
      const uint32_t kb = smem_addr(ring + stage * STAGE), vb = kb + HALF;
      if (++stage == STAGES) stage = 0;
      const int key0 = kt * TILE + warp * SLICE;
      float s[MT][2][4];
#pragma unroll
      for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int n = 0; n < 2; ++n)
#pragma unroll
          for (int x = 0; x < 4; ++x) s[m][n][x] = 0.f;
      {
        const int r = (lane & 7) + ((lane >> 4) << 3);
#pragma unroll
        for (int k = 0; k < KS; ++k) {
          uint32_t b[4];
          ldsm4(kb + r * ROW + (((k * 2 + ((lane >> 3) & 1)) ^ (r & 7)) << 4), b);
#pragma unroll
          for (int m = 0; m < MT; ++m) { mma(s[m][0], qf[m][k], b[0], b[1]); mma(s[m][1], qf[m][k], b[2], b[3]); }
        }
      }
      const bool masked = key0 + SLICE > all_see;
      uint32_t pf[MT][4];
#pragma unroll
      for (int m = 0; m < MT; ++m) {
        float up[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          float v[4] = {s[m][0][2 * h], s[m][0][2 * h + 1], s[m][1][2 * h], s[m][1][2 * h + 1]};
          if (masked) {
#pragma unroll
            for (int x = 0; x < 4; ++x) if (key0 + t4 * 2 + (x & 1) + (x >> 1) * 8 >= limit[m][h]) v[x] = -INFINITY;
          }
          float top = fmaxf(fmaxf(v[0], v[1]), fmaxf(v[2], v[3]));
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2)) * sl2;
          const float mn = fmaxf(mx[m][h], top), base = mn == -INFINITY ? 0.f : mn;
          up[h] = ex2(mx[m][h] - base);
          mx[m][h] = mn;
          float p[4];
#pragma unroll
          for (int x = 0; x < 4; ++x) p[x] = ex2(fmaf(v[x], sl2, -base));
          l[m][h] = l[m][h] * up[h] + ((p[0] + p[1]) + (p[2] + p[3]));
          pf[m][h] = pack2(p[0], p[1]); pf[m][2 + h] = pack2(p[2], p[3]);     // probabilities are rounded to bf16 for the tensor product
        }
        if (__any_sync(0xffffffffu, up[0] != 1.0f || up[1] != 1.0f)) {
#pragma unroll
          for (int n = 0; n < NT; ++n) { o[m][n][0] *= up[0]; o[m][n][1] *= up[0]; o[m][n][2] *= up[1]; o[m][n][3] *= up[1]; }
        }
      }
#pragma unroll
      for (int n = 0; n < NT; n += 2) {
        const int r = lane & 15;
        uint32_t b[4];
        ldsm4t(vb + r * ROW + (((n + (lane >> 4)) ^ (r & 7)) << 4), b);
#pragma unroll
        for (int m = 0; m < MT; ++m) { mma(o[m][n], pf[m], b[0], b[1]); mma(o[m][n + 1], pf[m], b[2], b[3]); }
      }
    }
    // ---- the four warps' parts: maxima and sums first, then the outputs one warp after the other (a fixed order)
    const bool whole = w.whole();
    float *slot = whole ? nullptr : paged_slot(a, c, pl.kt == 0);
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        l[m][h] += __shfl_xor_sync(0xffffffffu, l[m][h], 1);
        l[m][h] += __shfl_xor_sync(0xffffffffu, l[m][h], 2);
        if (t4 == 0) { sm_m[warp][m * 16 + g + 8 * h] = mx[m][h]; sm_l[warp][m * 16 + g + 8 * h] = l[m][h]; }
      }
    __syncthreads();
#pragma unroll
    for (int m = 0; m < MT; ++m) {
      float f[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int r = m * 16 + g + 8 * h;
        const float top = fmaxf(fmaxf(sm_m[0][r], sm_m[1][r]), fmaxf(sm_m[2][r], sm_m[3][r]));
        f[h] = top == -INFINITY ? 0.f : ex2(mx[m][h] - top);
      }
      // blocks of up to 8 (4) rows leave room for two (four) warps' parts side by side, and take as many rounds less
      const int n_rows = min(16, pl.q.ql * a.plan.G - m * 16), side = n_rows <= 4 ? 4 : n_rows <= 8 ? 2 : 1, part = 16 / side;
      for (int x = 0; x < WARPS; x += side) {
        if (warp / side == x / side) {
          float *mine = sO + (warp % side) * part * OST;
#pragma unroll
          for (int h = 0; h < 2; ++h)
            if (g + 8 * h < part) {
#pragma unroll
              for (int n = 0; n < NT; ++n) {
                float2 *d = (float2 *)(mine + (g + 8 * h) * OST + n * 8 + t4 * 2);
                float2 y = x ? *d : make_float2(0.f, 0.f);
                y.x = fmaf(o[m][n][2 * h], f[h], y.x); y.y = fmaf(o[m][n][2 * h + 1], f[h], y.y);
                *d = y;
              }
            }
        }
        __syncthreads();
      }
      for (int i = tid; i < n_rows * CH; i += THREADS) {
        const int r = m * 16 + i / CH, d = (i % CH) * 8;
        int row, head, pos;
        if (!paged_row(a, pl, r, row, head, pos)) continue;
        const float top = fmaxf(fmaxf(sm_m[0][r], sm_m[1][r]), fmaxf(sm_m[2][r], sm_m[3][r])), base = top == -INFINITY ? 0.f : top;
        float sum = 0.f;
#pragma unroll
        for (int x = 0; x < WARPS; ++x) sum = fmaf(sm_l[x][r], ex2(sm_m[x][r] - base), sum);
        const float *src = sO + (r & 15) * OST + d;
        float4 y0 = *(const float4 *)src, y1 = *(const float4 *)(src + 4);
        for (int x = 1; x < side; ++x) {
          const float4 z0 = *(const float4 *)(src + x * part * OST), z1 = *(const float4 *)(src + x * part * OST + 4);
          y0.x += z0.x; y0.y += z0.y; y0.z += z0.z; y0.w += z0.w; y1.x += z1.x; y1.y += z1.y; y1.z += z1.z; y1.w += z1.w;
        }
        if (whole) {
          const float inv = sum > 0.f ? 1.0f / sum : 0.f;
          const uint4 out = make_uint4(pack2(y0.x * inv, y0.y * inv), pack2(y0.z * inv, y0.w * inv), pack2(y1.x * inv, y1.y * inv), pack2(y1.z * inv, y1.w * inv));
          *(uint4 *)((bf16 *)a.o + (size_t)row * a.ld_o + (size_t)head * HD + d) = out;
          if (d == 0 && a.lse) a.lse[(size_t)row * a.nH + head] = sum > 0.f ? (top + log2f(sum)) / PAGED_LOG2E : -INFINITY;
        } else {
          *(float4 *)(slot + (size_t)r * HD + d) = y0; *(float4 *)(slot + (size_t)r * HD + d + 4) = y1;
          if (d == 0) { slot[(size_t)a.slot_rows * HD + r] = top; slot[(size_t)a.slot_rows * (HD + 1) + r] = sum; }
        }
      }
      __syncthreads();
    }
  }
  if (a.beside) pdl_wait();
}

template <int HD, int MT>
int launch_t(b200_ctx *ctx, const PagedAttnArgs &a) {
  constexpr int smem = WARPS * STAGES * 2 * SLICE * HD * 2 + 16 * (HD + 4) * 4;
  static std::atomic<unsigned long long> attr{0};
  const unsigned long long bit = 1ull << (ctx->device & 63);
  if (!(attr.load() & bit)) { B200_CUDA(ctx, cudaFuncSetAttribute(paged_attn_few_kernel<HD, MT>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem)); attr.fetch_or(bit); }
  B200_CUDA(ctx, launch_pdl(ctx, paged_attn_few_kernel<HD, MT>, dim3((unsigned)a.n_cta), dim3(THREADS), (size_t)smem, 0, a));
  B200_LAUNCHED(ctx);
  return B200_OK;
}

}  // namespace

// 16-byte rows of queries, outputs and pages.
bool paged_attn_few_supported(const b200_paged_cache *c, const void *q, size_t ld_q, const void *o, size_t ld_o) {
  if (c->dtype != B200_BF16 || (c->head_dim != 64 && c->head_dim != 128)) return false;
  return ((uintptr_t)q | (uintptr_t)o | (uintptr_t)c->k | (uintptr_t)c->v) % 16 == 0 && (ld_q | ld_o | c->page_stride | c->token_stride | c->head_stride) % 8 == 0;
}

int paged_attn_few_launch(b200_ctx *ctx, PagedAttnArgs &a, int G, bool beside) {
  const bool two = (long long)a.b.max_q * G > 16;
  // extra 3: a block's start and end cost three tiles' time (against 123 us then, 2: 125, 1: 143, 4: as 3, at the ragged step above); runs of
  // at least two tiles (against 14.9 us then, 1: 17.9, 4: 18.9, 8: 23.8 for the four short sequences)
  a.plan = paged::Plan{G, 0, two ? 32 : 16, 6, 3, 0, two ? PAGED_FEW_ROWS : 16};
  a.n_cta = 2 * ctx->sm_count; a.min_units = 2; a.slot_rows = two ? 32 : 16; a.vec_out = 1; a.beside = beside ? 1 : 0;
  if (a.b.hd == 128) return two ? launch_t<128, 2>(ctx, a) : launch_t<128, 1>(ctx, a);
  return two ? launch_t<64, 2>(ctx, a) : launch_t<64, 1>(ctx, a);
}
