// Attention over a paged cache for sequences with many rows (chunks of a prompt), bf16, head_dim 64 or 128, tcgen05.
//
// Bound by the tensor cores and the exponentials.  The organisation of the framework's dense forward kernel (attention_fwd2_tc.cu:
// two 128-row tiles per CTA that alternate on the tensor pipe, probabilities written back over the scores in tensor memory, the
// output accumulated there and rescaled only when a row's maximum grew by more than 2^8), with three differences:
//   * a tile's rows are (token, query head of the group), token by token: all heads that share keys are in one tile, so a chunk of 64
//     tokens already fills both tiles at four heads a group, and each key tile is loaded once for the group.  Queries come as boxes
//     [tokens][group][64] of a three-dimensional tensor map;
//   * a key tile is gathered from pages: one box of gcd(page_size, 128) positions per lane of the load warp, page ids looked up a tile
//     ahead.  Rows behind the sequence's end are boxes out of bounds (zeros) or, inside the last page, whatever was there: scores are
//     masked, and one warp overwrites those value rows with zeros before the product (0 x NaN is NaN);
//   * the grid is one CTA per SM, and each walks its equal run of (sequence, KV head, block, key tile): a run that cuts a block leaves a
//     partial result for the join.
// A block with rows for one tile only leaves the other idle; giving both alternate key tiles of the same rows was no faster (two buffers
// of keys and of values then hold no tile ahead: 3.2 thousand cycles a key tile against 4.2, and 6 thousand more to join the two; mixed batch 150 us
// against 127 then, 119 now).
// 1024 tokens over 30011 positions, 32 query and 8 KV heads of 128: 490 us by itself (1.01 PFLOP/s), 600 us in a loop of its own at the power limit
// (0.82 PFLOP/s, half the matrix rate).  A key tile takes 2.3 to 2.5 us for 256 rows in long runs; a block's start and end about 5 us (a CTA's
// first 7), which is what bounds batches of short chunks.  Asking the L2 cache for tiles two ahead made it slower (mixed batch 149 -> 190 us, before the last two steps): the boxes of
// small pages already fill the copy engine's issue rate.
// Tensor memory: [S_A 128 | O_A 128 | S_B 128 | O_B 128] columns.  Warps 0-3 softmax of tile A, 4-7 of tile B, 8 MMA issue, 9 loads, 10 value rows.
#include "attention_tc.cuh"
#include "paged_attn.cuh"
#include <algorithm>
#include <atomic>

using namespace attn;

namespace {

constexpr int TC_THREADS = 384, TC_WARPS = TC_THREADS / 32, FIX_WARP = 10;
struct alignas(16) TcShared {
  uint64_t q_full, q_empty, k_full[2], k_empty[2], v_full[2], v_empty[2], fix_ask[2], fix_done[2], s_full[2], p_full[2], o_full[2];
  uint32_t tmem_base;
  int abort_flag;
  long long red[33];
  paged::Place place;
  paged::Walk walk[TC_WARPS];      // each warp's own, to save registers (with 208 for the softmax warps and the walk in them, spills in the tile loop cost 20 %)
};

constexpr float RESCALE_THRESHOLD = 8.0f;      // log2 units: P stays below 2^8
constexpr int REGS_SOFTMAX = 216, REGS_SERVICE = 72;      // 8 x 32 x 216 + 4 x 32 x 72 = 384 x 168, the launch's share
template <int N> __device__ __forceinline__ void setmaxnreg_inc() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N)); }
template <int N> __device__ __forceinline__ void setmaxnreg_dec() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N)); }
__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

// What a CTA does of one block: key tiles [k0, k1); row tile X takes part in those below n[X] (0: it has no rows).
struct Segment {
  int k0, k1, n[2];
  __device__ __forceinline__ Segment(const PagedAttnArgs &a, const paged::Walk &w) {
    const int half = a.plan.tokens_per_block / 2, t0 = w.pl.block * a.plan.tokens_per_block;
    k0 = w.pl.kt; k1 = w.k1;
#pragma unroll
    for (int X = 0; X < 2; ++X) {
      const int first = t0 + X * half, last = min(w.pl.q.ql, first + half);          // tokens [first, last)
      n[X] = first < w.pl.q.ql ? max(1, (min(max(w.pl.q.base + last, 0), w.pl.q.len) + TK - 1) / TK) : 0;
    }
  }
  __device__ __forceinline__ int end(int X) const { return max(k0, min(k1, n[X])); }
  __device__ __forceinline__ bool last_reader(int X) const { return X == 1 || n[1] == 0; }      // B, where it has rows, sees every tile that A sees
  // the value tile with rows behind the sequence's end, or -1
  __device__ __forceinline__ int ragged(const paged::Place &pl) const {
    const int j = pl.q.len / TK;
    return pl.q.len % TK != 0 && j >= k0 && j < k1 ? j : -1;
  }
};

template <int HD>
__global__ void __launch_bounds__(TC_THREADS, 1)
paged_attn_tc_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
                     PagedAttnArgs a, int box_rows) {
  constexpr int TILE_BYTES = 128 * HD * 2;
  extern __shared__ __align__(1024) uint8_t smem[];
  uint8_t *sQ = smem, *sK = sQ + 2 * TILE_BYTES, *sV = sK + 2 * TILE_BYTES;
  TcShared *sh = (TcShared *)(sV + 2 * TILE_BYTES);
  uint8_t *stage = (uint8_t *)(sh + 1);          // 8 softmax warps x 2 KiB: transposition buffers of the output stores
  int *status = a.b.status;
  if (tc::smem_u32(smem) & 1023u) {              // swizzled tiles need 1024-byte alignment: refuse rather than corrupt
    if (threadIdx.x == 0) atomicCAS(status, 0, 298);
    return;
  }
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  volatile int *abort_flag = &sh->abort_flag;
  pdl_wait();
  pdl_launch_dependents();                       // behind the wait: a few-row kernel that follows does not wait for this one
  const paged::Run run = paged::line_run<TC_THREADS>(a.b, a.plan, blockIdx.x, a.n_cta, a.min_units, sh->red, &sh->place);
  if (threadIdx.x == 0) paged_write_head(a, run, sh->place, blockIdx.x);
  if (run.u == run.end) return;
  if (threadIdx.x == 0) {
    tc::mbar_init(&sh->q_full, 1); tc::mbar_init(&sh->q_empty, 1);
    for (int i = 0; i < 2; ++i) {
      tc::mbar_init(&sh->k_full[i], 1); tc::mbar_init(&sh->k_empty[i], 1);
      tc::mbar_init(&sh->v_full[i], 1); tc::mbar_init(&sh->v_empty[i], 1);
      tc::mbar_init(&sh->fix_ask[i], 1); tc::mbar_init(&sh->fix_done[i], 1);
      tc::mbar_init(&sh->s_full[i], 1); tc::mbar_init(&sh->p_full[i], 4); tc::mbar_init(&sh->o_full[i], 1);
    }
    sh->abort_flag = 0;
    tc::fence_barrier_init();
    tc::fence_proxy_async();
  }
  if (warp == MMA_WARP) tc::tmem_alloc(&sh->tmem_base, 512);
  tc::tc_fence_before();
  __syncthreads();
  tc::tc_fence_after();
  const uint32_t tmem_base = sh->tmem_base;
  const long long end = run.end;
  paged::Walk &w = sh->walk[warp];
  if (lane == 0) w.start(a.plan, sh->place, end);
  __syncwarp();
  const paged::Place &pl = w.pl;
  auto next = [&] { __syncwarp(); if (lane == 0) w.next(a.b, a.plan, end); __syncwarp(); };
  int seg = 0;                                   // segments so far
  bool ok = true;

  if (warp >= 8) {
    setmaxnreg_dec<REGS_SERVICE>();
    if (warp == TMA_WARP) {
      const int half = a.plan.tokens_per_block / 2, boxes = TK / box_rows;
      const uint32_t q_bytes = (uint32_t)(half * a.plan.G * HD * 2);
      int it = 0;                                // key tiles so far
      for (; w.more && ok; ++seg) {
        const Segment g(a, w);
        if (lane == 0 && seg > 0) ok = tc::mbar_wait(&sh->q_empty, (seg - 1) & 1, status, abort_flag, 261);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        if (lane == 0) {
          const int row0 = pl.q.q0 + pl.block * a.plan.tokens_per_block;
          tc::mbar_expect_tx(&sh->q_full, g.n[1] ? 2 * q_bytes : q_bytes);
#pragma unroll
          for (int c = 0; c < HD / 64; ++c) {
            tc::tma_load_3d(sQ + c * 16384, &map_q, c * 64, pl.kvh * a.plan.G, row0, &sh->q_full);
            if (g.n[1]) tc::tma_load_3d(sQ + TILE_BYTES + c * 16384, &map_q, c * 64, pl.kvh * a.plan.G, row0 + half, &sh->q_full);
          }
        }
        // box of lane i: positions kt * 128 + i * box_rows .. of one page; a page id out of bounds reads as zeros
        auto box_page = [&](int j) -> int {
          const int pos = j * TK + lane * box_rows;
          const int id = lane < boxes && j < g.k1 && pos < pl.q.len ? paged::page_of(a.b, pl.seq, pos) : -1;
          return id < 0 ? a.b.n_pages : id;
        };
        const int ragged = g.ragged(pl);
        int page = box_page(g.k0);
        for (int j = g.k0; j < g.k1; ++j, ++it) {
          const int s = it & 1, at = (j * TK + lane * box_rows) % a.b.page_size;
          const uint32_t ph = (uint32_t)(it >> 1) & 1;
          const int next = box_page(j + 1);
          if (lane == 0) {
            ok = tc::mbar_wait(&sh->k_empty[s], ph ^ 1, status, abort_flag, 262);
            if (ok) tc::mbar_expect_tx(&sh->k_full[s], TILE_BYTES);
          }
          ok = __all_sync(0xffffffffu, ok);
          if (!ok) break;
          if (lane < boxes) {
#pragma unroll
            for (int c = 0; c < HD / 64; ++c) tma_load_4d(sK + s * TILE_BYTES + c * 16384 + lane * box_rows * 128, &map_k, c * 64, at, pl.kvh, page, &sh->k_full[s]);
          }
          if (lane == 0) {
            ok = tc::mbar_wait(&sh->v_empty[s], ph ^ 1, status, abort_flag, 263);
            if (ok) tc::mbar_expect_tx(&sh->v_full[s], TILE_BYTES);
          }
          ok = __all_sync(0xffffffffu, ok);
          if (!ok) break;
          if (lane < boxes) {
#pragma unroll
            for (int c = 0; c < HD / 64; ++c) tma_load_4d(sV + s * TILE_BYTES + c * 16384 + lane * box_rows * 128, &map_v, c * 64, at, pl.kvh, page, &sh->v_full[s]);
          }
          if (lane == 0 && j == ragged) tc::mbar_arrive(&sh->fix_ask[s]);
          page = next;
        }
        next();
      }
      if (*abort_flag) { long long t0 = clock64(); while (clock64() - t0 < 2000000ll) {} }      // copies in flight land before the CTA ends
    } else if (warp == MMA_WARP) {
      if (lane == 0) {
        constexpr uint32_t idesc_s = tc::make_idesc_bf16(128, 128, false, false);
        constexpr uint32_t idesc_o = tc::make_idesc_bf16(128, HD, false, true);
        const uint32_t q_addr[2] = {tc::smem_u32(sQ), tc::smem_u32(sQ + TILE_BYTES)};
        int it = 0, fixes[2] = {0, 0}, done[2] = {0, 0};  // done[X]: products with V issued for row tile X; fixes: per buffer
        for (; w.more && ok; ++seg) {
          const Segment g(a, w);
          const int e[2] = {g.end(0), g.end(1)}, ragged = g.ragged(pl);
          bool fixed = false;
          ok = tc::mbar_wait(&sh->q_full, seg & 1, status, abort_flag, 264);
          tc::tc_fence_after();
          auto issue_s = [&](int X, int j) -> bool {
            const int i = it + j - g.k0, s = i & 1;
            if (!tc::mbar_wait(&sh->k_full[s], (uint32_t)(i >> 1) & 1, status, abort_flag, 265)) return false;
            tc::tc_fence_after();
            const uint32_t k_addr = tc::smem_u32(sK + s * TILE_BYTES);
#pragma unroll
            for (int k = 0; k < HD / 16; ++k)
              tc::umma_ss(tmem_base + X * 256, desc_kmajor(q_addr[X], k), desc_kmajor(k_addr, k), idesc_s, k ? 1u : 0u);
            tc::umma_commit(&sh->s_full[X]);
            if (g.last_reader(X)) {
              tc::umma_commit(&sh->k_empty[s]);
              if (j == g.k1 - 1) tc::umma_commit(&sh->q_empty);
            }
            return true;
          };
          auto issue_pv = [&](int X, int j) -> bool {
            const int i = it + j - g.k0, s = i & 1;
            if (!tc::mbar_wait(&sh->p_full[X], (uint32_t)done[X] & 1, status, abort_flag, 266)) return false;
            if (!tc::mbar_wait(&sh->v_full[s], (uint32_t)(i >> 1) & 1, status, abort_flag, 267)) return false;
            if (j == ragged && !fixed) {
              if (!tc::mbar_wait(&sh->fix_done[s], (uint32_t)fixes[s] & 1, status, abort_flag, 268)) return false;
              ++fixes[s]; fixed = true;
            }
            tc::tc_fence_after();
            const uint32_t v_addr = tc::smem_u32(sV + s * TILE_BYTES);
#pragma unroll
            for (int k = 0; k < TK / 16; ++k)
              tc::umma_ts(tmem_base + X * 256 + 128, tmem_base + X * 256 + k * 8, desc_mnmajor(v_addr, k), idesc_o, (j > g.k0 || k > 0) ? 1u : 0u);
            tc::umma_commit(&sh->o_full[X]);
            if (g.last_reader(X)) tc::umma_commit(&sh->v_empty[s]);
            ++done[X];
            return true;
          };
          if (ok && g.k0 < e[0]) ok = issue_s(0, g.k0);
          if (ok && g.k0 < e[1]) ok = issue_s(1, g.k0);
          for (int j = g.k0; j < g.k1 && ok; ++j) {
            if (j < e[0]) { ok = issue_pv(0, j); if (ok && j + 1 < e[0]) ok = issue_s(0, j + 1); }
            if (ok && j < e[1]) { ok = issue_pv(1, j); if (ok && j + 1 < e[1]) ok = issue_s(1, j + 1); }
          }
          it += g.k1 - g.k0;
          w.next(a.b, a.plan, end);
        }
      }
    } else if (warp == FIX_WARP) {
      // The load warp asks, per buffer, once the tile's copy is under way: a buffer is not loaded again before its repair was used, so
      // neither side of these barriers, nor the full barrier waited for here, can be more than one phase away.
      int it = 0, fixes[2] = {0, 0};
      while (w.more && ok) {
        const Segment g(a, w);
        const int j = g.ragged(pl);
        if (j >= 0) {
          const int i = it + j - g.k0, s = i & 1;
          ok = __all_sync(0xffffffffu, tc::mbar_wait(&sh->fix_ask[s], (uint32_t)fixes[s] & 1, status, abort_flag, 273));
          if (!ok) break;
          ++fixes[s];
          ok = __all_sync(0xffffffffu, tc::mbar_wait(&sh->v_full[s], (uint32_t)(i >> 1) & 1, status, abort_flag, 269));
          if (!ok) break;
          const int r0 = pl.q.len - j * TK;
          for (int x = r0 * 8 + lane; x < TK * 8; x += 32) {
#pragma unroll
            for (int c = 0; c < HD / 64; ++c) *reinterpret_cast<uint4 *>(sV + s * TILE_BYTES + c * 16384 + x * 16) = make_uint4(0, 0, 0, 0);
          }
          tc::fence_proxy_async();
          __syncwarp();
          if (lane == 0) tc::mbar_arrive(&sh->fix_done[s]);
        }
        it += g.k1 - g.k0;
        next();
      }
    }
  } else {
    setmaxnreg_inc<REGS_SOFTMAX>();
    // ---- softmax: warpgroup X owns row tile X, one thread per row
    const int X = warp >> 2, quarter = warp & 3, r = X * 128 + quarter * 32 + lane;
    const float sl2 = a.scale * PAGED_LOG2E;
    const uint32_t tS = tmem_base + ((uint32_t)(quarter * 32) << 16) + X * 256, tO = tS + 128;
    int cnt = 0;                                           // tiles of this row tile so far
    while (w.more && ok) {
      const Segment g(a, w);
      const int jx = g.end(X);
      int row, head, pos;
      const bool has = paged_row(a, pl, r, row, head, pos);
      const int limit = min(max(pos + 1, 0), pl.q.len);    // keys the row sees
      const int all_see = min(max(pl.q.base + pl.block * a.plan.tokens_per_block + X * (a.plan.tokens_per_block / 2) + 1, 0), pl.q.len);
      float m_used = -1e30f, l = 0.f;                      // a finite start: rows that see nothing stay there with l = 0
      for (int j = g.k0; j < jx; ++j, ++cnt) {
        ok = __all_sync(0xffffffffu, tc::mbar_wait(&sh->s_full[X], cnt & 1, status, abort_flag, 270));
        if (!ok) break;                                    // the tensor-memory accesses below are warp-collective
        tc::tc_fence_after();
        const int k0 = j * TK;
        uint32_t v[128];
#pragma unroll
        for (int c = 0; c < 4; ++c) tc::tmem_ld_32x32(tS + c * 32, v + c * 32);
        tc::tmem_ld_wait();
        if (k0 + TK > all_see) {
#pragma unroll
          for (int i = 0; i < 128; ++i)
            if (k0 + i >= limit) v[i] = 0xff800000u;       // -inf: exp2 gives exactly 0 below
        }
        float mx4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int i = 0; i < 128; i += 8) {
          mx4[0] = max3(mx4[0], __uint_as_float(v[i]), __uint_as_float(v[i + 1]));
          mx4[1] = max3(mx4[1], __uint_as_float(v[i + 2]), __uint_as_float(v[i + 3]));
          mx4[2] = max3(mx4[2], __uint_as_float(v[i + 4]), __uint_as_float(v[i + 5]));
          mx4[3] = max3(mx4[3], __uint_as_float(v[i + 6]), __uint_as_float(v[i + 7]));
        }
        const float m_new = fmaxf(m_used, fmaxf(fmaxf(mx4[0], mx4[1]), fmaxf(mx4[2], mx4[3])) * sl2);
        const bool need = (m_new - m_used) > RESCALE_THRESHOLD;
        if (j == g.k0) {
          m_used = m_new;                                  // nothing accumulated yet
        } else if (__any_sync(0xffffffffu, need)) {
          // a row outgrew the maximum in use: rescale its accumulator (the product of the tile before must have landed; this
          // tile's cannot start before p_full below)
          ok = __all_sync(0xffffffffu, tc::mbar_wait(&sh->o_full[X], (cnt - 1) & 1, status, abort_flag, 271));
          if (!ok) break;
          tc::tc_fence_after();
          const float f = need ? fast_exp2(m_used - m_new) : 1.0f;
#pragma unroll
          for (int c = 0; c < HD / 32; ++c) {
            uint32_t o[32];
            tc::tmem_ld_32x32(tO + c * 32, o);
            tc::tmem_ld_wait();
#pragma unroll
            for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * f);
            tc::tmem_st_32x32(tO + c * 32, o);
          }
          tc::tmem_st_wait();
          l *= f;
          if (need) m_used = m_new;
        }
        // probabilities, rounded to bf16 for the tensor product, over the first half of the score columns (all 128 were read above)
        float rs4[4] = {0.f, 0.f, 0.f, 0.f};
        uint32_t pk[64];
#pragma unroll
        for (int i = 0; i < 128; i += 2) {
          const float e0 = fast_exp2(__uint_as_float(v[i]) * sl2 - m_used), e1 = fast_exp2(__uint_as_float(v[i + 1]) * sl2 - m_used);
          rs4[(i >> 1) & 3] += e0 + e1;
          pk[i >> 1] = pack_bf16(e0, e1);
        }
        tc::tmem_st_32x32(tS, pk);
        tc::tmem_st_32x32(tS + 32, pk + 32);
        l += (rs4[0] + rs4[1]) + (rs4[2] + rs4[3]);
        tc::tmem_st_wait();
        tc::tc_fence_before();
        __syncwarp();
        if (lane == 0) tc::mbar_arrive(&sh->p_full[X]);
      }
      if (!ok) break;
      // ---- the block's end, or the run's: normalised rows, or a partial result
      const bool whole = w.whole(), any = jx > g.k0;
      if (any) {
        ok = __all_sync(0xffffffffu, tc::mbar_wait(&sh->o_full[X], (cnt - 1) & 1, status, abort_flag, 272));
        if (!ok) break;
        tc::tc_fence_after();
      }
      const float inv = whole ? (l > 0.f ? 1.0f / l : 0.f) : 1.0f;
      const long long off = !has ? -1 : whole ? (long long)row * a.ld_o + (long long)head * HD : (long long)r * HD;
      float *slot = whole ? nullptr : paged_slot(a, blockIdx.x, g.k0 == 0);
      uint8_t *stg = stage + warp * 2048;
      const bool writes = g.n[X] > 0;
#pragma unroll 1
      for (int c = 0; writes && c < HD / 32; ++c) {
        uint32_t v[32];
        if (any) {
          tc::tmem_ld_32x32(tO + c * 32, v);
          tc::tmem_ld_wait();
        } else {
#pragma unroll
          for (int x = 0; x < 32; ++x) v[x] = 0u;
        }
        // transposed through a warp-private buffer so that a store instruction writes whole 64-byte pieces of eight rows
        if (whole) {
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            uint4 y;
            y.x = pack_bf16(__uint_as_float(v[x * 8 + 0]) * inv, __uint_as_float(v[x * 8 + 1]) * inv);
            y.y = pack_bf16(__uint_as_float(v[x * 8 + 2]) * inv, __uint_as_float(v[x * 8 + 3]) * inv);
            y.z = pack_bf16(__uint_as_float(v[x * 8 + 4]) * inv, __uint_as_float(v[x * 8 + 5]) * inv);
            y.w = pack_bf16(__uint_as_float(v[x * 8 + 6]) * inv, __uint_as_float(v[x * 8 + 7]) * inv);
            *reinterpret_cast<uint4 *>(stg + lane * 64 + ((x ^ ((lane >> 1) & 3)) << 4)) = y;
          }
          __syncwarp();
#pragma unroll
          for (int x = 0; x < 4; ++x) {
            const int rr = 8 * x + (lane >> 2), q = lane & 3;
            const uint4 y = *reinterpret_cast<const uint4 *>(stg + rr * 64 + ((q ^ ((rr >> 1) & 3)) << 4));
            const long long o = __shfl_sync(0xffffffffu, off, rr);
            if (o >= 0) *reinterpret_cast<uint4 *>((bf16 *)a.o + o + c * 32 + q * 8) = y;
          }
          __syncwarp();
        } else {
#pragma unroll
          for (int h = 0; h < 2; ++h) {
#pragma unroll
            for (int x = 0; x < 4; ++x)
              *reinterpret_cast<uint4 *>(stg + lane * 64 + ((x ^ ((lane >> 1) & 3)) << 4)) = make_uint4(v[h * 16 + 4 * x], v[h * 16 + 4 * x + 1], v[h * 16 + 4 * x + 2], v[h * 16 + 4 * x + 3]);
            __syncwarp();
#pragma unroll
            for (int x = 0; x < 4; ++x) {
              const int rr = 8 * x + (lane >> 2), q = lane & 3;
              const uint4 y = *reinterpret_cast<const uint4 *>(stg + rr * 64 + ((q ^ ((rr >> 1) & 3)) << 4));
              const long long o = __shfl_sync(0xffffffffu, off, rr);
              if (o >= 0) *reinterpret_cast<uint4 *>(slot + o + c * 32 + h * 16 + q * 4) = y;
            }
            __syncwarp();
          }
        }
      }
      if (writes && has) {
        if (!whole) {
          slot[(size_t)256 * HD + r] = l > 0.f ? m_used : -INFINITY;
          slot[(size_t)256 * (HD + 1) + r] = l;
        } else if (a.lse) a.lse[(long long)row * a.nH + head] = l > 0.f ? (m_used + log2f(l)) / PAGED_LOG2E : -INFINITY;
      }
      tc::tc_fence_before();
      next();
    }
  }
  tc::tc_fence_before();
  __syncthreads();
  if (warp == MMA_WARP) {
    __syncwarp();
    tc::tc_fence_after();
    tc::tmem_dealloc(tmem_base, 512);
  }
}

int box_rows_of(size_t page_size) {                        // gcd(page_size, 128)
  int b = 128;
  while (page_size % b) b /= 2;
  return b;
}

template <int HD>
int launch_t(b200_ctx *ctx, const PagedAttnArgs &a) {
  const int G = a.plan.G, half = a.plan.tokens_per_block / 2, box = box_rows_of((size_t)a.b.page_size);
  CUtensorMap mq, mk, mv;
  if (tc_make_map_3d(&mq, a.q, HD, (uint64_t)a.nH, (uint64_t)a.b.rows, HD * 2, (uint64_t)a.ld_q * 2, 64, (uint32_t)G, (uint32_t)half) ||
      tc_make_map_4d(&mk, a.k, HD, (uint64_t)a.b.page_size, (uint64_t)a.b.n_kv, (uint64_t)a.b.n_pages, (uint64_t)a.b.token_stride * 2, (uint64_t)a.b.head_stride * 2, (uint64_t)a.b.page_stride * 2, 64, (uint32_t)box) ||
      tc_make_map_4d(&mv, a.v, HD, (uint64_t)a.b.page_size, (uint64_t)a.b.n_kv, (uint64_t)a.b.n_pages, (uint64_t)a.b.token_stride * 2, (uint64_t)a.b.head_stride * 2, (uint64_t)a.b.page_stride * 2, 64, (uint32_t)box))
    return b200_fail(ctx, B200_ERR_CUDA, "cuTensorMapEncodeTiled failed for the paged cache");
  constexpr int smem = 6 * 128 * HD * 2 + (int)sizeof(TcShared) + 8 * 2048;
  static_assert(smem <= 232448, "tiles exceed the 227 KiB of shared memory per CTA");
  static std::atomic<unsigned long long> attr{0};
  const unsigned long long bit = 1ull << (ctx->device & 63);
  if (!(attr.load() & bit)) { B200_CUDA(ctx, cudaFuncSetAttribute(paged_attn_tc_kernel<HD>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem)); attr.fetch_or(bit); }
  B200_CUDA(ctx, launch_pdl(ctx, paged_attn_tc_kernel<HD>, dim3((unsigned)a.n_cta), dim3(TC_THREADS), (size_t)smem, 0, mq, mk, mv, a, box));
  B200_LAUNCHED(ctx);
  return B200_OK;
}

}  // namespace

// 16-byte rows; pages of a multiple of eight positions (a box of the gather is whole swizzle atoms); groups of at most 128 heads (a tile
// holds whole tokens).
bool paged_attn_tc_supported(const b200_paged_cache *c, size_t n_heads, const void *q, size_t ld_q, const void *o, size_t ld_o) {
  return paged_attn_few_supported(c, q, ld_q, o, ld_o) && c->page_size % 8 == 0 && n_heads / c->n_kv <= 128;
}

int paged_attn_tc_launch(b200_ctx *ctx, PagedAttnArgs &a, int G, int min_rows) {
  // a block's start and end cost three tiles' time; runs of at least two tiles
  a.plan = paged::Plan{G, 2 * (128 / G), 0, 7, 3, min_rows, 0x7fffffff};
  a.n_cta = ctx->sm_count; a.min_units = 2; a.slot_rows = 256; a.vec_out = 1; a.beside = 0;
  return a.b.hd == 128 ? launch_t<128>(ctx, a) : launch_t<64>(ctx, a);
}
