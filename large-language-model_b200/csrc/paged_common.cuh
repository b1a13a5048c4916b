// What the kernels over a paged key/value cache share: the ragged batch, its checks on the device, and the division of its
// attention work into equal runs.
//
// The lengths and the page table live on the device (a captured step replays with new ones), so the host knows only upper
// bounds and nothing the kernels read may be trusted: every length is clamped to the arrays it indexes, every page id is
// compared with the page count before it is used, and the first violation is recorded in the context's status word.
#pragma once
#include "common.cuh"

constexpr int PAGED_BAD_BATCH = 3;      // status code: a page id or a length of the batch is out of range

struct PagedArgs {
  const int *q_start, *kv_len, *table;  // [n_seq + 1], [n_seq], [n_seq, table_ld]
  int n_seq, table_ld, rows, max_q;
  int page_size, n_pages, n_kv, hd;
  long long page_stride, token_stride, head_stride;   // elements
  int *status;
};

struct DeviceGuard {                    // entry points may be called with another device current
  int prev = -1;
  bool ok = true;
  explicit DeviceGuard(const b200_ctx *ctx) {
    if (cudaGetDevice(&prev) != cudaSuccess) { ok = false; return; }
    if (prev == ctx->device) prev = -1;
    else ok = cudaSetDevice(ctx->device) == cudaSuccess;
  }
  ~DeviceGuard() { if (prev >= 0) cudaSetDevice(prev); }
};

// Programmatic launch whatever the context's setting: these operators are chains of short kernels, each of which waits for the one before in its
// first instruction (or says why not) and lets the next one launch behind that.
template <class... K, class... A>
inline cudaError_t launch_pdl(b200_ctx *ctx, void (*kern)(K...), dim3 grid, dim3 block, size_t smem, int cluster_x, A... args) {
  const bool pdl = ctx->pdl;
  ctx->pdl = true;
  const cudaError_t e = launch_k(ctx, kern, grid, block, smem, cluster_x, args...);
  ctx->pdl = pdl;
  return e;
}

// Host checks of the two descriptors; fills `a`.
int paged_args(b200_ctx *ctx, const b200_paged_cache *cache, const b200_paged_batch *batch, PagedArgs *a);

namespace paged {

struct Seq { int q0, ql, base, len; };  // first row, rows, position of row 0, cached positions

// The checks and the stepping below also compile for the host, where the CPU tests run them.
__host__ __device__ __forceinline__ void bad_batch(const PagedArgs &a) {
#ifdef __CUDA_ARCH__
  atomicCAS(a.status, 0, PAGED_BAD_BATCH);
#else
  *a.status = PAGED_BAD_BATCH;
#endif
}
__host__ __device__ __forceinline__ int lesser(int a, int b) { return a < b ? a : b; }
__host__ __device__ __forceinline__ int greater(int a, int b) { return a > b ? a : b; }

__host__ __device__ __forceinline__ Seq load_seq(const PagedArgs &a, int s) {
  const int r0 = a.q_start[s], r1 = a.q_start[s + 1], l = a.kv_len[s];
  const long long room = (long long)a.table_ld * a.page_size;
  Seq q;
  q.q0 = lesser(greater(r0, 0), a.rows);
  const int q1 = lesser(greater(r1, q.q0), a.rows), n = q1 - q.q0;
  q.ql = lesser(n, a.max_q);
  q.len = l < 0 ? 0 : l > room ? (int)room : l;
  q.base = q.len - n;
  if (q.q0 != r0 || q1 != r1 || q.ql != n || q.len != l) bad_batch(a);
  return q;
}
// Page of position `pos`, or -1 (recorded) when the table holds an id outside the cache.
__host__ __device__ __forceinline__ int page_of(const PagedArgs &a, int s, int pos) {
  const int id = a.table[(long long)s * a.table_ld + pos / a.page_size];
  if ((unsigned)id < (unsigned)a.n_pages) return id;
  bad_batch(a);
  return -1;
}

// ---- division of the work ---------------------------------------------------------------------------------------------
// A sequence's rows (token, query head of the group) are cut into blocks; a block walks the key tiles its last row can see.
// All (sequence, KV head, block, tile) in this order form one line; a block takes `extra` units (its start and end, in tiles' time)
// and one per tile.  The line is cut into n runs of equal length (the first total % n have one unit more): every SM gets the same amount of work
// whatever the lengths are (without the extra, CTAs whose run held dozens of short sequences took 1.8 times the others' time).
// A block that crosses a border leaves partial results (unnormalised output, maximum, sum) that a second kernel joins in CTA order.
struct Plan {
  int G, tokens_per_block, rows_per_block;   // rows_per_block > 0: blocks of consecutive rows; else blocks of whole tokens
  int tile_log2, extra, min_rows, max_rows;  // keys per tile; only sequences with min_rows <= rows <= max_rows take part
  __host__ __device__ __forceinline__ bool takes(int ql) const { const long long r = (long long)ql * G; return ql > 0 && r >= min_rows && r <= max_rows; }
  __host__ __device__ __forceinline__ int blocks(int ql) const {
    if (max_rows <= rows_per_block) return 1;
    if (!rows_per_block) return (int)((unsigned)(ql + tokens_per_block - 1) / (unsigned)tokens_per_block);
    const unsigned long long r = (unsigned long long)ql * G + rows_per_block - 1;
    return r >> 32 ? (int)(r / rows_per_block) : (int)((unsigned)r / (unsigned)rows_per_block);      // (a 64-bit division costs a microsecond in a loop)
  }
  __host__ __device__ __forceinline__ int tiles(const Seq &q, int block) const {
    int last = q.ql;                                                     // rows up to the block's end
    if (!rows_per_block) { const long long end = (long long)(block + 1) * tokens_per_block; last = end < q.ql ? (int)end : q.ql; }
    else if (max_rows > rows_per_block) {
      const unsigned long long r = (unsigned long long)(block + 1) * rows_per_block - 1;
      const unsigned long long end = (r >> 32 ? r / G : (unsigned)r / (unsigned)G) + 1;
      last = end < (unsigned long long)q.ql ? (int)end : q.ql;
    }
    const int seen = lesser(greater(q.base + last, 0), q.len);
    return greater(1, (int)(((long long)seen + (1 << tile_log2) - 1) >> tile_log2));   // a block that sees nothing still writes its empty rows
  }
};
// Divisions of positions on the line are 32-bit ones wherever it is that short.
__host__ __device__ __forceinline__ long long quotient(long long a, int b) { return a >> 32 ? a / b : (long long)((unsigned)a / (unsigned)b); }
__host__ __device__ __forceinline__ long long block_units(const Plan &p, const Seq &q, int block) { return (long long)p.tiles(q, block) + p.extra; }
struct Place { int seq, kvh, block, kt; Seq q; long long first; };   // tile kt of a block, which begins at unit `first`

__host__ __device__ __forceinline__ long long seq_units(const PagedArgs &a, const Plan &p, int s) {
  const Seq q = load_seq(a, s);
  if (!p.takes(q.ql)) return 0;
  long long u = 0;
  for (int b = p.blocks(q.ql) - 1; b >= 0; --b) u += block_units(p, q, b);
  return u * a.n_kv;
}

// Unit u of the line, which is in sequence s, whose units begin at `at` and number `units`.
__host__ __device__ __forceinline__ Place place_in(const PagedArgs &a, const Plan &p, int s, long long units, long long at, long long u) {
  const long long per_head = quotient(units, a.n_kv);
  Place pl;
  pl.seq = s; pl.q = load_seq(a, s); pl.kvh = per_head >> 31 ? (int)((u - at) / per_head) : (int)quotient(u - at, (int)per_head);
  pl.first = at + pl.kvh * per_head;
  int b = 0;
  long long t = block_units(p, pl.q, 0);
  while (u - pl.first >= t) { pl.first += t; t = block_units(p, pl.q, ++b); }
  pl.block = b; pl.kt = greater(0, (int)(u - pl.first) - p.extra);
  return pl;
}

// Exclusive prefix over the CTA's threads and the CTA total; `red` is shared [33].  All threads must call.
template <int THREADS>
__device__ __forceinline__ long long block_scan(long long v, long long *red, long long &sum) {
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  long long inc = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) { const long long t = __shfl_up_sync(0xffffffffu, inc, o); if (lane >= o) inc += t; }
  __syncthreads();
  if (lane == 31) red[w] = inc;
  __syncthreads();
  long long before = 0; sum = 0;
#pragma unroll
  for (int i = 0; i < THREADS / 32; ++i) { if (i < w) before += red[i]; sum += red[i]; }
  return before + inc - v;
}

// CTAs that take part: at most n_max, and few enough that each gets min_units.
__host__ __device__ __forceinline__ int line_ctas(long long total, int n_max, int min_units) {
  const long long n = quotient(total, min_units);        // (rounded down: no CTA gets less)
  return n < 1 ? 1 : n < n_max ? (int)n : n_max;
}
__host__ __device__ __forceinline__ long long line_at(long long total, int n, int c) {      // the first total % n CTAs have one unit more
  const long long each = quotient(total, n);
  const int more = (int)(total - each * n);
  return each * c + lesser(c, more);
}
__host__ __device__ __forceinline__ int line_cta(long long total, int n, long long u) {      // the CTA of unit u
  const long long each = quotient(total, n);
  const int more = (int)(total - each * n);
  const long long longer = (each + 1) * more;
  return u < longer ? (int)((u >> 32) || each >> 31 ? u / (each + 1) : (unsigned)u / (unsigned)(each + 1))
                    : more + (int)(((u - longer) >> 32) || each >> 31 ? (u - longer) / each : (unsigned)(u - longer) / (unsigned)each);
}
struct Run { long long u, end, total; int n; };          // units [u, end) of CTA c; n CTAs take part

// The run of CTA c, and the place of unit u in *out (shared) unless the run is empty.  All threads must call; ends with a barrier.
template <int THREADS>
__device__ Run line_run(const PagedArgs &a, const Plan &p, int c, int n_max, int min_units, long long *red, Place *out) {
  const int tid = (int)threadIdx.x;
  const long long first = tid < a.n_seq ? seq_units(a, p, tid) : 0;
  long long mine = first, total;
  for (int s = tid + THREADS; s < a.n_seq; s += THREADS) mine += seq_units(a, p, s);
  long long at = block_scan<THREADS>(mine, red, total);
  Run r;
  r.total = total; r.n = line_ctas(total, n_max, min_units);
  r.u = r.end = 0;
  if (total == 0 || c >= r.n) return r;
  r.u = line_at(total, r.n, c); r.end = line_at(total, r.n, c + 1);
  if (a.n_seq <= THREADS) {                                // each thread has one sequence: the scan above is the line
    if (r.u >= at && r.u < at + mine) *out = place_in(a, p, tid, mine, at, r.u);
  } else {
    long long done = 0;
    for (int s0 = 0; s0 < a.n_seq; s0 += THREADS) {
      const int s = s0 + tid;
      const long long m = s0 == 0 ? first : s < a.n_seq ? seq_units(a, p, s) : 0;
      long long sum;
      at = done + block_scan<THREADS>(m, red, sum);
      if (r.u >= at && r.u < at + m) *out = place_in(a, p, s, m, at, r.u);
      done += sum;
      if (done > r.u) break;                               // the same for all threads
    }
  }
  __syncthreads();
  return r;
}
// Steps through a run block by block: tiles [pl.kt, k1) of the block's `tiles`.
struct Walk {
  Place pl;
  int tiles, k1;
  bool more;
  __host__ __device__ __forceinline__ void start(const Plan &p, const Place &at, long long end) { pl = at; set(p, end); }
  __host__ __device__ __forceinline__ void set(const Plan &p, long long end) {
    tiles = p.tiles(pl.q, pl.block);
    const long long room = end - pl.first - p.extra;
    k1 = room < tiles ? (int)room : tiles;
    more = k1 > pl.kt;                                     // a run that ends in a block's extra leaves it to the next CTA
  }
  __host__ __device__ __forceinline__ bool whole() const { return pl.kt == 0 && k1 == tiles; }
  __host__ __device__ __forceinline__ void next(const PagedArgs &a, const Plan &p, long long end) {
    pl.first += block_units(p, pl.q, pl.block);
    pl.kt = 0;
    if (pl.first >= end) { more = false; return; }
    if (++pl.block >= p.blocks(pl.q.ql)) {
      pl.block = 0;
      if (++pl.kvh >= a.n_kv) {
        pl.kvh = 0;
        while (++pl.seq < a.n_seq) {
          pl.q = load_seq(a, pl.seq);
          if (p.takes(pl.q.ql)) break;
        }
        if (pl.seq >= a.n_seq) { more = false; return; }
      }
    }
    set(p, end);
  }
};
// How many CTAs, from c - 1 on, have parts of the block that run c begins in; 0 unless c is the first border inside that block.
__host__ __device__ __forceinline__ int parts_at(const Plan &p, const Run &r, const Place &pl, int c) {
  if (c == 0 || pl.kt == 0 || line_at(r.total, r.n, c - 1) > pl.first + p.extra) return 0;
  return line_cta(r.total, r.n, pl.first + block_units(p, pl.q, pl.block) - 1) - c + 2;
}

}  // namespace paged
