// Shared by the attention kernels over a paged cache: arguments, the layout of partial results, the launcher of the join.
#pragma once
#include "paged_common.cuh"

struct PagedAttnArgs {
  PagedArgs b;
  paged::Plan plan;
  const void *k, *v, *q;
  void *o;
  float *lse, *ws;                       // ws: the join's heads, then the partial results
  long long ld_q, ld_o;
  int nH, n_cta, min_units, slot_rows;   // slot_rows: rows of one partial result
  int vec_out;                           // rows of o are 16-byte aligned
  int beside;                            // do not wait for the kernel before
  float scale;
};

constexpr int PAGED_FEW_ROWS = 32;
constexpr float PAGED_LOG2E = 1.4426950408889634f;

// Partial result of a block: [slot_rows][hd] output in units of 2^maximum, then [slot_rows] maxima (log2 units), [slot_rows] sums.
// A part whose maximum is -inf saw no key; its output is not read.  CTA c owns two: slot 2c for a block that began before its run, 2c + 1 for one that begins in it and ends behind it.
__host__ __device__ __forceinline__ size_t paged_slot_floats(int slot_rows, int hd) { return (size_t)slot_rows * (hd + 2); }
// What the join needs of the border before run c: written by CTA c (every CTA of the grid writes its own).
struct alignas(16) JoinHead { int parts; paged::Place pl; };
constexpr int JOIN_HEAD_FLOATS = 16;
static_assert(sizeof(JoinHead) <= JOIN_HEAD_FLOATS * 4, "join head");
__device__ __forceinline__ JoinHead *paged_head(const PagedAttnArgs &a, int cta) { return reinterpret_cast<JoinHead *>(a.ws + (size_t)cta * JOIN_HEAD_FLOATS); }
__device__ __forceinline__ void paged_write_head(const PagedAttnArgs &a, const paged::Run &run, const paged::Place &pl, int c) {
  JoinHead *h = paged_head(a, c);
  const int parts = run.u == run.end ? 0 : paged::parts_at(a.plan, run, pl, c);
  h->parts = parts;
  if (parts) h->pl = pl;
}
__device__ __forceinline__ float *paged_slot(const PagedAttnArgs &a, int cta, bool begins) {
  return a.ws + (size_t)a.n_cta * JOIN_HEAD_FLOATS + (size_t)(2 * cta + (begins ? 1 : 0)) * paged_slot_floats(a.slot_rows, a.b.hd);
}
// (row of q / o, query head) of row r of a block; false where the block has no such row.
__device__ __forceinline__ bool paged_row(const PagedAttnArgs &a, const paged::Place &pl, int r, int &row, int &head, int &pos) {
  int tok, g;
  if (a.plan.rows_per_block) {
    const long long f = (long long)pl.block * a.plan.rows_per_block + r;
    tok = (int)(f / a.plan.G); g = (int)(f - (long long)tok * a.plan.G);
  } else {
    // two tiles of 128 rows, each of whole tokens
    const int half = a.plan.tokens_per_block / 2, t = (r & 127) / a.plan.G;
    tok = pl.block * a.plan.tokens_per_block + (r >> 7) * half + t; g = (r & 127) - t * a.plan.G;
    if (t >= half) return false;
  }
  row = pl.q.q0 + tok; head = pl.kvh * a.plan.G + g; pos = pl.q.base + tok;
  return tok < pl.q.ql;
}

// Joins what one or two kernels left (b may be null).
int paged_join_launch(b200_ctx *ctx, const PagedAttnArgs &a, const PagedAttnArgs *b, b200_dtype dt);
bool paged_attn_few_supported(const b200_paged_cache *c, const void *q, size_t ld_q, const void *o, size_t ld_o);
// The launchers complete `a` (the join needs it); its workspace begins at a.ws.
// beside: the kernel before it on the stream works on other sequences of the same call and has waited for what came before the call, so this one
// starts without waiting and fills the SMs that the other leaves; it waits for the other before it ends, so that what follows it follows both.
int paged_attn_few_launch(b200_ctx *ctx, PagedAttnArgs &a, int G, bool beside);
bool paged_attn_tc_supported(const b200_paged_cache *c, size_t n_heads, const void *q, size_t ld_q, const void *o, size_t ld_o);
int paged_attn_tc_launch(b200_ctx *ctx, PagedAttnArgs &a, int G, int min_rows);
