// Sampling from given random numbers: per-row temperature, top-k, top-p and min-p, the id by inversion of the cumulative
// weights.  Beside b200_sample (one setting for all rows, its own random numbers, cpp/python rules of the reference).
//
//   w_i = exp((l_i - max l) / T); ids in the order (l descending, id ascending); top-k keeps the first k; top-p keeps a survivor
//   while the weight before it is below p x the weight of all top-k survivors; min-p keeps w_i >= min_p; the id is the least
//   kept one whose cumulative kept weight (in id order) exceeds u x the kept weight.
//
// The answer is a whole number, so it has to be the right one and not nearly so: weights are computed in 64 bits and added as
// fixed-point integers (2^-44 of the largest weight at up to 2^18 ids), which makes every sum exact and independent of order.
// Nothing is sorted.  A cluster of CTAs holds a row, each its slice in shared memory (one read of the logits).  One histogram
// of 2048 value bins below the maximum (count and weight) locates the bin where the k-th id or the p-th part falls; the bin's few
// ids are ranked against each other.  A bin with more ids than the list holds is cut again by the bits of its values, at most
// three times; equal values are settled by arithmetic.  The kept set is a prefix of the order: a least value and the number of
// ids of that value, lowest ids first.
// Bound by latency at usual sizes (a dozen exchanges within the cluster of 0.5 us) and by the 64-bit exponentials for large
// vocabularies; the floor is one read of the logits.
#include "paged_common.cuh"
#include <algorithm>
#include <atomic>
#include <cooperative_groups.h>

namespace cg = cooperative_groups;

namespace {

constexpr int THREADS = 512, WARPS = THREADS / 32, BINS = 2048, LIST = 512, MAX_CLUSTER = 8;
typedef unsigned long long u64;

struct GivenArgs {
  const void *logits;
  long long ld;
  int V, slice, fixed_bits, in_smem;      // slice: ids per CTA, a multiple of 16
  const float *temperature, *top_p, *min_p, *uniform;
  const int *top_k;
  int32_t *tokens, *kept;
  float *prob;
};

struct Mail { u64 a, b, c, d; };
struct Entry { uint32_t key, id; u64 q; };
struct Shared {
  uint32_t cnt[BINS], lo[BINS], hi[BINS];    // this CTA's histogram; a bin's weight is hi : lo
  uint32_t tot_cnt[BINS];                    // the cluster's sums of this CTA's part of the bins
  u64 tot_mass[BINS];
  double table[64];                          // 2^(j / 64)
  Mail mail[2][MAX_CLUSTER];
  u64 found[2][8];
  u64 warp_mail[MAX_CLUSTER * WARPS];
  uint32_t warp_eq[MAX_CLUSTER * WARPS];
  u64 red[WARPS], red2[WARPS];
  Entry list[LIST];
  int list_n;
  u64 res[4];
};

__device__ __forceinline__ uint32_t key_of(float x) { const uint32_t b = __float_as_uint(x); return b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u); }
// -0 is 0; NaN counts as masked
__device__ __forceinline__ float clean(float x) { return x == x ? x + 0.0f : -INFINITY; }

// exp(z) for z2 = z / ln 2 <= 0: 2^(k/64) from a table times a polynomial of the rest (|rest| <= 2^-7, degree 5: error 3e-17).
__device__ __forceinline__ double weight(double z2, const double *table) {
  if (!(z2 > -1020.0)) return 0.0;
  const double shift = 6755399441055744.0;      // 1.5 * 2^52: adding it rounds to an integer held in the low bits
  const double t = z2 * 64.0 + shift;
  const int k = __double2loint(t);
  const double r = (z2 - (t - shift) * 0.015625) * 0.69314718055994530942;
  const double p = fma(r, fma(r, fma(r, fma(r, fma(r, 1.0 / 120, 1.0 / 24), 1.0 / 6), 0.5), 1.0), 1.0);
  const double m = p * table[k & 63];           // in (0.99, 2.01)
  return __hiloint2double(__double2hiint(m) + ((k >> 6) << 20), __double2loint(m));
}

template <int C>
struct Group {                                   // the CTAs of a row
  Shared *s;
  int rank, par;
  __device__ __forceinline__ void sync() { if constexpr (C > 1) cg::this_cluster().sync(); else __syncthreads(); }
  template <class P> __device__ __forceinline__ P *peer(P *p, int r) { if constexpr (C > 1) return cg::this_cluster().map_shared_rank(p, r); else return p; }
  // Every CTA posts one Mail; all see all.  Two mailboxes in turn: a CTA cannot be two exchanges ahead of a peer that still reads.
  __device__ __forceinline__ const Mail *exchange(const Mail &m) {
    par ^= 1;
    if (threadIdx.x < C) *peer(&s->mail[par][rank], threadIdx.x) = m;
    sync();
    return s->mail[par];
  }
};

__device__ __forceinline__ u64 warp_sum64(u64 v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
__device__ __forceinline__ u64 block_sum64(u64 v, u64 *red) {
  v = warp_sum64(v);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  u64 t = 0;
#pragma unroll
  for (int i = 0; i < WARPS; ++i) t += red[i];
  return t;
}
__device__ __forceinline__ uint32_t block_max32(uint32_t v, u64 *red) {
  v = __reduce_max_sync(0xffffffffu, v);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  uint32_t t = 0;
#pragma unroll
  for (int i = 0; i < WARPS; ++i) t = max(t, (uint32_t)red[i]);
  return t;
}

struct Find { u64 above_c, above_m, cnt, mass, total; int bin; };

template <class T, int C>
struct Row {
  Group<C> g;
  Shared *s;
  const T *x;          // this CTA's slice
  int n, id0;          // ids in the slice, first id
  float mx;
  double z_scale;      // log2(e) / T
  int fixed_bits;

  __device__ __forceinline__ double w_of(float v) const { return v == mx ? 1.0 : weight(((double)v - (double)mx) * z_scale, s->table); }
  __device__ __forceinline__ u64 q_of(double w) const { return (u64)(w * (double)(1ll << fixed_bits) + 0.5); }

  // f(value, index in the slice) for every id
  template <class F> __device__ __forceinline__ void each(F f) const {
    constexpr int N = 16 / sizeof(T);
    if (((uintptr_t)x & 15) == 0) {
      const int nv = n / N;
      for (int i = threadIdx.x; i < nv; i += THREADS) {
        Vec16<T> v;
        float e[N];
        v.load(x + i * N); v.unpack(e);
#pragma unroll
        for (int j = 0; j < N; ++j) f(clean(e[j]), i * N + j);
      }
      for (int i = nv * N + threadIdx.x; i < n; i += THREADS) f(clean(to_f(x[i])), i);
    } else {
      for (int i = threadIdx.x; i < n; i += THREADS) f(clean(to_f(x[i])), i);
    }
  }
  __device__ __forceinline__ void clear() {
    for (int i = threadIdx.x; i < BINS; i += THREADS) { s->cnt[i] = 0; s->lo[i] = 0; s->hi[i] = 0; }
    __syncthreads();
  }
  __device__ __forceinline__ void add(int bin, u64 q, bool mass) {
    atomicAdd(&s->cnt[bin], 1u);
    if (!mass) return;
    const uint32_t l = (uint32_t)q, h = (uint32_t)(q >> 32);
    uint32_t carry = 0;
    if (l) carry = atomicAdd(&s->lo[bin], l) > 0xffffffffu - l;
    if (h + carry) atomicAdd(&s->hi[bin], h + carry);
  }
  // Sums the CTAs' histograms: CTA r takes bins [r, r + 1) * BINS / C.
  __device__ __forceinline__ void collect() {
    g.sync();
    constexpr int PART = BINS / C;
    for (int i = threadIdx.x; i < PART; i += THREADS) {
      uint32_t c = 0;
      u64 m = 0;
#pragma unroll
      for (int r = 0; r < C; ++r) {
        const Shared *o = g.peer(s, r);
        const int b = g.rank * PART + i;
        c += o->cnt[b]; m += ((u64)o->hi[b] << 32) + o->lo[b];
      }
      s->tot_cnt[i] = c; s->tot_mass[i] = m;
    }
    __syncthreads();
  }
  // The bin where the running total of counts (by_mass false) or weights from the top reaches the target: above < target <= above + bin.
  // frac >= 0: the target is frac x the weight in all bins.  `start_c` / `start_m` lie above the first bin.
  __device__ Find search(bool by_mass, double target, double frac, u64 start_c, u64 start_m) {
    constexpr int PART = BINS / C, PER = (PART + THREADS - 1) / THREADS;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, b0 = threadIdx.x * PER;
    u64 c = 0, m = 0;
    for (int j = 0; j < PER; ++j) if (b0 + j < PART) { c += s->tot_cnt[b0 + j]; m += s->tot_mass[b0 + j]; }
    u64 ic = c, im = m;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const u64 tc_ = __shfl_up_sync(0xffffffffu, ic, o), tm = __shfl_up_sync(0xffffffffu, im, o);
      if (lane >= o) { ic += tc_; im += tm; }
    }
    __syncthreads();
    if (lane == 31) { s->red[warp] = ic; s->red2[warp] = im; }
    __syncthreads();
    u64 before_c = 0, before_m = 0, sum_c = 0, sum_m = 0;
#pragma unroll
    for (int i = 0; i < WARPS; ++i) {
      if (i < warp) { before_c += s->red[i]; before_m += s->red2[i]; }
      sum_c += s->red[i]; sum_m += s->red2[i];
    }
    before_c += ic - c; before_m += im - m;
    const Mail *all = g.exchange(Mail{sum_c, sum_m, 0, 0});
    u64 total = 0;
    before_c += start_c; before_m += start_m;
#pragma unroll
    for (int r = 0; r < C; ++r) { if (r < g.rank) { before_c += all[r].a; before_m += all[r].b; } total += all[r].b; }
    if (frac >= 0.0) target = frac * (double)total;
    const int par = g.par;
    for (int j = 0; j < PER; ++j)
      if (b0 + j < PART) {
        const u64 bc = s->tot_cnt[b0 + j], bm = s->tot_mass[b0 + j];
        const double lo = by_mass ? (double)before_m : (double)before_c, hi = by_mass ? (double)(before_m + bm) : (double)(before_c + bc);
        if (bc && lo < target && target <= hi) {
#pragma unroll
          for (int r = 0; r < C; ++r) {
            u64 *f = g.peer(s->found[par], r);
            f[0] = before_c; f[1] = before_m; f[2] = bc; f[3] = bm; f[4] = (u64)(g.rank * PART + b0 + j);
          }
        }
        before_c += bc; before_m += bm;
      }
    g.sync();
    const u64 *f = s->found[par];
    return Find{f[0], f[1], f[2], f[3], total, (int)f[4]};
  }

  // Settles the border inside a bin: the least kept value (key), how many ids of that value are kept, how many have it, and the weight
  // of the kept prefix.  `member(value, key)` selects the bin's ids.
  struct Border { uint32_t key; u64 ties, equal, mass; };
  template <class M>
  __device__ Border settle(M member, Find f, bool by_mass, double target, bool level0) {
    bool narrowed = !level0;
    uint32_t kl = 0, kh = 0xffffffffu;
    for (int round = 0; round < 5; ++round) {
      auto inside = [&](float v, uint32_t k) { return narrowed ? k >= kl && k <= kh : member(v, k); };
      if (f.cnt <= LIST) {
        if (threadIdx.x == 0) s->list_n = 0;
        g.sync();
        Shared *first = g.peer(s, 0);
        each([&](float v, int i) {
          const uint32_t k = key_of(v);
          if (v > -INFINITY && inside(v, k)) {
            const int at = atomicAdd(&first->list_n, 1);
            if (at < LIST) first->list[at] = Entry{k, (uint32_t)(id0 + i), q_of(w_of(v))};
          }
        });
        g.sync();
        if (g.rank == 0) {
          const int n_list = min(s->list_n, LIST);
          for (int i = threadIdx.x; i < n_list; i += THREADS) {      // LIST == THREADS: one entry a thread
            const Entry e = s->list[i];
            u64 rank_c = f.above_c, rank_m = f.above_m;
            u64 eq_before = 0, equal = 0;
            for (int j = 0; j < n_list; ++j) {
              const Entry o = s->list[j];
              const bool ahead = o.key > e.key || (o.key == e.key && o.id < e.id);
              if (ahead) { ++rank_c; rank_m += o.q; }
              if (o.key == e.key) { ++equal; eq_before += ahead; }
            }
            const double lo = by_mass ? (double)rank_m : (double)rank_c, hi = by_mass ? (double)(rank_m + e.q) : (double)(rank_c + 1);
            if (lo < target && target <= hi) {
#pragma unroll
              for (int r = 0; r < C; ++r) { u64 *o = g.peer(s->res, r); o[0] = e.key; o[1] = eq_before + 1; o[2] = equal; o[3] = rank_m + e.q; }
            }
          }
        }
        g.sync();
        return Border{(uint32_t)s->res[0], s->res[1], s->res[2], s->res[3]};
      }
      if (!narrowed) {                                      // the bin's range of values
        uint32_t hi_ = 0, lo_ = 0;                          // lo_ holds ~key
        each([&](float v, int) { const uint32_t k = key_of(v); if (v > -INFINITY && member(v, k)) { hi_ = max(hi_, k); lo_ = max(lo_, ~k); } });
        hi_ = block_max32(hi_, s->red); lo_ = block_max32(lo_, s->red);
        const Mail *all = g.exchange(Mail{hi_, lo_, 0, 0});
        uint32_t h = 0, l = 0;
#pragma unroll
        for (int r = 0; r < C; ++r) { h = max(h, (uint32_t)all[r].a); l = max(l, (uint32_t)all[r].b); }
        kh = h; kl = ~l; narrowed = true;
      }
      if (kl == kh) {                                       // equal values
        const u64 q = by_mass || f.mass ? f.mass / f.cnt : 0;
        u64 t;
        if (by_mass) {
          const double need = target - (double)f.above_m;
          t = q ? (u64)ceil(need / (double)q) : 1;
          t = t < 1 ? 1 : t > f.cnt ? f.cnt : t;
        } else t = (u64)target - f.above_c;
        return Border{kl, t, f.cnt, f.above_m + t * q};
      }
      const uint32_t span = kh - kl;
      const int sh = max(0, 21 - __clz(span));              // (span >> sh) < 2048
      clear();
      each([&](float v, int) {
        const uint32_t k = key_of(v);
        if (v > -INFINITY && k >= kl && k <= kh) add((int)((kh - k) >> sh), q_of(w_of(v)), true);
      });
      collect();
      f = search(by_mass, target, -1.0, f.above_c, f.above_m);
      const uint32_t top = kh - ((uint32_t)f.bin << sh);
      const u64 low = (u64)((uint32_t)f.bin + 1) << sh;
      kl = low > (u64)(kh - kl) ? kl : kh - (uint32_t)low + 1;
      kh = top;
    }
    return Border{kl, f.cnt, f.cnt, f.above_m + f.mass};    // not reached: three cuts leave one value
  }
};

template <class T, int C>
__global__ void __launch_bounds__(THREADS)
sample_given_kernel(GivenArgs a) {
  pdl_launch_dependents();
  pdl_wait();
  extern __shared__ __align__(16) uint8_t dyn[];
  Shared *s = (Shared *)dyn;
  T *copy = (T *)(dyn + ((sizeof(Shared) + 15) & ~(size_t)15));
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, b = blockIdx.x / C;
  Row<T, C> row;
  row.s = s; row.g.s = s; row.g.par = 0; row.fixed_bits = a.fixed_bits;
  row.g.rank = C > 1 ? (int)(blockIdx.x % C) : 0;
  row.id0 = min(a.V, row.g.rank * a.slice); row.n = min(a.V, row.id0 + a.slice) - row.id0;
  const T *src = (const T *)a.logits + (size_t)b * a.ld + row.id0;
  row.x = src;
  if (tid < 64) s->table[tid] = exp2(tid * 0.015625);
  // ---- one read of the slice: a copy in shared memory, the largest and the smallest finite value
  uint32_t hi = 0, lo = 0;
  row.each([&](float v, int i) {
    if (a.in_smem) copy[i] = from_f<T>(v);
    if (v > -INFINITY) { const uint32_t k = key_of(v); hi = max(hi, k); lo = max(lo, ~k); }
  });
  hi = block_max32(hi, s->red); lo = block_max32(lo, s->red);
  if (a.in_smem) row.x = copy;
  if (C > 1) row.g.sync();                                   // every CTA of the cluster runs before its memory is written
  {
    const Mail *all = row.g.exchange(Mail{hi, lo, 0, 0});
#pragma unroll
    for (int r = 0; r < C; ++r) { hi = max(hi, (uint32_t)all[r].a); lo = max(lo, (uint32_t)all[r].b); }
  }
  if (hi == 0) {                                             // nothing to draw from
    if (row.g.rank == 0 && tid == 0) { a.tokens[b] = -1; if (a.kept) a.kept[b] = 0; if (a.prob) a.prob[b] = 0.f; }
    row.g.sync();
    return;
  }
  auto value = [](uint32_t k) { return __uint_as_float(k & 0x80000000u ? k ^ 0x80000000u : ~k); };
  row.mx = value(hi);
  const float mn = value(~lo), T_ = a.temperature ? a.temperature[b] : 1.0f;
  if (!(T_ > 0.f)) {                                         // greedy: the lowest id of the maximum
    uint32_t best = 0;                                       // ~id
    row.each([&](float v, int i) { if (v == row.mx) best = max(best, ~(uint32_t)(row.id0 + i)); });
    best = block_max32(best, s->red);
    const Mail *all = row.g.exchange(Mail{best, 0, 0, 0});
#pragma unroll
    for (int r = 0; r < C; ++r) best = max(best, (uint32_t)all[r].a);
    if (row.g.rank == 0 && tid == 0) { a.tokens[b] = (int)~best; if (a.kept) a.kept[b] = 1; if (a.prob) a.prob[b] = 1.f; }
    row.g.sync();
    return;
  }
  row.z_scale = 1.44269504088896340736 / (double)T_;
  const int k = a.top_k ? a.top_k[b] : 0;
  const float p = a.top_p ? a.top_p[b] : 1.f, mp = a.min_p ? a.min_p[b] : 0.f, u_ = a.uniform[b];
  const bool by_k = k > 0 && k < a.V, by_p = p < 1.f, by_m = mp > 0.f;
  const double min_w = by_m ? fmin((double)mp, 1.0) : 0.0;
  // ---- the kept prefix
  uint32_t vkey = 0;                                         // keep keys above it, and `ties` of the ids that have it
  u64 ties = 0, equal = 0;
  if (by_k || by_p) {
    const float range = fminf(row.mx - mn, 32.0f * T_), scale = range > 0.f && range < INFINITY ? (float)(BINS - 1) / range : 0.f;
    auto bin_of = [&](float v) {
      const float t = v == row.mx ? 0.f : (row.mx - v) * scale;
      return t < (float)(BINS - 1) ? (int)t : BINS - 1;
    };
    row.clear();
    row.each([&](float v, int) { if (v > -INFINITY) row.add(bin_of(v), by_p ? row.q_of(row.w_of(v)) : 0, by_p); });
    row.collect();
    bool have_k = false;
    u64 mass_k = 0;
    if (by_k) {
      // fewer finite ids than k: nothing to cut
      u64 mine = 0;
      for (int i = tid; i < BINS / C; i += THREADS) mine += s->tot_cnt[i];
      mine = block_sum64(mine, s->red);
      const Mail *all = row.g.exchange(Mail{mine, 0, 0, 0});
      u64 n_all = 0;
#pragma unroll
      for (int r = 0; r < C; ++r) n_all += all[r].a;
      if ((u64)k < n_all) {
        const Find f = row.search(false, (double)k, -1.0, 0, 0);
        const auto bd = row.settle([&](float v, uint32_t) { return bin_of(v) == f.bin; }, f, false, (double)k, true);
        vkey = bd.key; ties = bd.ties; equal = bd.equal; mass_k = bd.mass; have_k = true;
        if (by_p && f.cnt > LIST) {                          // the cut inside the bin took the histogram: build it again
          row.clear();
          row.each([&](float v, int) { if (v > -INFINITY) row.add(bin_of(v), row.q_of(row.w_of(v)), true); });
          row.collect();
        }
      }
    }
    if (by_p) {
      const double frac = p > 0.f ? (double)p : 0.0;         // p <= 0 keeps the first id
      Find f;
      double target;
      if (have_k) { target = fmax(frac * (double)mass_k, 0.5); f = row.search(true, target, -1.0, 0, 0); }
      else {
        u64 mine = 0;
        for (int i = tid; i < BINS / C; i += THREADS) mine += s->tot_mass[i];
        mine = block_sum64(mine, s->red);
        const Mail *all = row.g.exchange(Mail{mine, 0, 0, 0});
        u64 total = 0;
#pragma unroll
        for (int r = 0; r < C; ++r) total += all[r].a;
        target = fmax(frac * (double)total, 0.5);
        f = row.search(true, target, -1.0, 0, 0);
      }
      const auto bd = row.settle([&](float v, uint32_t) { return bin_of(v) == f.bin; }, f, true, target, true);
      vkey = bd.key; ties = bd.ties; equal = bd.equal;
    }
  }
  // ---- the draw, in id order: warp w of CTA r owns a run of ids
  constexpr int N = 16 / sizeof(T);
  const int run = ((row.n + WARPS - 1) / WARPS + N - 1) / N * N, i0 = min(row.n, warp * run), i1 = min(row.n, i0 + run);
  const bool count_eq = ties < equal;                        // only some ids of the least value are kept
  u64 eq_before = 0;
  if (count_eq) {
    uint32_t c = 0;
    for (int i = i0 + lane; i < i1; i += 32) c += key_of(clean(to_f(row.x[i]))) == vkey;
    c = __reduce_add_sync(0xffffffffu, c);
    if (lane == 0)
      for (int r = 0; r < C; ++r) *row.g.peer(&s->warp_eq[row.g.rank * WARPS + warp], r) = c;
    row.g.sync();
    for (int i = 0; i < row.g.rank * WARPS + warp; ++i) eq_before += s->warp_eq[i];
  }
  // the weight of a kept id (0: not kept); eq counts ids of the least value before it.  32 consecutive ids per call.
  auto kept_weight = [&](int i, u64 &eq, bool &is_kept) -> u64 {
    const float v = i < i1 ? clean(to_f(row.x[i])) : -INFINITY;
    const uint32_t key = key_of(v);
    bool keep = v > -INFINITY && key >= vkey;
    if (count_eq) {
      const unsigned same = __ballot_sync(0xffffffffu, v > -INFINITY && key == vkey);
      if (key == vkey) keep = keep && eq + __popc(same & ((1u << lane) - 1)) < ties;
      eq += __popc(same);
    }
    is_kept = keep;
    if (!keep) return 0;
    const double w = row.w_of(v);
    is_kept = w > 0.0 && w >= min_w;
    return is_kept ? row.q_of(w) : 0;
  };
  u64 mine = 0, eq = eq_before;
  uint32_t n_kept = 0;
  for (int i = i0; i < i1; i += 32) { bool kp; mine += kept_weight(i + lane, eq, kp); n_kept += kp; }
  mine = warp_sum64(mine);
  n_kept = __reduce_add_sync(0xffffffffu, n_kept);
  if (lane == 0)
    for (int r = 0; r < C; ++r) { *row.g.peer(&s->warp_mail[row.g.rank * WARPS + warp], r) = mine; }
  const u64 cta_kept = block_sum64(lane == 0 ? n_kept : 0, s->red);
  const Mail *all = row.g.exchange(Mail{cta_kept, 0, 0, 0});
  u64 total = 0, before = 0, kept = 0;
  for (int i = 0; i < C * WARPS; ++i) { if (i < row.g.rank * WARPS + warp) before += s->warp_mail[i]; total += s->warp_mail[i]; }
#pragma unroll
  for (int r = 0; r < C; ++r) kept += all[r].a;
  const float uc = u_ > 0.f ? fminf(u_, 0.99999994f) : 0.f;
  const u64 target = (u64)((double)uc * (double)total);      // cumulative > u * total, both whole: cumulative > floor
  if (before <= target && target < before + mine) {
    eq = eq_before;
    u64 at = before;
    for (int i = i0; i < i1; i += 32) {
      bool kp;
      const u64 q = kept_weight(i + lane, eq, kp);
      u64 inc = q;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) { const u64 t = __shfl_up_sync(0xffffffffu, inc, o); if (lane >= o) inc += t; }
      const unsigned hit = __ballot_sync(0xffffffffu, q > 0 && at + inc > target);
      if (hit) {
        if (lane == __ffs(hit) - 1) {
          a.tokens[b] = row.id0 + i + lane;
          if (a.prob) a.prob[b] = (float)((double)q / (double)total);
        }
        break;
      }
      at += __shfl_sync(0xffffffffu, inc, 31);
    }
  }
  if (row.g.rank == 0 && tid == 0 && a.kept) a.kept[b] = (int)kept;
  row.g.sync();                                              // no CTA leaves while a peer may still read its memory
}

template <class T, int C>
int launch_t(b200_ctx *ctx, const GivenArgs &a, size_t batch, size_t smem) {
  static std::atomic<unsigned long long> attr{0};
  const unsigned long long bit = 1ull << (ctx->device & 63);
  if (!(attr.load() & bit)) { B200_CUDA(ctx, cudaFuncSetAttribute(sample_given_kernel<T, C>, cudaFuncAttributeMaxDynamicSharedMemorySize, 220 * 1024)); attr.fetch_or(bit); }
  B200_CUDA(ctx, launch_k(ctx, sample_given_kernel<T, C>, dim3((unsigned)(batch * C)), dim3(THREADS), smem, C > 1 ? C : 0, a));
  B200_LAUNCHED(ctx);
  return B200_OK;
}

}  // namespace

extern "C" int b200_sample_given(b200_ctx *ctx, const void *logits, b200_dtype dt, size_t batch, size_t vocab, size_t ld, const float *temperature,
                                 const int32_t *top_k, const float *top_p, const float *min_p, const float *uniform, int32_t *out_tokens,
                                 int32_t *out_kept, float *out_prob) {
  if (!ctx) return B200_ERR_INVALID;
  B200_REQUIRE(ctx, dt == B200_F32 || dt == B200_BF16, "sample_given: unknown dtype");
  if (batch == 0) return B200_OK;
  B200_REQUIRE(ctx, logits && uniform && out_tokens, "sample_given: null pointer");
  B200_REQUIRE(ctx, vocab >= 1 && vocab <= ((size_t)1 << 24) && ld >= vocab, "sample_given: vocabulary of 1 .. 2^24 ids, rows at least that long");
  B200_REQUIRE(ctx, batch <= ((size_t)1 << 24), "sample_given: at most 2^24 rows");
  DeviceGuard guard(ctx);
  B200_REQUIRE(ctx, guard.ok, "sample_given: the context's device cannot be selected");
  GivenArgs a = {};
  a.logits = logits; a.ld = (long long)ld; a.V = (int)vocab;
  a.temperature = temperature; a.top_k = top_k; a.top_p = top_p; a.min_p = min_p; a.uniform = uniform;
  a.tokens = out_tokens; a.kept = out_kept; a.prob = out_prob;
  int bits = 0;
  while (((size_t)1 << bits) < vocab) ++bits;
  a.fixed_bits = std::min(44, 62 - bits);
  // CTAs per row: until the rows fill the SMs twice (two CTAs share one), not below 1024 ids each, and more where a slice would not fit
  const size_t es = dtype_size(dt), room = 220 * 1024 - sizeof(Shared) - 64;
  int C = 1;
  while (C < MAX_CLUSTER && (batch * C < (size_t)ctx->sm_count || vocab * es / C > room / 2) && vocab / C > 2048) C *= 2;
  a.slice = (int)(((vocab + C - 1) / C + 15) / 16 * 16);
  a.in_smem = (size_t)a.slice * es <= room;
  const size_t smem = ((sizeof(Shared) + 15) & ~(size_t)15) + (a.in_smem ? (size_t)a.slice * es : 0);
  if (dt == B200_BF16) return C == 1 ? launch_t<bf16, 1>(ctx, a, batch, smem) : C == 2 ? launch_t<bf16, 2>(ctx, a, batch, smem) : C == 4 ? launch_t<bf16, 4>(ctx, a, batch, smem) : launch_t<bf16, 8>(ctx, a, batch, smem);
  return C == 1 ? launch_t<float, 1>(ctx, a, batch, smem) : C == 2 ? launch_t<float, 2>(ctx, a, batch, smem) : C == 4 ? launch_t<float, 4>(ctx, a, batch, smem) : launch_t<float, 8>(ctx, a, batch, smem);
}
