// Sampling from given random numbers: per-row temperature, top-k, top-p and min-p, the id by inversion of the cumulative
// weights.  Beside b200_sample (one setting for all rows, its own random numbers, cpp/python rules of the reference).
//
//   w_i = exp((l_i - max l) / T); ids in the order (l descending, id ascending); top-k keeps the first k; top-p keeps a survivor
//   while the weight before it is below p x the weight of all top-k survivors; min-p keeps w_i >= min_p; the id is the least
//   kept one whose cumulative kept weight (in id order) exceeds u x the kept weight.
//
// The answer is a whole number, so it has to be the right one and not nearly so: weights that decide are computed in 64 bits and
// added as fixed-point integers (2^-44 of the largest weight at up to 2^18 ids), which makes every sum exact and independent of order.
// Nothing is sorted.  A cluster of CTAs holds a row, each its slice in shared memory (one read of the logits).
//   * A histogram of 2048 value bins below the maximum counts ids (32-bit arithmetic only) and gives the bin of the k-th id.
//   * Where that leaves at most 256 candidates, the first CTA ranks them against each other and does everything else among them.
//   * top-p otherwise: the counts and the bins' edges bound the border between two bins; one pass adds the exact weights above and
//     in all, and builds a second, finer histogram, of weights, between the bounds alone (weights in all 2048 bins cost three
//     shared-memory atomics per id, 12 us at 32 x 100256).
//   * The ids of a border's bin are ranked against each other; a bin with more ids than the list holds is cut again by the bits of
//     its values, at most three times; equal values are settled by arithmetic.
// The kept set is a prefix of the order: a least value and the number of ids of that value, lowest ids first.
// Bound by latency at usual sizes (five to ten exchanges within the cluster) and by the 64-bit exponentials for large vocabularies;
// the floor is one read of the logits.
#include "paged_common.cuh"
#include <algorithm>
#include <atomic>
#include <cooperative_groups.h>

namespace cg = cooperative_groups;

namespace {

constexpr int THREADS = 512, WARPS = THREADS / 32, BINS = 2048, PER = BINS / THREADS, LIST = 512, SMALL = 256, MAX_CLUSTER = 8;
static_assert(LIST <= THREADS && PER == 4, "one list entry and one 16-byte vector of bins a thread");
constexpr float RANGE = 32.0f;            // in units of the temperature: below max - 32 T a weight is under half of 2^-44
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

struct alignas(16) Entry { uint32_t key, id; u64 q; };
struct alignas(16) Mail { u64 a, b; };
struct Found { u64 above_c, above_m, cnt, mass; int bin; };
struct alignas(16) Shared {
  uint32_t cnt[BINS], lo[BINS], hi[BINS];    // this CTA's histogram; a bin's weight is hi : lo
  Entry list[LIST];
  double table[64];                          // 2^(j / 64)
  Mail mail[2][MAX_CLUSTER];
  Mail warp_mail[MAX_CLUSTER * WARPS];
  uint32_t warp_eq[MAX_CLUSTER * WARPS];
  u64 red[WARPS], red2[WARPS], sums[2], res[4];
  Found found;
  int bounds[2];
  int list_n;
};

__device__ __forceinline__ uint32_t key_of(float x) { const uint32_t b = __float_as_uint(x); return b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u); }
__device__ __forceinline__ float value_of(uint32_t k) { return __uint_as_float(k & 0x80000000u ? k ^ 0x80000000u : ~k); }
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

template <class V> __device__ __forceinline__ V warp_add(V v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
__device__ __forceinline__ u64 block_add(u64 v, u64 *red) {
  v = warp_add(v);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  u64 t = 0;
#pragma unroll
  for (int i = 0; i < WARPS; ++i) t += red[i];
  return t;
}
__device__ __forceinline__ void block_max2(uint32_t &a, uint32_t &b, u64 *red) {
  a = __reduce_max_sync(0xffffffffu, a); b = __reduce_max_sync(0xffffffffu, b);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = ((u64)a << 32) | b;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < WARPS; ++i) { a = max(a, (uint32_t)(red[i] >> 32)); b = max(b, (uint32_t)red[i]); }
}
// exclusive prefixes over the threads, and the totals, of two values
template <class V>
__device__ __forceinline__ void block_scan2(V &a, V &b, V &sum_a, V &sum_b, V *red, V *red2) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  V ia = a, ib = b;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const V ta = __shfl_up_sync(0xffffffffu, ia, o), tb = __shfl_up_sync(0xffffffffu, ib, o);
    if (lane >= o) { ia += ta; ib += tb; }
  }
  __syncthreads();
  if (lane == 31) { red[warp] = ia; red2[warp] = ib; }
  __syncthreads();
  V before_a = 0, before_b = 0;
  sum_a = sum_b = 0;
#pragma unroll
  for (int i = 0; i < WARPS; ++i) {
    if (i < warp) { before_a += red[i]; before_b += red2[i]; }
    sum_a += red[i]; sum_b += red2[i];
  }
  a = before_a + ia - a; b = before_b + ib - b;
}

// The CTAs of a row.
template <int C>
struct Group {
  Shared *s;
  int rank, par;
  __device__ __forceinline__ void sync() { if constexpr (C > 1) cg::this_cluster().sync(); else __syncthreads(); }
  template <class P> __device__ __forceinline__ P *peer(P *p, int r) { if constexpr (C > 1) return cg::this_cluster().map_shared_rank(p, r); else return p; }
  // Every CTA posts one Mail; all see all.  Two mailboxes in turn: a CTA cannot be two exchanges ahead of a peer that still reads.
  __device__ __forceinline__ const Mail *exchange(u64 a, u64 b) {
    par ^= 1;
    if (threadIdx.x < C) *peer(&s->mail[par][rank], threadIdx.x) = Mail{a, b};
    sync();
    return s->mail[par];
  }
};

struct Border { uint32_t key; u64 ties, equal, mass; };   // least kept value; kept ids of it, all ids of it; weight of the kept prefix

template <class T, int C>
struct Row {
  Group<C> g;
  Shared *s;
  const T *x;          // this CTA's slice
  int n, id0;          // ids in the slice, first id
  float mx, far, scale;   // far: values below mx - far have weight 0; scale: bins per unit of the logits
  double z_scale, one;    // log2(e) / T; the weight 1 in fixed point

  __device__ __forceinline__ double w_of(float v) const { return v == mx ? 1.0 : weight(((double)v - (double)mx) * z_scale, s->table); }
  // exp(..) > 0 in 64 bits; weight() gives 0 from 2^-1020 on, which no sum and no min_p (a 32-bit number) can tell from 0
  __device__ __forceinline__ bool positive(float v) const { return v == mx || ((double)v - (double)mx) * z_scale > -1075.0; }
  __device__ __forceinline__ u64 q_of(double w) const { return (u64)(w * one + 0.5); }
  __device__ __forceinline__ u64 q_at(float v) const { return v == mx || mx - v < far ? q_of(w_of(v)) : 0; }
  // distance from the maximum in bins; what lies behind the last bin is in it
  __device__ __forceinline__ float t_of(float v) const { const float t = v == mx ? 0.f : (mx - v) * scale; return t < (float)(BINS - 1) ? t : (float)(BINS - 1); }

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
    const uint4 z = make_uint4(0, 0, 0, 0);
    reinterpret_cast<uint4 *>(s->cnt)[threadIdx.x] = z; reinterpret_cast<uint4 *>(s->lo)[threadIdx.x] = z; reinterpret_cast<uint4 *>(s->hi)[threadIdx.x] = z;
  }
  __device__ __forceinline__ void add(int bin, u64 q) {
    atomicAdd(&s->cnt[bin], 1u);
    const uint32_t l = (uint32_t)q;
    uint32_t h = (uint32_t)(q >> 32);
    if (l && atomicAdd(&s->lo[bin], l) > 0xffffffffu - l) ++h;
    if (h) atomicAdd(&s->hi[bin], h);
  }
  // The cluster's sums of this thread's PER bins (call after a sync; the histograms must stay until the next one).
  __device__ __forceinline__ void counts(u64 (&c)[PER]) {
#pragma unroll
    for (int j = 0; j < PER; ++j) c[j] = 0;
#pragma unroll
    for (int r = 0; r < C; ++r) {
      const uint4 v = reinterpret_cast<const uint4 *>(g.peer(s->cnt, r))[threadIdx.x];
      c[0] += v.x; c[1] += v.y; c[2] += v.z; c[3] += v.w;
    }
  }
  __device__ __forceinline__ void weights(u64 (&m)[PER]) {
#pragma unroll
    for (int j = 0; j < PER; ++j) m[j] = 0;
#pragma unroll
    for (int r = 0; r < C; ++r) {
      const uint4 l = reinterpret_cast<const uint4 *>(g.peer(s->lo, r))[threadIdx.x], h = reinterpret_cast<const uint4 *>(g.peer(s->hi, r))[threadIdx.x];
      m[0] += ((u64)h.x << 32) + l.x; m[1] += ((u64)h.y << 32) + l.y; m[2] += ((u64)h.z << 32) + l.z; m[3] += ((u64)h.w << 32) + l.w;
    }
  }
  // The bin where the running total from the top reaches the target: above < target <= above + bin.  Every CTA finds it for itself.
  __device__ Found search(const u64 (&c)[PER], const u64 (&m)[PER], bool by_mass, double target, u64 start_c, u64 start_m) {
    u64 bc = 0, bm = 0, sc, sm;
#pragma unroll
    for (int j = 0; j < PER; ++j) { bc += c[j]; bm += m[j]; }
    block_scan2<u64>(bc, bm, sc, sm, s->red, s->red2);
    bc += start_c; bm += start_m;
#pragma unroll
    for (int j = 0; j < PER; ++j) {
      const double lo = by_mass ? (double)bm : (double)bc, hi = by_mass ? (double)(bm + m[j]) : (double)(bc + c[j]);
      if (c[j] && lo < target && target <= hi) s->found = Found{bc, bm, c[j], m[j], (int)threadIdx.x * PER + j};
      bc += c[j]; bm += m[j];
    }
    __syncthreads();
    const Found f = s->found;
    __syncthreads();
    return f;
  }

  // Sends the ids that `member` selects to the first CTA's list; returns after the list is complete.
  template <class M> __device__ __forceinline__ void gather(M member) {
    Shared *first = g.peer(s, 0);
    each([&](float v, int i) {
      const uint32_t k = key_of(v);
      if (v > -INFINITY && member(v, k)) {
        const int at = atomicAdd(&first->list_n, 1);
        if (at < LIST) *reinterpret_cast<uint2 *>(&first->list[at]) = make_uint2(k, (uint32_t)(id0 + i));
      }
    });
    g.sync();
  }
  // The first CTA: each entry's weight, then the ids and the weight ahead of this thread's entry in the order.  All its threads call.
  __device__ __forceinline__ int rank_list(Entry &e, u64 &ahead_c, u64 &ahead_m, u64 &eq_ahead, u64 &equal) {
    const int n_list = min(s->list_n, LIST), i = threadIdx.x;
    e = Entry{0, 0, 0};
    if (i < n_list) { e = s->list[i]; e.q = q_at(value_of(e.key)); s->list[i].q = e.q; }
    __syncthreads();
    ahead_c = ahead_m = eq_ahead = equal = 0;
    if (i < n_list) {
      uint32_t c = 0, q = 0, eq = 0;
#pragma unroll 4
      for (int j = 0; j < n_list; ++j) {
        const Entry o = s->list[j];
        const bool same = o.key == e.key, ahead = o.key > e.key || (same && o.id < e.id);
        c += ahead; q += same && ahead; eq += same;
        ahead_m += ahead ? o.q : 0;
      }
      ahead_c = c; eq_ahead = q; equal = eq;
    }
    return n_list;
  }

  // Settles the border inside a bin.  `member(value, key)` selects the bin's ids; the list must be empty (and is again afterwards).
  template <class M>
  __device__ Border settle(M member, Found f, bool by_mass, double target) {
    bool narrowed = false;
    uint32_t kl = 0, kh = 0xffffffffu;
    for (int round = 0; round < 5; ++round) {
      if (f.cnt <= LIST) {
        if (narrowed) gather([&](float, uint32_t k) { return k >= kl && k <= kh; });
        else gather(member);
        if (g.rank == 0) {
          Entry e;
          u64 rc, rm, eq_before, equal;
          const int n_list = rank_list(e, rc, rm, eq_before, equal);
          rc += f.above_c; rm += f.above_m;
          const double lo = by_mass ? (double)rm : (double)rc, hi = by_mass ? (double)(rm + e.q) : (double)(rc + 1);
          if ((int)threadIdx.x < n_list && lo < target && target <= hi) {
#pragma unroll
            for (int r = 0; r < C; ++r) { u64 *o = g.peer(s->res, r); o[0] = e.key; o[1] = eq_before + 1; o[2] = equal; o[3] = rm + e.q; }
          }
          if (threadIdx.x == 0) s->list_n = 0;
        }
        g.sync();
        return Border{(uint32_t)s->res[0], s->res[1], s->res[2], s->res[3]};
      }
      if (!narrowed) {                                      // the bin's range of values
        uint32_t h = 0, l = 0;                              // l holds ~key
        each([&](float v, int) { const uint32_t k = key_of(v); if (v > -INFINITY && member(v, k)) { h = max(h, k); l = max(l, ~k); } });
        block_max2(h, l, s->red);
        const Mail *all = g.exchange(h, l);
#pragma unroll
        for (int r = 0; r < C; ++r) { h = max(h, (uint32_t)all[r].a); l = max(l, (uint32_t)all[r].b); }
        kh = h; kl = ~l; narrowed = true;
      }
      if (kl == kh) {                                       // equal values
        const u64 q = q_at(value_of(kl));
        u64 t;
        if (by_mass) {
          const double need = target - (double)f.above_m;
          t = q ? (u64)ceil(need / (double)q) : 1;
          t = t < 1 ? 1 : t > f.cnt ? f.cnt : t;
        } else t = (u64)target - f.above_c;
        return Border{kl, t, f.cnt, f.above_m + t * q};
      }
      const int sh = max(0, 21 - __clz(kh - kl));           // (kh - kl) >> sh is below 2048
      g.sync();                                             // all have read the histograms that go now
      clear();
      __syncthreads();
      each([&](float v, int) {
        const uint32_t k = key_of(v);
        if (v > -INFINITY && k >= kl && k <= kh) add((int)((kh - k) >> sh), q_at(v));
      });
      g.sync();
      u64 c[PER], m[PER];
      counts(c); weights(m);
      f = search(c, m, by_mass, target, f.above_c, f.above_m);
      const uint32_t top = kh - ((uint32_t)f.bin << sh);
      const u64 low = (u64)((uint32_t)f.bin + 1) << sh;
      kl = low > (u64)(kh - kl) ? kl : kh - (uint32_t)low + 1;
      kh = top;
    }
    return Border{kl, f.cnt, f.cnt, f.above_m + f.mass};    // not reached: three cuts leave one value
  }
};

template <class T, int C>
__global__ void __launch_bounds__(THREADS, 1)
sample_given_kernel(GivenArgs a) {
  pdl_launch_dependents();
  pdl_wait();
  extern __shared__ __align__(16) uint8_t dyn[];
  Shared *s = (Shared *)dyn;
  T *copy = (T *)(dyn + sizeof(Shared));
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, b = blockIdx.x / C;
  Row<T, C> row;
  row.s = s; row.g.s = s; row.g.par = 0; row.one = (double)(1ll << a.fixed_bits);
  row.g.rank = C > 1 ? (int)(blockIdx.x % C) : 0;
  row.id0 = min(a.V, row.g.rank * a.slice); row.n = min(a.V, row.id0 + a.slice) - row.id0;
  row.x = (const T *)a.logits + (size_t)b * a.ld + row.id0;
  const float T_ = a.temperature ? a.temperature[b] : 1.0f, p = a.top_p ? a.top_p[b] : 1.f, mp = a.min_p ? a.min_p[b] : 0.f, u_ = a.uniform[b];
  const int k = a.top_k ? a.top_k[b] : 0;
  if (tid < 64) s->table[tid] = exp2(tid * 0.015625);
  if (tid == 0) s->list_n = 0;
  row.clear();
  // ---- one read of the slice: a copy in shared memory, the largest and the smallest finite value
  uint32_t hi = 0, lo = 0;
  {
    constexpr int N = 16 / sizeof(T);
    auto see = [&](float v) { if (v > -INFINITY) { const uint32_t key = key_of(v); hi = max(hi, key); lo = max(lo, ~key); } };
    if (((uintptr_t)row.x & 15) == 0) {
      const int nv = row.n / N;
      constexpr int U = 4;                                   // loads in flight
      for (int i0 = tid; i0 < nv; i0 += U * THREADS) {
        Vec16<T> v[U];
#pragma unroll
        for (int j = 0; j < U; ++j) if (i0 + j * THREADS < nv) v[j].load(row.x + (size_t)(i0 + j * THREADS) * N);
#pragma unroll
        for (int j = 0; j < U; ++j)
          if (i0 + j * THREADS < nv) {
            float e[N];
            v[j].unpack(e);
#pragma unroll
            for (int y = 0; y < N; ++y) { e[y] = clean(e[y]); see(e[y]); }
            if (a.in_smem) { v[j].pack(e); v[j].store(copy + (size_t)(i0 + j * THREADS) * N); }
          }
      }
      for (int i = nv * N + tid; i < row.n; i += THREADS) { const float v = clean(to_f(row.x[i])); see(v); if (a.in_smem) copy[i] = from_f<T>(v); }
    } else {
      for (int i = tid; i < row.n; i += THREADS) { const float v = clean(to_f(row.x[i])); see(v); if (a.in_smem) copy[i] = from_f<T>(v); }
    }
  }
  block_max2(hi, lo, s->red);
  if (a.in_smem) row.x = copy;
  if (C > 1) {
    row.g.sync();                                            // every CTA of the cluster runs before its memory is written
    const Mail *all = row.g.exchange(hi, lo);
#pragma unroll
    for (int r = 0; r < C; ++r) { hi = max(hi, (uint32_t)all[r].a); lo = max(lo, (uint32_t)all[r].b); }
  }
  if (hi == 0) {                                             // nothing to draw from
    if (row.g.rank == 0 && tid == 0) { a.tokens[b] = -1; if (a.kept) a.kept[b] = 0; if (a.prob) a.prob[b] = 0.f; }
    row.g.sync();
    return;
  }
  row.mx = value_of(hi);
  const float mn = value_of(~lo);
  if (!(T_ > 0.f)) {                                         // greedy: the lowest id of the maximum
    uint32_t best = 0, none = 0;                             // ~id
    row.each([&](float v, int i) { if (v == row.mx) best = max(best, ~(uint32_t)(row.id0 + i)); });
    block_max2(best, none, s->red);
    const Mail *all = row.g.exchange(best, 0);
#pragma unroll
    for (int r = 0; r < C; ++r) best = max(best, (uint32_t)all[r].a);
    if (row.g.rank == 0 && tid == 0) { a.tokens[b] = (int)~best; if (a.kept) a.kept[b] = 1; if (a.prob) a.prob[b] = 1.f; }
    row.g.sync();
    return;
  }
  row.z_scale = 1.44269504088896340736 / (double)T_;
  row.far = RANGE * T_;
  const bool by_k = k > 0 && k < a.V, by_p = p < 1.f;
  const double min_w = mp > 0.f ? fmin((double)mp, 1.0) : 0.0, frac = p > 0.f ? (double)p : 0.0;      // p <= 0 keeps the first id
  const double u = u_ > 0.f ? (double)fminf(u_, 0.99999994f) : 0.0;
  // ---- the kept prefix
  uint32_t vkey = 0;                                         // keep keys above it, and `ties` of the ids that have it
  u64 ties = 0, equal = 0;
  if (by_k || by_p) {
    const float range = fminf(row.mx - mn, row.far);
    row.scale = range > 0.f && range < INFINITY ? (float)(BINS - 1) / range : 0.f;
    if (!(row.scale < INFINITY)) row.scale = 0.f;            // a temperature next to 0: one bin, cut by the bits of the values
    row.each([&](float v, int) { if (v > -INFINITY) atomicAdd(&s->cnt[(int)row.t_of(v)], 1u); });
    row.g.sync();
    u64 c[PER], zero[PER] = {0, 0, 0, 0};
    row.counts(c);
    bool have_k = false;
    u64 mass_k = 0;
    int last_bin = BINS - 1;
    if (by_k) {
      u64 all_c = 0;
#pragma unroll
      for (int j = 0; j < PER; ++j) all_c += c[j];
      if ((u64)k < block_add(all_c, s->red)) {               // else fewer ids than k: nothing to cut
        const Found f = row.search(c, zero, false, (double)k, 0, 0);
        last_bin = f.bin;
        have_k = true;
        if (f.above_c + f.cnt <= SMALL) {
          // few candidates: the first CTA does the rest among them
          row.gather([&](float v, uint32_t) { return (int)row.t_of(v) <= f.bin; });
          if (row.g.rank == 0) {
            Entry e;
            u64 rank, before, d0, d1;
            const int n_list = row.rank_list(e, rank, before, d0, d1);
            const bool in_k = tid < n_list && rank < (u64)k;
            const u64 mass = block_add(in_k ? e.q : 0, s->red);
            const double w = in_k ? row.w_of(value_of(e.key)) : 0.0;
            const bool keep = in_k && (!by_p || rank == 0 || (double)before < frac * (double)mass) && row.positive(value_of(e.key)) && w >= min_w;
            const u64 mine = keep ? e.q : 0, total = block_add(mine, s->red);
            if (tid < n_list) s->list[tid].q = mine;
            const u64 n_kept = block_add(keep, s->red);      // its barriers order the list's new weights before the loop
            const u64 target = (u64)(u * (double)total);
            if (mine) {
              u64 at = 0;
              for (int j = 0; j < n_list; ++j) { const Entry o = s->list[j]; at += o.id < e.id ? o.q : 0; }
              if (at <= target && target < at + mine) {
                a.tokens[b] = (int)e.id;
                if (a.prob) a.prob[b] = (float)((double)mine / (double)total);
              }
            }
            if (tid == 0 && a.kept) a.kept[b] = (int)n_kept;
          }
          return;                                            // nobody reads another CTA's memory any more
        }
        const Border bd = row.settle([&](float v, uint32_t) { return (int)row.t_of(v) == f.bin; }, f, false, (double)k);
        vkey = bd.key; ties = bd.ties; equal = bd.equal;
      }
    }
    if (by_p) {
      // Bounds of the border from counts and edges.  A bin's weights lie between those of its edges (2^-12 more on either side covers the
      // rounding of the edges and of the sums); the last bin has no lower edge; a cut by k may take any part of its bin.
      double up = 0.0, dn = 0.0, u4[PER], d4[PER], sum_up, sum_dn;
      const float step = row.scale > 0.f ? (float)(row.z_scale) / row.scale : 0.f;
#pragma unroll
      for (int j = 0; j < PER; ++j) {
        const int bin = tid * PER + j;
        const double n_bin = bin <= last_bin ? (double)c[j] : 0.0;
        u4[j] = n_bin * (row.scale > 0.f ? (double)exp2f(-step * (float)bin) * (1.0 + 0x1p-12) : 1.0);
        d4[j] = bin < last_bin && bin < BINS - 1 && row.scale > 0.f ? n_bin * (double)exp2f(-step * (float)(bin + 1)) * (1.0 - 0x1p-12) : 0.0;
        up += u4[j]; dn += d4[j];
      }
      block_scan2<double>(up, dn, sum_up, sum_dn, (double *)s->red, (double *)s->red2);
      if (tid == 0) { s->bounds[0] = last_bin; s->bounds[1] = last_bin; }
      __syncthreads();
      const double want_lo = frac * sum_dn * (1.0 - 0x1p-12), want_hi = frac * sum_up * (1.0 + 0x1p-12);
      int first_up = BINS, first_dn = BINS;                  // the first bins where the running totals reach the bounds
#pragma unroll
      for (int j = PER - 1; j >= 0; --j) {
        double at_up = up, at_dn = dn;
#pragma unroll
        for (int y = 0; y <= j; ++y) { at_up += u4[y]; at_dn += d4[y]; }
        if (at_up >= want_lo) first_up = tid * PER + j;
        if (at_dn >= want_hi) first_dn = tid * PER + j;
      }
      first_up = __reduce_min_sync(0xffffffffu, first_up); first_dn = __reduce_min_sync(0xffffffffu, first_dn);
      if (lane == 0) { atomicMin(&s->bounds[0], first_up); atomicMin(&s->bounds[1], first_dn); }
      __syncthreads();
      const int b0 = s->bounds[0], b1 = max(b0, s->bounds[1]);
      const float fine = (float)(BINS / (b1 - b0 + 1));
      auto fine_bin = [&](float v) { return min(BINS - 1, (int)((row.t_of(v) - (float)b0) * fine)); };
      auto between = [&](float v, uint32_t key) { const int bin = (int)row.t_of(v); return bin >= b0 && bin <= b1 && key >= vkey; };
      row.g.sync();                                          // all have read the counts
      row.clear();
      __syncthreads();
      u64 above = 0, all_q = 0, above_c = 0;
      row.each([&](float v, int) {
        const uint32_t key = key_of(v);
        if (!(v > -INFINITY) || key < vkey) return;
        const int bin = (int)row.t_of(v);
        const u64 q = row.q_at(v);
        if (!have_k || key > vkey) all_q += q;
        if (bin < b0) { above += q; ++above_c; }
        else if (bin <= b1) row.add(fine_bin(v), q);
      });
      above = block_add(above, s->red); all_q = block_add(all_q, s->red);
      const Mail *all = row.g.exchange(above, all_q);        // its sync also completes the histograms
      above = all_q = 0;
#pragma unroll
      for (int r = 0; r < C; ++r) { above += all[r].a; all_q += all[r].b; }
      if (have_k) all_q += ties * row.q_at(value_of(vkey));
      const double target = fmax(frac * (double)all_q, 0.5);
      u64 m[PER];
      row.counts(c); row.weights(m);
      const Found f = row.search(c, m, true, target, 0, above);
      const Border bd = row.settle([&](float v, uint32_t key) { return between(v, key) && fine_bin(v) == f.bin; }, f, true, target);
      vkey = bd.key; ties = bd.ties; equal = bd.equal;
    }
  }
  // ---- the draw, in id order: warp w of CTA r owns a run of ids
  constexpr int N = 16 / sizeof(T);
  const int run = ((row.n + WARPS - 1) / WARPS + N - 1) / N * N, i0 = min(row.n, warp * run), i1 = min(row.n, i0 + run), slot = row.g.rank * WARPS + warp;
  const bool count_eq = ties < equal;                        // only some ids of the least value are kept
  u64 eq_before = 0;
  if (count_eq) {
    uint32_t c = 0;
    for (int i = i0 + lane; i < i1; i += 32) c += key_of(clean(to_f(row.x[i]))) == vkey;
    c = __reduce_add_sync(0xffffffffu, c);
    if (lane < C) *row.g.peer(&s->warp_eq[slot], lane) = c;
    row.g.sync();
    for (int i = lane; i < slot; i += 32) eq_before += s->warp_eq[i];
    eq_before = warp_add(eq_before);
  }
  auto weigh = [&](float v, bool keep, uint32_t &n_kept) -> u64 {
    if (!keep) return 0;
    const bool near = v == row.mx || row.mx - v < row.far;
    if (min_w == 0.0 && !near) { n_kept += row.positive(v); return 0; }
    const double w = row.w_of(v);
    if (w < min_w) return 0;
    n_kept += row.positive(v);
    return near ? row.q_of(w) : 0;
  };
  // the weight of a kept id (0: not kept); eq counts ids of the least value before it.  32 consecutive ids per call.
  auto ordered = [&](int i, u64 &eq, uint32_t &n_kept) -> u64 {
    const float v = i < i1 ? clean(to_f(row.x[i])) : -INFINITY;
    const uint32_t key = key_of(v);
    bool keep = v > -INFINITY && key >= vkey;
    if (count_eq) {
      const unsigned same = __ballot_sync(0xffffffffu, v > -INFINITY && key == vkey);
      if (key == vkey) keep = keep && eq + __popc(same & ((1u << lane) - 1)) < ties;
      eq += __popc(same);
    }
    return weigh(v, keep, n_kept);
  };
  u64 mine = 0, eq = eq_before;
  uint32_t n_kept = 0;
  if (count_eq || ((uintptr_t)row.x & 15)) {
    for (int i = i0; i < i1; i += 32) mine += ordered(i + lane, eq, n_kept);
  } else {                                                   // every id of the least value is kept: any order
    for (int i = i0 + lane * N; i < i1; i += 32 * N) {
      if (i + N <= i1) {
        Vec16<T> v;
        float e[N];
        v.load(row.x + i); v.unpack(e);
#pragma unroll
        for (int j = 0; j < N; ++j) { const float y = clean(e[j]); mine += weigh(y, y > -INFINITY && key_of(y) >= vkey, n_kept); }
      } else {
        for (int j = i; j < i1; ++j) { const float y = clean(to_f(row.x[j])); mine += weigh(y, y > -INFINITY && key_of(y) >= vkey, n_kept); }
      }
    }
  }
  mine = warp_add(mine);
  n_kept = __reduce_add_sync(0xffffffffu, n_kept);
  if (lane < C) *row.g.peer(&s->warp_mail[slot], lane) = Mail{mine, n_kept};
  row.g.sync();
  u64 before = 0, total = 0, kept = 0;
  for (int i = lane; i < C * WARPS; i += 32) { const Mail m = s->warp_mail[i]; if (i < slot) before += m.a; total += m.a; kept += m.b; }
  before = warp_add(before); total = warp_add(total); kept = warp_add(kept);
  const u64 target = (u64)(u * (double)total);               // cumulative > u * total, the cumulative whole: > its floor
  if (before <= target && target < before + mine) {
    eq = eq_before;
    u64 at = before;
    for (int i = i0; i < i1; i += 32) {
      const u64 q = ordered(i + lane, eq, n_kept);
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
  if (slot == 0 && lane == 0 && a.kept) a.kept[b] = (int)kept;
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
  // CTAs per row: as many as still run at once, one per SM (clusters of eight fit 15 times on 148 SMs, of four 32 times), not below 1024
  // ids each; more where a slice would not fit in shared memory.  At 32 x 100256 in 32 bits, clusters of eight ran in three waves (96 us).
  const size_t es = dtype_size(dt), room = 220 * 1024 - sizeof(Shared);
  auto fit = [&](int C) { return (size_t)(C == 2 ? ctx->sm_count : C == 4 ? ctx->sm_count - 20 : ctx->sm_count - 28); };
  int C = 1;
  while (C < MAX_CLUSTER && (batch * 2 * C <= fit(2 * C) || vocab * es / C > room) && vocab / C > 2048) C *= 2;
  a.slice = (int)(((vocab + C - 1) / C + 15) / 16 * 16);
  a.in_smem = (size_t)a.slice * es <= room;
  const size_t smem = sizeof(Shared) + (a.in_smem ? (size_t)a.slice * es : 0);
  if (dt == B200_BF16) return C == 1 ? launch_t<bf16, 1>(ctx, a, batch, smem) : C == 2 ? launch_t<bf16, 2>(ctx, a, batch, smem) : C == 4 ? launch_t<bf16, 4>(ctx, a, batch, smem) : launch_t<bf16, 8>(ctx, a, batch, smem);
  return C == 1 ? launch_t<float, 1>(ctx, a, batch, smem) : C == 2 ? launch_t<float, 2>(ctx, a, batch, smem) : C == 4 ? launch_t<float, 4>(ctx, a, batch, smem) : launch_t<float, 8>(ctx, a, batch, smem);
}
