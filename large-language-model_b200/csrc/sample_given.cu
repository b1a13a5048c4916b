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
// Bound by latency at usual sizes (64 rows of 32000 ids in bf16 with all filters: 13.9 us, five exchanges within the cluster) and by instructions, the
// 64-bit exponentials above all, for large vocabularies (32 rows of 100256 ids in 32 bits, nucleus alone: 38 us); the floor is one read of
// the logits (0.6 and 2 us).
#include "paged_common.cuh"
#include <algorithm>
#include <atomic>
#include <cfloat>
#include <cooperative_groups.h>

namespace cg = cooperative_groups;

namespace {

// 1024 threads at 64 registers: 512 at 128 take 56 us where these take 46 (32 x 100256).
constexpr int THREADS = 1024, WARPS = THREADS / 32, BINS = 2048, PER = BINS / THREADS, LIST = 512, SMALL = 256, HELD = 2048, CHUNK = 128, MAX_CLUSTER = 8;
static_assert(LIST <= THREADS && PER % 2 == 0, "one list entry and pairs of bins a thread");
constexpr float RANGE = 32.0f;            // in units of the temperature: from max - 32 T on a weight is under a quarter of 2^-44
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
  uint32_t coarse[BINS];                     // this CTA's counts below the maximum
  uint32_t cnt[BINS], lo[BINS], hi[BINS];    // its finer histogram; a bin's weight is hi : lo
  Entry list[LIST];
  uint2 held[HELD];                          // (key, id) of the ids between the bounds of top-p's border
  double table[64];                          // 2^(j / 64)
  Mail mail[2][MAX_CLUSTER];
  u64 red[WARPS], red2[WARPS], res[4];
  Found found;
  float edges[2];
  int bounds[2], list_n, held_n, pick_chunk;
  uint32_t last_id;
  u64 pick_before;
};

__device__ __forceinline__ uint32_t key_of(float x) { const uint32_t b = __float_as_uint(x); return b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u); }
__device__ __forceinline__ float value_of(uint32_t k) { return __uint_as_float(k & 0x80000000u ? k ^ 0x80000000u : ~k); }
// -0 is 0; NaN counts as masked
__device__ __forceinline__ float clean(float x) { return x == x ? x + 0.0f : -INFINITY; }

// 2^z2 for z2 in [-1020, 0]: 2^(k/64) from a table times the exponential series in (rest ln 2), |rest| <= 2^-7, to degree 5 (error 3e-17).
__device__ __forceinline__ double weight(double z2, const double *table) {
  constexpr double L = 0.69314718055994530942, L2 = L * L, L3 = L2 * L, L4 = L3 * L, L5 = L4 * L;
  const double shift = 6755399441055744.0;      // 1.5 * 2^52: adding it rounds to an integer held in the low bits
  const double t = fma(z2, 64.0, shift);
  const int k = __double2loint(t);
  const double r = fma(t - shift, -0.015625, z2);
  const double p = fma(r, fma(r, fma(r, fma(r, fma(r, L5 / 120, L4 / 24), L3 / 6), L2 / 2), L), 1.0);
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
  return warp_add((threadIdx.x & 31) < WARPS ? red[threadIdx.x & 31] : 0ull);
}
__device__ __forceinline__ void block_max2(uint32_t &a, uint32_t &b, u64 *red) {
  a = __reduce_max_sync(0xffffffffu, a); b = __reduce_max_sync(0xffffffffu, b);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = ((u64)a << 32) | b;
  __syncthreads();
  const u64 v = (threadIdx.x & 31) < WARPS ? red[threadIdx.x & 31] : 0ull;
  a = __reduce_max_sync(0xffffffffu, (uint32_t)(v >> 32)); b = __reduce_max_sync(0xffffffffu, (uint32_t)v);
}
// exclusive prefixes over the threads, and the totals, of two values
template <class V>
__device__ __forceinline__ void block_scan2(V &a, V &b, V &sum_a, V &sum_b, V *red, V *red2) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  auto scan = [&](V &x, V &y) {
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const V tx = __shfl_up_sync(0xffffffffu, x, o), ty = __shfl_up_sync(0xffffffffu, y, o);
      if (lane >= o) { x += tx; y += ty; }
    }
  };
  V ia = a, ib = b;
  scan(ia, ib);
  __syncthreads();
  if (lane == 31) { red[warp] = ia; red2[warp] = ib; }
  __syncthreads();
  V wa = lane < WARPS ? red[lane] : V(0), wb = lane < WARPS ? red2[lane] : V(0);
  scan(wa, wb);
  sum_a = __shfl_sync(0xffffffffu, wa, 31); sum_b = __shfl_sync(0xffffffffu, wb, 31);
  const V pa = __shfl_sync(0xffffffffu, wa, max(warp - 1, 0)), pb = __shfl_sync(0xffffffffu, wb, max(warp - 1, 0));
  a = (warp ? pa : V(0)) + ia - a; b = (warp ? pb : V(0)) + ib - b;
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

struct Border { uint32_t key, last_id; };   // least kept value, and the last id of it that is kept

template <class T, int C>
struct Row {
  Group<C> g;
  Shared *s;
  const T *x;          // this CTA's slice
  int n, id0;          // ids in the slice, first id
  float mx, low, scale;   // low = mx - 32 T: ids above it need no look at how small their weight is; scale: bins per unit of the logits
  double mxd, z_scale, one;    // mx; log2(e) / T; the weight 1 in fixed point
  bool inf_max, dirty;    // the maximum is infinite: only the ids that reach it count; values not cleaned yet

  __device__ __forceinline__ double z2_of(float v) const { return ((double)v - mxd) * z_scale; }
  // in 64 bits; weights below 2^-1020, which no sum and no min_p (a 32-bit number) can tell from 0, are 0
  __device__ __forceinline__ double w_of(float v) const { const double z2 = z2_of(v); return z2 > -1020.0 ? weight(z2, s->table) : 0.0; }
  __device__ __forceinline__ bool positive(float v) const { return v > low || z2_of(v) > -1075.0; }      // exp(..) > 0 in 64 bits
  // the weight as a whole multiple of 2^-fixed_bits: rounded next to 2^52, so the low bits of that sum are it.  What lies below 2^-46.5, masked
  // ids among it, is taken as that, which rounds to 0.
  __device__ __forceinline__ double at_2_52(float v) const { return fma(weight(fmax(z2_of(v), -46.5), s->table), one, 4503599627370496.0); }
  __device__ __forceinline__ double qd_at(float v) const { return at_2_52(v) - 4503599627370496.0; }
  __device__ __forceinline__ u64 q_at(float v) const { return (u64)(__double_as_longlong(at_2_52(v)) - 0x4330000000000000ll); }
  // distance from the maximum in bins; what lies behind the last bin is in it
  __device__ __forceinline__ float t_of(float v) const { return fminf(fmaxf((mx - v) * scale, 0.f), (float)(BINS - 1)); }

  // ids i .. i + 3 of the slice, -inf from `end` on; i is a multiple of four
  __device__ __forceinline__ void load4(int i, int end, float (&e)[4]) const {
    if (i + 4 <= end && ((uintptr_t)x & (4 * sizeof(T) - 1)) == 0) {
      if constexpr (sizeof(T) == 4) { const float4 v = *reinterpret_cast<const float4 *>(x + i); e[0] = v.x; e[1] = v.y; e[2] = v.z; e[3] = v.w; }
      else {
        const uint2 v = *reinterpret_cast<const uint2 *>(x + i);
        e[0] = __uint_as_float(v.x << 16); e[1] = __uint_as_float(v.x & 0xffff0000u); e[2] = __uint_as_float(v.y << 16); e[3] = __uint_as_float(v.y & 0xffff0000u);
      }
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j) e[j] = i + j < end ? to_f(x[i + j]) : -INFINITY;
    }
    if (dirty) {
#pragma unroll
      for (int j = 0; j < 4; ++j) e[j] = clean(e[j]);
    }
    if (inf_max) {
#pragma unroll
      for (int j = 0; j < 4; ++j) e[j] = e[j] == INFINITY ? 0.f : -INFINITY;
    }
  }
  __device__ __forceinline__ float one_of(int i, int end) const {
    const float v = i < end ? clean(to_f(x[i])) : -INFINITY;
    return !inf_max ? v : v == INFINITY ? 0.f : -INFINITY;
  }
  // f(values, index of the first in the slice): four consecutive ids at a time
  template <class F> __device__ __forceinline__ void each4(F f) const {
    for (int i = threadIdx.x * 4; i < n; i += THREADS * 4) {
      float e[4];
      load4(i, n, e);
      f(e, i);
    }
  }
  // f(value, index in the slice) for every finite id of at least `least`
  template <class F> __device__ __forceinline__ void each(float least, F f) const {
    each4([&](const float (&e)[4], int i) {
      if (!(fmaxf(fmaxf(e[0], e[1]), fmaxf(e[2], e[3])) >= least)) return;
#pragma unroll
      for (int j = 0; j < 4; ++j) if (e[j] >= least && e[j] > -INFINITY) f(e[j], i + j);
    });
  }
  // The least finite value with t_of(value) < t, infinity where there is none.  A warp calls: 32 probes a step over the bits of the values.
  __device__ float edge(float t) const {
    uint32_t lo = key_of(-FLT_MAX), hi = key_of(mx);
    if (!(t > 0.f)) return INFINITY;                       // t_of(mx) = 0
    while (lo < hi) {
      const uint32_t step = max(1u, (hi - lo) / 32), probe = min(lo + (threadIdx.x & 31) * step, hi);
      const unsigned yes = __ballot_sync(0xffffffffu, t_of(value_of(probe)) < t);
      if (yes & 1) { hi = lo; break; }
      const int f = yes ? __ffs(yes) - 1 : 32;
      const uint32_t below_ = min(lo + (uint32_t)(f - 1) * step, hi);
      if (f < 32) hi = min(lo + (uint32_t)f * step, hi);
      lo = min(below_ + 1, hi);
    }
    return value_of(hi);
  }
  // a value below every id of bins 0 .. bin
  __device__ __forceinline__ float below(int bin) const {
    if (bin >= BINS - 1 || !(scale > 0.f)) return -INFINITY;
    return mx - (float)(bin + 2) / scale;
  }
  __device__ __forceinline__ void clear() {
    for (int i = threadIdx.x; i < BINS; i += THREADS) s->cnt[i] = s->lo[i] = s->hi[i] = 0;
  }
  __device__ __forceinline__ void add(int bin, u64 q) {
    atomicAdd(&s->cnt[bin], 1u);
    const uint32_t l = (uint32_t)q;
    uint32_t h = (uint32_t)(q >> 32);
    if (l && atomicAdd(&s->lo[bin], l) > 0xffffffffu - l) ++h;
    if (h) atomicAdd(&s->hi[bin], h);
  }
  // The cluster's sums of this thread's PER bins (call after a sync; the histograms must stay until the next one).
  __device__ __forceinline__ void counts(uint32_t *from, u64 (&c)[PER]) {
#pragma unroll
    for (int j = 0; j < PER; ++j) c[j] = 0;
#pragma unroll
    for (int r = 0; r < C; ++r)
#pragma unroll
      for (int j = 0; j < PER; j += 2) {
        const uint2 v = *reinterpret_cast<const uint2 *>(g.peer(from, r) + threadIdx.x * PER + j);
        c[j] += v.x; c[j + 1] += v.y;
      }
  }
  __device__ __forceinline__ void weights(u64 (&m)[PER]) {
#pragma unroll
    for (int j = 0; j < PER; ++j) m[j] = 0;
#pragma unroll
    for (int r = 0; r < C; ++r)
#pragma unroll
      for (int j = 0; j < PER; j += 2) {
        const uint2 l = *reinterpret_cast<const uint2 *>(g.peer(s->lo, r) + threadIdx.x * PER + j), h = *reinterpret_cast<const uint2 *>(g.peer(s->hi, r) + threadIdx.x * PER + j);
        m[j] += ((u64)h.x << 32) + l.x; m[j + 1] += ((u64)h.y << 32) + l.y;
      }
  }
  // The bin where the running total from the top reaches the target: above < target <= above + bin.  Every CTA finds it for itself.
  __device__ Found search(const u64 (&c)[PER], const u64 (&m)[PER], bool by_mass, double target, u64 start_c, u64 start_m) {
    u64 bc = 0, bm = 0, sc, sm;
    if (threadIdx.x == 0) s->found = Found{0, 0, 0, 0, 0};  // (the scan's barriers come before the one that finds it)
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

  // Sends the ids that `member` selects to the first CTA's list; returns after the list is complete.  From the held ids where `held`.
  template <class M> __device__ __forceinline__ void gather(float least, bool held, M member) {
    Shared *first = g.peer(s, 0);
    auto send = [&](uint32_t k, uint32_t id) {
      const int at = atomicAdd(&first->list_n, 1);
      if (at < LIST) *reinterpret_cast<uint2 *>(&first->list[at]) = make_uint2(k, id);
    };
    if (held) {
      for (int i = threadIdx.x; i < s->held_n; i += THREADS) { const uint2 h = s->held[i]; if (member(value_of(h.x), h.x)) send(h.x, h.y); }
    } else {
      each(least, [&](float v, int i) { const uint32_t k = key_of(v); if (member(v, k)) send(k, (uint32_t)(id0 + i)); });
    }
    g.sync();
  }
  // The first CTA: each entry's weight, then the ids and the weight ahead of this thread's entry in the order.  All its threads call.
  __device__ __forceinline__ int rank_list(Entry &e, u64 &ahead_c, u64 &ahead_m) {
    const int n_list = min(s->list_n, LIST), i = threadIdx.x;
    e = Entry{0, 0, 0};
    if (i < n_list) { e = s->list[i]; e.q = q_at(value_of(e.key)); s->list[i].q = e.q; }
    __syncthreads();
    ahead_c = ahead_m = 0;
    if (i < n_list) {
      uint32_t c = 0;
#pragma unroll 4
      for (int j = 0; j < n_list; ++j) {
        const Entry o = s->list[j];
        const bool ahead = o.key > e.key || (o.key == e.key && o.id < e.id);
        c += ahead;
        ahead_m += ahead ? o.q : 0;
      }
      ahead_c = c;
    }
    return n_list;
  }

  // The t-th id, in id order, of those with this value.  Each warp counts a run of ids, then one walks its own.
  __device__ uint32_t nth_equal(uint32_t key, u64 t) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, run = (n + WARPS - 1) / WARPS, i0 = min(n, warp * run), i1 = min(n, i0 + run);
    uint32_t mine = 0;
    for (int i = i0 + lane; i < i1; i += 32) mine += key_of(one_of(i, i1)) == key;
    mine = __reduce_add_sync(0xffffffffu, mine);
    u64 before = lane == 0 ? mine : 0, none = 0, sum, zero;
    block_scan2<u64>(before, none, sum, zero, s->red, s->red2);
    before = __shfl_sync(0xffffffffu, before, 0);
    const Mail *all = g.exchange(sum, 0);
    for (int r = 0; r < g.rank; ++r) before += all[r].a;
    if (before < t && t <= before + mine) {
      u64 at = before;
      for (int i = i0; i < i1; i += 32) {
        const unsigned same = __ballot_sync(0xffffffffu, i + lane < i1 && key_of(one_of(i + lane, i1)) == key);
        if (at + __popc(same) >= t) {
          if ((same >> lane & 1) && at + __popc(same & ((2u << lane) - 1)) == t)
            for (int r = 0; r < C; ++r) *g.peer(&s->last_id, r) = (uint32_t)(id0 + i + lane);
          break;
        }
        at += __popc(same);
      }
    }
    g.sync();
    return s->last_id;
  }

  // Settles the border inside a bin.  `member(value, key)` selects the bin's ids, all of them at least `least` and, where `held`, among the held
  // ones; the list must be empty (and is again afterwards).  by_k: the target is a count.
  template <class M>
  __device__ Border settle(float least, bool held, M member, Found f, bool by_mass, double target) {
    bool narrowed = false;
    uint32_t kl = 0, kh = 0xffffffffu;
    for (int round = 0; round < 5; ++round) {
      if (f.cnt <= LIST) {
        if (narrowed) gather(value_of(kl), held, [&](float, uint32_t k) { return k >= kl && k <= kh; });
        else gather(least, held, member);
        if (g.rank == 0) {
          Entry e;
          u64 rc, rm;
          const int n_list = rank_list(e, rc, rm);
          rc += f.above_c; rm += f.above_m;
          const double lo = by_mass ? (double)rm : (double)rc, hi = by_mass ? (double)(rm + e.q) : (double)(rc + 1);
          if ((int)threadIdx.x < n_list && lo < target && target <= hi) {
#pragma unroll
            for (int r = 0; r < C; ++r) { u64 *o = g.peer(s->res, r); o[0] = e.key; o[1] = e.id; }
          }
          if (threadIdx.x == 0) s->list_n = 0;
        }
        g.sync();
        return Border{(uint32_t)s->res[0], (uint32_t)s->res[1]};
      }
      if (!narrowed) {                                      // the bin's range of values
        uint32_t h = 0, l = 0;                              // l holds ~key
        each(least, [&](float v, int) { const uint32_t k = key_of(v); if (member(v, k)) { h = max(h, k); l = max(l, ~k); } });
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
        return Border{kl, nth_equal(kl, t)};
      }
      const int sh = max(0, 21 - __clz(kh - kl));           // (kh - kl) >> sh is below 2048
      g.sync();                                             // all have read the histograms that go now
      clear();
      __syncthreads();
      each(value_of(kl), [&](float v, int) {
        const uint32_t k = key_of(v);
        if (k >= kl && k <= kh) add((int)((kh - k) >> sh), q_at(v));
      });
      g.sync();
      u64 c[PER], m[PER];
      counts(s->cnt, c); weights(m);
      f = search(c, m, by_mass, target, f.above_c, f.above_m);
      const uint32_t top = kh - ((uint32_t)f.bin << sh);
      const u64 low_ = (u64)((uint32_t)f.bin + 1) << sh;
      kl = low_ > (u64)(kh - kl) ? kl : kh - (uint32_t)low_ + 1;
      kh = top;
    }
    return Border{kl, 0xffffffffu};                         // not reached: three cuts leave one value
  }
};

template <class T, int C>
__global__ void __launch_bounds__(THREADS, 1)
sample_given_kernel(GivenArgs a) {
  pdl_launch_dependents();
  pdl_wait();
  extern __shared__ __align__(16) uint8_t dyn[];
  Shared *s = (Shared *)dyn;
  u64 *chunk = (u64 *)(dyn + sizeof(Shared));               // kept weight of each 128 ids of the slice
  T *copy = (T *)(chunk + (a.slice + CHUNK - 1) / CHUNK + (((a.slice + CHUNK - 1) / CHUNK) & 1));
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, b = blockIdx.x / C;
  Row<T, C> row;
  row.s = s; row.g.s = s; row.g.par = 0; row.one = (double)(1ll << a.fixed_bits); row.inf_max = false;
  row.g.rank = C > 1 ? (int)(blockIdx.x % C) : 0;
  row.id0 = min(a.V, row.g.rank * a.slice); row.n = min(a.V, row.id0 + a.slice) - row.id0;
  row.x = (const T *)a.logits + (size_t)b * a.ld + row.id0;
  const float T_in = a.temperature ? a.temperature[b] : 1.0f, T_ = T_in > 0x1p100f ? 0x1p100f : T_in, p = a.top_p ? a.top_p[b] : 1.f, mp = a.min_p ? a.min_p[b] : 0.f, u_ = a.uniform[b];
  const int k = a.top_k ? a.top_k[b] : 0;
  if (tid < 64) s->table[tid] = exp2(tid * 0.015625);
  if (tid == 0) s->list_n = s->held_n = 0;
  row.clear();
  for (int i = tid; i < BINS; i += THREADS) s->coarse[i] = 0;
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
  row.dirty = !a.in_smem;
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
  float mn = value_of(~lo);
  if (row.mx == INFINITY) { row.inf_max = true; row.mx = mn = 0.f; }
  row.mxd = (double)row.mx;
  if (!(T_ > 0.f)) {                                         // greedy: the lowest id of the maximum
    uint32_t best = 0, none = 0;                             // ~id
    row.each(row.mx, [&](float v, int i) { if (v == row.mx) best = max(best, ~(uint32_t)(row.id0 + i)); });
    block_max2(best, none, s->red);
    const Mail *all = row.g.exchange(best, 0);
#pragma unroll
    for (int r = 0; r < C; ++r) best = max(best, (uint32_t)all[r].a);
    if (row.g.rank == 0 && tid == 0) { a.tokens[b] = (int)~best; if (a.kept) a.kept[b] = 1; if (a.prob) a.prob[b] = 1.f; }
    row.g.sync();
    return;
  }
  row.z_scale = 1.44269504088896340736 / (double)T_;
  row.low = row.mx - RANGE * T_;
  const bool by_k = k > 0 && k < a.V, by_p = p < 1.f;
  const double min_w = mp > 0.f ? fmin((double)mp, 1.0) : 0.0, frac = p > 0.f ? (double)p : 0.0;      // p <= 0 keeps the first id
  const double u = u_ > 0.f ? (double)fminf(u_, 0.99999994f) : 0.0;
  // ---- the kept prefix: values above `least`, and ids of that value up to last_id
  float least = -INFINITY;
  uint32_t last_id = 0xffffffffu;
  int b0 = 0, b1 = BINS - 1, last_bin = BINS - 1;
  bool have_k = false;
  u64 c[PER];
  if (by_k || by_p) {
    const float range = fminf(row.mx - mn, RANGE * T_);
    row.scale = range > 0.f && range < INFINITY ? (float)(BINS - 1) / range : 0.f;
    if (!(row.scale < INFINITY)) row.scale = 0.f;            // a temperature next to 0: one bin, cut by the bits of the values
    row.each4([&](const float (&e)[4], int) {
      int bin[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) bin[j] = (int)row.t_of(e[j]);
#pragma unroll
      for (int j = 0; j < 4; ++j) if (e[j] > -INFINITY) atomicAdd(&s->coarse[bin[j]], 1u);
    });
    row.g.sync();
    row.counts(s->coarse, c);
    if (by_k) {
      u64 all_c = 0, zero[PER] = {};
#pragma unroll
      for (int j = 0; j < PER; ++j) all_c += c[j];
      if ((u64)k < block_add(all_c, s->red)) {               // else fewer ids than k: nothing to cut
        const Found f = row.search(c, zero, false, (double)k, 0, 0);
        last_bin = f.bin;
        have_k = true;
        if (f.above_c + f.cnt <= SMALL) {
          // few candidates: the first CTA does the rest among them
          row.gather(row.below(f.bin), false, [&](float v, uint32_t) { return (int)row.t_of(v) <= f.bin; });
          if (row.g.rank == 0) {
            Entry e;
            u64 rank, before;
            const int n_list = row.rank_list(e, rank, before);
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
        const Border bd = row.settle(row.below(f.bin), false, [&](float v, uint32_t) { return (int)row.t_of(v) == f.bin; }, f, false, (double)k);
        least = value_of(bd.key); last_id = bd.last_id;
        if (by_p && f.cnt > LIST) { row.g.sync(); row.clear(); __syncthreads(); }      // the bin was cut again: its histogram goes
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
      if (lane == 0) { if (first_up < BINS) atomicMin(&s->bounds[0], first_up); if (first_dn < BINS) atomicMin(&s->bounds[1], first_dn); }
      __syncthreads();
      b0 = s->bounds[0]; b1 = max(b0, s->bounds[1]);
    }
  }
  const float t0 = (float)b0, t1 = (float)(b1 + 1), fine = (float)(BINS / (b1 - b0 + 1));
  auto fine_bin = [&](float v) { return min(BINS - 1, (int)((row.t_of(v) - t0) * fine)); };
  auto in_prefix = [&](float v, uint32_t id) { return v > least || (v == least && id <= last_id); };
  // The bounds as values: ids from v_above on lie above them, those from v_from on above or between.
  float v_above = -FLT_MAX, v_from = INFINITY;
  if (by_p) {
    if (warp < 2) {
      const float v = row.edge(warp ? t1 : t0);
      if (lane == 0) s->edges[warp] = v;
    }
    __syncthreads();
    v_above = s->edges[0]; v_from = s->edges[1];
  }

  // ---- weights, chunk by chunk of 128 ids (four a lane).  Weights are whole numbers whose sums stay below 2^53 in a thread, so sums of
  // 64-bit floats are exact there, and those of integers beyond.  With top-p's border still open (bounded), ids above its bounds go into
  // the chunks and the ids between them are held.
  u64 above = 0, all_q = 0, n_kept = 0;
  auto weigh = [&](bool bounded) {
    double above_d = 0.0, all_d = 0.0;
    uint32_t n_thread = 0;
    const bool cut = least > -INFINITY, look = min_w == 0.0 && !(v_above > row.low);      // look: some weights may be 0 in 64 bits
    for (int ch = warp; ch * CHUNK < row.n; ch += WARPS) {
      const int i = ch * CHUNK + lane * 4;
      float e[4];
      row.load4(i, row.n, e);
      if (cut) {
#pragma unroll
        for (int j = 0; j < 4; ++j) if (!in_prefix(e[j], (uint32_t)(row.id0 + i + j))) e[j] = -INFINITY;
        if (!__any_sync(0xffffffffu, fmaxf(fmaxf(e[0], e[1]), fmaxf(e[2], e[3])) > -INFINITY)) {
          if (lane == 0) chunk[ch] = 0;
          continue;
        }
      }
      double q[4], sum = 0.0;
#pragma unroll
      for (int j = 0; j < 4; ++j) q[j] = row.qd_at(e[j]);
      unsigned hold = 0;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        bool in = e[j] >= v_above;
        if (bounded) {
          all_d += q[j];
          hold |= (unsigned)(e[j] >= v_from && !in) << j;
        }
        if (min_w > 0.0) {
          above_d += in ? q[j] : 0.0;
          in = in && row.w_of(e[j]) >= min_w;
        } else if (look) in = in && row.positive(e[j]);
        sum += in ? q[j] : 0.0;
        n_thread += in;
      }
      if (bounded && __any_sync(0xffffffffu, hold)) {
        const int n_lane = __popc(hold);
        int at = n_lane;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) { const int t = __shfl_up_sync(0xffffffffu, at, o); if (lane >= o) at += t; }
        int base = 0;
        if (lane == 31) base = atomicAdd(&s->held_n, at);                  // one a warp: single ones crowd the one address
        at += __shfl_sync(0xffffffffu, base, 31) - n_lane;
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (hold >> j & 1) { if (at < HELD) s->held[at] = make_uint2(key_of(e[j]), (uint32_t)(row.id0 + i + j)); ++at; }
      }
      const u64 in_chunk = warp_add((u64)sum);
      if (lane == 0) chunk[ch] = in_chunk;
      if (min_w == 0.0 && lane == 0) above += in_chunk;
    }
    if (min_w > 0.0) above = (u64)above_d;
    all_q = (u64)all_d; n_kept = n_thread;
  };
  weigh(by_p);
  if (by_p) {
    above = block_add(above, s->red); all_q = block_add(all_q, s->red);
    const bool held_all = s->held_n <= HELD;                 // else the ids between the bounds are looked up again
    if (held_all) { for (int i = tid; i < s->held_n; i += THREADS) { const float v = value_of(s->held[i].x); row.add(fine_bin(v), row.q_at(v)); } }
    else row.each(fmaxf(v_from, least), [&](float v, int i) { if (v < v_above && in_prefix(v, (uint32_t)(row.id0 + i))) row.add(fine_bin(v), row.q_at(v)); });
    const Mail *all = row.g.exchange(above | (held_all ? 0 : 1ull << 63), all_q);      // its sync also completes the histograms
    above = all_q = 0;
    bool held = true;
#pragma unroll
    for (int r = 0; r < C; ++r) { above += all[r].a & ~(1ull << 63); all_q += all[r].b; held = held && !(all[r].a >> 63); }
    const double target = fmax(frac * (double)all_q, 0.5);
    u64 m[PER];
    row.counts(s->cnt, c); row.weights(m);
    const Found f = row.search(c, m, true, target, 0, above);
    const float k_least = least;
    const Border bd = row.settle(fmaxf(v_from, k_least), held, [&](float v, uint32_t) { return v >= k_least && v >= v_from && v < v_above && fine_bin(v) == f.bin; }, f, true, target);
    least = value_of(bd.key); last_id = bd.last_id;
    if (held) {                                              // the held ids that stay join their chunks
      for (int i = tid; i < s->held_n; i += THREADS) {
        const uint2 h = s->held[i];
        const float v = value_of(h.x);
        if (in_prefix(v, h.y) && (min_w > 0.0 ? row.w_of(v) >= min_w : row.positive(v))) {
          atomicAdd(&chunk[((int)h.y - row.id0) / CHUNK], row.q_at(v));
          ++n_kept;
        }
      }
    } else {
      v_above = -FLT_MAX;
      weigh(false);
    }
  }
  // ---- the draw: the chunk, in id order, then the id in it
  const int n_chunks = (row.n + CHUNK - 1) / CHUNK, per = (n_chunks + THREADS - 1) / THREADS;
  n_kept = block_add(n_kept, s->red);                        // (a barrier before the chunks are read)
  u64 mine = 0, none = 0, sum, zero;
  for (int j = 0; j < per; ++j) if (tid * per + j < n_chunks) mine += chunk[tid * per + j];
  u64 before = mine;
  block_scan2<u64>(before, none, sum, zero, s->red, s->red2);
  const Mail *all = row.g.exchange(sum, n_kept);
  u64 total = 0, kept = 0;
#pragma unroll
  for (int r = 0; r < C; ++r) { if (r < row.g.rank) before += all[r].a; total += all[r].a; kept += all[r].b; }
  if (row.g.rank == 0 && tid == 0 && a.kept) a.kept[b] = (int)kept;
  const u64 target = (u64)(u * (double)total);               // cumulative > u * total, the cumulative whole: > its floor
  if (tid == 0) s->pick_chunk = -1;
  __syncthreads();
  if (before <= target && target < before + mine) {
    int ch = tid * per;
    while (ch + 1 < n_chunks && before + chunk[ch] <= target) before += chunk[ch++];
    s->pick_chunk = ch; s->pick_before = before;
  }
  __syncthreads();
  if (warp == 0 && s->pick_chunk >= 0) {
    const int i = s->pick_chunk * CHUNK + lane * 4;
    float e[4];
    row.load4(i, row.n, e);
    u64 q[4], own = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      bool keep = e[j] > -INFINITY && (!(least > -INFINITY) || in_prefix(e[j], (uint32_t)(row.id0 + i + j)));
      if (min_w > 0.0) keep = keep && row.w_of(e[j]) >= min_w;
      q[j] = keep ? row.q_at(e[j]) : 0;
      own += q[j];
    }
    u64 at = own;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) { const u64 t = __shfl_up_sync(0xffffffffu, at, o); if (lane >= o) at += t; }
    at += s->pick_before - own;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (at <= target && target < at + q[j]) {
        a.tokens[b] = row.id0 + i + j;
        if (a.prob) a.prob[b] = (float)((double)q[j] / (double)total);
      }
      at += q[j];
    }
  }
}

template <class T, int C>
int launch_t(b200_ctx *ctx, const GivenArgs &a, size_t batch, size_t smem) {
  static std::atomic<unsigned long long> attr{0};
  const unsigned long long bit = 1ull << (ctx->device & 63);
  if (!(attr.load() & bit)) { B200_CUDA(ctx, cudaFuncSetAttribute(sample_given_kernel<T, C>, cudaFuncAttributeMaxDynamicSharedMemorySize, 220 * 1024)); attr.fetch_or(bit); }
  B200_CUDA(ctx, launch_pdl(ctx, sample_given_kernel<T, C>, dim3((unsigned)(batch * C)), dim3(THREADS), smem, C > 1 ? C : 0, a));
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
  const size_t es = dtype_size(dt), room = 220 * 1024;
  auto slice = [&](int C) { return ((vocab + C - 1) / C + 15) / 16 * 16; };
  auto fixed = [&](int C) { const size_t n = (slice(C) + CHUNK - 1) / CHUNK; return sizeof(Shared) + 8 * (n + (n & 1)); };
  auto at_once = [&](int C) { return (size_t)(C == 2 ? ctx->sm_count : C == 4 ? ctx->sm_count - 20 : ctx->sm_count - 28); };
  int C = 1;
  while (C < MAX_CLUSTER && (batch * 2 * C <= at_once(2 * C) || fixed(C) + slice(C) * es > room) && vocab / C > 2048) C *= 2;
  a.slice = (int)slice(C);
  a.in_smem = fixed(C) + a.slice * es <= room;
  const size_t smem = fixed(C) + (a.in_smem ? a.slice * es : 0);      // at most 198 KiB of it fixed (2^24 ids over eight CTAs)
  if (dt == B200_BF16) return C == 1 ? launch_t<bf16, 1>(ctx, a, batch, smem) : C == 2 ? launch_t<bf16, 2>(ctx, a, batch, smem) : C == 4 ? launch_t<bf16, 4>(ctx, a, batch, smem) : launch_t<bf16, 8>(ctx, a, batch, smem);
  return C == 1 ? launch_t<float, 1>(ctx, a, batch, smem) : C == 2 ? launch_t<float, 2>(ctx, a, batch, smem) : C == 4 ? launch_t<float, 4>(ctx, a, batch, smem) : launch_t<float, 8>(ctx, a, batch, smem);
}
