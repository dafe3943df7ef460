// Sampling with temperature, top-k, top-p and min-p from one given uniform per row (include/csm_ops.h).
//   w_i = exp((x_i - max) / T);  rows ordered by (x descending, index ascending);  every filter keeps a PREFIX of that order, so the kept set
//   is "key > cut, and the first `ties` entries with key == cut";  the token is where the running sum of kept w (index order) passes u * total.
// Sums are uint64 fixed point (w scaled by 2^min(62 - ceil log2 V, 51)) of weights computed in fp64: exact integer additions, so neither the
// split over threads nor any order of arrival changes a result, and what is rounded away per weight is below 2^-45 of the largest.
//
// One workgroup per row.  No sort: a cut is found by narrowing an interval of order keys (count and mass at or above a probe, one block sum per
// step; the probe alternates between the middle VALUE, which a smooth row needs few of, and the middle KEY, which bounds any row) until at most
// 64 entries or one single key are left, which a wave then ranks exactly.
//   V <= 16 384: the row lives in registers (up to 16 consecutive entries per thread), read once.
//   larger V:    one pass for the maximum, one for the mass (only where top-p needs the whole row's) and for the entries above a threshold that 4 096
//                samples put near the 12 288th largest; these are compacted in index order and treated like a short row.  Where that list
//                is not enough (a flat row whose nucleus is larger), the same search streams over the row.
#include "ops_common.h"
#include <math.h>

struct SampleOpArgs {
  const void* logits;
  int64_t stride;
  int V, shift;   // shift: binary point of the fixed-point weights
  const float *uniform, *temperatures, *top_ps, *min_ps;
  const int32_t* topks;
  float temperature, top_p, min_p;
  int topk;
  int32_t* out;
};
constexpr int E = 16;                     // entries per thread
constexpr int LIST = 1024 * E;            // entries of a compacted list
constexpr int SAMPLES = 4096, AIM = LIST * 3 / 4;   // the list's threshold is a sample's order statistic that aims at this many entries: at V = 131 072
                                                    // their number scatters by 613, LIST is 6.7 of that away

__device__ __forceinline__ uint32_t order_key(float x) {   // larger float = larger key
  const uint32_t u = __float_as_uint(x);
  return u ^ ((u >> 31) ? 0xffffffffu : 0x80000000u);
}
__device__ __forceinline__ float key_value(uint32_t k) { return __uint_as_float((k >> 31) ? k ^ 0x80000000u : ~k); }
template <typename T>
__device__ __forceinline__ float logit(const T* x, int i) {   // NaN counts as -inf, -0 as +0
  const float v = to_f32(x[i]) + 0.f;
  return v != v ? -INFINITY : v;
}
constexpr uint32_t NEG_INF_KEY = 0x007fffffu;   // order_key(-inf); keys at or below it are no entries

// w * 2^shift as an integer.  2^t = 2^n 2^f with f in [-1/2, 1/2] from its power series (12 terms: below 2^-52); adding 2^52 leaves the rounded
// integer in the mantissa (shift <= 51).
struct Weigh {
  float mx;
  double k2;   // log2(e) / T
  int shift;
  __device__ __forceinline__ uint64_t operator()(float x) const {
    if (x == mx) return 1ull << shift;
    if (x == -INFINITY || mx == INFINITY) return 0;
    const double t = fmax(((double)x - (double)mx) * k2, -1200.0), n = rint(t), f = (t - n) * 0.69314718055994530942;
    double p = 1.0 / 479001600.0;
    p = __fma_rn(p, f, 1.0 / 39916800.0); p = __fma_rn(p, f, 1.0 / 3628800.0); p = __fma_rn(p, f, 1.0 / 362880.0);
    p = __fma_rn(p, f, 1.0 / 40320.0); p = __fma_rn(p, f, 1.0 / 5040.0); p = __fma_rn(p, f, 1.0 / 720.0); p = __fma_rn(p, f, 1.0 / 120.0);
    p = __fma_rn(p, f, 1.0 / 24.0); p = __fma_rn(p, f, 1.0 / 6.0); p = __fma_rn(p, f, 0.5); p = __fma_rn(p, f, 1.0); p = __fma_rn(p, f, 1.0);
    return (uint64_t)__double_as_longlong(ldexp(p, (int)n + shift) + 4503599627370496.0) & 0xfffffffffffffull;
  }
};

// ---- block sums -------------------------------------------------------------------------------------------------------------------------
__device__ __forceinline__ uint64_t wave_sum64(uint64_t v) {
#pragma unroll
  for (int d = 32; d; d >>= 1) v += __shfl_xor((unsigned long long)v, d);
  return v;
}
__device__ __forceinline__ uint32_t wave_sum32(uint32_t v) {
#pragma unroll
  for (int d = 32; d; d >>= 1) v += __shfl_xor(v, d);
  return v;
}
struct Red { uint64_t m[2][16]; uint32_t c[2][16]; };   // two generations: one barrier per sum

template <int NT>
struct Block {
  Red* r;
  int gen = 0;
  __device__ __forceinline__ void sum(uint32_t& cnt, uint64_t& mass, bool want_mass) {
    cnt = wave_sum32(cnt);
    if (want_mass) mass = wave_sum64(mass);
    const int g = gen ^= 1;
    if ((threadIdx.x & 63) == 0) { r->c[g][threadIdx.x >> 6] = cnt; r->m[g][threadIdx.x >> 6] = mass; }
    __syncthreads();
    cnt = 0;
#pragma unroll
    for (int i = 0; i < NT / 64; ++i) cnt += r->c[g][i];
    if (want_mass) {
      mass = 0;
#pragma unroll
      for (int i = 0; i < NT / 64; ++i) mass += r->m[g][i];
    }
  }
  // sum over the threads before this one, and over all
  __device__ __forceinline__ uint64_t before(uint64_t v, uint64_t& total) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    uint64_t x = v;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const uint64_t y = __shfl_up((unsigned long long)x, d);
      if (lane >= d) x += y;
    }
    const int g = gen ^= 1;
    if (lane == 63) r->m[g][wave] = x;
    __syncthreads();
    uint64_t b = 0;
    total = 0;
#pragma unroll
    for (int i = 0; i < NT / 64; ++i) {
      if (i < wave) b += r->m[g][i];
      total += r->m[g][i];
    }
    return b + x - v;
  }
};

// ---- the search ---------------------------------------------------------------------------------------------------------------------------
struct Cut { uint32_t key; uint32_t ties; };   // kept: keys above `key`, and the first `ties` entries equal to it
struct Few { uint64_t w[64]; uint32_t key[64]; int n; };

// Largest interval end `lo` whose entries at or above it reach the target -- a count (MASS false) or a mass -- narrowed to the exact entry.
// At entry: everything in [lo, ...) reaches it, nothing at or above hi does (cnt_hi / mass_hi are what lies there).
template <int NT, bool MASS, typename Src>
__device__ __forceinline__ Cut find_cut(Src& src, Block<NT>& blk, Few* few, const Weigh& weigh, uint32_t lo, uint32_t cnt_lo, uint32_t hi, uint32_t want_n, double want_m) {
  uint32_t cnt_hi = 0;
  uint64_t mass_hi = 0;
  for (int step = 0; cnt_lo - cnt_hi > 64 && hi - lo > 1; ++step) {
    uint32_t mid = lo + (hi - lo) / 2;
    if (!(step & 1)) {
      const float v = 0.5f * key_value(lo) + 0.5f * key_value(hi - 1);
      const uint32_t kv = order_key(v + 0.f);
      if (v == v && kv > lo && kv < hi) mid = kv;
    }
    uint32_t cnt;
    uint64_t mass = 0;
    src.template stat<MASS>(mid, cnt, mass);
    blk.sum(cnt, mass, MASS);
    if (MASS ? (double)mass >= want_m : cnt >= want_n) { lo = mid; cnt_lo = cnt; }
    else { hi = mid; cnt_hi = cnt; mass_hi = mass; }
  }
  if (hi - lo <= 1) {   // one key: equal entries, equal weights
    if (!MASS) return {lo, want_n - cnt_hi};
    const uint64_t each = weigh(key_value(lo));
    const double q = each ? ceil((want_m - (double)mass_hi) / (double)each) : 1.0;
    const uint32_t n = cnt_lo - cnt_hi;
    return {lo, q < 1.0 ? 1u : q > (double)n ? n : (uint32_t)q};
  }
  if (threadIdx.x == 0) few->n = 0;
  __syncthreads();
  src.gather(lo, hi, few);
  __syncthreads();
  // every wave ranks the (at most 64) entries itself
  const int lane = threadIdx.x & 63, n = min(few->n, 64);
  const uint32_t key = lane < n ? few->key[lane] : 0;
  const uint64_t w = lane < n && MASS ? weigh(key_value(key)) : 0;
  if (MASS && threadIdx.x < 64) few->w[lane] = w;
  if (MASS) __syncthreads();
  uint32_t rank = 0, above = 0;
  uint64_t before = mass_hi;
  for (int j = 0; j < n; ++j) {
    const uint32_t kj = few->key[j];
    const bool first = kj > key || (kj == key && j < lane);
    rank += first;
    above += kj > key;
    if (MASS && first) before += few->w[j];
  }
  const bool here = lane < n && (MASS ? (double)before < want_m && (double)(before + w) >= want_m : cnt_hi + rank == want_n - 1);
  const uint64_t at = __ballot(here);
  const int src_lane = at ? __ffsll((unsigned long long)at) - 1 : 0;
  Cut r;
  r.key = __builtin_amdgcn_readlane(key, src_lane);
  r.ties = __builtin_amdgcn_readlane(rank - above, src_lane) + 1;
  __syncthreads();   // `few` may be filled again
  return r;
}

// a row (or list) in registers: thread t holds entries t * per .. t * per + per - 1; key 0 = not (or no longer) an entry
struct RegRow {
  uint32_t key[E];
  uint64_t w[E];
  int per;
  template <bool MASS>
  __device__ __forceinline__ void stat(uint32_t c, uint32_t& cnt, uint64_t& mass) const {
    cnt = 0;
#pragma unroll
    for (int e = 0; e < E; ++e)
      if (e < per) {
        const bool in = key[e] >= c;
        cnt += in;
        if (MASS) mass += in ? w[e] : 0;
      }
  }
  __device__ __forceinline__ void gather(uint32_t lo, uint32_t hi, Few* few) const {
#pragma unroll
    for (int e = 0; e < E; ++e)
      if (e < per && key[e] >= lo && key[e] < hi) {
        const int at = atomicAdd(&few->n, 1);
        if (at < 64) few->key[at] = key[e];
      }
  }
};

// drop what a cut does not keep
template <int NT>
__device__ __forceinline__ void apply(RegRow& r, Block<NT>& blk, const Cut& c) {
  uint32_t mine = 0;
#pragma unroll
  for (int e = 0; e < E; ++e)
    if (e < r.per) mine += r.key[e] == c.key;
  uint32_t all = mine;
  uint64_t unused = 0;
  blk.sum(all, unused, false);
  uint64_t rank = 0, total;
  if (all > c.ties) rank = blk.before(mine, total);
#pragma unroll
  for (int e = 0; e < E; ++e)
    if (e < r.per) {
      bool keep = r.key[e] >= c.key;
      if (r.key[e] == c.key) keep = rank++ < c.ties;
      if (!keep) { r.key[e] = 0; r.w[e] = 0; }
    }
}

struct Setting {
  float T, top_p, min_p, u;
  int k;   // 0 = off
};
__device__ __forceinline__ Setting setting(const SampleOpArgs& a, int row) {
  Setting s;
  s.T = a.temperatures ? a.temperatures[row] : a.temperature;
  s.top_p = a.top_ps ? a.top_ps[row] : a.top_p;
  s.min_p = a.min_ps ? a.min_ps[row] : a.min_p;
  s.u = a.uniform[row];
  s.k = a.topks ? a.topks[row] : a.topk;
  if (!(s.T > 0.f)) { s.T = 0.f; s.k = 1; }
  if (s.k <= 0 || s.k >= a.V) s.k = a.V == 1 ? 1 : 0;
  if (!(s.top_p >= 0.f)) s.top_p = 0.f;
  if (!(s.min_p >= 0.f)) s.min_p = 0.f;
  if (s.min_p > 1.f) s.min_p = 1.f;
  if (!(s.u >= 0.f)) s.u = 0.f;
  if (s.u >= 1.f) s.u = 0.99999994f;
  return s;
}
__device__ __forceinline__ double target(float top_p, uint64_t base) { return fmax((double)top_p * (double)base, 1.0); }   // at least one entry

// filters and draw on entries in registers; returns the place (e, in the thread that owns it) or -1.  `base`: the mass that top_p refers to when
// top-k is off (0: that of these entries).  `enough` comes back false when these entries cannot hold the nucleus.
template <int NT>
__device__ __forceinline__ int filter_and_draw(RegRow& r, Block<NT>& blk, Few* few, const Weigh& weigh, const Setting& s, uint32_t n, uint32_t key_min, uint32_t key_max, uint64_t base, bool& enough) {
  enough = true;
  if (s.k && (uint32_t)s.k < n) {
    apply(r, blk, find_cut<NT, false>(r, blk, few, weigh, key_min, n, key_max + 1, (uint32_t)s.k, 0.0));
    n = (uint32_t)s.k;
  }
  if (s.top_p < 1.f) {
    uint32_t cnt = 0;
    uint64_t mass = 0;
    r.stat<true>(1u, cnt, mass);
    blk.sum(cnt, mass, true);
    const double want = target(s.top_p, base ? base : mass);
    if ((double)mass < want) { enough = false; return -1; }
    apply(r, blk, find_cut<NT, true>(r, blk, few, weigh, key_min, n, key_max + 1, 0u, want));
  }
  uint64_t mine = 0, total;
  const double least = (double)s.min_p * (double)(1ull << weigh.shift);
#pragma unroll
  for (int e = 0; e < E; ++e)
    if (e < r.per) {
      if ((double)r.w[e] < least) r.w[e] = 0;
      mine += r.w[e];
    }
  const uint64_t before = blk.before(mine, total);
  const double want = (double)s.u * (double)total;
  if (!((double)before > want) && (double)(before + mine) > want) {
    uint64_t run = before;
#pragma unroll
    for (int e = 0; e < E; ++e)
      if (e < r.per) {
        run += r.w[e];
        if ((double)run > want) return e;
      }
  }
  return -1;
}

template <int NT>
__device__ __forceinline__ float block_max(float v, float* s) {
  v = wave_max(v);
  if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = v;
  __syncthreads();
  float m = s[0];
#pragma unroll
  for (int i = 1; i < NT / 64; ++i) m = fmaxf(m, s[i]);
  return m;
}

// rows of at most NT * E entries
template <int NT, typename XT>
__global__ __launch_bounds__(NT) void sample_short_kernel(SampleOpArgs a) {
  __shared__ Red red;
  __shared__ Few few;
  __shared__ float mx_s[2][NT / 64];
  __shared__ int best;
  const int row = blockIdx.x, tid = threadIdx.x;
  const XT* x = reinterpret_cast<const XT*>(a.logits) + row * a.stride;
  const Setting s = setting(a, row);
  Block<NT> blk{&red};
  RegRow r;
  r.per = (a.V + NT - 1) / NT;
  const int first = tid * r.per;
  float v[E], mx = -INFINITY, mn = INFINITY;
#pragma unroll
  for (int e = 0; e < E; ++e)
    if (e < r.per) v[e] = logit(x, min(first + e, a.V - 1));
  uint32_t n = 0;
#pragma unroll
  for (int e = 0; e < E; ++e)
    if (e < r.per) {
      if (first + e >= a.V) v[e] = -INFINITY;
      mx = fmaxf(mx, v[e]);
      if (v[e] > -INFINITY) { mn = fminf(mn, v[e]); ++n; }
    }
  mx = block_max<NT>(mx, mx_s[0]);
  if (mx == -INFINITY) {
    if (tid == 0) a.out[row] = -1;
    return;
  }
  if (s.k == 1) {   // the first entry of the order
    if (tid == 0) best = a.V;
    __syncthreads();
#pragma unroll
    for (int e = E - 1; e >= 0; --e)
      if (e < r.per && v[e] == mx) atomicMin(&best, first + e);
    __syncthreads();
    if (tid == 0) a.out[row] = best;
    return;
  }
  mn = -block_max<NT>(-mn, mx_s[1]);
  const Weigh weigh{mx, 1.4426950408889634074 / (double)s.T, a.shift};
#pragma unroll
  for (int e = 0; e < E; ++e) {
    r.key[e] = 0; r.w[e] = 0;
    if (e < r.per && v[e] > -INFINITY) { r.key[e] = order_key(v[e]); r.w[e] = weigh(v[e]); }
  }
  uint64_t none = 0;
  blk.sum(n, none, false);
  bool enough;
  const int e = filter_and_draw<NT>(r, blk, &few, weigh, s, n, order_key(mn), order_key(mx), 0, enough);
  if (e >= 0) a.out[row] = first + e;
}

// ---- long rows ------------------------------------------------------------------------------------------------------------------------------
// A wave owns a run of consecutive entries (a multiple of 64 * VEC); lanes take VEC consecutive ones at a time, 16-byte loads where the row allows.
template <typename XT, bool ALIGNED>
struct LongRow {
  static constexpr int VEC = 8;
  const XT* x;
  int V, seg;
  const Weigh* weigh;
  uint32_t floor_key;   // entries below are not counted
  template <typename F>
  __device__ __forceinline__ void each(int from, int to, F f) const {   // f(index of the first, values): every lane of the wave takes part
    const int lane = threadIdx.x & 63;
    for (int i0 = from; i0 < to; i0 += 64 * VEC) {
      const int i = i0 + lane * VEC;
      float v[VEC];
      if (ALIGNED && i + VEC <= V) {
        W8<XT> w;
        w.load(x + i);
#pragma unroll
        for (int e = 0; e < VEC; ++e) { const float y = w.get(e) + 0.f; v[e] = y != y ? -INFINITY : y; }
      } else {
#pragma unroll
        for (int e = 0; e < VEC; ++e) v[e] = i + e < V ? logit(x, i + e) : -INFINITY;
      }
      f(i, v);
    }
  }
  __device__ __forceinline__ int begin() const { return min((int)(threadIdx.x >> 6) * seg, V); }
  __device__ __forceinline__ int end() const { return min((int)(threadIdx.x >> 6) * seg + seg, V); }
  template <bool MASS>
  __device__ __forceinline__ void stat(uint32_t c, uint32_t& cnt, uint64_t& mass) const {
    uint32_t n = 0;
    uint64_t m = 0;
    each(begin(), end(), [&](int, const float (&v)[VEC]) {
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        const uint32_t key = order_key(v[e]);
        if (key >= c && key >= floor_key) { ++n; if (MASS) m += (*weigh)(v[e]); }
      }
    });
    cnt = n;
    mass = m;
  }
  __device__ __forceinline__ void gather(uint32_t lo, uint32_t hi, Few* few) const {
    each(begin(), end(), [&](int, const float (&v)[VEC]) {
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        const uint32_t key = order_key(v[e]);
        if (key >= lo && key < hi && key >= floor_key) {
          const int at = atomicAdd(&few->n, 1);
          if (at < 64) few->key[at] = key;
        }
      }
    });
  }
};
struct ListLds { float x[LIST]; int32_t i[LIST]; };

template <typename XT, bool ALIGNED>
__global__ __launch_bounds__(1024) void sample_long_kernel(SampleOpArgs a) {
  constexpr int NT = 1024;
  extern __shared__ __attribute__((aligned(16))) char dyn[];
  ListLds* list = reinterpret_cast<ListLds*>(dyn);
  __shared__ Red red;
  __shared__ Few few;
  __shared__ float mx_s[2][NT / 64];
  __shared__ int best;
  __shared__ uint32_t cnt_s[NT / 64], tie_s[NT / 64];
  __shared__ uint64_t mass_s[NT / 64];
  const int row = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const Setting s = setting(a, row);
  Block<NT> blk{&red};
  LongRow<XT, ALIGNED> src;
  constexpr int VEC = LongRow<XT, ALIGNED>::VEC;
  src.x = reinterpret_cast<const XT*>(a.logits) + row * a.stride;
  src.V = a.V;
  src.seg = (a.V + NT * VEC - 1) / (NT * VEC) * (64 * VEC);
  src.floor_key = NEG_INF_KEY + 1;
  const int from = src.begin(), to = src.end();

  float mx = -INFINITY, mn = INFINITY;
  src.each(from, to, [&](int, const float (&v)[VEC]) {
#pragma unroll
    for (int e = 0; e < VEC; ++e) { mx = fmaxf(mx, v[e]); mn = v[e] > -INFINITY ? fminf(mn, v[e]) : mn; }
  });
  mx = block_max<NT>(mx, mx_s[0]);
  if (mx == -INFINITY) {
    if (tid == 0) a.out[row] = -1;
    return;
  }
  if (s.k == 1) {
    if (tid == 0) best = a.V;
    __syncthreads();
    src.each(from, to, [&](int i, const float (&v)[VEC]) {
#pragma unroll
      for (int e = VEC - 1; e >= 0; --e)
        if (v[e] == mx) atomicMin(&best, i + e);
    });
    __syncthreads();
    if (tid == 0) a.out[row] = best;
    return;
  }
  mn = -block_max<NT>(-mn, mx_s[1]);
  const Weigh weigh{mx, 1.4426950408889634074 / (double)s.T, a.shift};
  src.weigh = &weigh;
  const uint32_t key_min = order_key(mn), key_max = order_key(mx);
  const bool filtered = s.k || s.top_p < 1.f;
  Cut cut{0u, 0u};      // what the streaming draw keeps
  uint32_t n = 0;
  if (filtered) {
    // threshold of the list, from samples spread over the row
    RegRow r;
    uint32_t ns = 0;
    r.per = SAMPLES / NT;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      r.key[e] = 0; r.w[e] = 0;
      if (e < SAMPLES / NT) {
        const float v = logit(src.x, (int)((int64_t)(tid * (SAMPLES / NT) + e) * a.V / SAMPLES));
        if (v > -INFINITY) { r.key[e] = order_key(v); ++ns; }
      }
    }
    uint64_t none = 0;
    blk.sum(ns, none, false);
    uint32_t thr = key_min;
    const uint32_t rank = max(1u, (uint32_t)((int64_t)AIM * SAMPLES / a.V));
    if (ns > rank) thr = find_cut<NT, false>(r, blk, &few, weigh, NEG_INF_KEY + 1, ns, key_max + 1, rank, 0.0).key;
    // count what the list would take; the whole row's mass where top-p refers to it
    const bool want_mass = s.top_p < 1.f && !s.k;
    uint32_t take = 0, more = 0, all = 0;
    uint64_t base = 0;
    src.each(from, to, [&](int, const float (&v)[VEC]) {
#pragma unroll
      for (int e = 0; e < VEC; ++e) {
        const uint32_t key = order_key(v[e]);
        take += key >= thr && key > NEG_INF_KEY;
        more += key > thr;
        all += key > NEG_INF_KEY;
        if (want_mass) base += weigh(v[e]);
      }
    });
    uint32_t total_take = take, total_more = more;
    n = all;
    blk.sum(n, base, want_mass);
    blk.sum(total_take, none, false);
    blk.sum(total_more, none, false);
    if (total_take > LIST) { ++thr; take = more; total_take = total_more; }   // (a crowd of equals at the threshold stays out)
    const bool list_ok = total_take <= LIST && (s.k == 0 || (uint32_t)s.k <= total_take || total_take == n);
    bool enough = false;
    if (list_ok && total_take) {
      const uint32_t wave_take = wave_sum32(take);
      if (lane == 0) cnt_s[wave] = wave_take;
      __syncthreads();
      uint32_t at = 0;
      for (int w = 0; w < wave; ++w) at += cnt_s[w];
      src.each(from, to, [&](int i, const float (&v)[VEC]) {
        uint32_t mine = 0;
#pragma unroll
        for (int e = 0; e < VEC; ++e) { const uint32_t key = order_key(v[e]); mine += key >= thr && key > NEG_INF_KEY; }
        uint32_t upto = mine;
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
          const uint32_t y = __shfl_up(upto, d);
          if (lane >= d) upto += y;
        }
        uint32_t p = at + upto - mine;
        at += __builtin_amdgcn_readlane(upto, 63);
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          const uint32_t key = order_key(v[e]);
          if (key >= thr && key > NEG_INF_KEY) { list->x[p] = v[e]; list->i[p] = i + e; ++p; }
        }
      });
      __syncthreads();
      r.per = (int)((total_take + NT - 1) / NT);
#pragma unroll
      for (int e = 0; e < E; ++e) {
        r.key[e] = 0; r.w[e] = 0;
        const uint32_t p = tid * r.per + e;
        if (e < r.per && p < total_take) { const float v = list->x[p]; r.key[e] = order_key(v); r.w[e] = weigh(v); }
      }
      const int e = filter_and_draw<NT>(r, blk, &few, weigh, s, total_take, thr > key_min ? thr : key_min, key_max, s.k ? 0 : base, enough);
      if (e >= 0) a.out[row] = list->i[tid * r.per + e];
    }
    if (enough) return;
    // the list does not hold the answer: the same search over the row itself
    if (s.k && (uint32_t)s.k < n) cut = find_cut<NT, false>(src, blk, &few, weigh, key_min, n, key_max + 1, (uint32_t)s.k, 0.0);
    if (s.top_p < 1.f) {
      uint32_t cnt;
      uint64_t above;
      src.template stat<true>(cut.key + 1, cnt, above);
      blk.sum(cnt, above, true);
      const uint64_t each = cut.ties ? weigh(key_value(cut.key)) : 0;
      const double want = target(s.top_p, above + each * cut.ties);
      if ((double)above >= want) {
        src.floor_key = max(src.floor_key, cut.key + 1);
        cut = find_cut<NT, true>(src, blk, &few, weigh, max(key_min, src.floor_key), cnt, key_max + 1, 0u, want);
        src.floor_key = NEG_INF_KEY + 1;
      } else {
        const double q = each ? ceil((want - (double)above) / (double)each) : 1.0;
        if (q < (double)cut.ties) cut.ties = q < 1.0 ? 1u : (uint32_t)q;
      }
    }
  }
  // draw by streaming: mass and ties of every wave's run, then the one run that holds the target
  const double least = (double)s.min_p * (double)(1ull << weigh.shift);
  auto value = [&](float v) { const uint64_t w = weigh(v); return (double)w < least ? 0ull : w; };
  uint64_t mass = 0;
  uint32_t ties = 0;
  src.each(from, to, [&](int, const float (&v)[VEC]) {
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      const uint32_t key = order_key(v[e]);
      if (key > cut.key && key > NEG_INF_KEY) mass += value(v[e]);
      ties += key == cut.key;
    }
  });
  mass = wave_sum64(mass);
  ties = wave_sum32(ties);
  const uint64_t each = cut.ties ? value(key_value(cut.key)) : 0;
  if (lane == 0) { mass_s[wave] = mass; tie_s[wave] = ties; }
  __syncthreads();
  uint64_t total = 0, run_before = 0;
  uint32_t tie_before = 0;
  for (int w = 0; w < NT / 64; ++w) {
    const uint32_t t = min(tie_s[w], cut.ties - min(cut.ties, tie_before));
    total += mass_s[w] + t * each;
    tie_before += tie_s[w];
  }
  const double want = (double)s.u * (double)total;
  int at = 0;
  tie_before = 0;
  for (int w = 0; w < NT / 64; ++w) {
    const uint32_t t = min(tie_s[w], cut.ties - min(cut.ties, tie_before));
    const uint64_t m = mass_s[w] + t * each;
    at = w;
    if ((double)(run_before + m) > want) break;
    run_before += m;
    tie_before += tie_s[w];
  }
  // all threads on that run, consecutive entries each
  const int lo = min(at * src.seg, a.V), hi = min(lo + src.seg, a.V), per = (hi - lo + NT - 1) / NT;
  const int i0 = min(lo + tid * per, hi), i1 = min(i0 + per, hi);
  uint64_t my_ties = 0, unused;
  for (int i = i0; i < i1; ++i) my_ties += order_key(logit(src.x, i)) == cut.key;
  const uint64_t seen0 = tie_before + blk.before(my_ties, unused);
  uint64_t seen = seen0, mine = 0;
  auto kept = [&](int i) -> uint64_t {
    const float v = logit(src.x, i);
    const uint32_t key = order_key(v);
    if (key <= NEG_INF_KEY || key < cut.key || (key == cut.key && seen++ >= cut.ties)) return 0;
    return value(v);
  };
  for (int i = i0; i < i1; ++i) mine += kept(i);
  const uint64_t before = run_before + blk.before(mine, unused);
  if (!((double)before > want) && (double)(before + mine) > want) {
    uint64_t run = before;
    seen = seen0;
    for (int i = i0; i < i1; ++i) {
      run += kept(i);
      if ((double)run > want) { a.out[row] = i; break; }
    }
  }
}

extern "C" int csm_ops_sample_filtered(const csm_ops_sample_t* p, void* stream) {
  if (!p) return ops_fail(CSM_OPS_ERR_ARG, "null argument");
  if (p->x_dtype != CSM_OPS_F32 && p->x_dtype != CSM_OPS_BF16) return ops_fail(CSM_OPS_ERR_ARG, "unknown dtype %d", p->x_dtype);
  if (p->rows < 0 || p->V < 1) return ops_fail(CSM_OPS_ERR_ARG, "rows must not be negative and V must be positive");
  if (p->V > (1 << 24)) return ops_fail(CSM_OPS_ERR_CAPACITY, "V = %d: at most 2^24", p->V);
  if (!p->temperatures && !(p->temperature >= 0.f && p->temperature < INFINITY)) return ops_fail(CSM_OPS_ERR_ARG, "temperature must be finite and not negative");
  if (!p->topks && (p->topk < 0 || p->topk > p->V)) return ops_fail(CSM_OPS_ERR_ARG, "selected index k out of range");
  if (!p->top_ps && !(p->top_p > 0.f && p->top_p <= 1.f)) return ops_fail(CSM_OPS_ERR_ARG, "top_p must lie in (0, 1]");
  if (!p->min_ps && !(p->min_p >= 0.f && p->min_p <= 1.f)) return ops_fail(CSM_OPS_ERR_ARG, "min_p must lie in [0, 1]");
  if (!p->rows) return 0;
  if (!p->logits || !p->uniform || !p->out) return ops_fail(CSM_OPS_ERR_ARG, "null pointer");
  SampleOpArgs a;
  a.logits = p->logits; a.stride = p->logits_stride; a.V = p->V; a.uniform = p->uniform; a.temperatures = p->temperatures;
  a.top_ps = p->top_ps; a.min_ps = p->min_ps; a.topks = p->topks; a.temperature = p->temperature; a.top_p = p->top_p; a.min_p = p->min_p;
  a.topk = p->topk; a.out = p->out;
  int bits = 0;
  while ((1 << bits) < p->V) ++bits;
  a.shift = 62 - bits < 51 ? 62 - bits : 51;   // V weights of at most 1 stay below 2^62
  hipStream_t st = (hipStream_t)stream;
  const bool b = p->x_dtype == CSM_OPS_BF16;
  const dim3 grid(p->rows);
  if (p->V <= 256 * E) {
    if (b) hipLaunchKernelGGL((sample_short_kernel<256, bf16_t>), grid, dim3(256), 0, st, a);
    else hipLaunchKernelGGL((sample_short_kernel<256, float>), grid, dim3(256), 0, st, a);
  } else if (p->V <= 1024 * E) {
    if (b) hipLaunchKernelGGL((sample_short_kernel<1024, bf16_t>), grid, dim3(1024), 0, st, a);
    else hipLaunchKernelGGL((sample_short_kernel<1024, float>), grid, dim3(1024), 0, st, a);
  } else {
    const bool al = ops_aligned(p->logits) && (p->rows == 1 || ops_stride16(p->logits_stride, p->x_dtype));
    const void* f = b ? (al ? (const void*)sample_long_kernel<bf16_t, true> : (const void*)sample_long_kernel<bf16_t, false>)
                      : (al ? (const void*)sample_long_kernel<float, true> : (const void*)sample_long_kernel<float, false>);
    OPS_HIP(hipFuncSetAttribute(f, hipFuncAttributeMaxDynamicSharedMemorySize, sizeof(ListLds)));
    void* args[] = {&a};
    OPS_HIP(hipLaunchKernel(f, grid, dim3(1024), args, sizeof(ListLds), st));
  }
  OPS_HIP(hipGetLastError());
  return 0;
}
