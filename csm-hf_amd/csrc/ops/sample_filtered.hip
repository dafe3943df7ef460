// Sampling with temperature, top-k, top-p and min-p from one given uniform per row (include/csm_ops.h).
//   w_i = exp((x_i - max) / T);  rows ordered by (x descending, index ascending);  every filter keeps a PREFIX of that order, so the kept set
//   is "key > cut, and the first `ties` entries with key == cut";  the token is where the running sum of kept w (index order) passes u * total.
// Sums are uint64 fixed point of weights computed in fp64: exact integer additions, so neither the split over threads nor any order of arrival
// changes a result.  The scale of a weight is 2^min(62 - ceil log2 n, 51) where at most n entries are summed (a row in registers, a list, a chunk: n <= 16 384),
// and 2^min(61 - floor log2 mass, 51) where a long row is streamed, `mass` its total in units of the largest weight: what is rounded away per weight is
// below 2^-49 of the largest, or 2^-61 of the total.
//
// No sort of the row: a histogram over its values (counts and masses, a few bins per thread, LDS atomics on integers) is summed from the top, the bin in
// which a cut falls is gathered (at most 64 entries) and ranked exactly by one wave.  Rows whose values crowd in one bin go the long way:
// an interval of order keys is narrowed by false position and bisection, one block sum per step, until 64 entries or one single key are left.
//   V <= 16 384: one workgroup, the row in registers (4 or 16 consecutive entries per thread), read once.  Such a launch is a chain of dependent
//                steps over code that runs once, so its loops carry no branches and its sums stay on the DPP path.  A top-k of at most 64 narrows
//                the row to 64 entries at once, and one wave does the rest without a barrier.
//   larger V:    three launches, so that few rows still use many CUs: a threshold near the 12 288th largest from 4 096 samples; per chunk of
//                8 192 entries its maximum, its mass and the entries above the threshold; per row the cuts and the draw on those entries.
//                Where they are not enough (a flat row whose nucleus is larger), the same search streams over the row, one workgroup a row with an fp64
//                exponential per entry and step: 64 rows of 128 256 with deviation 1 (nucleus of 0.9: some 73 000) take 1.3 ms, one row 1.2.
//
// What bounds it: not the bytes.  One row of 2051 fp32: 6.5 us, the chain of steps; 512 of them, each with its own filters: 13 us for 4.2 MB (0.9 at the rate
// of a large copy) -- two workgroups a CU, whose steps overlap little.  64 rows of 128 256 bf16, top_p alone: 7.4 + 17 + 17.1 us for 16.4 MB (3.4); the
// chunks' 8.2 million fp64 exponentials (13 operations of 8 clocks a wave) take some 8 of the 17, in the list's 17 are 4 to fetch it, 5 for the histogram, 3
// for the draw and the heads' sums.
#include "ops_common.h"
#include <math.h>

struct SampleOpArgs {
  const void* logits;
  int64_t stride;
  int V, shift;   // shift: binary point of the weights where the whole row may be summed, whatever it holds
  const float *uniform, *temperatures, *top_ps, *min_ps;
  const int32_t* topks;
  float temperature, top_p, min_p;
  int topk;
  int32_t* out;
  // long rows: workspace
  int chunks;
  uint32_t* thr;           // [rows]
  struct ChunkHead* heads; // [rows][chunks]
  uint2* lists;            // [rows][chunks][CHUNK] (key, index)
};
constexpr int LIST = 1024 * 16;           // entries that fit the registers of a workgroup
constexpr int SHORT = 256 * 16;           // entries that fit those of a small one
constexpr int LIST_SHIFT = 48;            // binary point of their weights: 2^14 of them stay within 2^62
constexpr int SAMPLES = 4096, AIM = LIST * 3 / 4;   // the list's threshold is a sample's order statistic that aims at this many entries: at V = 131 072
                                                    // their number scatters by 613, LIST is 6.7 of that away
// (a chunk of 8192 is 32 entries a thread: 16 chunks of a row of 128 256, so that 16 rows already fill the CUs).  Any chunk may list all it has, so the
// list fails by its total alone, wherever in the row the large values stand.  The rows that stream for it: a nucleus (or what min-p keeps) larger than the list;
// more equal values at the threshold than fit; a sample far off -- the total scatters by sqrt(3 (V - 12 288)), so LIST is 4.7 of that away at V = 2^18, but
// 2.3 at 2^20 and 1.6 at 2^21 (one row in a hundred, in twenty).  Chunk lists of 2048 overflowed in every row below V = 49 152, and where one chunk held 2.6 times
// its share: 64 rows under top_p 0.9 (us, then / now) 177 / 48 at V = 16 385, 217 / 36 at 32 000, 432 / 42 at 50 257, 773 / 44 at 128 256 with the
// largest values in the first chunk.
constexpr int CHUNK = 8192, MAX_V = 1 << 21, MAX_CHUNKS = MAX_V / CHUNK;
struct ChunkHead { double mass; float mx; int32_t at; uint32_t count, pad; };   // mass relative to the chunk's own maximum, `at` its first place

// Order keys: larger value = larger key, one key per value of the type (a search that must end on a single key needs 16 fewer steps where
// values are bf16).  value() of a key that no number has is a NaN.  Keys at or below NONE are no entries.
template <typename T>
struct Keys;
template <>
struct Keys<float> {
  static constexpr uint32_t NONE = 0x007fffffu;   // of -inf
  static __device__ __forceinline__ uint32_t key(float x) {
    const uint32_t u = __float_as_uint(x);
    return u ^ ((u >> 31) ? 0xffffffffu : 0x80000000u);
  }
  static __device__ __forceinline__ float value(uint32_t k) { return __uint_as_float((k >> 31) ? k ^ 0x80000000u : ~k); }
};
template <>
struct Keys<bf16_t> {
  static constexpr uint32_t NONE = Keys<float>::NONE >> 16;
  static __device__ __forceinline__ uint32_t key(float x) { return Keys<float>::key(x) >> 16; }   // (other values than the type's: the next key below)
  static __device__ __forceinline__ float value(uint32_t k) { return Keys<float>::value(k << 16 | ((k >> 15) ? 0u : 0xffffu)); }
};
template <typename T>
__device__ __forceinline__ float logit(const T* x, int i) {   // NaN counts as -inf, -0 as +0
  const float v = to_f32(x[i]) + 0.f;
  return v != v ? -INFINITY : v;
}
// w * 2^shift as an integer.  2^t = 2^n 2^f with f in [-1/2, 1/2] from its power series (up to f^11: below 2^-47); adding 2^52 leaves the rounded
// integer in the mantissa (shift <= 51).  -inf ends as 0 without a test (the maximum also drops the NaN of 0 * -inf).
struct Weigh {
  float mx;
  double k2;   // log2(e) / T
  int shift;
  __device__ __forceinline__ uint64_t operator()(float x) const {
    if (mx == INFINITY) return x == INFINITY ? 1ull << shift : 0ull;
    const double t = fmax(((double)x - (double)mx) * k2, -1200.0), n = rint(t), f = t - n;
    double p = 4.4455382718708116e-10;   // ln(2)^i / i!, i = 11 .. 0
    p = __fma_rn(p, f, 7.0549116208011233e-09); p = __fma_rn(p, f, 1.0178086009239700e-07); p = __fma_rn(p, f, 1.3215486790144309e-06);
    p = __fma_rn(p, f, 1.5252733804059840e-05); p = __fma_rn(p, f, 1.5403530393381610e-04); p = __fma_rn(p, f, 1.3333558146428443e-03);
    p = __fma_rn(p, f, 9.6181291076284772e-03); p = __fma_rn(p, f, 5.5504108664821580e-02); p = __fma_rn(p, f, 2.4022650695910071e-01);
    p = __fma_rn(p, f, 6.9314718055994531e-01); p = __fma_rn(p, f, 1.0);
    return (uint64_t)__double_as_longlong(ldexp(p, (int)n + shift) + 4503599627370496.0) & 0xfffffffffffffull;
  }
};

// The same where millions of them bound the launch: 2^t = 2^(n / 32) 2^f with |f| <= 1/64, the root from a table in LDS (no two of its entries share a bank),
// f to the 5th power (below 2^-48).  Adding 1.5 * 2^47 leaves n in the low mantissa; 13 fp64 operations instead of 20, 43.8 -> 41.4 us for 64 rows of
// 128 256 bf16 logits.  Where an exponential is one link of a chain of steps, the shorter way without a table to wait for is Weigh's.
__device__ const double roots[32] = {  // 2^(i / 32)
    1.0, 1.0218971486541166, 1.0442737824274138, 1.0671404006768237, 1.0905077326652577, 1.1143867425958924, 1.1387886347566916, 1.1637248587775775,
    1.189207115002721, 1.215247359980469, 1.241857812073484, 1.2690509571917332, 1.2968395546510096, 1.3252366431597413, 1.3542555469368927, 1.383909881963832,
    1.4142135623730951, 1.4451808069770467, 1.4768261459394993, 1.5091644275934228, 1.5422108254079407, 1.5759808451078865, 1.6104903319492543, 1.645755478153965,
    1.681792830507429, 1.718619298122478, 1.7562521603732995, 1.7947090750031072, 1.8340080864093424, 1.8741676341103, 1.9152065613971474, 1.9571441241754002};
struct WeighMany {
  float mx;
  double k2;
  int shift;
  const double* table;   // in LDS
  __device__ __forceinline__ uint64_t operator()(float x) const {
    if (mx == INFINITY) return x == INFINITY ? 1ull << shift : 0ull;
    const double t = fmax(((double)x - (double)mx) * k2, -1000.0), whole = t + 211106232532992.0, f = t - (whole - 211106232532992.0);
    const int n = (int)(uint32_t)__double_as_longlong(whole);
    const double root = table[n & 31];
    double p = 0.0013333558146428441;   // ln(2)^i / i!, i = 5 .. 0
    p = __fma_rn(p, f, 0.009618129107628477); p = __fma_rn(p, f, 0.055504108664821576); p = __fma_rn(p, f, 0.2402265069591007);
    p = __fma_rn(p, f, 0.6931471805599453); p = __fma_rn(p, f, 1.0);
    const double scale = __hiloint2double(__double2hiint(root) + (((n >> 5) + shift) << 20), __double2loint(root));
    return (uint64_t)__double_as_longlong(__fma_rn(p, scale, 4503599627370496.0)) & 0xfffffffffffffull;
  }
};

// ---- block sums -------------------------------------------------------------------------------------------------------------------------
// running sum over the lanes on the DPP path (row shifts, then the two row broadcasts): no trip through the LDS crossbar
template <int CTRL, int ROWS>
__device__ __forceinline__ uint32_t dpp0(uint32_t v) { return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, ROWS, 0xf, false); }
template <int CTRL, int ROWS>
__device__ __forceinline__ uint64_t dpp0(uint64_t v) { return (uint64_t)dpp0<CTRL, ROWS>((uint32_t)v) | ((uint64_t)dpp0<CTRL, ROWS>((uint32_t)(v >> 32)) << 32); }
template <int CTRL>
__device__ __forceinline__ uint32_t dpp_any(uint32_t v) { return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xf, 0xf, true); }
template <int CTRL>
__device__ __forceinline__ uint64_t dpp_any(uint64_t v) { return (uint64_t)dpp_any<CTRL>((uint32_t)v) | ((uint64_t)dpp_any<CTRL>((uint32_t)(v >> 32)) << 32); }
template <int CTRL, int ROWS>
__device__ __forceinline__ double dpp0(double v) { return __longlong_as_double((long long)dpp0<CTRL, ROWS>((uint64_t)__double_as_longlong(v))); }
template <typename T>
__device__ __forceinline__ T row_upto(T v) {   // within 16 lanes
  v += dpp0<0x111, 0xf>(v); v += dpp0<0x112, 0xf>(v); v += dpp0<0x114, 0xf>(v); v += dpp0<0x118, 0xf>(v);
  return v;
}
template <typename T>
__device__ __forceinline__ T wave_upto(T v) {
  v = row_upto(v);
  v += dpp0<0x142, 0xa>(v); v += dpp0<0x143, 0xc>(v);
  return v;
}
__device__ __forceinline__ uint32_t lane_value(uint32_t v, int lane) { return (uint32_t)__builtin_amdgcn_readlane((int)v, lane); }
__device__ __forceinline__ uint64_t lane_value(uint64_t v, int lane) { return (uint64_t)lane_value((uint32_t)v, lane) | ((uint64_t)lane_value((uint32_t)(v >> 32), lane) << 32); }
template <typename T>
__device__ __forceinline__ T wave_total(T v) { return lane_value(wave_upto(v), 63); }
struct Red { uint64_t m[2][16]; uint32_t c[2][16]; };   // two generations: one barrier per sum

// sum over the W (4 or 16) entries that the waves left in LDS, in every lane
template <int W, typename T>
__device__ __forceinline__ T over_waves(T v) {
  v += dpp_any<0xB1>(v); v += dpp_any<0x4E>(v);
  if (W > 4) { v += dpp_any<0x141>(v); v += dpp_any<0x140>(v); }
  return v;
}

template <int NT>
struct Block {
  static constexpr int W = NT / 64;
  static_assert(W == 4 || W == 16, "");
  Red* r;
  int gen = 0;
  // totals over the waves: cnt is already the wave's, mass is per lane
  template <bool MASS>
  __device__ __forceinline__ void sum(uint32_t& cnt, uint64_t& mass) {
    if (MASS) mass = wave_total(mass);
    const int g = gen ^= 1, lane = threadIdx.x & 63;
    if (lane == 0) { r->c[g][threadIdx.x >> 6] = cnt; if (MASS) r->m[g][threadIdx.x >> 6] = mass; }
    __syncthreads();
    cnt = lane_value(over_waves<W>(r->c[g][lane % W]), 0);
    if (MASS) mass = lane_value(over_waves<W>(r->m[g][lane % W]), 0);
  }
  __device__ __forceinline__ uint32_t count(uint32_t wave_cnt) {
    uint64_t none = 0;
    sum<false>(wave_cnt, none);
    return wave_cnt;
  }
  // sums over the threads before this one, and over all
  __device__ __forceinline__ void before2(uint32_t& c, uint64_t& m, uint32_t& all_c, uint64_t& all_m) {
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const uint32_t x = wave_upto(c);
    const uint64_t y = wave_upto(m);
    const int g = gen ^= 1;
    if (lane == 63) { r->c[g][wave] = x; r->m[g][wave] = y; }
    __syncthreads();
    const uint32_t wc = r->c[g][lane % W];
    const uint64_t wm = r->m[g][lane % W];
    all_c = lane_value(over_waves<W>(wc), 0);
    all_m = lane_value(over_waves<W>(wm), 0);
    c = lane_value(over_waves<W>(lane % W < wave ? wc : 0u), 0) + x - c;
    m = lane_value(over_waves<W>(lane % W < wave ? wm : (uint64_t)0), 0) + y - m;
  }
  template <typename T>
  __device__ __forceinline__ T before(T v, T& total) {
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const T x = wave_upto(v);
    const int g = gen ^= 1;
    if (lane == 63) r->m[g][wave] = x;
    __syncthreads();
    const T w = (T)r->m[g][lane % W];
    total = lane_value(over_waves<W>(w), 0);
    return lane_value(over_waves<W>(lane % W < wave ? w : (T)0), 0) + x - v;
  }
};

// ---- one wave's sort of 64 values, descending by lane: a bitonic network whose exchanges are DPP moves and row swaps ----------------------------
template <int D>
__device__ __forceinline__ uint32_t lane_xor(uint32_t v) {
  if constexpr (D == 1) return dpp_any<0xB1>(v);
  if constexpr (D == 2) return dpp_any<0x4E>(v);
  if constexpr (D == 4) {   // banks 1 and 3 of a row from 4 lanes below, 0 and 2 from 4 lanes above
    const int up = __builtin_amdgcn_update_dpp(0, (int)v, 0x114, 0xf, 0xa, false);
    return (uint32_t)__builtin_amdgcn_update_dpp(up, (int)v, 0x104, 0xf, 0x5, false);
  }
  if constexpr (D == 8) return dpp_any<0x128>(v);
  if constexpr (D == 16) { const auto r = __builtin_amdgcn_permlane16_swap(v, v, false, false); return threadIdx.x & 16 ? r[0] : r[1]; }
  if constexpr (D == 32) { const auto r = __builtin_amdgcn_permlane32_swap(v, v, false, false); return threadIdx.x & 32 ? r[0] : r[1]; }
}
template <int D>
__device__ __forceinline__ uint64_t lane_xor(uint64_t v) { return (uint64_t)lane_xor<D>((uint32_t)v) | ((uint64_t)lane_xor<D>((uint32_t)(v >> 32)) << 32); }
template <int SIZE, int D, typename T>
__device__ __forceinline__ void sort_merge(T& v) {
  const T o = lane_xor<D>(v);
  const int lane = threadIdx.x & 63;
  const bool big = ((lane & D) == 0) == ((lane & SIZE) == 0);   // this lane keeps the larger of the two (SIZE 64: descending throughout)
  v = (v > o) == big ? v : o;
  if constexpr (D > 1) sort_merge<SIZE, D / 2>(v);
}
template <typename T>
__device__ __forceinline__ void wave_sort(T& v) {
  sort_merge<2, 1>(v); sort_merge<4, 2>(v); sort_merge<8, 4>(v); sort_merge<16, 8>(v); sort_merge<32, 16>(v); sort_merge<64, 32>(v);
}

// ---- the search ---------------------------------------------------------------------------------------------------------------------------
struct Cut { uint32_t key; uint32_t ties, same; };   // kept: keys above `key`, and the first `ties` of the `same` entries equal to it
struct Few { uint32_t key[64]; int n; };

// The interval of a search and where to look next: a false-position step over the values (with the Illinois rule: an end that stays twice has its
// residual halved), every fourth time the middle key -- few steps on a smooth row, a bound on any.  y: the measure's distance from its target
// in a scale that is straight enough (counts: their logarithm, a tail falls fast; masses: themselves).
template <typename K>
struct Interval {
  uint32_t lo, hi;      // the target is reached at lo, not at hi
  float y_lo, y_hi;
  int step = 0, side = 0;
  __device__ __forceinline__ uint32_t probe() const {   // lo < probe < hi
    const float a = K::value(lo), b = K::value(hi - 1);
    const float part = fminf(fmaxf(y_lo / (y_lo - y_hi), 0.03f), 0.97f);
    const uint32_t kv = K::key((1.f - part) * a + part * b + 0.f);
    return (step & 3) != 3 && kv > lo && kv < hi ? kv : lo + (hi - lo) / 2;   // (a NaN's key is above any hi)
  }
  __device__ __forceinline__ void take(uint32_t mid, float y, bool reached) {
    ++step;
    if (reached) { lo = mid; y_lo = y; if (side == 1) y_hi *= 0.5f; side = 1; }
    else { hi = mid; y_hi = y; if (side == -1) y_lo *= 0.5f; side = -1; }
  }
};
__device__ __forceinline__ float log_count(uint32_t n) { return __log2f(fmaxf((float)n, 0.5f)); }

// The exact cut among the gathered entries, above which lie `above` entries of mass `mass`; every wave does it for itself.  kept: the mass that stays
template <typename K, bool MASS>
__device__ __forceinline__ void rank_few(Few* few, const Weigh& weigh, uint32_t above, uint64_t mass, uint32_t want_n, double want_m, Cut& cut, uint64_t& kept) {
  const int lane = threadIdx.x & 63, n = min(few->n, 64);
  uint32_t key = lane < n ? few->key[lane] : 0;
  wave_sort(key);
  const uint64_t upto = mass + wave_upto(lane < n ? weigh(K::value(key)) : (uint64_t)0);
  const uint64_t at = __ballot(lane < n && (MASS ? (double)upto >= want_m : above + lane + 1 >= want_n));
  const int first = at ? __ffsll((unsigned long long)at) - 1 : 0;
  cut.key = lane_value(key, first);
  kept = lane_value(upto, first);
  const uint64_t equal = __ballot(key == cut.key);
  cut.same = __popcll(equal);
  cut.ties = __popcll(equal & ((2ull << first) - 1));
  __syncthreads();   // `few` may be filled again
}

// Largest interval end `lo` whose entries at or above it reach the target -- a count (MASS false) or a mass -- narrowed to the exact entry.
// At entry: everything in [lo, ...) reaches it (cnt_lo entries, mass_lo), nothing at or above hi does.
template <typename K, bool MASS, int NT, typename Src>
__device__ __forceinline__ Cut find_cut(Src& src, Block<NT>& blk, Few* few, const Weigh& weigh, uint32_t lo, uint32_t cnt_lo, uint64_t mass_lo, uint32_t hi, uint32_t want_n, double want_m) {
  uint32_t cnt_hi = 0;
  uint64_t mass_hi = 0;
  const float goal = MASS ? 0.f : log_count(want_n);
  Interval<K> in{lo, hi, MASS ? (float)((double)mass_lo - want_m) : log_count(cnt_lo) - goal, MASS ? -(float)want_m : -1.f - goal};
  while (cnt_lo - cnt_hi > 64 && in.hi - in.lo > 1) {
    const uint32_t mid = in.probe();
    uint32_t cnt;
    uint64_t mass = 0;
    src.template stat<MASS>(mid, cnt, mass);
    blk.template sum<MASS>(cnt, mass);
    const bool reached = MASS ? (double)mass >= want_m : cnt >= want_n;
    in.take(mid, MASS ? (float)((double)mass - want_m) : log_count(cnt) - goal, reached);
    if (reached) cnt_lo = cnt;
    else { cnt_hi = cnt; mass_hi = mass; }
  }
  lo = in.lo; hi = in.hi;
  if (hi - lo <= 1) {   // one key: equal entries, equal weights
    const uint32_t same = cnt_lo - cnt_hi;
    if (!MASS) return {lo, want_n - cnt_hi, same};
    const uint64_t each = weigh(K::value(lo));
    const double q = each ? ceil((want_m - (double)mass_hi) / (double)each) : 1.0;
    return {lo, q < 1.0 ? 1u : q > (double)same ? same : (uint32_t)q, same};
  }
  if (threadIdx.x == 0) few->n = 0;
  __syncthreads();
  src.gather(lo, hi, few);
  __syncthreads();
  Cut cut;
  uint64_t kept;
  rank_few<K, MASS>(few, weigh, cnt_hi, mass_hi, want_n, want_m, cut, kept);
  return cut;
}

// a row (or list) in registers: thread t holds entries t * per .. t * per + per - 1; key 0, w 0 = not (or no longer) an entry
// BINS: the entries' bins of the histogram built last are kept too (a row of 2051 under a small top-k 7.7 -> 7.1 us); not where 1024 threads hold a whole row
// with its values, whose registers that would spill (19.1 -> 19.8)
template <int E, bool BINS = true>
struct RegRow {
  uint32_t key[E], bin[BINS ? E : 1];
  uint64_t w[E];
  int per;
  template <typename K>
  __device__ __forceinline__ void weigh_all(const Weigh& weigh) {
#pragma unroll
    for (int e = 0; e < E; ++e) {
      w[e] = 0;
      if (e < per && key[e]) w[e] = weigh(K::value(key[e]));
    }
  }
  template <bool MASS>
  __device__ __forceinline__ void stat(uint32_t c, uint32_t& cnt, uint64_t& mass) const {   // cnt: of the wave
    cnt = 0;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      if (E > 4 && e % 4 == 0 && e >= per) break;   // (uniform; in steps of four)
      const bool in = key[e] >= c;
      cnt += __popcll(__ballot(in));
      if (MASS) mass += in ? w[e] : 0;
    }
  }
  __device__ __forceinline__ void gather(uint32_t lo, uint32_t hi, Few* few) const {
    uint64_t in[E];
    uint32_t n = 0;
#pragma unroll
    for (int e = 0; e < E; ++e) {
      in[e] = __ballot(key[e] - lo < hi - lo);
      n += __popcll(in[e]);
    }
    if (!n) return;
    uint32_t at = 0;
    if ((threadIdx.x & 63) == 0) at = atomicAdd(&few->n, (int)n);   // one reservation per wave; the order does not matter, they are sorted
    at = lane_value(at, 0);
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const uint32_t p = at + __builtin_amdgcn_mbcnt_hi((uint32_t)(in[e] >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)in[e], 0));
      if (key[e] - lo < hi - lo && p < 64) few->key[p] = key[e];
      at += __popcll(in[e]);
    }
  }
};

// of the entries equal to a cut, drop those that it does not keep (entries below it are left: they lie under every later probe)
template <int E, bool BINS, int NT>
__device__ __forceinline__ void drop_ties(RegRow<E, BINS>& r, Block<NT>& blk, const Cut& c) {
  if (c.ties >= c.same) return;
  uint32_t mine = 0, total;
#pragma unroll
  for (int e = 0; e < E; ++e) mine += r.key[e] == c.key;
  uint32_t rank = blk.before(mine, total);
#pragma unroll
  for (int e = 0; e < E; ++e) {
    const bool eq = r.key[e] == c.key, drop = eq && rank >= c.ties;
    rank += eq;
    r.key[e] = drop ? 0 : r.key[e];
    r.w[e] = drop ? 0 : r.w[e];
  }
}

// ---- histogram of a row in registers ----------------------------------------------------------------------------------------------------------
// Bins count from the top.  Where the row spans few enough keys a bin is a key; otherwise it is a slice of the value range.
template <int NT>
struct HistLds { uint32_t c[4 * NT]; uint64_t m[4 * NT]; uint32_t bin[2], above[2], in[2]; uint64_t mass[2]; };
struct Where { uint32_t bin, above, in; uint64_t mass; };   // the bin of a cut, its entries, and what lies above it

template <typename K, int NT>
struct Hist {
  static constexpr int N = 4 * NT;
  HistLds<NT>* h;
  uint32_t key_min, key_max, c[4], cb, all_c;   // this thread's four bins and what lies above them
  uint64_t m[4], mb, all_m;
  float top, inv;
  bool exact, usable;
  int turn = 0;
  __device__ __forceinline__ Hist(HistLds<NT>* lds, uint32_t lo, uint32_t hi) : h(lds), key_min(lo), key_max(hi) {
    exact = hi - lo < N;
    top = K::value(hi);
    const float span = top - K::value(lo);
    inv = (float)N / span;
    usable = exact || (span > 0.f && span < INFINITY && inv < INFINITY);
  }
  __device__ __forceinline__ uint32_t bin(uint32_t key) const { return exact ? key_max - key : min((uint32_t)((top - K::value(key)) * inv), (uint32_t)N - 1); }
  template <int E, bool BINS>
  __device__ __forceinline__ uint32_t bin_of(const RegRow<E, BINS>& r, int e) const { return BINS ? r.bin[e] : bin(r.key[e]); }
  // TABLE, and a bin is a key: the weights are not there yet.  Each is computed once per key, not once per entry, and a bin's mass is count * weight --
  // the bf16 list of a long row holds 12 000 entries of some 250 keys (64 rows of 128 256, top_p 0.9: 48.5 -> 43.3 us; whole rows seldom span few
  // enough keys, there the second way only makes the code longer: 12.2 -> 12.7)
  template <bool MASS, bool TABLE, int E, bool BINS>
  __device__ __forceinline__ void build(RegRow<E, BINS>& r, Block<NT>& blk, const Weigh& weigh) {
    const bool table = TABLE && exact;
    const int tid = threadIdx.x;
#pragma unroll
    for (int i = 0; i < 4; ++i) { h->c[i * NT + tid] = 0; if (MASS && !table) h->m[i * NT + tid] = 0; }
    __syncthreads();
#pragma unroll
    for (int e = 0; e < E; ++e) {
      if (E > 4 && e % 4 == 0 && e >= r.per) break;
      if (r.key[e]) {
        const uint32_t b = bin(r.key[e]);
        if (BINS) r.bin[e] = b;
        atomicAdd(&h->c[b], 1u);
        if (MASS && !table) atomicAdd(reinterpret_cast<unsigned long long*>(&h->m[b]), (unsigned long long)r.w[e]);
      }
    }
    __syncthreads();
    cb = 0; mb = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      c[i] = h->c[4 * tid + i];
      m[i] = MASS && !table ? h->m[4 * tid + i] : 0;
      if (table && c[i]) {
        const uint64_t each = weigh(K::value(key_max - (4 * tid + i)));
        h->m[4 * tid + i] = each;
        m[i] = c[i] * each;
      }
      cb += c[i];
      mb += m[i];
    }
    if (MASS) blk.before2(cb, mb, all_c, all_m);   // (its barrier is between the weights and their use)
    else cb = blk.before(cb, all_c);
    if (table) {
#pragma unroll
      for (int e = 0; e < E; ++e) r.w[e] = r.key[e] ? h->m[key_max - r.key[e]] : 0;
    }
  }
  // the bin in which the running count (or mass) from the top first reaches its target, which the row does reach
  template <bool MASS>
  __device__ __forceinline__ Where locate(uint32_t want_n, double want_m) {
    uint32_t run = cb;
    uint64_t mass = mb;
    const int t = turn;
    turn ^= 1;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const bool here = MASS ? (double)mass < want_m && (double)(mass + m[i]) >= want_m : run < want_n && run + c[i] >= want_n;
      if (here) { h->bin[t] = 4 * threadIdx.x + i; h->above[t] = run; h->in[t] = c[i]; h->mass[t] = mass; }
      run += c[i];
      mass += m[i];
    }
    __syncthreads();
    return {h->bin[t], h->above[t], h->in[t], h->mass[t]};
  }
  // the exact cut in that bin; false: more than 64 entries of several keys crowd there
  template <bool MASS, int E, bool BINS>
  __device__ __forceinline__ bool resolve(const RegRow<E, BINS>& r, const Where& w, Few* few, const Weigh& weigh, uint32_t want_n, double want_m, Cut& cut, uint64_t& kept) {
    if (exact) {
      cut.key = key_max - w.bin;
      cut.same = w.in;
      const uint64_t each = weigh(K::value(cut.key));
      const double q = each ? ceil((want_m - (double)w.mass) / (double)each) : 1.0;
      cut.ties = MASS ? q < 1.0 ? 1u : q > (double)w.in ? w.in : (uint32_t)q : want_n - w.above;
      kept = w.mass + cut.ties * each;
      return true;
    }
    if (w.in > 64) return false;
    if (threadIdx.x == 0) few->n = 0;
    __syncthreads();
#pragma unroll
    for (int e = 0; e < E; ++e) {
      if (E > 4 && e % 4 == 0 && e >= r.per) break;
      if (r.key[e] && bin_of(r, e) == w.bin) {
        const int at = atomicAdd(&few->n, 1);
        if (at < 64) few->key[at] = r.key[e];
      }
    }
    __syncthreads();
    rank_few<K, MASS>(few, weigh, w.above, w.mass, want_n, want_m, cut, kept);
    return true;
  }
};

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
__device__ __forceinline__ double target(float top_p, double base) { return fmax((double)top_p * base, 1.0); }   // at least one entry

// All filters and the draw on at most 64 entries in index order, by one wave: lane i holds entry i (key 0: none), the first `k` of the order
// count.  The entries are sorted with their places, cut, and their weights sent back to their places for the draw; the result is a place.
template <typename K>
__device__ __forceinline__ int draw_few(uint32_t key, uint32_t k, const Weigh& weigh, const Setting& s) {
  const int lane = threadIdx.x & 63;
  uint64_t c = (uint64_t)key << 32 | (uint32_t)(63 - lane);
  wave_sort(c);
  const uint32_t sorted = (uint32_t)(c >> 32);
  const uint64_t w = sorted && (uint32_t)lane < k ? weigh(K::value(sorted)) : 0, upto = wave_upto(w);
  const double reach = target(s.top_p, (double)lane_value(upto, 63));
  const bool keep = w && (s.top_p >= 1.f || (double)(upto - w) < reach) && (double)w >= (double)s.min_p * (double)(1ull << weigh.shift);
  const int place = 63 - (int)(uint32_t)c;
  const uint64_t v = keep ? w : 0;
  const uint64_t back = (uint64_t)(uint32_t)__builtin_amdgcn_ds_permute(place * 4, (int)(uint32_t)v) | (uint64_t)(uint32_t)__builtin_amdgcn_ds_permute(place * 4, (int)(v >> 32)) << 32;
  const uint64_t cum = wave_upto(back);
  const double want = (double)s.u * (double)lane_value(cum, 63);
  return __ffsll((unsigned long long)__ballot(back && (double)cum > want)) - 1;
}

// The short way for a small top-k: the top bins that hold k entries and no more than 64 go in index order to one wave.  -2: too many crowd in the last
// of these bins.  Otherwise the place (e, in the thread that owns it) or -1.  Needs keys only.
struct FewOrder { uint32_t key[64]; int hit; };
template <typename K, int E, bool BINS, int NT>
__device__ __forceinline__ int draw_small(RegRow<E, BINS>& r, Block<NT>& blk, HistLds<NT>* lds, FewOrder* few, const Weigh& weigh, const Setting& s, uint32_t n, uint32_t k, uint32_t key_min, uint32_t key_max) {
  uint32_t cnt = n, last = ~0u;   // the listed bins end with `last`
  Hist<K, NT> hist(lds, key_min, key_max);
  if (n > 64) {
    if (!hist.usable) return -2;
    hist.template build<false, false>(r, blk, Weigh{});
    const Where w = hist.template locate<false>(k, 0.0);
    cnt = w.above + w.in;
    last = w.bin;
    if (cnt > 64) return -2;
  }
  uint32_t in = 0, total;   // which of this thread's entries are listed
#pragma unroll
  for (int e = 0; e < E; ++e) {
    if (E > 4 && e % 4 == 0 && e >= r.per) break;
    if (r.key[e] && (last == ~0u || hist.bin_of(r, e) <= last)) in |= 1u << e;
  }
  const uint32_t mine = __popc(in), first = blk.before(mine, total);
  if (mine) {
    uint32_t p = first;
#pragma unroll
    for (int e = 0; e < E; ++e)
      if ((in >> e) & 1) few->key[p++] = r.key[e];
  }
  __syncthreads();
  if (threadIdx.x < 64) {
    const int lane = threadIdx.x;
    const int hit = draw_few<K>(lane < (int)cnt ? few->key[lane] : 0u, k, weigh, s);
    if (lane == 0) few->hit = hit;
  }
  __syncthreads();
  uint32_t nth = (uint32_t)few->hit - first;
  if (nth >= mine) return -1;
  for (; nth; --nth) in &= in - 1;
  return __ffs(in) - 1;
}

// filters and draw on entries in registers, with their weights unless TABLE; returns the place (e, in the thread that owns it) or -1.  `base`: the mass that top_p refers to when
// it is not that of these entries (< 0: it is).  `enough` comes back false when these entries cannot hold the nucleus.
template <typename K, bool TABLE, int E, bool BINS, int NT>
__device__ __forceinline__ int filter_and_draw(RegRow<E, BINS>& r, Block<NT>& blk, HistLds<NT>* lds, Few* few, const Weigh& weigh, const Setting& s, uint32_t n, uint32_t key_min, uint32_t key_max, double base, bool& enough) {
  enough = true;
  Cut cut{key_min, 1u, 1u};
  const bool cut_k = s.k && (uint32_t)s.k < n;
  Hist<K, NT> hist(lds, key_min, key_max);
  bool binned = hist.usable && (cut_k || s.top_p < 1.f);
  uint64_t mass = 0;
  if (TABLE && !(binned && hist.exact)) r.template weigh_all<K>(weigh);
  if (binned) {
    hist.template build<true, TABLE>(r, blk, weigh);
    mass = hist.all_m;
  }
  if (cut_k) {
    if (binned) binned = hist.template resolve<false>(r, hist.template locate<false>((uint32_t)s.k, 0.0), few, weigh, (uint32_t)s.k, 0.0, cut, mass);
    if (!binned) cut = find_cut<K, false>(r, blk, few, weigh, key_min, n, 0, key_max + 1, (uint32_t)s.k, 0.0);
    drop_ties(r, blk, cut);
    n = (uint32_t)s.k;
  }
  if (s.top_p < 1.f) {
    if (!binned) {
      uint32_t cnt;
      mass = 0;
      r.template stat<true>(cut.key, cnt, mass);
      blk.template sum<true>(cnt, mass);
    }
    const double want = target(s.top_p, base < 0.0 ? (double)mass : base);
    if ((double)mass < want) { enough = false; return -1; }
    uint64_t kept;
    if (binned) binned = hist.template resolve<true>(r, hist.template locate<true>(0u, want), few, weigh, 0u, want, cut, kept);
    if (!binned) cut = find_cut<K, true>(r, blk, few, weigh, cut.key, n, mass, key_max + 1, 0u, want);
    drop_ties(r, blk, cut);
  }
  uint64_t mine = 0, total;
  const double least = (double)s.min_p * (double)(1ull << weigh.shift);
#pragma unroll
  for (int e = 0; e < E; ++e) {
    r.w[e] = r.key[e] < cut.key || (double)r.w[e] < least ? 0 : r.w[e];
    mine += r.w[e];
  }
  const uint64_t before = blk.before(mine, total);
  const double want = (double)s.u * (double)total;
  if ((double)before > want || !((double)(before + mine) > want)) return -1;
  uint64_t run = before + mine;
  int found = 0;
#pragma unroll
  for (int e = E - 1; e >= 0; --e) {   // the first place whose running sum is past the target
    found = (double)run > want && r.w[e] ? e : found;
    run -= r.w[e];
  }
  return found;
}

// maximum, minimum and count of the entries (values above -inf) of a block, in one exchange
struct Extremes { float mx, mn; uint32_t n; };
struct ExtremesLds { float mx[16], mn[16]; uint32_t n[16]; };
template <int NT, int E>
__device__ __forceinline__ Extremes extremes(const float (&v)[E], ExtremesLds* s) {
  float mx = -INFINITY, mn = INFINITY;
  uint32_t n = 0;
#pragma unroll
  for (int e = 0; e < E; ++e) {
    mx = fmaxf(mx, v[e]);
    mn = v[e] > -INFINITY ? fminf(mn, v[e]) : mn;
    n += __popcll(__ballot(v[e] > -INFINITY));
  }
  mx = wave_max(mx);
  mn = -wave_max(-mn);
  const int lane = threadIdx.x & 63;
  if (lane == 0) { s->mx[threadIdx.x >> 6] = mx; s->mn[threadIdx.x >> 6] = mn; s->n[threadIdx.x >> 6] = n; }
  __syncthreads();
  constexpr int W = NT / 64;
  mx = s->mx[lane % W]; mn = -s->mn[lane % W];
  n = over_waves<W>(s->n[lane % W]);
  auto all = [](float m) { m = fmaxf(m, dpp_all<0xB1>(m)); m = fmaxf(m, dpp_all<0x4E>(m)); m = fmaxf(m, dpp_all<0x141>(m)); return fmaxf(m, dpp_all<0x140>(m)); };
  auto uni = [](float m) { return __int_as_float(__builtin_amdgcn_readfirstlane(__float_as_int(m))); };
  return {uni(all(mx)), -uni(all(mn)), lane_value(n, 0)};
}

// rows of at most NT * E entries
template <int NT, int E, typename XT>
__global__ __launch_bounds__(NT) void sample_short_kernel(SampleOpArgs a) {
  using K = Keys<XT>;
  __shared__ Red red;
  __shared__ Few few;
  __shared__ FewOrder order;
  __shared__ ExtremesLds ext;
  __shared__ HistLds<NT> hist;
  __shared__ int best;
  const int row = blockIdx.x, tid = threadIdx.x;
  const XT* x = reinterpret_cast<const XT*>(a.logits) + row * a.stride;
  const Setting s = setting(a, row);
  Block<NT> blk{&red};
  RegRow<E, NT == 256> r;
  r.per = (a.V + NT - 1) / NT;
  const int first = tid * r.per, mine = min(r.per, a.V - first);   // (mine <= 0 behind the row's end)
  float v[E];
#pragma unroll
  for (int e = 0; e < E; ++e) v[e] = logit(x, min(first + e, a.V - 1));
#pragma unroll
  for (int e = 0; e < E; ++e) v[e] = e < mine ? v[e] : -INFINITY;
  const Extremes ex = extremes<NT>(v, &ext);
  const float mx = ex.mx;
  const uint32_t n = ex.n;
  if (mx == -INFINITY) {
    if (tid == 0) a.out[row] = -1;
    return;
  }
  if (s.k == 1) {   // the first entry of the order
    if (tid == 0) best = a.V;
    __syncthreads();
    int at = a.V;
#pragma unroll
    for (int e = E - 1; e >= 0; --e) at = v[e] == mx ? first + e : at;
    if (at < a.V) atomicMin(&best, at);
    __syncthreads();
    if (tid == 0) a.out[row] = best;
    return;
  }
  const Weigh weigh{mx, 1.4426950408889634074 / (double)s.T, a.shift};
  const uint32_t key_min = K::key(ex.mn), key_max = K::key(mx), k = s.k && (uint32_t)s.k < n ? (uint32_t)s.k : n;
#pragma unroll
  for (int e = 0; e < E; ++e) r.key[e] = v[e] > -INFINITY ? K::key(v[e]) : 0;
  int e = -2;
  if (k <= 64) e = draw_small<K>(r, blk, &hist, &order, weigh, s, n, k, key_min, key_max);
  if (e == -2) {
#pragma unroll
    for (int i = 0; i < E; ++i) {
      r.w[i] = 0;
      if (i < r.per) r.w[i] = weigh(v[i]);
    }
    bool enough;
    e = filter_and_draw<K, false>(r, blk, &hist, &few, weigh, s, n, key_min, key_max, -1.0, enough);
  }
  if (e >= 0) a.out[row] = first + e;
}

// ---- long rows ------------------------------------------------------------------------------------------------------------------------------
template <typename XT>
__device__ __forceinline__ void gather8(W8<XT>& r, const XT* x, int i, int V);   // x[i .. i + 7] one by one, -inf past the row's end
template <>
__device__ __forceinline__ void gather8<float>(W8<float>& r, const float* x, int i, int V) {
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const float v = i + e < V ? x[min(i + e, V - 1)] : -INFINITY;
    if (e < 4) r.a[e] = v; else r.b[e - 4] = v;
  }
}
template <>
__device__ __forceinline__ void gather8<bf16_t>(W8<bf16_t>& r, const bf16_t* x, int i, int V) {
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const uint32_t lo = i + 2 * e < V ? x[min(i + 2 * e, V - 1)] : 0xff80u, hi = i + 2 * e + 1 < V ? x[min(i + 2 * e + 1, V - 1)] : 0xff80u;
    r.r[e] = lo | (hi << 16);
  }
}
// The row as it lies in memory, for the search that streams.  A wave owns a run of consecutive entries (a multiple of 64 * VEC).
template <typename XT, bool ALIGNED>
struct LongRow {
  using K = Keys<XT>;
  static constexpr int VEC = 8;
  const XT* x;
  int V, seg;
  const Weigh* weigh;
  uint32_t floor_key;   // entries below are not counted
  template <typename F>
  __device__ __forceinline__ void each(int from, int to, F f) const {   // f(index, value, whether the index is in the run): every lane takes part
    const int lane = threadIdx.x & 63;
    for (int i0 = from; i0 < to; i0 += 64 * VEC) {
      const int i = i0 + lane * VEC;
      W8<XT> w;
      if (ALIGNED && i + VEC <= V) w.load(x + i);
      else gather8(w, x, i, V);
#pragma unroll 2
      for (int e = 0; e < VEC; ++e) { const float y = w.get(e) + 0.f; f(i + e, y != y ? -INFINITY : y, i + e < to); }
    }
  }
  __device__ __forceinline__ int begin() const { return min((int)(threadIdx.x >> 6) * seg, V); }
  __device__ __forceinline__ int end() const { return min((int)(threadIdx.x >> 6) * seg + seg, V); }
  template <bool MASS>
  __device__ __forceinline__ void stat(uint32_t c, uint32_t& cnt, uint64_t& mass) const {
    uint32_t n = 0;
    uint64_t m = 0;
    each(begin(), end(), [&](int, float v, bool) {
      const uint32_t key = K::key(v);
      const bool in = key >= c && key >= floor_key;
      n += __popcll(__ballot(in));
      if (MASS) { const uint64_t w = (*weigh)(v); m += in ? w : 0; }
    });
    cnt = n;
    mass = m;
  }
  __device__ __forceinline__ void gather(uint32_t lo, uint32_t hi, Few* few) const {
    each(begin(), end(), [&](int, float v, bool) {
      const uint32_t key = K::key(v);
      if (key >= lo && key < hi && key >= floor_key) {
        const int at = atomicAdd(&few->n, 1);
        if (at < 64) few->key[at] = key;
      }
    });
  }
};

// ---- launch 1 of a long row: the list's threshold, from samples spread over the row.  ~0 = no list
template <typename XT>
__global__ __launch_bounds__(256) void sample_threshold_kernel(SampleOpArgs a) {
  using K = Keys<XT>;
  constexpr int NT = 256;
  __shared__ Red red;
  __shared__ Few few;
  __shared__ ExtremesLds ext;
  __shared__ HistLds<NT> lds;
  const int row = blockIdx.x, tid = threadIdx.x;
  const XT* x = reinterpret_cast<const XT*>(a.logits) + row * a.stride;
  const Setting s = setting(a, row);
  uint32_t thr = ~0u;
  if (s.k != 1 && (s.k || s.top_p < 1.f || s.min_p > 0.f)) {
    constexpr int E = SAMPLES / NT;
    Block<NT> blk{&red};
    RegRow<E> r;
    r.per = E;
    float v[E];
#pragma unroll
    for (int e = 0; e < E; ++e) v[e] = logit(x, (int)((int64_t)(e * NT + tid) * a.V / SAMPLES));
#pragma unroll
    for (int e = 0; e < E; ++e) r.key[e] = v[e] > -INFINITY ? K::key(v[e]) : 0;
    const Extremes ex = extremes<NT>(v, &ext);
    const uint32_t n = ex.n;
    const int aim = s.k && s.k < AIM / 4 - 512 ? 4 * s.k + 2048 : AIM;   // a short top-k needs a short list
    const uint32_t rank = max(1u, (uint32_t)((int64_t)aim * SAMPLES / a.V));
    thr = K::NONE + 1;
    if (n > rank) {   // (the lower end of the bin is near enough, unless too many crowd there)
      Hist<K, NT> hist(&lds, K::key(ex.mn), K::key(ex.mx));
      Where w{0, 0, ~0u, 0};
      if (hist.usable) {
        hist.template build<false, false>(r, blk, Weigh{});
        w = hist.template locate<false>(rank, 0.0);
      }
      if (hist.exact) thr = hist.key_max - w.bin;
      else if (w.in <= 64) thr = K::key(hist.top - (float)(w.bin + 1) / hist.inv + 0.f);
      else thr = find_cut<K, false>(r, blk, &few, Weigh{}, K::key(ex.mn), n, 0, K::key(ex.mx) + 1, rank, 0.0).key;
    }
  }
  if (tid == 0) a.thr[row] = thr;
}

// ---- launch 2: a workgroup per chunk.  A thread owns 32 consecutive entries.
template <typename XT, bool ALIGNED>
__global__ __launch_bounds__(256) void sample_chunk_kernel(SampleOpArgs a) {
  using K = Keys<XT>;
  constexpr int PER = CHUNK / 256;
  __shared__ float mx_s[4];
  __shared__ double mass_s[4];
  __shared__ uint32_t cnt_s[4];
  __shared__ int at_s;
  __shared__ double roots_s[32];
  const int row = blockIdx.x / a.chunks, chunk = blockIdx.x - row * a.chunks, tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const XT* x = reinterpret_cast<const XT*>(a.logits) + row * a.stride;
  const Setting s = setting(a, row);
  const int i0 = chunk * CHUNK + tid * PER;
  W8<XT> raw[PER / 8];
  if (ALIGNED && i0 + PER <= a.V) {
#pragma unroll
    for (int j = 0; j < PER / 8; ++j) raw[j].load(x + i0 + 8 * j);
  } else {
#pragma unroll
    for (int j = 0; j < PER / 8; ++j) gather8(raw[j], x, i0 + 8 * j, a.V);
  }
  float v[PER];
#pragma unroll
  for (int e = 0; e < PER; ++e) {
    const float y = raw[e / 8].get(e % 8) + 0.f;
    v[e] = y != y ? -INFINITY : y;
  }
  if (tid == 0) at_s = a.V;
  if (tid < 32) roots_s[tid] = roots[tid];
  float mx = -INFINITY;
#pragma unroll
  for (int e = 0; e < PER; ++e) mx = fmaxf(mx, v[e]);
  const float my_mx = mx;
  mx = wave_max(mx);
  if (lane == 0) mx_s[wave] = mx;
  __syncthreads();
  mx = fmaxf(fmaxf(mx_s[0], mx_s[1]), fmaxf(mx_s[2], mx_s[3]));
  if (my_mx == mx) {
    int at = a.V;
#pragma unroll
    for (int e = PER - 1; e >= 0; --e) at = v[e] == mx ? i0 + e : at;
    atomicMin(&at_s, at);
  }
  const float thr = K::value(a.thr[row]);   // (~0 is a NaN: nothing is listed)
  uint32_t mine = 0;
#pragma unroll
  for (int e = 0; e < PER; ++e) mine += v[e] >= thr;
  const uint32_t upto = wave_upto(mine);
  // the chunk's mass where it counts: no top-k, and a nucleus or nothing at all to cut
  double mass = 0.0;
  if (!s.k && (s.top_p < 1.f || s.min_p == 0.f) && mx > -INFINITY) {
    const WeighMany weigh{mx, 1.4426950408889634074 / (double)s.T, 51, roots_s};
    uint64_t m = 0;
#pragma unroll
    for (int e = 0; e < PER; ++e) m += weigh(v[e]);
    m = wave_total(m);      // 64 * 32 weights of at most 2^51
    mass = (double)m * 0x1p-51;
  }
  if (lane == 63) { cnt_s[wave] = upto; mass_s[wave] = mass; }
  __syncthreads();
  uint32_t before = 0;
  for (int w = 0; w < wave; ++w) before += cnt_s[w];
  if (tid == 0) {
    ChunkHead h;
    h.mass = (mass_s[0] + mass_s[1]) + (mass_s[2] + mass_s[3]);
    h.mx = mx; h.at = at_s; h.count = cnt_s[0] + cnt_s[1] + cnt_s[2] + cnt_s[3]; h.pad = 0;
    a.heads[(int64_t)row * a.chunks + chunk] = h;
  }
  if (mine) {
    uint32_t p = before + upto - mine;
    uint2* list = a.lists + ((int64_t)row * a.chunks + chunk) * CHUNK;
#pragma unroll
    for (int e = 0; e < PER; ++e)
      if (v[e] >= thr) list[p++] = make_uint2(K::key(v[e]), (uint32_t)(i0 + e));
  }
}

// ---- launch 3: a workgroup per row
template <typename XT, bool ALIGNED>
__global__ __launch_bounds__(1024) void sample_list_kernel(SampleOpArgs a) {
  using K = Keys<XT>;
  constexpr int NT = 1024;
  extern __shared__ __attribute__((aligned(16))) uint32_t keys[];   // [LIST]
  __shared__ Red red;
  __shared__ Few few;
  __shared__ FewOrder order;
  __shared__ ExtremesLds ext;
  __shared__ HistLds<NT> hist;
  __shared__ int best;
  __shared__ uint32_t start_s[MAX_CHUNKS], tie_s[16];
  __shared__ uint64_t mass_s[16];
  __shared__ double cum_s[MAX_CHUNKS];
  constexpr int E = LIST / NT;
  const int row = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const Setting s = setting(a, row);
  const uint32_t thr = a.thr[row];
  Block<NT> blk{&red};
  const ChunkHead* heads = a.heads + (int64_t)row * a.chunks;
  ChunkHead h{0.0, -INFINITY, a.V, 0u, 0u};
  if (tid < a.chunks) h = heads[tid];
  if (tid == 0) best = a.V;
  const float hm[1] = {h.mx};
  const float mx = extremes<NT>(hm, &ext).mx;
  if (mx == -INFINITY) {
    if (tid == 0) a.out[row] = -1;
    return;
  }
  if (s.k == 1) {
    if (tid < a.chunks && h.mx == mx) atomicMin(&best, h.at);
    __syncthreads();
    if (tid == 0) a.out[row] = best;
    return;
  }
  const double k2 = 1.4426950408889634074 / (double)s.T;
  Weigh weigh{mx, k2, LIST_SHIFT};
  // masses of the chunks in one scale, summed by one wave in a fixed order: the same bits every time
  if (tid < a.chunks) cum_s[tid] = h.mx == mx ? h.mass : h.mx == -INFINITY || mx == INFINITY ? 0.0 : h.mass * exp2(fmax(((double)h.mx - (double)mx) * k2, -1200.0));
  uint64_t n_list;
  const uint64_t start = blk.before((uint64_t)(tid < a.chunks ? h.count : 0), n_list);
  if (tid < a.chunks) start_s[tid] = (uint32_t)start;
  __syncthreads();
  if (tid < 64) {   // 4 consecutive chunks a lane
    double c[4], run = 0.0;
#pragma unroll
    for (int i = 0; i < 4; ++i) c[i] = run += 4 * lane + i < a.chunks ? cum_s[4 * lane + i] : 0.0;
    const double before = wave_upto(run) - run;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (4 * lane + i < a.chunks) cum_s[4 * lane + i] = before + c[i];
  }
  __syncthreads();
  double all = cum_s[a.chunks - 1];
  const uint32_t key_max = K::key(mx);

  LongRow<XT, ALIGNED> src;
  constexpr int VEC = LongRow<XT, ALIGNED>::VEC;
  src.x = reinterpret_cast<const XT*>(a.logits) + row * a.stride;
  src.V = a.V;
  src.seg = (a.V + NT * VEC - 1) / (NT * VEC) * (64 * VEC);
  src.weigh = &weigh;
  src.floor_key = K::NONE + 1;

  if (!s.k && s.top_p >= 1.f && s.min_p == 0.f) {   // nothing is cut: the chunk that holds u * total, then its entries
    const double want = (double)s.u * all;
    int c = 0;
    while (c < a.chunks - 1 && !(cum_s[c] > want)) ++c;
    const double rest = (want - (c ? cum_s[c - 1] : 0.0)) * (double)(1ull << LIST_SHIFT);
    constexpr int PER = CHUNK / NT;
    const int i0 = c * CHUNK + tid * PER;
    uint64_t w[PER], mine = 0, total;
#pragma unroll
    for (int e = 0; e < PER; ++e) {
      w[e] = i0 + e < a.V ? weigh(logit(src.x, min(i0 + e, a.V - 1))) : 0;
      mine += w[e];
    }
    const uint64_t before = blk.before(mine, total);
    uint64_t run = before;
    int at = a.V, last = -1;
#pragma unroll
    for (int e = 0; e < PER; ++e) {
      run += w[e];
      if (w[e] && (double)run > rest && at == a.V) at = i0 + e;
      if (w[e]) last = i0 + e;
    }
    if (at < a.V) atomicMin(&best, at);
    __syncthreads();
    const bool none = best == a.V;      // (rounding left the target past the chunk's last entry)
    __syncthreads();
    if (none) {
      if (tid == 0) best = -1;
      __syncthreads();
      atomicMax(&best, last >= 0 ? last : -1);
      __syncthreads();
      if (tid == 0 && best < 0) best = heads[c].at;
      __syncthreads();
    }
    if (tid == 0) a.out[row] = best;
    return;
  }

  bool ok = n_list > 0 && n_list <= LIST;
  if (ok && s.k) ok = n_list >= (uint64_t)s.k || thr <= K::NONE + 1;
  if (ok && !s.k && s.top_p >= 1.f) ok = thr <= K::NONE + 1 || (double)weigh(K::value(thr)) < (double)s.min_p * (double)(1ull << LIST_SHIFT);   // min-p alone: all it keeps is listed
  if (ok) {
    const uint2* lists = a.lists + (int64_t)row * a.chunks * CHUNK;
    for (int c = wave; c < a.chunks; c += 16) {
      const uint32_t at = start_s[c], cnt = (c + 1 < a.chunks ? start_s[c + 1] : (uint32_t)n_list) - at;
#pragma unroll 8
      for (uint32_t i = lane; i < cnt; i += 64) keys[at + i] = lists[(int64_t)c * CHUNK + i].x;
    }
    __syncthreads();
    RegRow<E> r;
    const uint32_t n = (uint32_t)n_list;
    r.per = (int)((n + NT - 1) / NT);
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const uint32_t p = tid * r.per + e;
      r.key[e] = e < r.per && p < n ? keys[min(p, (uint32_t)LIST - 1)] : 0;
    }
    bool enough = true;
    int e = -2;
    if (s.k && s.k <= 64) e = draw_small<K>(r, blk, &hist, &order, weigh, s, n, min((uint32_t)s.k, n), thr, key_max);
    if (e == -2) {
      constexpr bool TABLE = sizeof(XT) == 2;
      if (!TABLE) r.template weigh_all<K>(weigh);
      e = filter_and_draw<K, TABLE>(r, blk, &hist, &few, weigh, s, n, thr, key_max, s.k ? -1.0 : all * (double)(1ull << LIST_SHIFT), enough);
    }
    if (e >= 0) {
      const uint32_t p = tid * r.per + e;
      int c = 0;
      while (c + 1 < a.chunks && start_s[c + 1] <= p) ++c;
      a.out[row] = (int)lists[(int64_t)c * CHUNK + (p - start_s[c])].y;
    }
    if (enough) return;
  }

  // the list does not hold the answer: the same search over the row itself
  Cut cut{0u, 0u, 0u};
  {
    uint32_t n;
    uint64_t sum = 0;
    if (!s.k && s.top_p < 1.f) {
      src.template stat<false>(K::NONE + 1, n, sum);
      n = blk.count(n);
    } else {   // the chunks' masses are not there: the total in the coarsest scale (2^21 weights within 2^-21 of it) finds the finest that holds it
      weigh.shift = a.shift;
      src.template stat<true>(K::NONE + 1, n, sum);
      blk.template sum<true>(n, sum);
      all = ldexp((double)sum, -a.shift);
    }
    weigh.shift = min(61 - ilogb(all), 51);
    if (s.k && (uint32_t)s.k < n) cut = find_cut<K, false>(src, blk, &few, weigh, K::NONE + 1, n, 0, key_max + 1, (uint32_t)s.k, 0.0);
  }
  if (s.top_p < 1.f) {
    uint32_t cnt;
    uint64_t above = 0;
    src.template stat<true>(cut.key + 1, cnt, above);
    blk.template sum<true>(cnt, above);
    const uint64_t each = cut.ties ? weigh(K::value(cut.key)) : 0;
    const double want = target(s.top_p, (double)(above + each * cut.ties));
    if ((double)above >= want) {
      src.floor_key = max(src.floor_key, cut.key + 1);
      cut = find_cut<K, true>(src, blk, &few, weigh, src.floor_key, cnt, above, key_max + 1, 0u, want);
      src.floor_key = K::NONE + 1;
    } else {
      const double q = each ? ceil((want - (double)above) / (double)each) : 1.0;
      if (q < (double)cut.ties) cut.ties = q < 1.0 ? 1u : (uint32_t)q;
    }
  }
  // draw by streaming: mass and ties of every wave's run, then the one run that holds the target
  const double least = (double)s.min_p * (double)(1ull << weigh.shift);
  auto value = [&](float v) { const uint64_t w = weigh(v); return (double)w < least ? 0ull : w; };
  uint64_t mass = 0;
  uint32_t ties = 0;
  src.each(src.begin(), src.end(), [&](int, float v, bool) {
    const uint32_t key = K::key(v);
    const uint64_t w = value(v);
    mass += key > cut.key && key > K::NONE ? w : 0;
    ties += key == cut.key;
  });
  mass = wave_total(mass);
  ties = wave_total(ties);
  const uint64_t each = cut.ties ? value(K::value(cut.key)) : 0;
  if (lane == 0) { mass_s[wave] = mass; tie_s[wave] = ties; }
  __syncthreads();
  uint64_t total = 0, run_before = 0;
  uint32_t tie_before = 0;
  for (int w = 0; w < 16; ++w) {
    const uint32_t t = min(tie_s[w], cut.ties - min(cut.ties, tie_before));
    total += mass_s[w] + t * each;
    tie_before += tie_s[w];
  }
  const double want = (double)s.u * (double)total;
  int at = 0;
  tie_before = 0;
  for (int w = 0; w < 16; ++w) {
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
  for (int i = i0; i < i1; ++i) my_ties += K::key(logit(src.x, i)) == cut.key;
  const uint64_t seen0 = tie_before + blk.before(my_ties, unused);
  uint64_t seen = seen0, mine = 0;
  auto kept = [&](int i) -> uint64_t {
    const float v = logit(src.x, i);
    const uint32_t key = K::key(v);
    if (key <= K::NONE || key < cut.key || (key == cut.key && seen++ >= cut.ties)) return 0;
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

static int check(const csm_ops_sample_t* p) {
  if (!p) return ops_fail(CSM_OPS_ERR_ARG, "null argument");
  if (p->x_dtype != CSM_OPS_F32 && p->x_dtype != CSM_OPS_BF16) return ops_fail(CSM_OPS_ERR_ARG, "unknown dtype %d", p->x_dtype);
  if (p->rows < 0 || p->V < 1) return ops_fail(CSM_OPS_ERR_ARG, "rows must not be negative and V must be positive");
  if (p->V > MAX_V) return ops_fail(CSM_OPS_ERR_CAPACITY, "V = %d: at most 2^21", p->V);
  const bool lists = p->V > LIST;
  if (!ops_launchable(p->rows, p->V > SHORT ? 1024 : 256) || (lists && !ops_launchable((int64_t)p->rows * ((p->V + CHUNK - 1) / CHUNK), 256))) return ops_fail(CSM_OPS_ERR_CAPACITY, "too many rows for one launch");
  if (!p->temperatures && !(p->temperature >= 0.f && p->temperature < INFINITY)) return ops_fail(CSM_OPS_ERR_ARG, "temperature must be finite and not negative");
  if (!p->topks && (p->topk < 0 || p->topk > p->V)) return ops_fail(CSM_OPS_ERR_ARG, "selected index k out of range");
  if (!p->top_ps && !(p->top_p > 0.f && p->top_p <= 1.f)) return ops_fail(CSM_OPS_ERR_ARG, "top_p must lie in (0, 1]");
  if (!p->min_ps && !(p->min_p >= 0.f && p->min_p <= 1.f)) return ops_fail(CSM_OPS_ERR_ARG, "min_p must lie in [0, 1]");
  return 0;
}
static size_t workspace(const csm_ops_sample_t* p, SampleOpArgs& a) {   // heads | lists | thresholds
  a.chunks = (p->V + CHUNK - 1) / CHUNK;
  if (p->V <= LIST) return 0;
  const size_t n = (size_t)p->rows * a.chunks;
  char* base = reinterpret_cast<char*>(p->workspace);
  a.heads = reinterpret_cast<ChunkHead*>(base);
  a.lists = reinterpret_cast<uint2*>(base + n * sizeof(ChunkHead));
  a.thr = reinterpret_cast<uint32_t*>(base + n * (sizeof(ChunkHead) + CHUNK * sizeof(uint2)));
  return n * (sizeof(ChunkHead) + CHUNK * sizeof(uint2)) + (size_t)p->rows * 4;
}

extern "C" int csm_ops_sample_workspace(const csm_ops_sample_t* p, size_t* bytes) {
  if (!bytes) return ops_fail(CSM_OPS_ERR_ARG, "null argument");
  if (const int r = check(p)) return r;
  SampleOpArgs a;
  *bytes = workspace(p, a);
  return 0;
}

template <typename XT, bool ALIGNED>
static int launch_long(const SampleOpArgs& a, int rows, hipStream_t st) {
  // the keys of a list (64 KB) and what stands beside them (52 KB, most of it the histogram): 116 KB of the CU's 160
  OPS_HIP(hipFuncSetAttribute(reinterpret_cast<const void*>(sample_list_kernel<XT, ALIGNED>), hipFuncAttributeMaxDynamicSharedMemorySize, LIST * sizeof(uint32_t)));
  hipLaunchKernelGGL((sample_threshold_kernel<XT>), dim3(rows), dim3(256), 0, st, a);
  hipLaunchKernelGGL((sample_chunk_kernel<XT, ALIGNED>), dim3((unsigned)rows * a.chunks), dim3(256), 0, st, a);
  hipLaunchKernelGGL((sample_list_kernel<XT, ALIGNED>), dim3(rows), dim3(1024), LIST * sizeof(uint32_t), st, a);
  OPS_HIP(hipGetLastError());
  return 0;
}

extern "C" int csm_ops_sample_filtered(const csm_ops_sample_t* p, void* stream) {
  if (const int r = check(p)) return r;
  if (!p->rows) return 0;
  if (!p->logits || !p->uniform || !p->out) return ops_fail(CSM_OPS_ERR_ARG, "null pointer");
  SampleOpArgs a;
  const size_t need = workspace(p, a);
  if (need && (!p->workspace || p->workspace_bytes < need || !ops_aligned(p->workspace)))
    return ops_fail(CSM_OPS_ERR_CAPACITY, "workspace of %zu bytes: %zu on 16 bytes are needed", p->workspace_bytes, need);
  a.logits = p->logits; a.stride = p->logits_stride; a.V = p->V; a.uniform = p->uniform; a.temperatures = p->temperatures;
  a.top_ps = p->top_ps; a.min_ps = p->min_ps; a.topks = p->topks; a.temperature = p->temperature; a.top_p = p->top_p; a.min_p = p->min_p;
  a.topk = p->topk; a.out = p->out;
  int bits = 0;
  while ((1 << bits) < p->V) ++bits;
  a.shift = 62 - bits < 51 ? 62 - bits : 51;   // V weights of at most 1 stay below 2^62
  hipStream_t st = (hipStream_t)stream;
  const bool b = p->x_dtype == CSM_OPS_BF16;
  const dim3 grid(p->rows);
  // as few waves as hold the row at 4 or 16 entries a thread: every wave repeats the scalar part of every step, and four waves on a SIMD take turns at it.
  // Rows of 2051 under top_p on 4 waves and on 16 (us): one 9.4 / 12.8, 512 of them 11.8 / 24.9; 512 of 1000 with 4 and with 16 entries 8.0 / 10.5
  if (p->V <= 256 * 4) {
    if (b) hipLaunchKernelGGL((sample_short_kernel<256, 4, bf16_t>), grid, dim3(256), 0, st, a);
    else hipLaunchKernelGGL((sample_short_kernel<256, 4, float>), grid, dim3(256), 0, st, a);
  } else if (p->V <= SHORT) {
    if (b) hipLaunchKernelGGL((sample_short_kernel<256, 16, bf16_t>), grid, dim3(256), 0, st, a);
    else hipLaunchKernelGGL((sample_short_kernel<256, 16, float>), grid, dim3(256), 0, st, a);
  } else if (p->V <= LIST) {
    if (b) hipLaunchKernelGGL((sample_short_kernel<1024, 16, bf16_t>), grid, dim3(1024), 0, st, a);
    else hipLaunchKernelGGL((sample_short_kernel<1024, 16, float>), grid, dim3(1024), 0, st, a);
  } else {
    const bool al = ops_aligned(p->logits) && (p->rows == 1 || ops_stride16(p->logits_stride, p->x_dtype));
    return b ? (al ? launch_long<bf16_t, true>(a, p->rows, st) : launch_long<bf16_t, false>(a, p->rows, st))
             : (al ? launch_long<float, true>(a, p->rows, st) : launch_long<float, false>(a, p->rows, st));
  }
  OPS_HIP(hipGetLastError());
  return 0;
}
