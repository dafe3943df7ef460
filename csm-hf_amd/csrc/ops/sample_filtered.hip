// Sampling with temperature, top-k, top-p and min-p from one given uniform per row (include/csm_ops.h).
//   w_i = exp((x_i - max) / T);  rows ordered by (x descending, index ascending);  every filter keeps a PREFIX of that order, so the kept set
//   is "key > cut, and the first `ties` entries with key == cut";  the token is where the running sum of kept w (index order) passes u * total.
// Sums are uint64 fixed point (w scaled by 2^(62 - ceil log2 V)) of weights computed in fp64: exact integer additions, so neither the split over
// threads nor any order of arrival changes a result, and what is rounded away per weight is below 2^-45 of the largest.
// First form: one workgroup per row; each cut by bisection of the 32-bit order key, one pass over the row per bit.
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
constexpr int ST = 256;

__device__ __forceinline__ uint32_t order_key(float x) {   // larger float = larger key; NaN was mapped to -inf, -0 to +0
  const uint32_t u = __float_as_uint(x);
  return u ^ ((u >> 31) ? 0xffffffffu : 0x80000000u);
}
template <typename T>
__device__ __forceinline__ float logit(const T* x, int i) {
  const float v = to_f32(x[i]) + 0.f;
  return v != v ? -INFINITY : v;
}
__device__ __forceinline__ double weight(float x, float mx, double T) {
  return x == -INFINITY ? 0.0 : x == mx ? 1.0 : exp(((double)x - (double)mx) / T);
}

__device__ __forceinline__ uint64_t block_sum(uint64_t v, uint64_t* s) {
  for (int d = 32; d; d >>= 1) v += __shfl_xor((unsigned long long)v, d);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = v;
  __syncthreads();
  return s[0] + s[1] + s[2] + s[3];
}
// sum over the threads before this one
__device__ __forceinline__ uint64_t block_before(uint64_t v, uint64_t* s, uint64_t& total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  uint64_t x = v;
  for (int d = 1; d < 64; d <<= 1) {
    const uint64_t y = __shfl_up((unsigned long long)x, d);
    if (lane >= d) x += y;
  }
  __syncthreads();
  if (lane == 63) s[wave] = x;
  __syncthreads();
  uint64_t before = 0;
  for (int i = 0; i < wave; ++i) before += s[i];
  total = s[0] + s[1] + s[2] + s[3];
  return before + x - v;
}

template <typename XT>
__global__ __launch_bounds__(ST) void sample_filtered_kernel(SampleOpArgs a) {
  __shared__ uint64_t red[4];
  __shared__ float mx_s[4];
  __shared__ int found;
  const int row = blockIdx.x, tid = threadIdx.x, V = a.V;
  const XT* x = reinterpret_cast<const XT*>(a.logits) + row * a.stride;
  float T = a.temperatures ? a.temperatures[row] : a.temperature;
  float top_p = a.top_ps ? a.top_ps[row] : a.top_p, min_p = a.min_ps ? a.min_ps[row] : a.min_p, u = a.uniform[row];
  int k = a.topks ? a.topks[row] : a.topk;
  if (!(T > 0.f)) k = 1;
  if (k <= 0 || k > V) k = V;
  if (!(top_p >= 0.f)) top_p = 0.f;
  if (!(min_p >= 0.f)) min_p = 0.f;
  if (min_p > 1.f) min_p = 1.f;
  if (!(u >= 0.f)) u = 0.f;
  if (u >= 1.f) u = 0.99999994f;
  const double Td = T > 0.f ? (double)T : 1.0, scale = (double)(1ull << a.shift);

  float mx = -INFINITY;
  for (int i = tid; i < V; i += ST) mx = fmaxf(mx, logit(x, i));
  mx = wave_max(mx);
  if ((tid & 63) == 0) mx_s[tid >> 6] = mx;
  __syncthreads();
  mx = fmaxf(fmaxf(mx_s[0], mx_s[1]), fmaxf(mx_s[2], mx_s[3]));
  if (mx == -INFINITY) {
    if (tid == 0) a.out[row] = -1;
    return;
  }
  auto fixed = [&](float v) { return (uint64_t)(weight(v, mx, Td) * scale + 0.5); };

  // top-k: the largest cut with at least k entries at or above it
  uint32_t cut = 0;
  uint64_t ties = (uint64_t)V;   // entries with key == cut that stay, in index order
  if (k < V) {
    for (int bit = 31; bit >= 0; --bit) {
      const uint32_t c = cut | (1u << bit);
      uint64_t n = 0;
      for (int i = tid; i < V; i += ST) n += order_key(logit(x, i)) >= c;
      if (block_sum(n, red) >= (uint64_t)k) cut = c;
    }
    uint64_t above = 0;
    for (int i = tid; i < V; i += ST) above += order_key(logit(x, i)) > cut;
    ties = (uint64_t)k - block_sum(above, red);
  }
  // top-p over what top-k kept: the largest cut at which the mass at or above it reaches top_p of the kept mass
  if (top_p < 1.f && T > 0.f) {
    uint64_t n = 0, tie_w = 0;
    for (int i = tid; i < V; i += ST) {
      const float v = logit(x, i);
      const uint32_t key = order_key(v);
      if (key > cut) n += fixed(v);
      else if (key == cut) tie_w = fixed(v);
    }
    uint64_t base = block_sum(n, red);
    uint64_t n_tie = 0;
    for (int i = tid; i < V; i += ST) n_tie += order_key(logit(x, i)) == cut;
    n_tie = block_sum(n_tie, red);
    if (n_tie < ties) ties = n_tie;
    // every tie has the same weight; a thread that met one knows it
    const uint64_t with = block_sum(tie_w ? 1 : 0, red), sum_w = block_sum(tie_w, red);
    const uint64_t each = with ? sum_w / with : 0;
    base += ties * each;
    const double want = (double)top_p * (double)base;
    uint32_t pc = 0;
    for (int bit = 31; bit >= 0; --bit) {
      const uint32_t c = pc | (1u << bit);
      uint64_t mass = 0;
      for (int i = tid; i < V; i += ST) {
        const float v = logit(x, i);
        const uint32_t key = order_key(v);
        if (key >= c && key > cut) mass += fixed(v);
      }
      mass = block_sum(mass, red);
      if (c <= cut) mass += ties * each;
      if ((double)mass >= want) pc = c;
    }
    if (pc > cut) {
      uint64_t above = 0, w = 0, cnt = 0;
      for (int i = tid; i < V; i += ST) {
        const float v = logit(x, i);
        const uint32_t key = order_key(v);
        if (key > pc) above += fixed(v);
        else if (key == pc) { w = fixed(v); ++cnt; }
      }
      above = block_sum(above, red);
      cnt = block_sum(cnt, red);
      const uint64_t met = block_sum(w ? 1 : 0, red), sw = block_sum(w, red), e = met ? sw / met : 0;
      uint64_t need = 1;
      if (e) { const double q = ceil((want - (double)above) / (double)e); need = q > 1.0 ? (uint64_t)q : 1; }
      cut = pc;
      ties = need < cnt ? need : cnt;
    } else if (each) {
      const double q = ceil((want - (double)(base - ties * each)) / (double)each);
      const uint64_t need = q > 1.0 ? (uint64_t)q : 1;
      if (need < ties) ties = need;
    }
  }
  // the draw: a thread owns a run of consecutive indices
  const int per = (V + ST - 1) / ST, lo = min(V, tid * per), hi = min(V, lo + per);
  uint64_t mine = 0, total = 0;
  for (int i = lo; i < hi; ++i) mine += order_key(logit(x, i)) == cut;
  const uint64_t ties_before = block_before(mine, red, total);
  auto kept = [&](int i, uint64_t& seen) -> uint64_t {
    const float v = logit(x, i);
    const uint32_t key = order_key(v);
    if (key < cut) return 0;
    if (key == cut && seen++ >= ties) return 0;
    const double w = weight(v, mx, Td);
    return w >= (double)min_p ? (T > 0.f ? (uint64_t)(w * scale + 0.5) : 1ull) : 0;
  };
  uint64_t seen = ties_before, mass = 0;
  for (int i = lo; i < hi; ++i) mass += kept(i, seen);
  const uint64_t before = block_before(mass, red, total);
  const double want = (double)u * (double)total;
  if (tid == 0) found = V;
  __syncthreads();
  if (mass && (double)(before + mass) > want) {
    uint64_t run = before;
    seen = ties_before;
    for (int i = lo; i < hi; ++i) {
      const uint64_t w = kept(i, seen);
      run += w;
      if (w && (double)run > want) { atomicMin(&found, i); break; }
    }
  }
  __syncthreads();
  if (tid == 0) a.out[row] = found;
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
  a.shift = 62 - bits < 52 ? 62 - bits : 52;   // V weights of at most 1 stay below 2^62; a double holds 2^52 and one half exactly
  hipStream_t st = (hipStream_t)stream;
  if (p->x_dtype == CSM_OPS_BF16) hipLaunchKernelGGL((sample_filtered_kernel<bf16_t>), dim3(p->rows), dim3(ST), 0, st, a);
  else hipLaunchKernelGGL((sample_filtered_kernel<float>), dim3(p->rows), dim3(ST), 0, st, a);
  OPS_HIP(hipGetLastError());
  return 0;
}
