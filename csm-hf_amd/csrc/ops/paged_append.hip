// Rotary embedding + append into a paged KV cache: raw q|k|v rows -> rotated q, rotated k and v in their cache slots, one launch.
//   y[i] = x[i] cos - x[i + d/2] sin,   y[i + d/2] = x[i + d/2] cos + x[i] sin,   angle of position pos_offset + slot
// Bound by memory: every input element is read once, every output written once, 1.5 flops per byte.  A thread owns 16 elements of one head:
// 8 of the lower half and the 8 they rotate with (q, k), or 16 consecutive ones (v), so that both partners are in its registers and all
// traffic is 16-byte vectors; consecutive threads take consecutive 8-element pieces of a row.
// Measured: 98.6 MB (4 sequences of some 2000 fp32 rows of 8 + 2 x 2 heads of 128) in 18.0 us, 5.5 TB/s, where a large copy reaches 4.9 with memory alone;
// 26.9 MB of bf16 rows (2162 of 32 + 2 x 8 heads of 64) in 6.6 us; 96 rows in 3.5 and one in 2.4, which are a launch and four dependent reads (length, page, row).
#include "ops_common.h"
#include <algorithm>

struct AppendArgs {
  Paged c;
  const void* qkv;
  void *k, *v, *q_out;
  const float *cos_t, *sin_t;
  int64_t qkv_stride, q_stride;
  int n_q, hd, units, total, rope_positions, pos_offset;   // units: 16-element pieces of a row; total = rows * units
};

constexpr int APPEND_THREADS = 256, CU_LDS = 1024;

template <typename T>
__device__ __forceinline__ void load8(const T* p, float (&x)[8]) {
  W8<T> w;
  w.load(p);
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] = w.get(i);
}
__device__ __forceinline__ void store8(float* p, const float (&x)[8]) {
  *reinterpret_cast<f32x4*>(p) = f32x4{x[0], x[1], x[2], x[3]};
  *reinterpret_cast<f32x4*>(p + 4) = f32x4{x[4], x[5], x[6], x[7]};
}
__device__ __forceinline__ void store8(bf16_t* p, const float (&x)[8]) {
  u32x4 w;
#pragma unroll
  for (int i = 0; i < 4; ++i) w[i] = (uint32_t)f32_to_bf16(x[2 * i]) | ((uint32_t)f32_to_bf16(x[2 * i + 1]) << 16);
  *reinterpret_cast<u32x4*>(p) = w;
}

template <typename XT, typename CT>
__global__ __launch_bounds__(APPEND_THREADS) void paged_append_kernel(AppendArgs a) {
  __shared__ int32_t cu_s[CU_LDS];
  const Paged& c = a.c;
  const int32_t* cu = c.cu;
  if (cu && c.n_seqs < CU_LDS) {   // the search is a chain of dependent reads: make them LDS reads
    for (int i = threadIdx.x; i <= c.n_seqs; i += APPEND_THREADS) cu_s[i] = cu[i];
    __syncthreads();
    cu = cu_s;
  }
  const int idx = blockIdx.x * APPEND_THREADS + threadIdx.x;
  if (idx >= a.total) return;
  const int row = idx / a.units, unit = idx - row * a.units;
  int seq = row, t = 0, n_new = 1;
  if (c.cu) {
    seq = ops_find_seq(cu, c.n_seqs, row);
    if (seq < 0) return;
    t = row - cu[seq];
    n_new = cu[seq + 1] - cu[seq];
  }
  const int len = c.lens[seq];
  const int64_t slot64 = (int64_t)len - n_new + t, pos = slot64 + a.pos_offset;
  if (len < 0 || slot64 < 0 || slot64 > 0x7fffffff || pos >= a.rope_positions) return;
  const int slot = (int)slot64;
  const int page = ops_page(c.table + seq * c.table_stride, c.width, c.n_pages, c.shift, slot);
  if (page < 0) return;
  const int per_head = a.hd >> 4, head = unit / per_head, piece = unit - head * per_head, half = a.hd >> 1;
  const int in_page = slot & ((1 << c.shift) - 1);
  const bool is_v = head >= a.n_q + c.n_kv;
  const int i0 = is_v ? 16 * piece : 8 * piece, i1 = is_v ? i0 + 8 : i0 + half;
  const XT* x = reinterpret_cast<const XT*>(a.qkv) + row * a.qkv_stride + (int64_t)head * a.hd;
  float lo[8], hi[8];
  load8(x + i0, lo);
  load8(x + i1, hi);
  if (!is_v) {
    float cs[8], sn[8];
    load8(a.cos_t + pos * half + i0, cs);
    load8(a.sin_t + pos * half + i0, sn);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float l = lo[i], h = hi[i];
      lo[i] = l * cs[i] - h * sn[i];
      hi[i] = h * cs[i] + l * sn[i];
    }
  }
  if (head < a.n_q) {
    XT* y = reinterpret_cast<XT*>(a.q_out) + row * a.q_stride + (int64_t)head * a.hd;
    store8(y + i0, lo);
    store8(y + i1, hi);
  } else {
    const int h = is_v ? head - a.n_q - c.n_kv : head - a.n_q;
    CT* y = is_v ? reinterpret_cast<CT*>(a.v) + page * c.vp + h * c.vh + in_page * c.vs : reinterpret_cast<CT*>(a.k) + page * c.kp + h * c.kh + in_page * c.ks;
    store8(y + i0, lo);
    store8(y + i1, hi);
  }
}

// Whether no two slots of the cache share memory, going by strides that nest: in ascending order each is at least what those below it span.  K and V of
// the same strides are taken as one more dimension, the distance between them, so that both may lie in one buffer in any order.
struct Dim { int64_t size, step; };
static bool nest(Dim* d, int n, int64_t span0) {
  std::sort(d, d + n, [](const Dim& a, const Dim& b) { return a.step < b.step; });
  __int128 span = span0;
  for (int i = 0; i < n; ++i) {
    if (d[i].size <= 1) continue;
    if (d[i].step < span) return false;
    span += (__int128)(d[i].size - 1) * d[i].step;
  }
  return true;
}
static bool apart(const csm_ops_paged_t& c) {
  Dim k[4] = {{c.n_pages, c.k_page_stride}, {c.n_kv, c.k_head_stride}, {c.page_size, c.k_slot_stride}}, v[3] = {{c.n_pages, c.v_page_stride}, {c.n_kv, c.v_head_stride}, {c.page_size, c.v_slot_stride}};
  bool alike = true;
  for (int i = 0; i < 3; ++i) alike &= k[i].size <= 1 || k[i].step == v[i].step;
  const int64_t bytes = (int64_t)((uintptr_t)c.v > (uintptr_t)c.k ? (uintptr_t)c.v - (uintptr_t)c.k : (uintptr_t)c.k - (uintptr_t)c.v);
  k[3] = {alike ? 2 : 1, bytes / (int64_t)ops_size(c.dtype)};
  return bytes && nest(k, 4, c.head_dim) && nest(v, 3, c.head_dim);
}

extern "C" int csm_ops_paged_rope_append(const csm_ops_rope_append_t* p, void* stream) {
  if (!p) return ops_fail(CSM_OPS_ERR_ARG, "null argument");
  const csm_ops_paged_t& c = p->c;
  if (const int r = ops_check_paged(c)) return r;
  if (p->x_dtype != CSM_OPS_F32 && p->x_dtype != CSM_OPS_BF16) return ops_fail(CSM_OPS_ERR_ARG, "unknown dtype %d", p->x_dtype);
  if (p->n_q < 1) return ops_fail(CSM_OPS_ERR_ARG, "n_q must be positive");
  if (c.head_dim % 16 || c.head_dim > 256) return ops_fail(CSM_OPS_ERR_ARG, "head_dim %d is not a multiple of 16 up to 256", c.head_dim);
  if (p->pos_offset < 0 || p->rope_positions < 0) return ops_fail(CSM_OPS_ERR_ARG, "negative position");
  if (!c.rows) return 0;
  if (!p->qkv || !p->q_out || !p->cos || !p->sin) return ops_fail(CSM_OPS_ERR_ARG, "null pointer");
  if (!ops_aligned(p->qkv) || !ops_aligned(p->q_out) || !ops_aligned(p->cos) || !ops_aligned(p->sin) || !ops_stride16(p->qkv_stride, p->x_dtype) ||
      !ops_stride16(p->q_out_stride, p->x_dtype))
    return ops_fail(CSM_OPS_ERR_ARG, "qkv, q_out, cos and sin must start on 16 bytes and have rows of multiples of 16 bytes");
  if (c.rows > 1 && p->q_out_stride < (int64_t)p->n_q * c.head_dim) return ops_fail(CSM_OPS_ERR_ARG, "rows of q_out overlap");
  if (c.n_pages && !apart(c)) return ops_fail(CSM_OPS_ERR_ARG, "slots of k_cache or v_cache overlap, or their strides do not nest");
  const int64_t units = (int64_t)(p->n_q + 2 * (int64_t)c.n_kv) * (c.head_dim / 16), total = units * c.rows;
  if (total > 0x7fffff00) return ops_fail(CSM_OPS_ERR_CAPACITY, "too many rows for one launch");
  AppendArgs a;
  a.c = ops_paged(c);
  a.qkv = p->qkv; a.k = c.k; a.v = c.v; a.q_out = p->q_out; a.cos_t = p->cos; a.sin_t = p->sin;
  a.qkv_stride = p->qkv_stride; a.q_stride = p->q_out_stride; a.n_q = p->n_q; a.hd = c.head_dim;
  a.units = (int)units; a.total = (int)total; a.rope_positions = p->rope_positions; a.pos_offset = p->pos_offset;
  const dim3 grid((unsigned)((total + APPEND_THREADS - 1) / APPEND_THREADS));
  hipStream_t st = (hipStream_t)stream;
  const bool xb = p->x_dtype == CSM_OPS_BF16, cb = c.dtype == CSM_OPS_BF16;
  if (xb && cb) hipLaunchKernelGGL((paged_append_kernel<bf16_t, bf16_t>), grid, dim3(APPEND_THREADS), 0, st, a);
  else if (xb) hipLaunchKernelGGL((paged_append_kernel<bf16_t, float>), grid, dim3(APPEND_THREADS), 0, st, a);
  else if (cb) hipLaunchKernelGGL((paged_append_kernel<float, bf16_t>), grid, dim3(APPEND_THREADS), 0, st, a);
  else hipLaunchKernelGGL((paged_append_kernel<float, float>), grid, dim3(APPEND_THREADS), 0, st, a);
  OPS_HIP(hipGetLastError());
  return 0;
}
