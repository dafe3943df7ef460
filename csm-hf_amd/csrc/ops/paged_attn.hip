// Attention of a batch over a shared prefix and each sequence's own pages (include/csm_ops.h).
//   out[r, h] = sum_j p_j v_j / sum_j p_j,   p_j = exp(scale q.k_j - m),   j over the prefix's slots and own slots 0 .. slot(r)
// First form: one wave per (row, head); the head's elements are spread over the lanes, one key at a time with a running maximum and sum.
#include "ops_common.h"
#include <math.h>

struct AttnOpArgs {
  Paged c;
  const void *q, *k, *v;
  void* out;
  const int32_t* prefix;
  int64_t q_stride, out_stride;
  int n_q, prefix_pages, prefix_len;
  float scale;
};

template <typename XT, typename CT, int HD>
__global__ __launch_bounds__(64) void paged_attn_simple_kernel(AttnOpArgs a) {
  constexpr int N = HD / 64;
  const Paged& c = a.c;
  const int row = blockIdx.x, h = blockIdx.y, lane = threadIdx.x, kvh = h / (a.n_q / c.n_kv);
  int seq = row, t = 0, n_new = 1;
  if (c.cu) {
    seq = ops_find_seq(c.cu, c.n_seqs, row);
    if (seq < 0) return;
    t = row - c.cu[seq];
    n_new = c.cu[seq + 1] - c.cu[seq];
  }
  const int len = c.lens[seq];
  if (len < 0) return;
  const int64_t seen64 = (int64_t)len - n_new + t + 1, cap = (int64_t)c.width << c.shift;
  const int own = (int)(seen64 < 0 ? 0 : seen64 > cap ? cap : seen64);
  float q[N], o[N] = {}, m = -INFINITY, l = 0.f;
#pragma unroll
  for (int i = 0; i < N; ++i) q[i] = to_f32(reinterpret_cast<const XT*>(a.q)[row * a.q_stride + (int64_t)h * HD + i * 64 + lane]) * a.scale;
  for (int j = 0; j < a.prefix_len + own; ++j) {
    const bool in_prefix = j < a.prefix_len;
    const int slot = in_prefix ? j : j - a.prefix_len;
    const int page = in_prefix ? ops_page(a.prefix, a.prefix_pages, c.n_pages, c.shift, slot) : ops_page(c.table + seq * c.table_stride, c.width, c.n_pages, c.shift, slot);
    if (page < 0) continue;
    const int at = slot & ((1 << c.shift) - 1);
    const CT* kp = reinterpret_cast<const CT*>(a.k) + page * c.kp + kvh * c.kh + at * c.ks;
    const CT* vp = reinterpret_cast<const CT*>(a.v) + page * c.vp + kvh * c.vh + at * c.vs;
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < N; ++i) s += q[i] * to_f32(kp[i * 64 + lane]);
    s = wave_sum(s);
    const float m_new = fmaxf(m, s), ref = m_new == -INFINITY ? 0.f : m_new, alpha = __expf(m - ref), p = __expf(s - ref);
    l = l * alpha + p;
#pragma unroll
    for (int i = 0; i < N; ++i) o[i] = o[i] * alpha + p * to_f32(vp[i * 64 + lane]);
    m = m_new;
  }
#pragma unroll
  for (int i = 0; i < N; ++i) store_kv(reinterpret_cast<XT*>(a.out) + row * a.out_stride + (int64_t)h * HD + i * 64 + lane, l == 0.f ? 0.f : o[i] / l);
}

static int check(const csm_ops_attention_t* p) {
  if (!p) return ops_fail(CSM_OPS_ERR_ARG, "null argument");
  const csm_ops_paged_t& c = p->c;
  if (const int r = ops_check_paged(c)) return r;
  if (p->x_dtype != CSM_OPS_F32 && p->x_dtype != CSM_OPS_BF16) return ops_fail(CSM_OPS_ERR_ARG, "unknown dtype %d", p->x_dtype);
  if (p->x_dtype == CSM_OPS_BF16 && c.dtype != CSM_OPS_BF16) return ops_fail(CSM_OPS_ERR_ARG, "bf16 queries need a bf16 cache");
  if (c.head_dim != 64 && c.head_dim != 128) return ops_fail(CSM_OPS_ERR_ARG, "head_dim %d: 64 or 128", c.head_dim);
  if (p->n_q < 1 || p->n_q % c.n_kv) return ops_fail(CSM_OPS_ERR_ARG, "n_q %d is not a multiple of n_kv %d", p->n_q, c.n_kv);
  if (p->prefix_len < 0 || p->prefix_pages < 0) return ops_fail(CSM_OPS_ERR_ARG, "negative size");
  if ((int64_t)p->prefix_pages * c.page_size < p->prefix_len) return ops_fail(CSM_OPS_ERR_ARG, "%d pages of %d slots do not hold a prefix of %d", p->prefix_pages, c.page_size, p->prefix_len);
  if ((int64_t)c.table_width * c.page_size + p->prefix_len > 0x7fffff00) return ops_fail(CSM_OPS_ERR_CAPACITY, "more than 2^31 slots");
  if (!isfinite(p->scale)) return ops_fail(CSM_OPS_ERR_ARG, "scale must be finite");
  if (!c.rows) return 0;
  if (!p->q || !p->out || (p->prefix_len && !p->prefix_table)) return ops_fail(CSM_OPS_ERR_ARG, "null pointer");
  if (!ops_aligned(p->q) || !ops_aligned(p->out) || !ops_stride16(p->q_stride, p->x_dtype) || !ops_stride16(p->out_stride, p->x_dtype))
    return ops_fail(CSM_OPS_ERR_ARG, "q and out must start on 16 bytes and have rows of multiples of 16 bytes");
  return 0;
}

extern "C" int csm_ops_paged_attention_workspace(const csm_ops_attention_t* p, size_t* bytes) {
  if (!bytes) return ops_fail(CSM_OPS_ERR_ARG, "null argument");
  if (const int r = check(p)) return r;
  *bytes = 0;
  return 0;
}

extern "C" int csm_ops_paged_prefix_attention(const csm_ops_attention_t* p, void* stream) {
  if (const int r = check(p)) return r;
  const csm_ops_paged_t& c = p->c;
  if (!c.rows) return 0;
  AttnOpArgs a;
  a.c = ops_paged(c);
  a.q = p->q; a.k = c.k; a.v = c.v; a.out = p->out; a.prefix = p->prefix_table; a.q_stride = p->q_stride; a.out_stride = p->out_stride;
  a.n_q = p->n_q; a.prefix_pages = p->prefix_pages; a.prefix_len = p->prefix_len; a.scale = p->scale;
  const dim3 grid(c.rows, p->n_q);
  hipStream_t st = (hipStream_t)stream;
  const bool xb = p->x_dtype == CSM_OPS_BF16, cb = c.dtype == CSM_OPS_BF16;
#define GO(HD)                                                                                                          \
  do {                                                                                                                  \
    if (xb) hipLaunchKernelGGL((paged_attn_simple_kernel<bf16_t, bf16_t, HD>), grid, dim3(64), 0, st, a);               \
    else if (cb) hipLaunchKernelGGL((paged_attn_simple_kernel<float, bf16_t, HD>), grid, dim3(64), 0, st, a);           \
    else hipLaunchKernelGGL((paged_attn_simple_kernel<float, float, HD>), grid, dim3(64), 0, st, a);                    \
  } while (0)
  if (c.head_dim == 64) GO(64);
  else GO(128);
#undef GO
  OPS_HIP(hipGetLastError());
  return 0;
}
