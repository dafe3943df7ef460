// Error text and the argument checks shared by the entry points of include/csm_ops.h.
#include "ops_common.h"
#include <stdio.h>

static thread_local char g_err[512] = "";

int ops_fail(int code, const char* fmt, ...) {
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(g_err, sizeof g_err, fmt, ap);
  va_end(ap);
  return code;
}
extern "C" const char* csm_ops_last_error(void) { return g_err; }
extern "C" int csm_ops_abi_version(void) { return CSM_OPS_ABI_VERSION; }

int ops_check_paged(const csm_ops_paged_t& c) {
  if (c.dtype != CSM_OPS_F32 && c.dtype != CSM_OPS_BF16) return ops_fail(CSM_OPS_ERR_ARG, "unknown cache dtype %d", c.dtype);
  if (c.rows < 0 || c.n_seqs < 0 || c.n_pages < 0 || c.table_width < 0) return ops_fail(CSM_OPS_ERR_ARG, "negative size");
  if (c.n_kv < 1 || c.head_dim < 1) return ops_fail(CSM_OPS_ERR_ARG, "n_kv and head_dim must be positive");
  if (c.page_size < 1 || (c.page_size & (c.page_size - 1)) || c.page_size > (1 << 20))
    return ops_fail(CSM_OPS_ERR_ARG, "page_size %d is not a power of two up to 2^20", c.page_size);
  if (!c.cu_rows && c.rows != c.n_seqs) return ops_fail(CSM_OPS_ERR_ARG, "without cu_rows every sequence has one row: %d rows, %d sequences", c.rows, c.n_seqs);
  if ((int64_t)c.table_width * c.page_size > 0x7fffffff) return ops_fail(CSM_OPS_ERR_CAPACITY, "a sequence's pages hold more than 2^31 slots");
  if (c.rows && (!c.seq_lens || (c.table_width && !c.page_table) || (c.n_pages && (!c.k || !c.v)))) return ops_fail(CSM_OPS_ERR_ARG, "null pointer");
  if (!ops_aligned(c.k) || !ops_aligned(c.v)) return ops_fail(CSM_OPS_ERR_ARG, "k_cache and v_cache must start on 16 bytes");
  const int64_t s[6] = {c.k_page_stride, c.k_head_stride, c.k_slot_stride, c.v_page_stride, c.v_head_stride, c.v_slot_stride};
  for (int64_t x : s)
    if (x < 0 || !ops_stride16(x, c.dtype)) return ops_fail(CSM_OPS_ERR_ARG, "cache strides must be multiples of 16 bytes");
  return 0;
}

Paged ops_paged(const csm_ops_paged_t& c) {
  Paged p;
  p.table = c.page_table; p.lens = c.seq_lens; p.cu = c.cu_rows; p.table_stride = c.table_stride;
  p.kp = c.k_page_stride; p.kh = c.k_head_stride; p.ks = c.k_slot_stride;
  p.vp = c.v_page_stride; p.vh = c.v_head_stride; p.vs = c.v_slot_stride;
  p.n_pages = c.n_pages; p.shift = __builtin_ctz((unsigned)c.page_size); p.width = c.table_width;
  p.n_seqs = c.n_seqs; p.rows = c.rows; p.n_kv = c.n_kv;
  return p;
}
