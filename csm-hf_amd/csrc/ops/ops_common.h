// Shared parts of the stand-alone operators (include/csm_ops.h): error text, argument checks, page lookup.
#pragma once
#include "../common.h"
#include "../../../include/csm_ops.h"
#include <stdarg.h>

int ops_fail(int code, const char* fmt, ...);           // records the message, returns `code`
int ops_check_paged(const csm_ops_paged_t& c);          // 0 or a recorded failure
inline bool ops_aligned(const void* p) { return ((uintptr_t)p & 15u) == 0; }
inline size_t ops_size(int dtype) { return dtype == CSM_OPS_BF16 ? 2 : 4; }
inline bool ops_stride16(int64_t s, int dtype) { return (s * (int64_t)ops_size(dtype)) % 16 == 0; }
// a launch has fewer than 2^32 threads in all: checked before the first launch of a call
inline bool ops_launchable(int64_t workgroups, int threads) { return workgroups * threads <= 0xffffffffll; }
#define OPS_HIP(call)                                                                             \
  do {                                                                                            \
    const hipError_t e_ = (call);                                                                 \
    if (e_ != hipSuccess) return ops_fail((int)e_, "%s: %s", #call, hipGetErrorString(e_));       \
  } while (0)

// What a kernel needs of csm_ops_paged_t, by value.
struct Paged {
  const int32_t *table, *lens, *cu;
  int64_t table_stride, kp, kh, ks, vp, vh, vs;
  int n_pages, shift, width, n_seqs, rows, n_kv;
};
Paged ops_paged(const csm_ops_paged_t& c);

// sequence that owns `row`: the last b with cu[b] <= row (cu in LDS or memory), -1 if no sequence does.  Whatever cu holds, b stays in
// [0, n_seqs).
__device__ __forceinline__ int ops_find_seq(const int32_t* cu, int n_seqs, int row) {
  if (n_seqs < 1 || row < cu[0] || row >= cu[n_seqs]) return -1;
  int lo = 0, hi = n_seqs;   // cu[lo] <= row < cu[hi]
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (cu[mid] <= row) lo = mid; else hi = mid;
  }
  return lo;
}
// page number of slot s of a sequence; -1 where the table ends or the page does not exist
__device__ __forceinline__ int ops_page(const int32_t* table, int width, int n_pages, int shift, int slot) {
  const unsigned i = (unsigned)slot >> shift;
  if (slot < 0 || i >= (unsigned)width) return -1;
  const int p = table[i];
  return (unsigned)p < (unsigned)n_pages ? p : -1;
}
