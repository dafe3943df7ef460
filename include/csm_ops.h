/*
 * csm_ops.h -- C ABI of libcsm_ops.so: stand-alone MI355X (gfx950) operators of a serving step over a PAGED KV cache.  They need no engine
 * (include/csm_hip.h): every call takes its tensors, its sizes and a stream, keeps nothing between calls, allocates nothing and does not
 * synchronise, so all of them may be captured into a hipGraph.  They continue what csm_rope_scatter, csm_attn_decode and csm_sample_topk
 * do for the engine's contiguous cache; the reference (thomasgauthier/csm-hf) has no counterpart of a paged cache.
 *
 * Conventions
 *   - return 0 on success; negative = CSM_OPS_ERR_*, positive = hipError_t.  Never throws.  csm_ops_last_error() returns a thread-local
 *     message for the last failure.
 *   - every pointer inside an argument struct is a DEVICE pointer of the device that is current on the calling thread; `stream` is a
 *     hipStream_t of it.  Argument structs live in host memory and are read before the call returns.
 *   - strides count ELEMENTS.  Rows, caches and tables must start on 16 bytes and their strides must keep 16-byte alignment where the
 *     struct says "16 B"; the innermost dimension is contiguous everywhere.  Inputs may share memory between rows (a stride of 0); rows
 *     of an output, and slots of a cache that is written, may not: its strides must nest (each at least what the smaller ones span), and K and V
 *     must lie apart.
 *   - what only the device knows (lengths, page numbers, row offsets) is bounds-checked by the kernels: nothing outside the given tensors
 *     is ever read or written, whatever these arrays hold.
 *
 * The paged cache.  k_cache / v_cache hold `n_pages` pages of `page_size` (a power of two) cache slots for `n_kv` heads of `head_dim`
 * elements; a page's heads and slots lie at the given strides, so [pages][heads][slots][dim] and [pages][slots][heads][dim] both work.
 * Sequence b keeps slot s in page page_table[b * table_stride + s / page_size].  Table entries past a sequence's length are not looked at.
 *
 * Rows.  The `rows` token rows of a call belong to the sequences in order: sequence b owns rows cu_rows[b] .. cu_rows[b+1] - 1, or row b
 * where cu_rows is NULL (one new token per sequence, rows == n_seqs).  seq_lens[b] counts the sequence's own slots INCLUDING these rows:
 * its row t of T sits in slot seq_lens[b] - T + t.  A sequence with seq_lens[b] < 0 is padding: its rows, like rows behind
 * cu_rows[n_seqs], are skipped and their outputs left as they were.
 */
#ifndef CSM_OPS_H
#define CSM_OPS_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define CSM_OPS_ABI_VERSION 1

enum { CSM_OPS_F32 = 0, CSM_OPS_BF16 = 1 };
enum {
  CSM_OPS_OK = 0,
  CSM_OPS_ERR_ARG = -1,       /* bad argument / unsupported shape, type, stride or alignment */
  CSM_OPS_ERR_CAPACITY = -3   /* sizes beyond what one launch covers, or a workspace that is too small */
};

typedef struct {
  void *k, *v;                                             /* 16 B */
  int32_t dtype;                                           /* CSM_OPS_F32 / CSM_OPS_BF16 */
  int32_t n_pages, page_size, n_kv, head_dim;
  int64_t k_page_stride, k_head_stride, k_slot_stride;     /* 16 B each */
  int64_t v_page_stride, v_head_stride, v_slot_stride;
  const int32_t* page_table;                               /* [n_seqs][table_width] at table_stride */
  int64_t table_stride;
  int32_t table_width, n_seqs;
  const int32_t* seq_lens;                                 /* [n_seqs] */
  const int32_t* cu_rows;                                  /* [n_seqs + 1] or NULL */
  int32_t rows;
} csm_ops_paged_t;

/* ---- rotary embedding + append.  Each row of `qkv` is n_q | n_kv | n_kv heads (q, k, v) as the packed projection leaves it.  q and k are
 * rotated in halves by the angle of position pos_offset + slot (cos / sin: fp32 tables [rope_positions][head_dim / 2]), fp32 arithmetic,
 * one rounding to the output's type; v is copied.  k and v go to the row's cache slot, q to q_out [rows][n_q][head_dim] (dtype of qkv; it
 * may be the q part of qkv itself).  head_dim: a multiple of 16 up to 256.  A row is skipped -- nothing written -- when its slot lies outside
 * the page table, its page outside the cache, or its position outside the tables. */
typedef struct {
  csm_ops_paged_t c;
  const void* qkv;                    /* 16 B */
  void* q_out;                        /* 16 B */
  int64_t qkv_stride, q_out_stride;   /* per row, 16 B */
  int32_t x_dtype, n_q;
  const float *cos, *sin;             /* 16 B */
  int32_t rope_positions, pos_offset;
} csm_ops_rope_append_t;
int csm_ops_paged_rope_append(const csm_ops_rope_append_t* a, void* stream);

/* ---- attention over a prefix shared by all rows and each sequence's own slots.  Row r of sequence b at slot s sees the prefix's
 * `prefix_len` slots (pages prefix_table[0 ..], same cache) and its own slots 0 .. s; out[r, h] = softmax(scale q.k) v over them, head h
 * reading kv head h / (n_q / n_kv).  The prefix is stored once for all sequences.  It is also read once
 * for every 128 query rows of a kv-head (64 with fp32 q), whichever sequences they are of, except where that would not pay: sequences that bring 32
 * query rows (rows * n_q / n_kv) each and more on average, and few sequences on a short axis, read it with their own slots.  A row that sees no key gives zeros; a
 * page number outside the cache hides its slots.  Slots that no row of the call sees may hold anything; a NaN or infinity in v of a slot
 * that some rows of a sequence see also reaches that sequence's earlier rows of the call (0 * NaN), never another sequence.  x_dtype (q and
 * out) bf16 needs a bf16 cache: products on the bf16 matrix pipe with fp32 sums; x_dtype fp32 takes either cache, fp32 throughout.
 * head_dim 64 or 128; any n_q that is a multiple of n_kv; at most 64 GB of cache, 2^24 pages, pages and slots less than 256 MB apart.
 * `workspace`: at least csm_ops_paged_attention_workspace bytes (16 B), contents undefined before and after; calls that may overlap in time
 * need one each.  out may be q. */
typedef struct {
  csm_ops_paged_t c;
  const void* q;                      /* 16 B; heads contiguous */
  void* out;
  int64_t q_stride, out_stride;       /* per row, 16 B */
  int32_t x_dtype, n_q;
  const int32_t* prefix_table;        /* [prefix_pages], NULL when prefix_len is 0 */
  int32_t prefix_pages, prefix_len;
  float scale;
  void* workspace;
  size_t workspace_bytes;
} csm_ops_attention_t;
int csm_ops_paged_attention_workspace(const csm_ops_attention_t* a, size_t* bytes_host);
int csm_ops_paged_prefix_attention(const csm_ops_attention_t* a, void* stream);

/* ---- sampling.  Per row: w_i = exp((x_i - max x) / temperature); order the row by x descending, equal values by index; keep the first
 * min(n_k, n_p, n_m) entries: n_k = topk, n_p = the fewest whose w reach top_p of the w of the first n_k, n_m = those with w >= min_p; the
 * token is the first index (in index order) at which the running sum of kept w exceeds u times their total.  temperature 0 = arg-max, the
 * lowest index of equals.  NaN logits count as -inf; several +inf share the row equally; a row of nothing but -inf gives -1.  u outside
 * [0, 1) is clamped to it.  The first entry is always kept.
 * The scalars hold for all rows and are checked: 0 <= temperature < inf, 0 <= topk <= V (0 or V: off), 0 < top_p <= 1 (1: off), 0 <= min_p <= 1 (0: off).
 * A pointer gives one value per row instead; the host does not see these, so any is taken: topk <= 0 or >= V, top_p >= 1, min_p <= 0 switch that
 * filter off, and others are read as the nearest that can be used (temperature < 0 or NaN: 0; top_p < 0 or NaN: 0; min_p > 1: 1, NaN: 0).  V up to 2^21.  Weights are
 * computed in fp64 and summed in 64-bit fixed point, chunks of a long row in fp64 in their order: the same input gives the same token.  A weight is
 * held to 2^-49 of the row's largest, or to 2^-61 of their sum where that is more; smaller ones count as 0. */
typedef struct {
  const void* logits;                 /* [rows][V] at logits_stride, any alignment */
  int64_t logits_stride;
  int32_t x_dtype, rows, V;
  const float* uniform;               /* [rows] */
  const float *temperatures, *top_ps, *min_ps;
  const int32_t* topks;
  float temperature, top_p, min_p;
  int32_t topk;
  int32_t* out;                       /* [rows] */
  void* workspace;                    /* csm_ops_sample_workspace bytes (16 B; 0 up to V = 16 384), undefined before and after, one per call in flight */
  size_t workspace_bytes;
} csm_ops_sample_t;
int csm_ops_sample_workspace(const csm_ops_sample_t* a, size_t* bytes_host);
int csm_ops_sample_filtered(const csm_ops_sample_t* a, void* stream);

const char* csm_ops_last_error(void);
int csm_ops_abi_version(void);

#ifdef __cplusplus
}
#endif
#endif /* CSM_OPS_H */
