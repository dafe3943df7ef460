// Attention of a batch over a shared prefix and each sequence's own pages (include/csm_ops.h).
//   out[r, h] = sum_j p_j v_j / sum_j p_j,   p_j = exp(scale q.k_j - m),   j over the prefix's slots and own slots 0 .. slot(r)
//
// The keys of a row form one axis: prefix slots 0 .. P-1, then own slots.  Query rows of one kv-head are FLATTENED to (token row, head of the
// group): f = row * rep + h.  A workgroup takes up to 128 (bf16) or 64 such rows and a range of the axis:
//   prefix item : rows of the WHOLE batch, range inside the prefix -- a prefix slot is fetched once per 128 rows, not once per sequence;
//   own item    : rows of one sequence, range inside its own slots (its prefix too, where every sequence brings rows enough of its own);
// and leaves (max, sum, unnormalised output) per row, which a second small launch joins.
//   up to 16 live rows (decode): the launch waits for memory.  The four waves split the keys, each streams its own, and they join through LDS.
//   more rows: 64-key tiles (32 fp32) of K and V are staged once per workgroup in LDS (two buffers), every wave takes 16-row tiles.
//   more rows in a tall workgroup (below; a text among single tokens): every wave streams all keys for its 16 rows.
// Measured: 128 sequences of some 1500 own slots behind 4096 (32 / 8 heads of 64, bf16): 416 MB in 83 + 5 us, 4.7 TB/s of the 4.9 that a large copy reaches.
// 2 sequences of 4096 new rows: 136 GFLOP in 184 us, 740 TFLOP/s of the 1330 that a large bf16 product reaches; 2162 ragged rows behind 2048 slots 540,
// where 664 workgroups share 256 CUs.  Without its exponentials that launch (at 220 us) took 14 percent less, without the second product 15, without half of the
// first 13, without fetching tiles 11: no single one bounds it.  One sequence behind 512 slots: two launches in 6.9 us, a chain of latencies.
//
// Per wave and 16 query rows, both products are transposed so that a lane owns one query row from score to result:
//   S^T[key][row] = K Q^T   lane (row = lane % 16, g = lane / 16) ends with the scores of keys 4g .. 4g+3 of each 16-key group
//   O^T[d][row]  += V^T P^T contracted over keys in exactly that order, so P never leaves its lane
// K goes from memory straight into the A operand (a lane's 16 bytes are 8 elements of one key); V passes through a wave-private LDS tile and
// ds_read_b64_tr_b16, which hands out the columns.  The running reference m moves only when a score exceeds it by 2^8 (p <= 256 is harmless in
// fp32 sums), so no cross-lane maximum and no rescaling happen in most tiles.
#include "ops_common.h"
#include <float.h>
#include <math.h>

typedef __attribute__((ext_vector_type(8))) short b16x8;
typedef __attribute__((ext_vector_type(4))) short b16x4;
typedef __attribute__((ext_vector_type(2))) float f2;
typedef __attribute__((ext_vector_type(2))) __bf16 b2;

struct AttnOpArgs {
  Paged c;
  const void *q, *k, *v;
  void* out;
  const int32_t* prefix;
  int64_t q_stride, out_stride;
  int n_q, rep, prefix_len;
  uint32_t kp16, ks16, vp16, vs16;   // page and slot strides in 16-byte units (below 2^24): a slot's place inside the cache fits 32 bits up to 64 GB
  int one_place;                     // K and V lie alike: one place serves both
  float c2;               // |scale| log2(e); the sign of scale is folded into q
  uint32_t q_flip;
  int np_tiles, nsp, no_tiles, nso, per_seq_tiles, with_prefix, tall, narrow, nsplit;   // nsplit = partial results per row
  float* part;            // [rows * n_q][nsplit][hd]
  float2* ml;             // [rows * n_q][nsplit] (reference in log2 units, sum)
};

constexpr int AT = 256, MAX_SPLIT = 64;
constexpr float LOG2E = 1.4426950408889634f;
constexpr int tile_rows(int x_dtype) { return x_dtype == CSM_OPS_BF16 ? 128 : 64; }
constexpr float SLACK = 8.f;

__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {   // round to nearest even
  const f2 v = {lo, hi};
  const b2 r = __builtin_convertvector(v, b2);
  return *reinterpret_cast<const uint32_t*>(&r);
}
__device__ __forceinline__ uint32_t pack_trunc(float lo, float hi) { return __builtin_amdgcn_perm(__float_as_uint(hi), __float_as_uint(lo), 0x07060302u); }
__device__ __forceinline__ float trunc_bf16(float x) { return __uint_as_float(__float_as_uint(x) & 0xffff0000u); }
__device__ __forceinline__ float xor16_max(float x) {
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
// 8 floats as N bf16 pieces: one rounded piece, or an exact sum of truncated ones (2: 16 bits, 3: all 24)
template <int N>
__device__ __forceinline__ void split8(const float (&x)[8], b16x8 (&out)[N]) {
  float r[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) r[i] = x[i];
#pragma unroll
  for (int n = 0; n < N; ++n) {
    u32x4 w;
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = n == N - 1 ? pack_bf16(r[2 * i], r[2 * i + 1]) : pack_trunc(r[2 * i], r[2 * i + 1]);
    if (n < N - 1) {
#pragma unroll
      for (int i = 0; i < 8; ++i) r[i] -= trunc_bf16(r[i]);
    }
    out[n] = *reinterpret_cast<const b16x8*>(&w);
  }
}

// ---- products of one wave, by type.  NG = 16-key groups per tile -------------------------------
template <typename XT, typename CT, int HD>
struct Prod;

// bf16 cache: v_mfma_f32_16x16x32_bf16.  bf16 queries: one piece of q; p in two bf16 pieces (16 bits), so that rounding p adds nothing to the one
// rounding of the result -- the launch waits for memory, the second product is free.  fp32 queries: q and p as three pieces each, exactly.
template <typename XT, int HD>
struct Prod<XT, bf16_t, HD> {
  static constexpr int NG = 2, NQ = sizeof(XT) == 2 ? 1 : 3, NP = sizeof(XT) == 2 ? 2 : 3, T = HD / 32, LPK = HD / 8, KPP = 64 / LPK, NV = 32 / KPP;
  static constexpr int LDS_BYTES = 32 * HD * 2;
  b16x8 q[NQ][T];
  struct Tile { u32x4 k[NG][T], v[NV]; };

  struct Raw { W8<XT> w[T]; };   // q as it lies in memory
  static __device__ __forceinline__ void load_q(Raw& raw, const XT* p, int g) {
#pragma unroll
    for (int t = 0; t < T; ++t) raw.w[t].zero();
    if (p)
#pragma unroll
      for (int t = 0; t < T; ++t) raw.w[t].load(p + 32 * t + 8 * g);
  }
  static __device__ __forceinline__ void make_q(const Raw& raw, b16x8 (&q)[NQ][T], uint32_t flip) {
#pragma unroll
    for (int t = 0; t < T; ++t) {
      float x[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = __uint_as_float(__float_as_uint(raw.w[t].get(i)) ^ flip);
      b16x8 f[NQ];
      split8<NQ>(x, f);
#pragma unroll
      for (int n = 0; n < NQ; ++n) q[n][t] = f[n];
    }
  }
  // ko[kt], vo[kt]: place of key 16 kt + lane % 16; kb, vb point at the lane's own piece of a slot
  static __device__ __forceinline__ int k_piece(int lane) { return 8 * (lane >> 4); }
  static __device__ __forceinline__ int v_piece(int lane) { return (lane % LPK) * 8; }
  static __device__ __forceinline__ void load(Tile& t, const char* kb, const char* vb, const uint32_t (&ko)[NG], const uint32_t (&vo)[NG], int lane) {
#pragma unroll
    for (int kt = 0; kt < NG; ++kt) {
      const char* p = kb + ((uint64_t)ko[kt] << 4);
#pragma unroll
      for (int s = 0; s < T; ++s) t.k[kt][s] = *reinterpret_cast<const u32x4*>(p + 64 * s);
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) {   // key i * KPP + lane / LPK
      const int kk = i * KPP, from = (kk & 15) + lane / LPK;
      t.v[i] = *reinterpret_cast<const u32x4*>(vb + ((uint64_t)__shfl(vo[kk >> 4], from) << 4));
    }
  }
  __device__ __forceinline__ void scores(const Tile& t, f32x4 (&s)[NG]) const {
#pragma unroll
    for (int kt = 0; kt < NG; ++kt) {
      s[kt] = (f32x4)(0.f);
#pragma unroll
      for (int n = NQ - 1; n >= 0; --n)
#pragma unroll
        for (int x = 0; x < T; ++x) s[kt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(*reinterpret_cast<const b16x8*>(&t.k[kt][x]), q[n][x], s[kt], 0, 0, 0);
    }
  }
  // 16-byte chunk ch of key kk lies at chunk ch ^ (kk & 7): the rows of a transposing read then cover all banks.  Key i * KPP + lane / LPK: only the
  // KPP part of the key moves the XOR
  static __device__ __forceinline__ void stage_v(const Tile& t, char* lds, int lane, uint32_t valid) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int kk = i * KPP + lane / LPK, ch = lane % LPK;
      u32x4 x = t.v[i];
      if (valid != 0xffffffffu && !((valid >> kk) & 1)) x = (u32x4)(0u);   // 0 * (what an unused slot holds) must be 0
      *reinterpret_cast<u32x4*>(lds + kk * HD * 2 + ((ch ^ (kk & 7)) << 4)) = x;
    }
  }
  // where a lane's transposing reads start: 4 keys from 4 g, columns 16 dt ..; the other columns of the row are an XOR away, keys + 16 a constant
  static __device__ __forceinline__ int v_place(int lane) {
    const int g = lane >> 4, li = lane & 15, k0 = 4 * g + (li >> 2);
    return k0 * HD * 2 + ((((li & 3) >> 1) ^ (k0 & 7)) << 4) + (li & 1) * 8;
  }
  static __device__ __forceinline__ void accumulate(const f32x4 (&p)[NG], char* lds, int place, f32x4 (&o)[HD / 16], int) {
    const float x[8] = {p[0][0], p[0][1], p[0][2], p[0][3], p[1][0], p[1][1], p[1][2], p[1][3]};
    b16x8 f[NP];
    split8<NP>(x, f);
#pragma unroll
    for (int dt = 0; dt < HD / 16; ++dt) {
      typedef __attribute__((address_space(3))) b16x4* lp;
      const b16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lp)(lds + (place ^ (dt << 5))));
      const b16x4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lp)(lds + (place ^ (dt << 5)) + 16 * HD * 2));
      const b16x8 v = {a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
#pragma unroll
      for (int n = NP - 1; n >= 0; --n) o[dt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(v, f[n], o[dt], 0, 0, 0);
    }
  }
};

// fp32 cache and queries: v_mfma_f32_16x16x4_f32, fp32 throughout.  Contraction step (u, e) of the scores takes d = 16 u + 4 g + e from lane
// group g, so that a lane's 16-byte loads of K and Q are operands as they are.
template <int HD>
struct Prod<float, float, HD> {
  static constexpr int NG = 1, U = HD / 16, LPK = HD / 4, KPP = 64 / LPK, NV = 16 / KPP, LD = HD + 4;   // LDS rows 4 floats longer: groups of rows on different banks
  static constexpr int LDS_BYTES = 16 * LD * 4;
  f32x4 q[U];
  struct Tile { f32x4 k[NG][U], v[NV]; };

  struct Raw { f32x4 w[U]; };
  static __device__ __forceinline__ void load_q(Raw& raw, const float* p, int g) {
#pragma unroll
    for (int u = 0; u < U; ++u) raw.w[u] = (f32x4)(0.f);
    if (p)
#pragma unroll
      for (int u = 0; u < U; ++u) raw.w[u] = *reinterpret_cast<const f32x4*>(p + 16 * u + 4 * g);
  }
  static __device__ __forceinline__ void make_q(const Raw& raw, f32x4 (&q)[U], uint32_t flip) {
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int e = 0; e < 4; ++e) q[u][e] = __uint_as_float(__float_as_uint(raw.w[u][e]) ^ flip);
  }
  static __device__ __forceinline__ int k_piece(int lane) { return 4 * (lane >> 4); }
  static __device__ __forceinline__ int v_piece(int lane) { return (lane % LPK) * 4; }
  static __device__ __forceinline__ void load(Tile& t, const char* kb, const char* vb, const uint32_t (&ko)[NG], const uint32_t (&vo)[NG], int lane) {
    const char* p = kb + ((uint64_t)ko[0] << 4);
#pragma unroll
    for (int u = 0; u < U; ++u) t.k[0][u] = *reinterpret_cast<const f32x4*>(p + 64 * u);
#pragma unroll
    for (int i = 0; i < NV; ++i) t.v[i] = *reinterpret_cast<const f32x4*>(vb + ((uint64_t)__shfl(vo[0], i * KPP + lane / LPK) << 4));
  }
  __device__ __forceinline__ void scores(const Tile& t, f32x4 (&s)[NG]) const {
    f32x4 a = (f32x4)(0.f);
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int e = 0; e < 4; ++e) a = __builtin_amdgcn_mfma_f32_16x16x4f32(t.k[0][u][e], q[u][e], a, 0, 0, 0);
    s[0] = a;
  }
  static __device__ __forceinline__ void stage_v(const Tile& t, char* lds, int lane, uint32_t valid) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int kk = i * KPP + lane / LPK;
      f32x4 x = t.v[i];
      if ((valid & 0xffffu) != 0xffffu && !((valid >> kk) & 1)) x = (f32x4)(0.f);
      *reinterpret_cast<f32x4*>(lds + (kk * LD + (lane % LPK) * 4) * 4) = x;
    }
  }
  static __device__ __forceinline__ int v_place(int lane) { return 4 * (lane >> 4) * LD + (lane & 15); }
  static __device__ __forceinline__ void accumulate(const f32x4 (&p)[NG], char* lds, int place, f32x4 (&o)[HD / 16], int) {
    const float* v = reinterpret_cast<const float*>(lds) + place;
#pragma unroll
    for (int dt = 0; dt < HD / 16; ++dt)
#pragma unroll
      for (int e = 0; e < 4; ++e) o[dt] = __builtin_amdgcn_mfma_f32_16x16x4f32(v[e * LD + 16 * dt], p[0][e], o[dt], 0, 0, 0);
  }
};

// ---- one wave over keys [k0, k1) of the axis, tiles first, first + step, ... -------------------------------------------------------------
struct KeyAxis {
  const int32_t *prefix, *own;
  int prefix_len;
  // the table entry that names axis position j's page, and its slot there.  The entry is only looked at when the tile is fetched, a tile later:
  // loads return in order, so a wait for it here would wait for every K and V load in flight
  __device__ __forceinline__ uint32_t entry(int j, const Paged& c, uint32_t& slot) const {
    const bool p = j < prefix_len;
    const uint32_t s = j - (p ? 0 : prefix_len);
    slot = s & ((1u << c.shift) - 1);
    return (uint32_t)(p ? prefix : own)[s >> c.shift];
  }
};

template <typename XT, typename CT, int HD>
__device__ __forceinline__ void wave_attend(const AttnOpArgs& a, const XT* qp, const KeyAxis& ax, int kvh, int k0, int k1, int first, int step,
                                            int lim, int lim_min, char* lds, f32x4 (&o)[HD / 16], float& m, float& l) {
  using P = Prod<XT, CT, HD>;
  constexpr int NG = P::NG, KT = 16 * NG;
  const int lane = threadIdx.x & 63, li = lane & 15, g = lane >> 4;
  const char* kb = reinterpret_cast<const char*>(reinterpret_cast<const CT*>(a.k) + kvh * a.c.kh + P::k_piece(lane));
  const char* vb = reinterpret_cast<const char*>(reinterpret_cast<const CT*>(a.v) + kvh * a.c.vh + P::v_piece(lane));
  const int place = P::v_place(lane);
  m = -INFINITY; l = 0.f;
#pragma unroll
  for (int i = 0; i < HD / 16; ++i) o[i] = (f32x4)(0.f);

  uint32_t pg[NG], sl[NG];
  auto look = [&](int j0) {
#pragma unroll
    for (int kt = 0; kt < NG; ++kt) {
      const int j = j0 + 16 * kt + li;
      pg[kt] = ~0u;
      sl[kt] = 0;
      if (j < k1) pg[kt] = ax.entry(j, a.c, sl[kt]);
    }
  };
  auto fetch = [&](typename P::Tile& t, uint32_t& valid) {
    uint32_t ko[NG], vo[NG];
    valid = 0;
#pragma unroll
    for (int kt = 0; kt < NG; ++kt) {
      const bool ok = pg[kt] < (uint32_t)a.c.n_pages;
      const uint32_t page = ok ? pg[kt] : 0;   // page 0 exists: callers have n_pages >= 1
      valid |= ((uint32_t)__ballot(ok) & 0xffffu) << (16 * kt);
      ko[kt] = __umul24(page, a.kp16) + __umul24(sl[kt], a.ks16);
      vo[kt] = ko[kt];
      if (!a.one_place) vo[kt] = __umul24(page, a.vp16) + __umul24(sl[kt], a.vs16);
    }
    P::load(t, kb, vb, ko, vo, lane);
  };
  int j = k0 + first * KT;
  const int hop = step * KT;
  if (j >= k1) return;
  typename P::Tile t;
  uint32_t valid;
  // a short launch is a chain of memory latencies: q is on its way while the page numbers and the first tile come
  P pr;
  typename P::Raw raw;
  look(j);
  P::load_q(raw, qp, g);
  fetch(t, valid);
  look(j + hop);
  P::make_q(raw, pr.q, a.q_flip);
  for (; j < k1; j += hop) {
    constexpr uint32_t ALL = NG == 2 ? 0xffffffffu : 0xffffu;
    f32x4 s[NG];
    P::stage_v(t, lds, lane, valid);
    pr.scores(t, s);
    if (valid != ALL || j + KT > lim_min) {
#pragma unroll
      for (int kt = 0; kt < NG; ++kt)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int kk = 16 * kt + 4 * g + e;
          s[kt][e] = ((valid >> kk) & 1) && j + kk < lim ? s[kt][e] : -INFINITY;
        }
    }
    if (j + hop < k1) {   // the tile's registers are free: the next one is in flight behind the softmax and the second product
      fetch(t, valid);
      look(j + 2 * hop);
    }
    float top = s[0][0];
#pragma unroll
    for (int kt = 0; kt < NG; ++kt)
#pragma unroll
      for (int e = 0; e < 4; ++e) top = fmaxf(top, s[kt][e]);
    top *= a.c2;
    if (__any(top > m + SLACK)) {   // (-inf + 8 = -inf: the first tile with a key always comes here)
      top = xor32_max(xor16_max(top));
      const float m_new = fmaxf(m, top), alpha = m_new == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m - m_new);
      l *= alpha;
#pragma unroll
      for (int i = 0; i < HD / 16; ++i) o[i] *= alpha;
      m = m_new;
    }
    const float ref = m == -INFINITY ? 0.f : m;
#pragma unroll
    for (int kt = 0; kt < NG; ++kt)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        s[kt][e] = __builtin_amdgcn_exp2f(__fmaf_rn(s[kt][e], a.c2, -ref));
        l += s[kt][e];
      }
    P::accumulate(s, lds, place, o, lane);
  }
  l = xor32_sum(xor16_sum(l));
}

// ---- many rows: tiles shared by the workgroup; bf16 cache: 64 keys ---------------------------------------------------------------------------
// bf16 queries: two 16-row tiles per wave, so that a K or V operand read from LDS feeds two products.  FINE: p in two bf16 pieces (16 bits), so that
// rounding p adds nothing to the one rounding of the result; otherwise in ONE piece, a second rounding of the size of the result's own (the sum l is of
// the same rounded p) against a third of the matrix instructions.  Two pieces / one (us; relative error 0.0017 / 0.0021-0.0023 throughout): prefix items of
// decode launches, which wait for memory beside the sequences' own items, 88.3 / 87.8 for 128 sequences of some 1500 slots behind 4096, 25.0 / 24.1 behind 2048,
// 14.8 / 13.7 for 32; many rows of their own, bound by issue slots, 89.7 / 70.1 for 2162 ragged rows, 252 / 187 for 2 x 4096.  So the decode launches
// (AttnOpArgs::narrow) take two and the others one.  fp32 queries: one tile per wave, q and p in three exact pieces.  l comes off the matrix pipe too, as
// a product with ones.
template <typename XT, typename CT, int HD, bool FINE>
struct Wide;
template <typename XT, int HD, bool FINE>
struct Wide<XT, bf16_t, HD, FINE> {
  static constexpr int RT = sizeof(XT) == 2 ? 2 : 1, NQ = sizeof(XT) == 2 ? 1 : 3, NP = sizeof(XT) == 2 && FINE ? 2 : NQ, T = HD / 32, KEYS = 64, CH = HD / 8, KPP = AT / CH, NL = KEYS / KPP;
  static constexpr int TILE = KEYS * HD * 2, LDS_BYTES = 4 * TILE;   // K, V, two buffers
  b16x8 q[RT][NQ][T];
  f32x4 o[RT][HD / 16], l4[RT];
  float m[RT];

  __device__ __forceinline__ void run(const AttnOpArgs& a, const XT* const (&qp)[RT], const KeyAxis& ax, int kvh, int k0, int k1, const int (&lim)[RT], const int (&lim_min)[RT], int n_rt, char* lds) {
    const int tid = threadIdx.x, lane = tid & 63, li = lane & 15, g = lane >> 4;
    const int ch = tid % CH, key0 = tid / CH;
    const char* kb = reinterpret_cast<const char*>(reinterpret_cast<const bf16_t*>(a.k) + kvh * a.c.kh + ch * 8);
    const char* vb = reinterpret_cast<const char*>(reinterpret_cast<const bf16_t*>(a.v) + kvh * a.c.vh + ch * 8);
#pragma unroll
    for (int r = 0; r < RT; ++r) {
      m[r] = -INFINITY;
      l4[r] = (f32x4)(0.f);
#pragma unroll
      for (int i = 0; i < HD / 16; ++i) o[r][i] = (f32x4)(0.f);
    }
    if (k0 >= k1) return;
    // every wave looks up the pages of a tile's 64 keys, lane = key; a thread stages chunk tid % CH of keys i * KPP + tid / CH
    uint32_t entry = 0, slot = 0;
    auto look = [&](int j0) {
      const int j = j0 + lane;
      entry = ~0u;
      slot = 0;
      if (j < k1) entry = ax.entry(j, a.c, slot);
    };
    u32x4 kr[NL], vr[NL];
    auto fetch = [&]() -> uint64_t {
      const bool ok = entry < (uint32_t)a.c.n_pages;
      const uint32_t page = ok ? entry : 0, ko = __umul24(page, a.kp16) + __umul24(slot, a.ks16);   // (page 0 exists)
      uint32_t kat[NL], vat[NL];
#pragma unroll
      for (int i = 0; i < NL; ++i) vat[i] = kat[i] = __shfl(ko, i * KPP + key0);
      if (!a.one_place) {
        const uint32_t vo = __umul24(page, a.vp16) + __umul24(slot, a.vs16);
#pragma unroll
        for (int i = 0; i < NL; ++i) vat[i] = __shfl(vo, i * KPP + key0);
      }
#pragma unroll
      for (int i = 0; i < NL; ++i) {
        kr[i] = *reinterpret_cast<const u32x4*>(kb + ((uint64_t)kat[i] << 4));
        vr[i] = *reinterpret_cast<const u32x4*>(vb + ((uint64_t)vat[i] << 4));
      }
      return __ballot(ok);
    };
    typename Prod<XT, bf16_t, HD>::Raw raw[RT];   // (on its way while the page numbers and the first tile come)
    look(k0);
#pragma unroll
    for (int r = 0; r < RT; ++r) Prod<XT, bf16_t, HD>::load_q(raw[r], qp[r], g);
    uint64_t valid = fetch();
    look(k0 + KEYS);
#pragma unroll
    for (int r = 0; r < RT; ++r) Prod<XT, bf16_t, HD>::make_q(raw[r], q[r], a.q_flip);
    // LDS places of this lane: what it stages (keys KPP apart), its K operands (16-key tiles and 32-element steps apart), its V columns
    int st[NL], kp[T], vp[HD / 16];
#pragma unroll
    for (int i = 0; i < NL; ++i) st[i] = (i * KPP + key0) * HD * 2 + ((ch ^ ((i * KPP + key0) & 7)) << 4);
#pragma unroll
    for (int x = 0; x < T; ++x) kp[x] = li * HD * 2 + (((4 * x + g) ^ (li & 7)) << 4);
#pragma unroll
    for (int dt = 0; dt < HD / 16; ++dt) vp[dt] = Prod<XT, bf16_t, HD>::v_place(lane) ^ (dt << 5);
    int buf = 0;
    for (int j = k0; j < k1; j += KEYS, buf ^= 1) {
      char* const ks = lds + buf * 2 * TILE;
      char* const vs = ks + TILE;
#pragma unroll
      for (int i = 0; i < NL; ++i) {
        if (valid != ~0ull && !((valid >> (i * KPP + key0)) & 1)) vr[i] = (u32x4)(0u);   // 0 * (what an unused slot holds) must be 0
        *reinterpret_cast<u32x4*>(ks + st[i]) = kr[i];
        *reinterpret_cast<u32x4*>(vs + st[i]) = vr[i];
      }
      __syncthreads();   // (one per tile: a buffer is written again only two tiles later)
      const uint64_t now = valid;
      if (j + KEYS < k1) {
        valid = fetch();
        look(j + 2 * KEYS);
      }
      if (n_rt) tile(a, ks, vs, kp, vp, now, j, g, lim, lim_min, n_rt);
    }
  }

  // One staged tile for the wave's first n_rt row tiles.  (A branch per product of the second one, not a copy without it: the copy let the scheduler hold
  // 30 registers more, and two waves per SIMD instead of three took 10 percent longer.)  The branches also keep the scheduler from moving LDS reads, so they
  // stand ahead by hand: K one 16-key tile, V two operands.  The further a wave is in its tile, the earlier it goes: the three waves of a SIMD then sit in
  // different phases, and one's exponentials run beside another's products.  2162 ragged rows behind 2048 slots 79 -> 70 us, 2 sequences of 4096 rows 193 -> 180;
  // reads ahead alone 77 -> 74.5 and 185 -> 194, priority for the second product alone 77 and 187.  (Four waves per SIMD need spills: 100 and 220)
  __device__ __forceinline__ void tile(const AttnOpArgs& a, const char* ks, char* vs, const int (&kp)[T], const int (&vp)[HD / 16], uint64_t now, int j, int g, const int (&lim)[RT], const int (&lim_min)[RT], int n_rt) {
    const b16x8 ones = (b16x8)((short)0x3f80);
    f32x4 s[RT][4];
    __builtin_amdgcn_s_setprio(1);
    b16x8 k[2][T];
    auto read_k = [&](int kt) {
#pragma unroll
      for (int x = 0; x < T; ++x) k[kt & 1][x] = *reinterpret_cast<const b16x8*>(ks + kp[x] + 16 * kt * HD * 2);
    };
    read_k(0);
#pragma unroll
    for (int kt = 0; kt < 4; ++kt) {
      if (kt < 3) read_k(kt + 1);
#pragma unroll
      for (int r = 0; r < RT; ++r) {
        if (r && n_rt < 2) break;
        s[r][kt] = (f32x4)(0.f);
#pragma unroll
        for (int n = NQ - 1; n >= 0; --n)
#pragma unroll
          for (int x = 0; x < T; ++x) s[r][kt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(k[kt & 1][x], q[r][n][x], s[r][kt], 0, 0, 0);
      }
    }
    __builtin_amdgcn_s_setprio(2);
    b16x8 p[RT][2][NP];
#pragma unroll
    for (int r = 0; r < RT; ++r) {
      if (r && n_rt < 2) break;
      if (now != ~0ull || j + KEYS > lim_min[r]) {
        const uint64_t seen = now >> (4 * g);
        const int left = lim[r] - j - 4 * g;
#pragma unroll
        for (int kt = 0; kt < 4; ++kt)
#pragma unroll
          for (int e = 0; e < 4; ++e) s[r][kt][e] = ((seen >> (16 * kt + e)) & 1) && 16 * kt + e < left ? s[r][kt][e] : -INFINITY;
      }
      float top = s[r][0][0];
#pragma unroll
      for (int kt = 0; kt < 4; ++kt)
#pragma unroll
        for (int e = 0; e < 4; ++e) top = fmaxf(top, s[r][kt][e]);
      top *= a.c2;
      if (__any(top > m[r] + SLACK)) {
        top = xor32_max(xor16_max(top));
        const float m_new = fmaxf(m[r], top), alpha = m_new == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m[r] - m_new);
        l4[r] *= alpha;
#pragma unroll
        for (int i = 0; i < HD / 16; ++i) o[r][i] *= alpha;
        m[r] = m_new;
      }
      const float ref = m[r] == -INFINITY ? 0.f : m[r];
#pragma unroll
      for (int kt = 0; kt < 4; ++kt)
#pragma unroll
        for (int e = 0; e < 4; ++e) s[r][kt][e] = __builtin_amdgcn_exp2f(__fmaf_rn(s[r][kt][e], a.c2, -ref));
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const float x[8] = {s[r][2 * h][0], s[r][2 * h][1], s[r][2 * h][2], s[r][2 * h][3], s[r][2 * h + 1][0], s[r][2 * h + 1][1], s[r][2 * h + 1][2], s[r][2 * h + 1][3]};
        split8<NP>(x, p[r][h]);
#pragma unroll
        for (int n = NP - 1; n >= 0; --n) l4[r] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(ones, p[r][h][n], l4[r], 0, 0, 0);
      }
    }
    __builtin_amdgcn_s_setprio(3);
    typedef __attribute__((address_space(3))) b16x4* lp;
    constexpr int NV = HD / 8, AHEAD = 2;
    b16x4 vx[AHEAD + 1], vy[AHEAD + 1];
    auto read_v = [&](int i) {
      const int h = i / (HD / 16), dt = i % (HD / 16), to = i % (AHEAD + 1);
      vx[to] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lp)(vs + vp[dt] + 32 * h * HD * 2));
      vy[to] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lp)(vs + vp[dt] + (32 * h + 16) * HD * 2));
    };
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) read_v(i);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      if (i + AHEAD < NV) read_v(i + AHEAD);
      const b16x4 x = vx[i % (AHEAD + 1)], y = vy[i % (AHEAD + 1)];
      const b16x8 v = {x[0], x[1], x[2], x[3], y[0], y[1], y[2], y[3]};
      const int h = i / (HD / 16), dt = i % (HD / 16);
#pragma unroll
      for (int r = 0; r < RT; ++r) {
        if (r && n_rt < 2) break;
#pragma unroll
        for (int n = NP - 1; n >= 0; --n) o[r][dt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(v, p[r][h][n], o[r][dt], 0, 0, 0);
      }
    }
    __builtin_amdgcn_s_setprio(0);
  }
};

// The same on an fp32 cache: 32-key tiles, 16 rows a wave, fp32 products.  Without the sharing each wave fetches every key for itself, and a workgroup of 64
// rows waits for four times the bytes: 2162 ragged rows behind 2048 slots 489 -> 410 us (92 TFLOP/s of the 154 that a large fp32 product reaches).  LDS rows are 4 floats longer than a key: the 16 keys of a K operand then
// cover all banks, and so do the 4 of a V operand.
template <int HD, bool FINE>
struct Wide<float, float, HD, FINE> {
  using P = Prod<float, float, HD>;
  static constexpr int RT = 1, KEYS = 32, CH = HD / 4, KPP = AT / CH, NL = KEYS / KPP, LD = P::LD, U = P::U;
  static constexpr int TILE = KEYS * LD * 4, LDS_BYTES = 4 * TILE;   // K, V, two buffers
  f32x4 q[U], o[RT][HD / 16], l4[RT];
  float m[RT];

  __device__ __forceinline__ void run(const AttnOpArgs& a, const float* const (&qp)[RT], const KeyAxis& ax, int kvh, int k0, int k1, const int (&lim)[RT], const int (&lim_min)[RT], int n_rt, char* lds) {
    const int tid = threadIdx.x, lane = tid & 63, li = lane & 15, g = lane >> 4;
    const int ch = tid % CH, key0 = tid / CH;
    const char* kb = reinterpret_cast<const char*>(reinterpret_cast<const float*>(a.k) + kvh * a.c.kh + ch * 4);
    const char* vb = reinterpret_cast<const char*>(reinterpret_cast<const float*>(a.v) + kvh * a.c.vh + ch * 4);
    m[0] = -INFINITY;
    l4[0] = (f32x4)(0.f);
#pragma unroll
    for (int i = 0; i < HD / 16; ++i) o[0][i] = (f32x4)(0.f);
    if (k0 >= k1) return;
    uint32_t entry = 0, slot = 0;   // of key lane % 32
    auto look = [&](int j0) {
      const int j = j0 + (lane & 31);
      entry = ~0u;
      slot = 0;
      if (j < k1) entry = ax.entry(j, a.c, slot);
    };
    f32x4 kr[NL], vr[NL];
    auto fetch = [&]() -> uint32_t {
      const bool ok = entry < (uint32_t)a.c.n_pages;
      const uint32_t page = ok ? entry : 0, ko = __umul24(page, a.kp16) + __umul24(slot, a.ks16);   // (page 0 exists)
      uint32_t kat[NL], vat[NL];
#pragma unroll
      for (int i = 0; i < NL; ++i) vat[i] = kat[i] = __shfl(ko, i * KPP + key0);
      if (!a.one_place) {
        const uint32_t vo = __umul24(page, a.vp16) + __umul24(slot, a.vs16);
#pragma unroll
        for (int i = 0; i < NL; ++i) vat[i] = __shfl(vo, i * KPP + key0);
      }
#pragma unroll
      for (int i = 0; i < NL; ++i) {
        kr[i] = *reinterpret_cast<const f32x4*>(kb + ((uint64_t)kat[i] << 4));
        vr[i] = *reinterpret_cast<const f32x4*>(vb + ((uint64_t)vat[i] << 4));
      }
      return (uint32_t)__ballot(ok);
    };
    typename P::Raw raw;
    look(k0);
    P::load_q(raw, qp[0], g);
    uint32_t valid = fetch();
    look(k0 + KEYS);
    P::make_q(raw, q, a.q_flip);
    const int st = (key0 * LD + ch * 4) * 4, kp = (li * LD + 4 * g) * 4;
    int buf = 0;
    for (int j = k0; j < k1; j += KEYS, buf ^= 1) {
      char* const ks = lds + buf * 2 * TILE;
      char* const vs = ks + TILE;
#pragma unroll
      for (int i = 0; i < NL; ++i) {
        if (valid != ~0u && !((valid >> (i * KPP + key0)) & 1)) vr[i] = (f32x4)(0.f);   // 0 * (what an unused slot holds) must be 0
        *reinterpret_cast<f32x4*>(ks + st + i * KPP * LD * 4) = kr[i];
        *reinterpret_cast<f32x4*>(vs + st + i * KPP * LD * 4) = vr[i];
      }
      __syncthreads();   // (one per tile: a buffer is written again only two tiles later)
      const uint32_t now = valid;
      if (j + KEYS < k1) {
        valid = fetch();
        look(j + 2 * KEYS);
      }
      if (n_rt) tile(a, ks, vs, kp, now, j, g, lane, lim[0], lim_min[0]);
    }
    l4[0] = (f32x4)(xor32_sum(xor16_sum(l4[0][0])));
  }

  __device__ __forceinline__ void tile(const AttnOpArgs& a, const char* ks, char* vs, int kp, uint32_t now, int j, int g, int lane, int lim, int lim_min) {
    f32x4 s[2];
    s[0] = s[1] = (f32x4)(0.f);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      f32x4 k[2];
#pragma unroll
      for (int kt = 0; kt < 2; ++kt) k[kt] = *reinterpret_cast<const f32x4*>(ks + kp + (16 * kt * LD + 16 * u) * 4);
#pragma unroll
      for (int e = 0; e < 4; ++e)
#pragma unroll
        for (int kt = 0; kt < 2; ++kt) s[kt] = __builtin_amdgcn_mfma_f32_16x16x4f32(k[kt][e], q[u][e], s[kt], 0, 0, 0);
    }
    if (now != ~0u || j + KEYS > lim_min) {
      const uint32_t seen = now >> (4 * g);
      const int left = lim - j - 4 * g;
#pragma unroll
      for (int kt = 0; kt < 2; ++kt)
#pragma unroll
        for (int e = 0; e < 4; ++e) s[kt][e] = ((seen >> (16 * kt + e)) & 1) && 16 * kt + e < left ? s[kt][e] : -INFINITY;
    }
    float top = s[0][0];
#pragma unroll
    for (int kt = 0; kt < 2; ++kt)
#pragma unroll
      for (int e = 0; e < 4; ++e) top = fmaxf(top, s[kt][e]);
    top *= a.c2;
    if (__any(top > m[0] + SLACK)) {
      top = xor32_max(xor16_max(top));
      const float m_new = fmaxf(m[0], top), alpha = m_new == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m[0] - m_new);
      l4[0][0] *= alpha;
#pragma unroll
      for (int i = 0; i < HD / 16; ++i) o[0][i] *= alpha;
      m[0] = m_new;
    }
    const float ref = m[0] == -INFINITY ? 0.f : m[0];
#pragma unroll
    for (int kt = 0; kt < 2; ++kt) {
      f32x4 p[1];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        p[0][e] = __builtin_amdgcn_exp2f(__fmaf_rn(s[kt][e], a.c2, -ref));
        l4[0][0] += p[0][e];
      }
      P::accumulate(p, vs, P::v_place(lane) + 16 * kt * LD, o[0], lane);
    }
  }
};

// ---- results ------------------------------------------------------------------------------------------------------------------------------
__device__ __forceinline__ void store4(float* p, const f32x4& v) { *reinterpret_cast<f32x4*>(p) = v; }
__device__ __forceinline__ void store4(bf16_t* p, const f32x4& v) { *reinterpret_cast<uint2*>(p) = make_uint2(pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3])); }
__device__ __forceinline__ float inverse(float l) { return l == 0.f ? 0.f : 1.f / l; }   // a row without a key: zeros

// sequence and tile of own item `tile` when rows are ragged: tiles are counted per sequence in order
template <int ROWS>
__device__ __forceinline__ bool find_tile(const AttnOpArgs& a, int tile, int& seq, int& first, int& n_rows, int& in_seq) {
  const Paged& c = a.c;
  const int lane = threadIdx.x & 63;
  int before = 0;
  for (int b0 = 0; b0 < c.n_seqs; b0 += 64) {
    const int b = b0 + lane;
    int lo = 0, n = 0;
    if (b < c.n_seqs) {
      lo = min(max(c.cu[b], 0), c.rows);
      n = min(max(c.cu[b + 1], lo), c.rows) - lo;
    }
    const int tiles = (n * a.rep + ROWS - 1) / ROWS;
    int upto = tiles;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const int y = __shfl_up(upto, d);
      if (lane >= d) upto += y;
    }
    const uint64_t past = __ballot(before + upto > tile);
    if (past) {
      const int w = __ffsll((unsigned long long)past) - 1;
      seq = b0 + w;
      first = __builtin_amdgcn_readlane(lo, w);
      n_rows = __builtin_amdgcn_readlane(n, w);
      in_seq = tile - before - __builtin_amdgcn_readlane(upto - tiles, w);
      return true;
    }
    before += __builtin_amdgcn_readlane(upto, 63);
  }
  return false;
}

// a finished 16-row tile: the result itself, or partial result number `slot`.  The lane holds elements 16 dt + 4 g .. + 3 of its row
template <typename XT, int HD>
__device__ __forceinline__ void put(const AttnOpArgs& a, int row, int head, int slot, int g, const f32x4 (&o)[HD / 16], float m, float l) {
  if (a.nsplit == 1) {
    const float inv = inverse(l);
    XT* y = reinterpret_cast<XT*>(a.out) + row * a.out_stride + (int64_t)head * HD + 4 * g;
#pragma unroll
    for (int dt = 0; dt < HD / 16; ++dt) store4(y + 16 * dt, o[dt] * inv);
  } else {
    const int64_t at = ((int64_t)row * a.n_q + head) * a.nsplit + slot;
#pragma unroll
    for (int dt = 0; dt < HD / 16; ++dt) store4(a.part + at * HD + 16 * dt + 4 * g, o[dt]);
    if (g == 0) a.ml[at] = make_float2(m, l);
  }
}

template <typename XT, typename CT, int HD, int NW, bool FINE>
__global__ __launch_bounds__(64 * NW, NW == 4 ? 2 : 1) void paged_attn_kernel(AttnOpArgs a) {
  using P = Prod<XT, CT, HD>;
  constexpr bool WIDE = NW == 4;
  constexpr int ROWS = tile_rows(sizeof(XT) == 2 ? CSM_OPS_BF16 : CSM_OPS_F32);
  constexpr int WAVE_LDS = P::LDS_BYTES > 16 * (HD + 4) * 4 ? P::LDS_BYTES : 16 * (HD + 4) * 4;   // V tile; at the end 16 rows of fp32 results
  constexpr int LDS = WIDE && Wide<XT, CT, HD, FINE>::LDS_BYTES > NW * WAVE_LDS ? Wide<XT, CT, HD, FINE>::LDS_BYTES : NW * WAVE_LDS;
  __shared__ __attribute__((aligned(16))) char lds[LDS];
  __shared__ float ml_s[NW][16][2];
  const Paged& c = a.c;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63, li = lane & 15, g = lane >> 4;
  const int kvh = blockIdx.x % c.n_kv;   // fastest: with 8 kv-heads the items of one head share an XCD's L2
  int it = blockIdx.x / c.n_kv;

  int row0, f0, live, slot_bias, k0, k1, split, axis_end;
  KeyAxis ax{a.prefix, nullptr, a.prefix_len};
  const bool own = it >= a.np_tiles * a.nsp;
  int len = 0, n_rows = 1;
  // keys that token row t of an own item sees, the prefix among them: its own slots are 0 .. slot_bias + t - 1, as far as the table goes
  const int cap = c.width << c.shift;
  auto sees = [&](int t) { return a.prefix_len + min(max(slot_bias + t, 0), cap); };
  if (!own) {
    split = it % a.nsp;
    f0 = (it / a.nsp) * ROWS;
    row0 = 0;
    live = min(ROWS, c.rows * a.rep - f0);
    slot_bias = 0;
    k0 = 0; axis_end = a.prefix_len;
  } else {
    it = a.np_tiles * a.nsp + a.no_tiles * a.nso - 1 - it;   // the last rows of a sequence see most keys: they start first
    split = it % a.nso;
    const int tile = it / a.nso;
    int seq, in_seq;
    if (c.cu) {
      if (!find_tile<ROWS>(a, tile, seq, row0, n_rows, in_seq)) return;
    } else {
      seq = tile / a.per_seq_tiles;
      in_seq = tile - seq * a.per_seq_tiles;
      row0 = seq;
    }
    len = c.lens[seq];
    if (len < 0) return;
    f0 = in_seq * ROWS;
    live = min(ROWS, n_rows * a.rep - f0);
    ax.own = c.table + seq * c.table_stride;
    slot_bias = len - n_rows + 1;
    k0 = a.with_prefix ? 0 : a.prefix_len;
    axis_end = sees((f0 + live - 1) / a.rep);
  }
  const int nsplit = own ? a.nso : a.nsp, slot0 = own ? a.nsplit - a.nso : 0;
  {
    constexpr int KT = 64;   // ranges of whole tiles
    const int span = max(axis_end - k0, 0), chunk = ((span + nsplit - 1) / nsplit + KT - 1) / KT * KT;
    k0 = min(k0 + split * chunk, axis_end);
    k1 = min(k0 + chunk, axis_end);
    if (c.n_pages == 0) k1 = k0;
  }
  const bool by_keys = live <= 16;
  if constexpr (WIDE) {
    if (!by_keys) {   // 16-row tiles wave, wave + 4
      using Wd = Wide<XT, CT, HD, FINE>;
      Wd w;
      int lim[Wd::RT], lim_min[Wd::RT], n_rt = 0;
      const XT* qp[Wd::RT];
#pragma unroll
      for (int r = 0; r < Wd::RT; ++r) {
        const int first = 16 * (wave + 4 * r), f = f0 + first + li;
        n_rt += first < live;
        lim[r] = own ? sees(f / a.rep) : a.prefix_len;
        lim_min[r] = own ? sees((f0 + first) / a.rep) : a.prefix_len;   // rows ascend: the first sees least
        const bool on = first + li < live;
        qp[r] = on ? reinterpret_cast<const XT*>(a.q) + (row0 + f / a.rep) * a.q_stride + (int64_t)(kvh * a.rep + f % a.rep) * HD : nullptr;
      }
      w.run(a, qp, ax, kvh, k0, k1, lim, lim_min, n_rt, lds);
#pragma unroll
      for (int r = 0; r < Wd::RT; ++r) {
        const int first = 16 * (wave + 4 * r), f = f0 + first + li;
        if (first + li >= live) continue;
        put<XT, HD>(a, row0 + f / a.rep, kvh * a.rep + f % a.rep, slot0 + split, g, w.o[r], w.m[r], w.l4[r][0]);
      }
      return;
    }
  }
  // rows of this wave: all waves the same 16 (keys split over the waves), or 16 each
  const int mine = by_keys ? 0 : 16 * wave, n_mine = min(16, live - mine);   // (ROWS <= 16 NW)
  char* my_lds = lds + wave * WAVE_LDS;
  f32x4 o[HD / 16];
  float m = -INFINITY, l = 0.f;
  const int f = f0 + mine + li, row = row0 + f / a.rep, head = kvh * a.rep + f % a.rep;
  const bool row_live = li < n_mine;
  if (n_mine > 0) {
    const XT* qp = row_live ? reinterpret_cast<const XT*>(a.q) + row * a.q_stride + (int64_t)head * HD : nullptr;
    const int lim = own ? sees(f / a.rep) : a.prefix_len, lim_min = own ? sees((f0 + mine) / a.rep) : a.prefix_len;   // rows ascend: the first sees least
    wave_attend<XT, CT, HD>(a, qp, ax, kvh, k0, k1, by_keys ? wave : 0, by_keys ? NW : 1, lim, lim_min, my_lds, o, m, l);
  }
  if (by_keys) {   // join the waves: every one rescales to the common reference and leaves its rows in LDS
    if (g == 0) { ml_s[wave][li][0] = m; ml_s[wave][li][1] = l; }
    __syncthreads();
    float top = -INFINITY;
#pragma unroll
    for (int w = 0; w < NW; ++w) top = fmaxf(top, ml_s[w][li][0]);
    const float alpha = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - top);
    float* mine_o = reinterpret_cast<float*>(my_lds) + li * (HD + 4);
#pragma unroll
    for (int dt = 0; dt < HD / 16; ++dt) store4(mine_o + 16 * dt + 4 * g, o[dt] * alpha);
    __syncthreads();
    for (int i = threadIdx.x; i < live * (HD / 4); i += 64 * NW) {
      const int r = i / (HD / 4), d = (i % (HD / 4)) * 4, ff = f0 + r;
      const int rr = row0 + ff / a.rep, hh = kvh * a.rep + ff % a.rep;
      f32x4 sum = (f32x4)(0.f);
      float top_r = -INFINITY, l_r = 0.f;
#pragma unroll
      for (int w = 0; w < NW; ++w) top_r = fmaxf(top_r, ml_s[w][r][0]);
#pragma unroll
      for (int w = 0; w < NW; ++w) {
        sum += *reinterpret_cast<const f32x4*>(reinterpret_cast<const float*>(lds + w * WAVE_LDS) + r * (HD + 4) + d);
        const float mw = ml_s[w][r][0];
        l_r += mw == -INFINITY ? ml_s[w][r][1] : ml_s[w][r][1] * __builtin_amdgcn_exp2f(mw - top_r);
      }
      const int64_t at = (int64_t)rr * a.n_q + hh;
      if (a.nsplit == 1) {
        store4(reinterpret_cast<XT*>(a.out) + rr * a.out_stride + (int64_t)hh * HD + d, sum * inverse(l_r));
      } else {
        store4(a.part + (at * a.nsplit + slot0 + split) * HD + d, sum);
        if (d == 0) a.ml[at * a.nsplit + slot0 + split] = make_float2(top_r, l_r);
      }
    }
    return;
  }
  if (row_live) put<XT, HD>(a, row, head, slot0 + split, g, o, m, l);
}

// join the partial results of a (row, head): one wave, its halves on alternate splits, lane = split for the weights
template <typename XT, int HD>
__global__ __launch_bounds__(AT) void paged_attn_join_kernel(AttnOpArgs a) {
  const Paged& c = a.c;
  constexpr int N = HD / 32;
  typedef __attribute__((ext_vector_type(N))) float vec;
  const int lane = threadIdx.x & 63, d = (lane & 31) * N;
  const int64_t at = (int64_t)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (at >= (int64_t)c.rows * a.n_q) return;
  const int row = (int)(at / a.n_q), head = (int)(at - (int64_t)row * a.n_q);
  const int seq = c.cu ? ops_find_seq(c.cu, c.n_seqs, row) : row;
  if (seq < 0) return;
  const int len = c.lens[seq];
  const float* p = a.part + at * a.nsplit * HD + d;
  // the first partial results are on their way while the weights are made (a padded sequence's hold anything, and are not stored)
  constexpr int AHEAD = 4;
  vec v[AHEAD];
#pragma unroll
  for (int i = 0; i < AHEAD; ++i) v[i] = *reinterpret_cast<const vec*>(p + (int64_t)min(2 * i + (lane >> 5), a.nsplit - 1) * HD);
  const float2 x = lane < a.nsplit ? a.ml[at * a.nsplit + lane] : make_float2(-INFINITY, 0.f);
  const float top = wave_max(x.x);
  const float w = x.x == -INFINITY ? (x.y == 0.f ? 0.f : 1.f) : __builtin_amdgcn_exp2f(x.x - top);   // (no key: sum 0; nothing but NaN: let it through)
  const float inv = inverse(wave_sum(w * x.y));
  vec o = (vec)(0.f);
  auto add = [&](int s0, const vec& val) {
    const float lo = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(w), s0));
    const float hi = s0 + 1 < a.nsplit ? __int_as_float(__builtin_amdgcn_readlane(__float_as_int(w), s0 + 1)) : 0.f;
    const float ws = lane < 32 ? lo : hi;
#pragma unroll
    for (int i = 0; i < N; ++i) o[i] += ws * val[i];
  };
#pragma unroll
  for (int i = 0; i < AHEAD; ++i)
    if (2 * i < a.nsplit) add(2 * i, v[i]);
#pragma unroll 4
  for (int s0 = 2 * AHEAD; s0 < a.nsplit; s0 += 2) add(s0, *reinterpret_cast<const vec*>(p + (int64_t)min(s0 + (lane >> 5), a.nsplit - 1) * HD));
  if (len < 0) return;
  XT* y = reinterpret_cast<XT*>(a.out) + row * a.out_stride + (int64_t)head * HD + d;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const float t = xor32_sum(o[i]) * inv;
    if (lane < 32) store_kv(y + i, t);
  }
}

// ---- entry points -----------------------------------------------------------------------------------------------------------------------
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
  if ((int64_t)c.table_width * c.page_size + p->prefix_len > 0x7fff0000) return ops_fail(CSM_OPS_ERR_CAPACITY, "more than 2^31 slots");
  if ((int64_t)c.rows * p->n_q > (1 << 28) || c.n_seqs > (1 << 28)) return ops_fail(CSM_OPS_ERR_CAPACITY, "too many rows for one launch");
  const int64_t unit = c.dtype == CSM_OPS_BF16 ? 8 : 4, most_k = (c.n_pages - 1) * c.k_page_stride + (c.page_size - 1) * c.k_slot_stride,
                most_v = (c.n_pages - 1) * c.v_page_stride + (c.page_size - 1) * c.v_slot_stride;
  if (c.n_pages && (most_k / unit > 0xffffffffll || most_v / unit > 0xffffffffll)) return ops_fail(CSM_OPS_ERR_CAPACITY, "a cache of more than 64 GB");
  const int64_t strides[4] = {c.k_page_stride, c.k_slot_stride, c.v_page_stride, c.v_slot_stride};
  for (int64_t x : strides)
    if (x / unit >= 1 << 24 || c.n_pages > 1 << 24) return ops_fail(CSM_OPS_ERR_CAPACITY, "more than 2^24 pages, or pages or slots 256 MB apart");
  if (!isfinite(p->scale * LOG2E)) return ops_fail(CSM_OPS_ERR_ARG, "scale must be finite, and so must scale * log2(e)");
  if (!c.rows) return 0;
  if (!p->q || !p->out || (p->prefix_len && !p->prefix_table)) return ops_fail(CSM_OPS_ERR_ARG, "null pointer");
  if (!ops_aligned(p->q) || !ops_aligned(p->out) || !ops_stride16(p->q_stride, p->x_dtype) || !ops_stride16(p->out_stride, p->x_dtype))
    return ops_fail(CSM_OPS_ERR_ARG, "q and out must start on 16 bytes and have rows of multiples of 16 bytes");
  if (c.rows > 1 && p->out_stride < (int64_t)p->n_q * c.head_dim) return ops_fail(CSM_OPS_ERR_ARG, "rows of out overlap");
  return 0;
}

// How the work is cut.  Items should fill 256 CUs (of two to four workgroups each), but a short item is mostly start-up, and every piece costs a
// partial result per row, written and read again.  Measured (us): 128 sequences behind 4096 slots, prefix in 4 / 8 / 16 pieces 86 / 88 / 96 (one rule for all of these takes 8), own slots in
// 1 / 2 / 3 / 5 pieces 92 / 88 / 90 / 92; 64 sequences of 128-wide heads behind 2048 slots, prefix in 4 / 8 / 16 pieces 25 / 18.5 / 22, own in 2 / 4 / 5
// pieces 18.7 / 18.5 / 19.8; 16 fp32 sequences behind 512 slots, prefix in 4 / 8 / 16 pieces 14 / 11.4 / 11.9; tiles of many rows whole / in 3 pieces 88 / 110.
static int plan(const csm_ops_attention_t* p, AttnOpArgs& a) {
  const csm_ops_paged_t& c = p->c;
  a.c = ops_paged(c);
  a.n_q = p->n_q; a.rep = p->n_q / c.n_kv; a.prefix_len = p->prefix_len;
  const int64_t flat = (int64_t)c.rows * a.rep;
  const int ROWS = tile_rows(p->x_dtype);
  a.per_seq_tiles = (a.rep + ROWS - 1) / ROWS;
  const int64_t own_tiles = c.cu_rows ? flat / ROWS + c.n_seqs : (int64_t)c.n_seqs * a.per_seq_tiles;
  const int64_t own_cap = (int64_t)c.table_width * c.page_size;
  a.narrow = c.n_seqs > 0 && flat / c.n_seqs <= 16;   // decode: items wait for memory and are cheap to cut; a tile of many rows has much to join
  const int64_t axis = p->prefix_len + own_cap;
  // few sequences and a short axis: ONE launch of tall workgroups (16 or 8 waves split the keys, the prefix among them) -- the prefix is read once per
  // sequence, from L2, and there is nothing to join.  The axis may be longer where the sequences alone give the CUs a workgroup each.  Measured (us, tall
  // against cut, 64 bf16 or fp32): 200 + 50 slots 6.2 / 6.7 and 8.4 / 7.1 for 1 sequence, 6.8 / 8.8 and 9.2 / 10.2 for 32; 512 + 130: 8.2 / 7.1 and
  // 13.6 / 8.0 for 1, 8.9 / 9.0 and 15.3 / 14.8 for 32; 512 + 1000: 12.5 / 11.1 and 25 / 18.5 for 16, 14.6 / 17.5 and 26.8 / 25.7 for 32; 128: 22 / 12 at 200 + 50
  const int64_t full = own_tiles * c.n_kv;
  a.tall = a.narrow && p->prefix_len > 0 && full <= 256 && axis * c.head_dim * (c.dtype == CSM_OPS_BF16 ? 2 : 4) <= 64 * 1024 + (full > 128 ? (full - 128) * 2048 : 0);
  // sequences that bring two tiles of 16 rows and more of their own read the prefix with them: nothing to share, nothing to join
  a.with_prefix = a.tall || (p->prefix_len > 0 && c.cu_rows && c.n_seqs > 0 && flat / c.n_seqs >= 32);
  const int64_t np = p->prefix_len && !a.with_prefix ? (flat + ROWS - 1) / ROWS : 0;
  const int64_t own_keys = own_cap + (a.with_prefix ? p->prefix_len : 0);
  // pieces of `keys` for each of `items`: up to `few` of them may be as short as `small` keys, up to `many` as short as 256
  auto splits = [](int64_t items, int64_t keys, int64_t few, int64_t small, int64_t many) {
    if (items < 1) items = 1;
    const int64_t a = few / items < (keys + small - 1) / small ? few / items : (keys + small - 1) / small;
    const int64_t b = many / items < (keys + 255) / 256 ? many / items : (keys + 255) / 256;
    const int64_t n = a > b ? a : b;
    return (int)(n < 1 ? 1 : n > MAX_SPLIT / 2 ? MAX_SPLIT / 2 : n);
  };
  a.nsp = np ? splits(np * c.n_kv, p->prefix_len, 64, 64, 256) : 0;
  a.nso = a.tall ? 1 : splits(own_tiles * c.n_kv, own_keys, 512, 128, a.narrow ? 2048 : 0);
  a.np_tiles = (int)np; a.no_tiles = (int)own_tiles; a.nsplit = a.nsp + a.nso;
  if (!ops_launchable(((int64_t)a.np_tiles * a.nsp + (int64_t)a.no_tiles * a.nso) * c.n_kv, a.tall ? 1024 : AT) ||
      (a.nsplit > 1 && !ops_launchable(((int64_t)c.rows * p->n_q + 3) / 4, AT)))
    return ops_fail(CSM_OPS_ERR_CAPACITY, "too many rows for one launch");
  return 0;
}
static size_t workspace(const csm_ops_attention_t* p, const AttnOpArgs& a) {
  if (a.nsplit <= 1) return 0;
  return (size_t)p->c.rows * p->n_q * a.nsplit * (p->c.head_dim * sizeof(float) + sizeof(float2));
}

extern "C" int csm_ops_paged_attention_workspace(const csm_ops_attention_t* p, size_t* bytes) {
  if (!bytes) return ops_fail(CSM_OPS_ERR_ARG, "null argument");
  if (const int r = check(p)) return r;
  AttnOpArgs a;
  *bytes = 0;
  if (!p->c.rows) return 0;
  if (const int r = plan(p, a)) return r;
  *bytes = workspace(p, a);
  return 0;
}

template <typename XT, typename CT, int HD>
static int launch(const AttnOpArgs& a, hipStream_t st) {
  const unsigned items = (unsigned)(((int64_t)a.np_tiles * a.nsp + (int64_t)a.no_tiles * a.nso) * a.c.n_kv);
  constexpr int TALL = HD == 64 ? 16 : 8;   // as many waves as their registers allow
  constexpr bool EXACT = sizeof(XT) == 4;   // fp32 queries: p is exact either way, one body
  if (a.tall) hipLaunchKernelGGL((paged_attn_kernel<XT, CT, HD, TALL, true>), dim3(items), dim3(64 * TALL), 0, st, a);
  else if (a.narrow || EXACT) hipLaunchKernelGGL((paged_attn_kernel<XT, CT, HD, 4, true>), dim3(items), dim3(AT), 0, st, a);
  else hipLaunchKernelGGL((paged_attn_kernel<XT, CT, HD, 4, EXACT>), dim3(items), dim3(AT), 0, st, a);
  OPS_HIP(hipGetLastError());
  if (a.nsplit > 1) {
    const unsigned n = (unsigned)(((int64_t)a.c.rows * a.n_q + 3) / 4);
    hipLaunchKernelGGL((paged_attn_join_kernel<XT, HD>), dim3(n), dim3(AT), 0, st, a);
    OPS_HIP(hipGetLastError());
  }
  return 0;
}

extern "C" int csm_ops_paged_prefix_attention(const csm_ops_attention_t* p, void* stream) {
  if (const int r = check(p)) return r;
  const csm_ops_paged_t& c = p->c;
  if (!c.rows) return 0;
  AttnOpArgs a;
  if (const int r = plan(p, a)) return r;
  const size_t need = workspace(p, a);
  if (need && (!p->workspace || p->workspace_bytes < need || !ops_aligned(p->workspace)))
    return ops_fail(CSM_OPS_ERR_CAPACITY, "workspace of %zu bytes: %zu on 16 bytes are needed", p->workspace_bytes, need);
  a.q = p->q; a.k = c.k; a.v = c.v; a.out = p->out; a.prefix = p->prefix_table; a.q_stride = p->q_stride; a.out_stride = p->out_stride;
  const int unit = c.dtype == CSM_OPS_BF16 ? 8 : 4;
  a.kp16 = (uint32_t)(c.k_page_stride / unit); a.ks16 = (uint32_t)(c.k_slot_stride / unit);
  a.vp16 = (uint32_t)(c.v_page_stride / unit); a.vs16 = (uint32_t)(c.v_slot_stride / unit);
  a.one_place = a.kp16 == a.vp16 && a.ks16 == a.vs16;
  a.part = reinterpret_cast<float*>(p->workspace);
  a.ml = need ? reinterpret_cast<float2*>(a.part + (size_t)c.rows * p->n_q * a.nsplit * c.head_dim) : nullptr;
  a.q_flip = p->scale < 0.f ? 0x80000000u : 0u;
  // a scale of 0 becomes the smallest there is: -inf times it is still -inf, and the largest finite score is 5e-7
  a.c2 = fmaxf(fabsf(p->scale) * LOG2E, FLT_TRUE_MIN);
  hipStream_t st = (hipStream_t)stream;
  const bool xb = p->x_dtype == CSM_OPS_BF16, cb = c.dtype == CSM_OPS_BF16;
  if (c.head_dim == 64) return xb ? launch<bf16_t, bf16_t, 64>(a, st) : cb ? launch<float, bf16_t, 64>(a, st) : launch<float, float, 64>(a, st);
  return xb ? launch<bf16_t, bf16_t, 128>(a, st) : cb ? launch<float, bf16_t, 128>(a, st) : launch<float, float, 128>(a, st);
}
