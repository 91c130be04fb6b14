// Attention in a sliding window along packed sequences, with a few first tokens that stay visible, and
// its gradient.
//
//   A sequence has n queries and m keys; query i stands at position p = i + m - n among the keys.
//   It sees key j where (j < sinks or |p - j| <= window) and (not causal or j <= p).
//   out = softmax(q k^T scale over the keys it sees) v; zeros where it sees none
// Gradient, with do = d out, dP = do v^T, r = do . out per query:
//   dv = P^T do;  dS = P (dP - r);  dq = scale dS k;  dk = scale dS^T q
//
// G = H / Hk query heads share a key head.  A block's rows are the (query, head of the group) pairs of one
// key head, row x = query x / G, head x % G: so a key head is read once for its G heads, a single token
// fills G rows of a tile, and a tile of 128 rows spans 128 / G positions only.
// The keys of a block's rows are two runs, the sinks and the window of the first to that of the last row
// (one run where they meet); tiles that all rows see take no mask.
// In the others a row and a key that do not see each other have P = 0, and dS = 0, by selection.  Their
// product with a row of v (k; do, q in dk / dv) that holds an infinity or NaN would be NaN still: tiles with
// masks look for those and take them as zeros, and a wave that met one adds them at the end to those of its
// rows that see them, so that the others have the bits they would have without them.

#include <float.h>

#include <algorithm>
#include <type_traits>

#include "attention_tiles.h"
#include "tsc_internal.h"

namespace tsc {
namespace {

constexpr int kNT = 256;  // 4 waves of 32 rows (or keys, in dk / dv)
constexpr int kBQ = 128;
constexpr int kBQ16 = 256;  // rows of a block of the forward pass in 16 bits: 4 waves of 64 (D = 64) or 8 of 32
constexpr int kBK = 32;   // keys of a tile

struct WaArgs {
  const void *q, *k, *v;
  int64_t ldq, ldk, ldv;
  const int32_t *cu_q, *cu_kv;
  int64_t total_q, total_kv;
  int32_t Hk, G, shift;  // G = 1 << shift, or shift < 0
  float sl2;             // scale * log2(e)
  int32_t window, sinks, causal, rest;
  // forward
  void *out, *lo;  // lo: what out's rounding left, in the same type, or null
  float* lse;      // (total_q, H): log2 of the sum of 2^(score sl2), or null
  int32_t splits;  // blocks that share a row tile's keys
  float* part;     // splits > 1: (splits, total_q, H, D) sums, then (splits, total_q, H, 2)
  // backward
  const void* dout;
  float* r;        // (total_q, H): do . out
  void *dq, *dk, *dv;
  int32_t own_sinks;   // dk / dv blocks leave out the sinks, which have blocks and scratch of their own:
  int32_t sink_keys;   // sinks of a sequence there is scratch for, whole tiles of 32
  int32_t sink_parts;  // blocks that share a tile's rows
  float* sink_sums;    // (parts, B, Hk, sink_keys, 2, D): dk without its scale, dv
};

// ---- rows, and what they see ----------------------------------------------------------------
__device__ __forceinline__ int query_of(const WaArgs& a, int x) {
  return a.shift >= 0 ? x >> a.shift : (int)((uint32_t)x / (uint32_t)a.G);
}
// Element offset of row x of key head h in a tensor of row stride ld.
__device__ __forceinline__ int64_t row_at(const WaArgs& a, int64_t ld, int h, int x, int D) {
  const int i = query_of(a, x);
  return (int64_t)i * ld + (int64_t)(h * a.G + x - i * a.G) * D;
}

// The keys that a query at position p sees: [lo, hi) and [0, sink).
struct Seen {
  int lo, hi, sink;
};
__device__ __forceinline__ Seen seen_from(const WaArgs& a, int p, int keys) {
  Seen s;
  s.lo = (int)max<int64_t>(0, (int64_t)p - a.window);
  s.hi = (int)max<int64_t>(s.lo, min<int64_t>(keys, a.causal ? (int64_t)p + 1 : (int64_t)p + a.window + 1));
  s.sink = max(0, min(min(a.sinks, keys), a.causal ? p + 1 : keys));
  return s;
}

// The key tiles, of BK keys, of rows at positions p0 to p1.
template <int BK>
struct Walk {
  int n1, n2;       // tiles of the two runs
  int end1, lo, hi; // the first run is [0, end1), the second [lo, hi)
  bool one;         // the sinks and the window are one run
  Seen first, last; // of p0 and p1
  __device__ __forceinline__ Walk(const WaArgs& a, int p0, int p1, int keys) {
    first = seen_from(a, p0, keys);
    last = seen_from(a, p1, keys);
    one = first.lo <= last.sink;
    end1 = one ? max(last.hi, last.sink) : last.sink;
    lo = first.lo;
    hi = last.hi;
    n1 = (end1 + BK - 1) / BK;
    n2 = one || hi <= lo ? 0 : (hi - lo + BK - 1) / BK;
  }
  __device__ __forceinline__ int tiles() const { return n1 + n2; }
  __device__ __forceinline__ void tile(int t, int* at, int* end) const {
    *at = t < n1 ? t * BK : lo + (t - n1) * BK;
    *end = t < n1 ? end1 : hi;
  }
  // Whether rows whose bounds are f (first) to l (last) see the first `keys` of tile t, all of which there
  // are; whether they see any of `keys` keys of it.
  __device__ __forceinline__ bool full(int t, const Seen& f, const Seen& l, int keys = BK) const {
    int at, end;
    tile(t, &at, &end);
    if (at + keys > end) return false;
    const bool sinks = t < n1 && at + keys <= f.sink;
    const bool win = (one || t >= n1) && at >= l.lo && at + keys <= f.hi;
    return sinks || win;
  }
  __device__ __forceinline__ bool any(int t, const Seen& f, const Seen& l, int from = 0, int keys = BK) const {
    int at, end;
    tile(t, &at, &end);
    at += from;
    const bool sinks = t < n1 && at < l.sink;
    const bool win = (one || t >= n1) && at < l.hi && at + keys > f.lo;
    return sinks || win;
  }
  // The longest run of tiles of which every row sees everything: of the window's, or of the sinks'.
  __device__ __forceinline__ void longest(int* from, int* to) const {
    const int t0 = one ? 0 : n1, k0 = one ? 0 : lo;
    *from = t0 + max(0, last.lo - k0 + BK - 1) / BK;
    *to = t0 + max(0, first.hi - k0) / BK;
    if (first.sink / BK > *to - *from) {
      *from = 0;
      *to = first.sink / BK;
    }
    if (*to <= *from) *from = *to = tiles();
  }
  // A row's bounds within the run that tile t belongs to.
  __device__ __forceinline__ Seen in_run(int t, Seen s) const {
    if (!one) {
      if (t < n1) s.hi = s.lo;
      else s.sink = 0;
    }
    return s;
  }
};
__device__ __forceinline__ bool sees(const Seen& s, int k) {
  return (uint32_t)(k - s.lo) < (uint32_t)(s.hi - s.lo) || k < s.sink;
}
__device__ __forceinline__ bool sees_any(const Seen& s) { return s.hi > s.lo || s.sink > 0; }

// ---- infinities and NaN where a row sees nothing ---------------------------------------------
// Not 0 if an element is not finite: whether each half of a word, or a word, has all of its exponent's bits
// set, by the carry out of them.
template <typename T>
__device__ __forceinline__ uint32_t odd(const F32x8& f) {
  uint32_t r = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) r |= (__float_as_uint(f.v[i]) & 0x7f800000u) + 0x00800000u & 0x80000000u;
  return r;
}
template <typename T>
__device__ __forceinline__ uint32_t odd(const u32x4_t& f) {
  constexpr uint32_t E = std::is_same<T, __bf16>::value ? 0x7f807f80u : 0x7c007c00u;
  constexpr uint32_t L = std::is_same<T, __bf16>::value ? 0x00800080u : 0x04000400u;
  uint32_t r = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) r |= (f[i] & E) + L & 0x80008000u;
  return r;
}
// A fragment with zeros in the place of what is not finite.
template <typename T>
__device__ __forceinline__ F32x8 finite(const F32x8& f) {
  F32x8 r;
#pragma unroll
  for (int i = 0; i < 8; ++i) r.v[i] = (__float_as_uint(f.v[i]) & 0x7f800000u) != 0x7f800000u ? f.v[i] : 0.f;
  return r;
}
template <typename T>
__device__ __forceinline__ u32x4_t finite(const u32x4_t& f) {
  constexpr uint32_t E = std::is_same<T, __bf16>::value ? 0x7f80u : 0x7c00u;
  u32x4_t r;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    r[i] = f[i] & (((f[i] & E) != E ? 0xffffu : 0u) | ((f[i] >> 16 & E) != E ? 0xffff0000u : 0u));
  return r;
}

// acc += sum over the 32 rows e of the tile of p[e] row_e; pf: p as two fragments, col: Tile's col_of.  With masks, what is not
// finite is left out, and met is set.
template <typename T, int D, bool MASK>
__device__ __forceinline__ void add_rows(const unsigned char* t, int col, const typename Frag<T>::type (&pf)[2],
                                         f32x16_t (&acc)[D / 32], bool& met) {
  typedef Frag<T> F;
  typedef typename F::type Fr;
  typedef Tile<T, D> Ti;
  constexpr int MT = D / 32;
#pragma unroll
  for (int g = 0; g < 2; ++g) {
    Fr v[MT];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) v[mt] = Ti::col_at(t, 0, col, g, mt);
    if constexpr (MASK) {
      uint32_t bad = 0;
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) bad |= odd<T>(v[mt]);
      if (__builtin_amdgcn_ballot_w64(bad != 0)) {
        met = true;
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) v[mt] = finite<T>(v[mt]);
      }
    }
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) F::mma(v[mt], pf[g], acc[mt]);
  }
}
// What such a row brings to a lane that sees it: a weight P > 0 times an infinity or NaN is that; dS of a
// score that is not finite is 0 or NaN, and makes NaN of it (NANS).
template <typename T, int D, bool NANS>
__device__ __forceinline__ void add_odd(const T* row, int hf, bool seen, f32x16_t (&acc)[D / 32]) {
#pragma unroll
  for (int mt = 0; mt < D / 32; ++mt)
#pragma unroll
    for (int j = 0; j < 16; ++j) {
      const float v = (float)row[32 * mt + 8 * (j >> 2) + 4 * hf + (j & 3)];
      if (seen && !(fabsf(v) < INFINITY)) acc[mt][j] += NANS ? NAN : v;
    }
}

// ------------------------------------------------------------------------------- forward
// add_odd for the keys of tiles t, t + step, .. below stop.
template <typename T, int D, bool NANS, int BK>
__device__ __forceinline__ void add_keys(const Walk<BK>& walk, const Seen& mine, int t, int stop, int step,
                                         const T* base, int64_t ld, int hf, f32x16_t (&acc)[D / 32]) {
  for (; t < stop; t += step) {
    int at, end;
    walk.tile(t, &at, &end);
    const Seen s = walk.in_run(t, mine);
    for (int k = at; k < min(at + BK, end); ++k) add_odd<T, D, NANS>(base + (int64_t)k * ld, hf, sees(s, k), acc);
  }
}

// One tile of 32 keys from k0 on, in LDS, for a wave's 32 rows; s: what the lane's row sees of it.
template <typename T, int D, bool MASK>
__device__ __forceinline__ void forward_step(const unsigned char* kt, const unsigned char* vt, int row, int col,
                                             int hf, int k0, const Seen& s, float sl2,
                                             const typename Frag<T>::type (&qf)[D / 16], float& m,
                                             float& l, f32x16_t (&o)[D / 32], bool& met) {
  typedef Frag<T> F;
  typedef Tile<T, D> Ti;
  constexpr int KS = D / 16, MT = D / 32;
  f32x16_t c;
  clear(c);
#pragma unroll
  for (int st = 0; st < KS; ++st) F::mma(Ti::row_at(kt, 0, row, st), qf[st], c);
  if constexpr (MASK) {
#pragma unroll
    for (int j = 0; j < 16; ++j)
      if (!sees(s, k0 + 8 * (j >> 2) + 4 * hf + (j & 3))) c[j] = -INFINITY;
  }
  float mx = c[0], p[16];
#pragma unroll
  for (int j = 1; j < 16; ++j) mx = fmaxf(mx, c[j]);
  mx = pair_max(mx) * sl2;
  if (__builtin_amdgcn_ballot_w64(mx > m)) {
    const float mn = fmaxf(m, mx), f = fast_exp2(m - mn);
    m = mn;
    l *= f;
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
      for (int j = 0; j < 16; ++j) o[mt][j] *= f;
  }
#pragma unroll
  for (int j = 0; j < 16; ++j) {
    p[j] = fast_exp2(fmaf(c[j], sl2, -m));
    l += p[j];
  }
  const typename F::type pf[2] = {F::pack(p), F::pack(p + 8)};
  add_rows<T, D, MASK>(vt, col, pf, o, met);
}

// 1 / l; l = 0: the row sees no key, and gets zeros, or its scores are all -inf, of which a softmax is NaN.
__device__ __forceinline__ float inverse(float l, bool some) { return l > 0.f || l != l ? 1.f / l : some ? NAN : 0.f; }
__device__ __forceinline__ float row_lse(float m, float l, bool some) {
  return l == 0.f ? (some ? NAN : INFINITY) : m + log2f(l);
}
// Writes a wave's finished rows: l summed over both halves; some: the row sees a key.
template <typename T, int D>
__device__ __forceinline__ void forward_store(const WaArgs& a, int64_t at, int hf, float l, bool some,
                                              f32x16_t (&o)[D / 32]) {
  const float inv = inverse(l, some);
#pragma unroll
  for (int mt = 0; mt < D / 32; ++mt) {
    T* p = (T*)a.out + at * D + 32 * mt;
    if (sizeof(T) == 2 && a.lo) {
#pragma unroll
      for (int j = 0; j < 16; ++j) o[mt][j] *= inv;
      store_dims(p, hf, o[mt], 1.f);
#pragma unroll
      for (int j = 0; j < 16; ++j) o[mt][j] -= (float)(T)o[mt][j];
      store_dims((T*)a.lo + at * D + 32 * mt, hf, o[mt], 1.f);
    } else {
      store_dims(p, hf, o[mt], inv);
    }
  }
}
__device__ __forceinline__ void store_lse(const WaArgs& a, int64_t at, int hf, float m, float l, bool some) {
  if (a.lse && hf == 0) a.lse[at] = row_lse(m, l, some);
}

// fp32: a block of 4 waves owns 128 rows and walks their keys in tiles of 32.  3500 tokens of 12 x 128, window 256: 226 us, 47
// of the 151 TFLOP/s of a large product by the pairs that are seen (80 % of a tile's).  Matrix cores busy 32 %, VALU 10 %,
// waves waiting 22 %: a wave has its SIMD for itself at D = 128 (416 registers), so 336 blocks take two rounds over the CUs of
// which the second fills a third, and in a wave products, exponentials and two barriers a tile follow one another.
template <int D>
__global__ void __launch_bounds__(kNT, D == 64 ? 2 : 1) wa_forward32_kernel(const WaArgs a) {
  typedef float T;
  typedef Frag<T> F;
  typedef Tile<T, D> Ti;
  constexpr int KS = D / 16, MT = D / 32;
  __shared__ __attribute__((aligned(16))) unsigned char kt[kBK * Ti::ROWB], vt[kBK * Ti::ROWB];
  int bx, h, bb;
  block_tile(a.cu_kv, &bx, &h, &bb);
  int q0, q_len, kv0, kv_len;
  segment(a.cu_q, bb, a.total_q, &q0, &q_len);
  segment(a.cu_kv, bb, a.total_kv, &kv0, &kv_len);
  const int tid = threadIdx.x, lane = tid & 63, l32 = lane & 31, hf = lane >> 5;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int H = a.Hk * a.G, n = q_len * a.G, off = kv_len - q_len;
  if (a.rest) zero_rest((T*)a.out, a.cu_q, a.total_q, bb, H, D, h * a.G, bx, gridDim.x, a.G);
  const T* qbase = (const T*)a.q + (int64_t)q0 * a.ldq;
  const T* kbase = (const T*)a.k + (int64_t)kv0 * a.ldk + (int64_t)h * D;
  const T* vbase = (const T*)a.v + (int64_t)kv0 * a.ldv + (int64_t)h * D;

  for (int64_t rt = (int64_t)bx * kBQ; rt < n; rt += (int64_t)gridDim.x * kBQ) {
    const int x0 = (int)rt, x = min(x0 + w * 32 + l32, n - 1);
    const bool live = x0 + w * 32 + l32 < n;
    typename F::type qf[KS];
    {
      const T* p = qbase + row_at(a, a.ldq, h, x, D) + 8 * hf;
#pragma unroll
      for (int st = 0; st < KS; ++st) qf[st] = F::load(p + 16 * st);
    }
    const Walk<kBK> walk(a, query_of(a, x0) + off, query_of(a, min(x0 + kBQ, n) - 1) + off, kv_len);
    const Seen mine = seen_from(a, query_of(a, x) + off, kv_len);
    const Seen wf = seen_from(a, query_of(a, min(x0 + w * 32, n - 1)) + off, kv_len);
    const Seen wl = seen_from(a, query_of(a, min(x0 + w * 32 + 31, n - 1)) + off, kv_len);
    const bool idle = x0 + w * 32 >= n;
    float m = -FLT_MAX, l = 0.f;  // a finite start: a tile of scores of -inf then adds nothing
    bool met = false;
    f32x16_t o[MT];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) clear(o[mt]);
    Stage<T, D, kBK, kNT> ks, vs;
    const int nt = walk.tiles();
    auto load = [&](int t) {
      if (t >= nt) return;
      int at, end;
      walk.tile(t, &at, &end);
      ks.load(kbase, a.ldk, at, end, tid);
      vs.load(vbase, a.ldv, at, end, tid);
    };
    int row = Ti::row_of(l32, hf), col = Ti::col_of(lane);
    load(0);
    for (int t = 0; t < nt; ++t) {
      asm volatile("" : "+v"(row), "+v"(col));  // no address made from them is kept from tile to tile
      int at, end;
      walk.tile(t, &at, &end);
      __syncthreads();
      ks.template store<false>(kt, tid);
      vs.template store<false>(vt, tid);
      __syncthreads();
      load(t + 1);
      if (idle || !walk.any(t, wf, wl)) continue;
      if (walk.full(t, wf, wl)) {
        forward_step<T, D, false>(kt, vt, row, col, hf, at, mine, a.sl2, qf, m, l, o, met);
      } else {
        forward_step<T, D, true>(kt, vt, row, col, hf, at, walk.in_run(t, mine), a.sl2, qf, m, l, o, met);
      }
    }
    if (met) add_keys<T, D, false>(walk, mine, 0, nt, 1, vbase, a.ldv, hf, o);
    l = pair_sum(l);
    if (live) {
      const int64_t at = q0 * (int64_t)H + row_at(a, H, h, x, 1);
      forward_store<T, D>(a, at, hf, l, sees_any(mine), o);
      store_lse(a, at, hf, m, l, sees_any(mine));
    }
  }
}

// 16 bits: one wave's softmax runs beside its matrix products.  A step of 32 keys has two phases, pinned in
// program order (left to itself the compiler gathers the products):
//   A  the next step's scores (matrix) beside the rest of this step's exponentials (VALU) and the transposed
//      reads of v
//   B  o += V^T P^T beside the next step's row maxima, the first half of its exponentials and the reads of k
//      for the step after
// Blocks of 64 keys come through LDS, k one block ahead of v (three buffers, two).  The longest run of them of
// which all rows see everything goes so; in the others, at the window's ends, a wave does one thing after the
// other, puts masks on the scores where it has to, and leaves out the keys of which its rows see nothing.
// Blocks of 256 rows: 16384 tokens of 12 x 128 bf16, window 512, take 171 us, in blocks of 128, of which LDS leaves one a CU,
// 220.  Masks inside the pipelined steps, or two halves of a block at once at the ends, spill 100 registers and more.
// Measured: 9000 + 6143 tokens, 12 x 128 bf16, window 512, 160 us, 580 of the 1117 TFLOP/s of a large product by the pairs
// that are seen (of a tile a fifth is not): matrix cores busy 24 %, VALU 31 %; 20011 + 4097 tokens, 16 / 4 x 64 f16, window
// 1023, causal, 160 us, 610 TFLOP/s, VALU 52 %.  What is left waits: a step's products for the exponentials before them, and
// the blocks at the ends, a third of the steps there, do one thing after the other.
// The sums of v are divided by the sum of the rounded P that they were made of.  KEEP (for the backward
// pass) also adds up the unrounded P: the log-sum-exps have to be those of the fp32 probabilities.
constexpr float kLazy = 8.f;  // log2 headroom before a running maximum is raised
template <typename T, int D, int QT, int NW, bool KEEP>
__global__ void __launch_bounds__(64 * NW, 2) wa_forward16_kernel(const WaArgs a) {
  typedef Tile<T, D> Ti;
  constexpr int BK = 64, NT = 64 * NW, BQ = 32 * NW * QT;
  constexpr int CPR = Ti::CPR, ROWB = Ti::ROWB, KS = D / 16, MT = D / 32;
  constexpr int RI = NT / CPR, NL = BK / RI;     // rows a load of the block covers; loads of a thread
  constexpr int NA = KS * QT, NB = 2 * MT * QT;  // products of the two phases
  static_assert(NL >= 1, "tile shape");
  __shared__ __attribute__((aligned(16))) unsigned char kbuf[3][BK * ROWB], vbuf[2][BK * ROWB];
  __shared__ uint32_t odd_in[2][NW];  // whether a wave's share of the v in vbuf holds what is not finite
  int bx, h, bb;
  block_tile(a.cu_kv, &bx, &h, &bb);
  int q0, q_len, kv0, kv_len;
  segment(a.cu_q, bb, a.total_q, &q0, &q_len);
  segment(a.cu_kv, bb, a.total_kv, &kv0, &kv_len);
  const int H = a.Hk * a.G, n = q_len * a.G, off = kv_len - q_len;
  if (a.rest) zero_rest((T*)a.out, a.cu_q, a.total_q, bb, H, D, h * a.G, bx, gridDim.x, a.G);
  const T* kbase = (const T*)a.k + (int64_t)kv0 * a.ldk + (int64_t)h * D;
  const T* vbase = (const T*)a.v + (int64_t)kv0 * a.ldv + (int64_t)h * D;
  const float sl2 = a.sl2;

  for (int64_t rt = (int64_t)bx * BQ; rt < n; rt += (int64_t)gridDim.x * BQ) {
    int tid = threadIdx.x;
    asm volatile("" : "+v"(tid));  // nothing derived from it is kept across row tiles
    const int lane = tid & 63, l32 = lane & 31, hf = lane >> 5;
    const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int x0 = (int)rt, xw = x0 + 32 * QT * w;  // first row of the block, of the wave
    const Walk<BK> walk(a, query_of(a, x0) + off, query_of(a, min(x0 + BQ, n) - 1) + off, kv_len);
    const int nblk = walk.tiles();
    const Seen wf = seen_from(a, query_of(a, min(xw, n - 1)) + off, kv_len);
    const Seen wl = seen_from(a, query_of(a, min(xw + 32 * QT, n) - 1) + off, kv_len);
    u32x4_t qf[QT][KS];
#pragma unroll
    for (int i = 0; i < QT; ++i) {
      const int x = min(xw + 32 * i + l32, n - 1);
      const T* p = (const T*)a.q + (int64_t)q0 * a.ldq + row_at(a, a.ldq, h, x, D) + 8 * hf;
#pragma unroll
      for (int st = 0; st < KS; ++st) qf[i][st] = *(const u32x4_t*)(p + 16 * st);
    }
    float mc[QT], l[QT], lu[QT], alpha[QT];  // mc: running maxima, times sl2
    f32x16_t o[QT][MT], sa[QT], sb[QT];
#pragma unroll
    for (int i = 0; i < QT; ++i) {
      mc[i] = -FLT_MAX;
      l[i] = lu[i] = 0.f;
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) clear(o[i][mt]);
    }
    auto row_sees = [&](int i) {  // the lane's row of tile i; made anew where it is needed, not kept in between
      int x = xw + 32 * i + l32;
      asm volatile("" : "+v"(x));
      return seen_from(a, query_of(a, min(x, n - 1)) + off, kv_len);
    };
    bool met = false;  // a row of v that is not finite, in a block with masks
    if (nblk > 0) {    // uniform over the block
      const int srow = tid / CPR, sc = tid % CPR;  // staging: chunk sc of rows srow + RI * i
      const uint32_t kst = (uint32_t)(2 * a.ldk), vst = (uint32_t)(2 * a.ldv);  // row bytes
      // Block t's rows; rows past a run's last key repeat it, a block past the end is block 0: no row sees them.
      u32x4_t kr[NL], vr[NL];
      auto load = [&](const T* base, uint32_t rb, int t, u32x4_t(&r)[NL]) {
        int at, end;
        walk.tile(t < nblk ? t : 0, &at, &end);
        const char* p = (const char*)base + (int64_t)at * rb;
        const uint32_t lim = (uint32_t)min(end - 1 - at, BK - 1) * rb + 16u * sc;
        const uint32_t o0 = (uint32_t)srow * rb + 16u * sc;
#pragma unroll
        for (int i = 0; i < NL; ++i) r[i] = *(const u32x4_t*)(p + min(o0 + (uint32_t)(RI * i) * rb, lim));
      };
      int kb = 0;  // the buffer of the current block's k
      auto later = [&](int by) { return kb + by < 3 ? kb + by : kb + by - 3; };
      auto store = [&](int t) {  // v of block t + 1, k of block t + 2
#pragma unroll
        for (int i = 0; i < NL; ++i) Ti::put(vbuf[~t & 1], srow + RI * i, sc, vr[i]);
#pragma unroll
        for (int i = 0; i < NL; ++i) Ti::put(kbuf[later(2)], srow + RI * i, sc, kr[i]);
      };
      u32x4_t kf[KS], vf[2][MT], pf[QT][2];
      float pr[16 * QT];
      int kfrag = Ti::row_of(l32, hf), vfrag = Ti::col_of(lane);
      auto read_k = [&](int buf, int half, int st) { kf[st] = Ti::row_at(kbuf[buf], 32 * half, kfrag, st); };
      auto read_v = [&](int buf, int half, int x) {
        vf[x / MT][x % MT] = Ti::col_at(vbuf[buf], 32 * half, vfrag, x / MT, x % MT);
      };
      // Masks the scores of 32 keys of block t, from its key `from` on.
      auto hide = [&](f32x16_t(&s)[QT], int t, int from, const Seen(&mine)[QT]) {
        int at, end;
        walk.tile(t, &at, &end);
        const int k0 = at + from + 4 * hf;
        const bool sinks = t < walk.n1 && at + from < wl.sink;  // uniform: most tiles with masks have none
#pragma unroll
        for (int i = 0; i < QT; ++i) {
          const Seen v = walk.in_run(t, mine[i]);
          const int lo = k0 - v.lo, sink = v.sink - k0;
          const uint32_t len = v.hi - v.lo;
          if (sinks) {
#pragma unroll
            for (int j = 0; j < 16; ++j) {
              const int c = 8 * (j >> 2) + (j & 3);
              if (!((uint32_t)(lo + c) < len || c < sink)) s[i][j] = -INFINITY;
            }
          } else {
#pragma unroll
            for (int j = 0; j < 16; ++j)
              if ((uint32_t)(lo + 8 * (j >> 2) + (j & 3)) >= len) s[i][j] = -INFINITY;
          }
        }
      };
      auto exp_one = [&](const f32x16_t(&s)[QT], int e) {
        pr[e] = fast_exp2(fmaf(s[e / 16][e % 16], sl2, -mc[e / 16]));
        if (KEEP) lu[e / 16] += pr[e];
      };
      auto pack_one = [&](int x) {  // x-th of 8 QT pairs -> rounded P and the denominator
        const int i = x / 8, e = 2 * (x % 8);
        const uint32_t p = Mma<T>::pack(pr[2 * x], pr[2 * x + 1]);
        pf[i][e / 8][(e / 2) % 4] = p;
        l[i] = Mma<T>::add2(p, l[i]);
      };
      auto max_part = [&](const f32x16_t(&s)[QT], int i, int part, float mx) {
#pragma unroll
        for (int j = 4 * part; j < 4 * part + 4; ++j) mx = fmaxf(mx, s[i][j]);
        return mx;
      };
      // Raises the running maxima of row tile i where a score exceeds one by more than 2^kLazy: those alone, so that
      // a row's bits do not depend on the scores of the rows beside it.  (The others' as -inf: with the comparison kept for
      // a selection, 29 registers spill where KEEP has 64 dimensions.)
      auto raise = [&](int i, float mx) {
        mx *= sl2;
        mx = mx > mc[i] + kLazy ? mx : -INFINITY;
        const bool up = __builtin_amdgcn_ballot_w64(mx > mc[i]) != 0;
        if (up) {
          const float mn = fmaxf(mc[i], mx);
          alpha[i] = fast_exp2(mc[i] - mn);
          mc[i] = mn;
          if (KEEP) lu[i] *= alpha[i];  // before the next exponentials are added to it
        }
        return up;
      };
      auto rescale = [&](int i) {
        l[i] *= alpha[i];
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
          for (int j = 0; j < 16; ++j) o[i][mt][j] *= alpha[i];
      };
      auto qk = [&](int x, f32x16_t(&s)[QT]) {
        const int st = x / QT, i = x % QT;
        if (st == 0) clear(s[i]);
        Mma<T>::run(kf[st], qf[i][st], s[i]);
      };
      auto pv = [&](int x) {
        const int g = x / (MT * QT), mt = (x / QT) % MT, i = x % QT;
        Mma<T>::run(vf[g][mt], pf[i][g], o[i][mt]);
      };
      // One step of the run: the scores of cur, half exponentiated, to the sums, beside those of nxt, whose k is
      // in kf; then the k of half khalf of buffer kbn.
      auto step = [&](f32x16_t(&cur)[QT], f32x16_t(&nxt)[QT], int t, int vhalf, int kbn, int khalf, auto stage) {
        constexpr bool STAGE = decltype(stage)::value;
        constexpr int EA = (8 * QT + NA - 1) / NA;    // exponentials and packed pairs per A group
        constexpr int VA = (2 * MT + NA - 1) / NA;    // v reads per A group
#pragma unroll
        for (int x = 0; x < NA; ++x) {
          qk(x, nxt);
#pragma unroll
          for (int y = 0; y < VA; ++y)
            if (x * VA + y < 2 * MT) read_v(t & 1, vhalf, x * VA + y);
#pragma unroll
          for (int y = 0; y < EA; ++y)
            if (x * EA + y < 8 * QT) exp_one(cur, 8 * QT + x * EA + y);
#pragma unroll
          for (int y = 0; y < EA; ++y)
            if (x * EA + y < 8 * QT) pack_one(x * EA + y);  // those made longest ago first
          __builtin_amdgcn_sched_barrier(0);
        }
        constexpr int KB = (KS + NB - 1) / NB;
        constexpr int M0 = NB / 8 > 0 ? NB / 8 : 1;  // groups before the row maxima (matrix latency)
        constexpr int MG = NB / 4;                   // groups of the row maxima
        constexpr int E0 = M0 + MG;
        constexpr int EB = (8 * QT + NB - E0 - 1) / (NB - E0);
        float mx[QT];
#pragma unroll
        for (int x = 0; x < E0; ++x) {
          pv(x);
#pragma unroll
          for (int y = 0; y < KB; ++y)
            if (x * KB + y < KS) read_k(kbn, khalf, x * KB + y);
          if (x == M0) {
#pragma unroll
            for (int i = 0; i < QT; ++i) mx[i] = nxt[i][0];
          }
          if (x >= M0) {
#pragma unroll
            for (int y = (x - M0) * 4 * QT / MG; y < (x - M0 + 1) * 4 * QT / MG; ++y)
              mx[y / 4] = max_part(nxt, y / 4, y % 4, mx[y / 4]);
          }
          __builtin_amdgcn_sched_barrier(0);
        }
        bool up[QT];
#pragma unroll
        for (int i = 0; i < QT; ++i) up[i] = raise(i, pair_max(mx[i]));
#pragma unroll
        for (int x = E0; x < NB; ++x) {
          pv(x);
#pragma unroll
          for (int y = 0; y < KB; ++y)
            if (x * KB + y < KS) read_k(kbn, khalf, x * KB + y);
#pragma unroll
          for (int y = 0; y < EB; ++y)
            if ((x - E0) * EB + y < 8 * QT) exp_one(nxt, (x - E0) * EB + y);
          if (STAGE && x == NB - NB / 4) store(t);
          __builtin_amdgcn_sched_barrier(0);
        }
#pragma unroll
        for (int i = 0; i < QT; ++i)
          if (up[i]) rescale(i);
      };
      // Scores of half `half` of the k in kbuf[b], and the maxima.
      auto scores = [&](f32x16_t(&s)[QT], int b, int half) {
#pragma unroll
        for (int st = 0; st < KS; ++st) read_k(b, half, st);
#pragma unroll
        for (int x = 0; x < NA; ++x) qk(x, s);
      };
      auto maxima = [&](f32x16_t(&s)[QT]) {
#pragma unroll
        for (int i = 0; i < QT; ++i) {
          float mx = s[i][0];
#pragma unroll
          for (int part = 0; part < 4; ++part) mx = max_part(s, i, part, mx);
          if (raise(i, pair_max(mx))) rescale(i);
        }
      };
      // The rest of a step whose first `done` exponentials are made; oddities: masked, and its v is not all finite.
      auto finish = [&](f32x16_t(&s)[QT], int t, int vhalf, int done, bool oddities) {
#pragma unroll
        for (int x = 0; x < 2 * MT; ++x) read_v(t & 1, vhalf, x);
#pragma unroll
        for (int e = 0; e < 16 * QT; ++e)
          if (e >= done) exp_one(s, e);
#pragma unroll
        for (int x = 0; x < 8 * QT; ++x) pack_one(x);
        if (oddities) {
          met = true;
#pragma unroll
          for (int x = 0; x < 2 * MT; ++x) vf[x / MT][x % MT] = finite<T>(vf[x / MT][x % MT]);
        }
#pragma unroll
        for (int x = 0; x < NB; ++x) pv(x);
      };
      auto fetch = [&](int t) {  // into registers, while block t is at work
        load(vbase, vst, t + 1, vr);
        load(kbase, kst, t + 2, kr);
      };
      auto next = [&]() {
        __syncthreads();
        kb = later(1);
      };
      auto check = [&](int t) {  // the v of block t, in vr
        uint32_t bad = 0;
#pragma unroll
        for (int i = 0; i < NL; ++i) bad |= odd<T>(vr[i]);
        const bool any = __builtin_amdgcn_ballot_w64(bad != 0) != 0;
        if (lane == 0) odd_in[t & 1][w] = any;
      };
      auto edges = [&](int t, int stop) __attribute__((always_inline)) {  // blocks t .. stop - 1, one thing after the other
        if (t >= stop) return;
        Seen mine[QT];
#pragma unroll
        for (int i = 0; i < QT; ++i) mine[i] = row_sees(i);
        for (; t < stop; ++t) {
          fetch(t);
          uint32_t bad = 0;
#pragma unroll
          for (int x = 0; x < NW; ++x) bad |= odd_in[t & 1][x];
          bad = __builtin_amdgcn_readfirstlane(bad);
#pragma unroll 1
          for (int half = 0; half < 2; ++half) {
            if (xw >= n || !walk.any(t, wf, wl, 32 * half, 32)) continue;
            const bool masked = !walk.full(t, wf, wl);
            scores(sa, kb, half);
            if (masked) hide(sa, t, 32 * half, mine);
            maxima(sa);
            finish(sa, t, half, 0, masked && bad);
          }
          check(t + 1);
          store(t);
          next();
        }
      };
      int from, to;
      walk.longest(&from, &to);
      {
        u32x4_t k1[NL];
        load(kbase, kst, 0, kr);
        load(vbase, vst, 0, vr);
        load(kbase, kst, 1, k1);
#pragma unroll
        for (int i = 0; i < NL; ++i) {
          Ti::put(kbuf[0], srow + RI * i, sc, kr[i]);
          Ti::put(vbuf[0], srow + RI * i, sc, vr[i]);
          Ti::put(kbuf[1], srow + RI * i, sc, k1[i]);
        }
        check(0);
      }
      __syncthreads();
      edges(0, from);
      if (from < to) {
        scores(sa, kb, 0);
        maxima(sa);
#pragma unroll
        for (int e = 0; e < 8 * QT; ++e) exp_one(sa, e);
#pragma unroll
        for (int st = 0; st < KS; ++st) read_k(kb, 1, st);
        for (int t = from; t < to - 1; ++t) {
          asm volatile("" : "+v"(kfrag), "+v"(vfrag));  // no address made from them is kept from block to block
          fetch(t);
          step(sa, sb, t, 0, later(1), 0, std::false_type());
          step(sb, sa, t, 1, later(1), 1, std::true_type());
          next();
        }
        fetch(to - 1);
        step(sa, sb, to - 1, 0, kb, 1, std::false_type());
        finish(sb, to - 1, 1, 8 * QT, false);
        check(to);
        store(to - 1);
        next();
        edges(to, nblk);
      }
    }
#pragma unroll
    for (int i = 0; i < QT; ++i) {
      const Seen mine = row_sees(i);
      if (met) add_keys<T, D, false>(walk, mine, 0, nblk, 1, vbase, a.ldv, hf, o[i]);
      const int x = xw + 32 * i + l32;
      l[i] = pair_sum(l[i]);
      if (KEEP) lu[i] = pair_sum(lu[i]);
      if (x < n) {
        const int64_t at = q0 * (int64_t)H + row_at(a, H, h, x, 1);
        forward_store<T, D>(a, at, hf, l[i], sees_any(mine), o[i]);
        if (KEEP) store_lse(a, at, hf, mc[i], lu[i], sees_any(mine));
      }
    }
    __syncthreads();  // the next row tile of this block stages over these buffers
  }
}

// Small grids: a block owns 32 rows, and its waves, and the blocks of a.splits parts, share out their key
// tiles.  Each wave brings its own tiles through its own piece of LDS, so none waits for another until
// the end, where their maxima, denominators and sums are joined.  Bound by latency: a wave's tile is loaded, brought
// through LDS and multiplied before the next.  One token each on 33 to 20011 keys (16 / 4 x 128 bf16, window 4095, 53 MB):
// 17 us, 3.3 TB/s, and 4 for the join; 311 + 1 + 150 tokens of 8 x 64 fp32 12 us.
__device__ __forceinline__ float* part_sums(const WaArgs& a, int sp, int64_t at, int D) {
  return a.part + ((int64_t)sp * a.total_q * a.Hk * a.G + at) * D;
}
__device__ __forceinline__ float2* part_stat(const WaArgs& a, int sp, int64_t at, int D) {
  return (float2*)part_sums(a, a.splits, 0, D) + (int64_t)sp * a.total_q * a.Hk * a.G + at;
}

template <typename T, int D>
__global__ void __launch_bounds__(kNT, D == 64 || sizeof(T) == 2 ? 2 : 1) wa_few_kernel(const WaArgs a) {
  typedef Frag<T> F;
  typedef Tile<T, D> Ti;
  constexpr int KS = D / 16, MT = D / 32, NW = kNT / 64;
  constexpr int TB = kBK * Ti::ROWB;
  constexpr int LB = NW * 2 * TB > 2 * MT * 4096 ? NW * 2 * TB : 2 * MT * 4096;  // the joined sums meet there too
  __shared__ __attribute__((aligned(16))) unsigned char lds[LB];
  __shared__ float sm[NW][32], sl[NW][32];
  int bx, h, bb;
  block_tile(a.cu_kv, &bx, &h, &bb);
  int q0, q_len, kv0, kv_len;
  segment(a.cu_q, bb, a.total_q, &q0, &q_len);
  segment(a.cu_kv, bb, a.total_kv, &kv0, &kv_len);
  const int lane = threadIdx.x & 63, l32 = lane & 31, hf = lane >> 5;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int sp = bx % a.splits, tile = bx / a.splits, tiles = gridDim.x / a.splits;
  const int H = a.Hk * a.G, n = q_len * a.G, off = kv_len - q_len;
  if (a.rest && sp == 0) zero_rest((T*)a.out, a.cu_q, a.total_q, bb, H, D, h * a.G, tile, tiles, a.G);
  const T* qbase = (const T*)a.q + (int64_t)q0 * a.ldq;
  const T* kbase = (const T*)a.k + (int64_t)kv0 * a.ldk + (int64_t)h * D;
  const T* vbase = (const T*)a.v + (int64_t)kv0 * a.ldv + (int64_t)h * D;
  unsigned char *kt = lds + w * 2 * TB, *vt = kt + TB;

  for (int64_t rt = (int64_t)tile * 32; rt < n; rt += (int64_t)tiles * 32) {
    const int x0 = (int)rt, x = min(x0 + l32, n - 1);
    typename F::type qf[KS];
    {
      const T* p = qbase + row_at(a, a.ldq, h, x, D) + 8 * hf;
#pragma unroll
      for (int st = 0; st < KS; ++st) qf[st] = F::load(p + 16 * st);
    }
    const Walk<kBK> walk(a, query_of(a, x0) + off, query_of(a, min(x0 + 32, n) - 1) + off, kv_len);
    const Seen mine = seen_from(a, query_of(a, x) + off, kv_len);
    float m = -FLT_MAX, l = 0.f;
    bool met = false;
    f32x16_t o[MT];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) clear(o[mt]);
    Stage<T, D, kBK, 64> ks, vs;
    const int nt = walk.tiles(), per = (nt + a.splits - 1) / a.splits;
    const int stop = min(nt, (sp + 1) * per);
    auto load = [&](int t) {
      if (t >= stop) return;
      int at, end;
      walk.tile(t, &at, &end);
      ks.load(kbase, a.ldk, at, end, lane);
      vs.load(vbase, a.ldv, at, end, lane);
    };
    // Whether there are registers for the next tile's rows.  (us, with / without: 16 x 64 bf16, 2048 tokens 20.6 / 21.8;
    // 12 x 128 36.9 / 35.1; one token on 33 to 20011 keys, 16 / 4 x 64 fp32 27.1 / 24.9.)
    constexpr bool AHEAD = sizeof(T) == 2 && D == 64;
    int t = sp * per + w, row = Ti::row_of(l32, hf), col = Ti::col_of(lane), from, to;
    walk.longest(&from, &to);
    if (AHEAD) load(t);
    // One loop for the tiles with masks and one for those without: with both in one, the registers of its two arms
    // do not fit.
    auto tiles = [&](int end_t, auto masked) __attribute__((always_inline)) {
      for (; t < end_t; t += NW) {
        asm volatile("" : "+v"(row), "+v"(col));  // no address made from them is kept from tile to tile
        if (!AHEAD) load(t);
        int at, end;
        walk.tile(t, &at, &end);
        // A wave's LDS operations are carried out in order; the compiler has to keep that order.
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        ks.template store<false>(kt, lane);
        vs.template store<false>(vt, lane);
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        if (AHEAD) load(t + NW);
        constexpr bool MASK = decltype(masked)::value;
        forward_step<T, D, MASK>(kt, vt, row, col, hf, at, MASK ? walk.in_run(t, mine) : mine, a.sl2, qf, m, l, o, met);
      }
    };
    tiles(min(from, stop), std::true_type());
    tiles(min(to, stop), std::false_type());
    tiles(stop, std::true_type());
    if (met) add_keys<T, D, false>(walk, mine, sp * per + w, stop, NW, vbase, a.ldv, hf, o);
    l = pair_sum(l);
    if (hf == 0) {
      sm[w][l32] = m;
      sl[w][l32] = l;
    }
    __syncthreads();  // every wave has left its tiles
    const float own = m;
    m = sm[0][l32];
#pragma unroll
    for (int y = 1; y < NW; ++y) m = fmaxf(m, sm[y][l32]);
    l = 0.f;
#pragma unroll
    for (int y = 0; y < NW; ++y) l = fmaf(sl[y][l32], fast_exp2(sm[y][l32] - m), l);
    const float f = fast_exp2(own - m);
#pragma unroll
    for (int mt = 0; mt < MT; ++mt)
#pragma unroll
      for (int j = 0; j < 16; ++j) o[mt][j] *= f;
    join_waves<MT>((float*)lds, w, lane, o);
    if (w != 0 || x0 + l32 >= n) continue;
    const int64_t at = q0 * (int64_t)H + row_at(a, H, h, x, 1);
    if (a.splits == 1) {
      forward_store<T, D>(a, at, hf, l, sees_any(mine), o);
      store_lse(a, at, hf, m, l, sees_any(mine));
    } else {
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) store_dims(part_sums(a, sp, at, D) + 32 * mt, hf, o[mt], 1.f);
      // A part without a weight of a row that sees a key has its maximum at -inf: the join tells such a row by it.
      if (hf == 0) *part_stat(a, sp, at, D) = make_float2(l == 0.f && sees_any(mine) ? -INFINITY : m, l);
    }
  }
}

// Joins the parts of the keys: one wave for a (query, head), D / 64 dims a lane.  Rows outside every
// sequence have no parts.
template <typename T, int D>
__global__ void __launch_bounds__(kNT) wa_join_kernel(const WaArgs a, int32_t B) {
  const int H = a.Hk * a.G;
  const int64_t at = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (at >= a.total_q * H) return;
  const int lane = threadIdx.x & 63;
  const int64_t row = at / H;
  bool in = false;
  for (int b = lane; b < B; b += 64) {
    int q0, ql;
    segment(a.cu_q, b, a.total_q, &q0, &ql);
    in |= row >= q0 && row < (int64_t)q0 + ql;
  }
  if (__builtin_amdgcn_ballot_w64(in) == 0) return;
  float m = -FLT_MAX, l = 0.f, o[D / 64] = {};
  bool some = false;
  for (int p = lane; p < a.splits; p += 64) m = fmaxf(m, part_stat(a, p, at, D)->x);
  for (int off = 32; off > 0; off >>= 1) m = fmaxf(m, __shfl_xor(m, off, 64));
#pragma unroll 4
  for (int p = 0; p < a.splits; ++p) {  // independent loads, one order of the sums
    const float2 st = *part_stat(a, p, at, D);
    const float* po = part_sums(a, p, at, D);
    const float f = fast_exp2(st.x - m);
    some |= st.x == -INFINITY;
    l = fmaf(st.y, f, l);
#pragma unroll
    for (int e = 0; e < D / 64; ++e) o[e] = fmaf(po[lane + 64 * e], f, o[e]);
  }
  const float inv = inverse(l, some);
#pragma unroll
  for (int e = 0; e < D / 64; ++e) {
    const int64_t p = at * D + lane + 64 * e;
    const float y = o[e] * inv;
    ((T*)a.out)[p] = (T)y;
    if (sizeof(T) == 2 && a.lo) ((T*)a.lo)[p] = (T)(y - (float)(T)y);
  }
  if (a.lse && lane == 0) a.lse[at] = row_lse(m, l, some);
}

// ------------------------------------------------------------------------------- backward
// Both gradient kernels: a block's waves own 32 rows (keys) each and share the tiles of the other side,
// through two buffers in LDS; or, where that leaves CUs idle (SHARE), all own the same 32 and take the
// tiles in turn, each through its own piece of LDS, and their sums are joined at the end.
template <bool SHARE>
__device__ __forceinline__ void tile_sync() {
  if (SHARE) __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  else __syncthreads();
}

// dq of 128 (32) rows, and r = do . out of each, which dk / dv read after it; out with what its rounding left:
// dS = P (dP - r) cancels where one key has most of a row, and out's rounding would be most of what is left.
// 15143 tokens of 12 x 128 bf16, window 256: 182 us, 500 MB to the L2s and 3.2 TB/s with its writes, matrix cores busy 18 %, VALU 27 %,
// waves waiting 47 %: two of 256 registers a SIMD (15 spilled), each with its products and its exponentials in turn.  r in a
// kernel of its own: 30 us less here, 25 there, and a launch more.
template <typename T, int D, bool SHARE>
__global__ void __launch_bounds__(kNT, D == 64 || (sizeof(T) == 2 && !SHARE) ? 2 : 1) wa_dq_kernel(const WaArgs a) {
  typedef Frag<T> F;
  typedef typename F::type Fr;
  typedef Tile<T, D> Ti;
  constexpr int KS = D / 16, MT = D / 32;
  constexpr int TB = kBK * Ti::ROWB, ROWS = SHARE ? 32 : kBQ, NT = SHARE ? 64 : kNT, BUFS = SHARE ? 4 : 2;
  constexpr int LB = !SHARE || BUFS * 2 * TB > 2 * MT * 4096 ? BUFS * 2 * TB : 2 * MT * 4096;
  __shared__ __attribute__((aligned(16))) unsigned char lds[LB];
  int bx, h, bb;
  block_tile(a.cu_kv, &bx, &h, &bb);
  int q0, q_len, kv0, kv_len;
  segment(a.cu_q, bb, a.total_q, &q0, &q_len);
  segment(a.cu_kv, bb, a.total_kv, &kv0, &kv_len);
  const int lane = threadIdx.x & 63, l32 = lane & 31, hf = lane >> 5;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), tid = SHARE ? lane : threadIdx.x;
  const int H = a.Hk * a.G, n = q_len * a.G, off = kv_len - q_len;
  if (a.rest) zero_rest((T*)a.dq, a.cu_q, a.total_q, bb, H, D, h * a.G, bx, gridDim.x, a.G);
  const T* kbase = (const T*)a.k + (int64_t)kv0 * a.ldk + (int64_t)h * D;
  const T* vbase = (const T*)a.v + (int64_t)kv0 * a.ldv + (int64_t)h * D;
  const float scale = a.sl2 / kLog2e;

  for (int64_t rt = (int64_t)bx * ROWS; rt < n; rt += (int64_t)gridDim.x * ROWS) {
    const int x0 = (int)rt, xw = SHARE ? x0 : x0 + w * 32, x = min(xw + l32, n - 1);
    const int64_t at = q0 * (int64_t)H + row_at(a, H, h, x, 1);
    Fr qf[KS], df[KS];
    {
      const T* p = (const T*)a.q + (int64_t)q0 * a.ldq + row_at(a, a.ldq, h, x, D) + 8 * hf;
      const T* d = (const T*)a.dout + at * D + 8 * hf;
#pragma unroll
      for (int st = 0; st < KS; ++st) {
        qf[st] = F::load(p + 16 * st);
        df[st] = F::load(d + 16 * st);
      }
    }
    float r = 0.f;
    {
      const T* o = (const T*)a.out + at * D + 8 * hf;
      const T* lo = (const T*)a.lo + at * D + 8 * hf;
#pragma unroll
      for (int st = 0; st < KS; ++st) {
        const Fr of = F::load(o + 16 * st), lf = F::load((sizeof(T) == 2 ? lo : o) + 16 * st);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          float y = (float)((const T*)&of)[e];
          if (sizeof(T) == 2) y += (float)((const T*)&lf)[e];
          r = fmaf((float)((const T*)&df[st])[e], y, r);
        }
      }
      r = pair_sum(r);
      if (hf == 0 && xw + l32 < n && (!SHARE || w == 0)) a.r[at] = r;
    }
    const float lse = a.lse[at];
    const Walk<kBK> walk(a, query_of(a, x0) + off, query_of(a, min(x0 + ROWS, n) - 1) + off, kv_len);
    const Seen mine = seen_from(a, query_of(a, x) + off, kv_len);
    const Seen wf = seen_from(a, query_of(a, min(xw, n - 1)) + off, kv_len);
    const Seen wl = seen_from(a, query_of(a, min(xw + 31, n - 1)) + off, kv_len);
    const bool idle = xw >= n;
    f32x16_t acc[MT];
    bool met = false;
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) clear(acc[mt]);
    Stage<T, D, kBK, NT> ks, vs;
    const int nt = walk.tiles();
    auto load = [&](int t) {
      if (t >= nt) return;
      int k0, end;
      walk.tile(t, &k0, &end);
      ks.load(kbase, a.ldk, k0, end, tid);
      vs.load(vbase, a.ldv, k0, end, tid);
    };
    constexpr int STEP = SHARE ? 4 : 1;
    // The next tile's rows on their way.  With SHARE the registers for them spill: both gradients, 1000 tokens of 12 x 128
    // bf16 78 us, 73 without; 8 / 2 x 64 fp32 149, 117.
    constexpr bool AHEAD = !SHARE;
    int row = Ti::row_of(l32, hf), col = Ti::col_of(lane);
    auto step = [&](const unsigned char* kt, const unsigned char* vt, auto masked, int k0, const Seen& s) __attribute__((always_inline)) {
      constexpr bool MASK = decltype(masked)::value;
      f32x16_t c, dp;
      clear(c);
      clear(dp);
#pragma unroll
      for (int st = 0; st < KS; ++st) {
        F::mma(Ti::row_at(kt, 0, row, st), qf[st], c);
        F::mma(Ti::row_at(vt, 0, row, st), df[st], dp);
      }
      float d[16];
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        d[j] = fast_exp2(fmaf(c[j], a.sl2, -lse)) * (dp[j] - r);
        if (MASK && !sees(s, k0 + 8 * (j >> 2) + 4 * hf + (j & 3))) d[j] = 0.f;
      }
      const Fr f[2] = {F::pack(d), F::pack(d + 8)};
      add_rows<T, D, MASK>(kt, col, f, acc, met);
    };
    int t = SHARE ? w : 0, buf = 0, from, to;
    walk.longest(&from, &to);
    if (AHEAD) load(t);
    // As in wa_few_kernel: tiles with masks, those without, and again with masks.
    auto tiles = [&](int stop, auto masked) __attribute__((always_inline)) {
      for (; t < stop; t += STEP, buf ^= 1) {
        asm volatile("" : "+v"(row), "+v"(col));  // no address made from them is kept from tile to tile
        unsigned char *kt = lds + (SHARE ? w : buf) * 2 * TB, *vt = kt + TB;
        if (!AHEAD) load(t);
        if (SHARE) tile_sync<SHARE>();
        ks.template store<false>(kt, tid);
        vs.template store<false>(vt, tid);
        tile_sync<SHARE>();
        if (AHEAD) load(t + STEP);
        int k0, end;
        walk.tile(t, &k0, &end);
        if (idle || (decltype(masked)::value && !walk.any(t, wf, wl))) continue;
        step(kt, vt, masked, k0, decltype(masked)::value ? walk.in_run(t, mine) : mine);
      }
    };
    tiles(from, std::true_type());
    tiles(to, std::false_type());
    tiles(nt, std::true_type());
    if (met) add_keys<T, D, true>(walk, mine, SHARE ? w : 0, nt, STEP, kbase, a.ldk, hf, acc);
    if (SHARE) join_waves<MT>((float*)lds, w, lane, acc);
    else __syncthreads();  // the next tile's rows go into these buffers
    if (xw + l32 < n && (!SHARE || w == 0)) {
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) store_dims((T*)a.dq + at * D + 32 * mt, hf, acc[mt], scale);
    }
  }
}

// The rows that see key k: one run [lo, hi).
struct Rows {
  int lo, hi;
};
__device__ __forceinline__ Rows rows_of(const WaArgs& a, int k, int off, int q_len) {
  const bool sink = k < a.sinks;
  int64_t lo = a.causal ? (int64_t)k - off : sink ? 0 : (int64_t)k - a.window - off;
  int64_t hi = sink ? q_len : (int64_t)k + a.window - off + 1;
  lo = min<int64_t>(max<int64_t>(lo, 0), q_len);
  hi = min<int64_t>(max<int64_t>(hi, lo), q_len);
  return {(int)lo * a.G, (int)hi * a.G};
}

// The rows that see any of the keys first .. last, and those, [lo, hi), that see each of them.  Along the keys both
// bounds grow, but for the sinks'.
struct Spans {
  Rows any;
  int lo, hi;
};
__device__ __forceinline__ Spans spans_of(const WaArgs& a, int first, int last, int off, int q_len) {
  const Rows f = rows_of(a, first, off, q_len), l = rows_of(a, last, off, q_len);
  const Rows m = first < a.sinks && last >= a.sinks ? rows_of(a, a.sinks, off, q_len) : f;
  Spans s;
  s.any = {min(f.lo, l.lo), max(max(f.hi, l.hi), f.lo)};
  s.lo = max(l.lo, f.lo);
  s.hi = min(min(f.hi, l.hi), m.hi);
  return s;
}

// dk and dv of 128 (32) keys of a key head, over the rows of all its query heads.  Every row sees the sinks: where
// that is many times what sees another key, they are left to SINKS blocks (32 keys, and of their rows one of
// sink_parts parts; 15143 tokens, 12 x 128 bf16, window 256, 16 sinks: the first tile's blocks took 28 times
// the others' rows and 970 of the step's 1374 us; now 32 and 4 for adding up the parts).  Spills up to 18 registers at
// D = 64 and two waves a SIMD, up to 27 in fp32 at D = 128 and one.
template <typename T, int D, bool SHARE, bool SINKS>
__global__ void __launch_bounds__(kNT, D == 64 && (sizeof(T) == 2 || SHARE) ? 2 : 1) wa_dkv_kernel(const WaArgs a) {
  static_assert(SHARE || !SINKS, "sinks: 32 keys");
  typedef Frag<T> F;
  typedef typename F::type Fr;
  typedef Tile<T, D> Ti;
  constexpr int BQ = 32;
  constexpr int KS = D / 16, MT = D / 32;
  constexpr int ROWS = SHARE ? 32 : 128, NT = SHARE ? 64 : kNT, BUFS = SHARE ? 4 : 2;
  constexpr int TB = BQ * Ti::ROWB;
  constexpr int LB = !SHARE || BUFS * 2 * TB > 2 * MT * 4096 ? BUFS * 2 * TB : 2 * MT * 4096;
  constexpr int NL = BQ * Ti::CPR / NT, EPC = 16 / sizeof(T);
  __shared__ __attribute__((aligned(16))) unsigned char lds[LB];
  __shared__ __attribute__((aligned(16))) float stats[BUFS][2][BQ];
  int bx, h, bb;
  block_tile(a.cu_q, &bx, &h, &bb);
  int q0, q_len, kv0, kv_len;
  segment(a.cu_q, bb, a.total_q, &q0, &q_len);
  segment(a.cu_kv, bb, a.total_kv, &kv0, &kv_len);
  const int lane = threadIdx.x & 63, l32 = lane & 31, hf = lane >> 5;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), tid = SHARE ? lane : threadIdx.x;
  const int H = a.Hk * a.G, off = kv_len - q_len;
  if (a.rest && !SINKS) {
    zero_rest((T*)a.dk, a.cu_kv, a.total_kv, bb, a.Hk, D, h, bx, gridDim.x, 1);
    zero_rest((T*)a.dv, a.cu_kv, a.total_kv, bb, a.Hk, D, h, bx, gridDim.x, 1);
  }
  const int part = SINKS ? bx % a.sink_parts : 0, bt = SINKS ? bx / a.sink_parts : bx;
  const int keys = SINKS ? min(kv_len, a.sinks) : kv_len;  // of this grid
  const int tiles = SINKS ? a.sink_keys / ROWS : gridDim.x;
  const int first = a.own_sinks && !SINKS ? a.sinks : 0;
  const T* qbase = (const T*)a.q + (int64_t)q0 * a.ldq;
  const T* dbase = (const T*)a.dout + (int64_t)q0 * H * D;
  const float scale = a.sl2 / kLog2e;

  for (int64_t ktile = (int64_t)bt * ROWS; ktile < keys; ktile += (int64_t)tiles * ROWS) {
    if (ktile + ROWS <= first) continue;
    const int k0 = max((int)ktile, first), kw = SHARE ? (int)ktile : (int)ktile + w * 32, ki = min(kw + l32, keys - 1);
    const int64_t krow = kv0 + ki;
    Fr kf[KS], vf[KS];
    {
      const T* p = (const T*)a.k + krow * a.ldk + (int64_t)h * D + 8 * hf;
      const T* d = (const T*)a.v + krow * a.ldv + (int64_t)h * D + 8 * hf;
#pragma unroll
      for (int st = 0; st < KS; ++st) {
        kf[st] = F::load(p + 16 * st);
        vf[st] = F::load(d + 16 * st);
      }
    }
    Spans all = spans_of(a, k0, (int)min(ktile + ROWS, (int64_t)keys) - 1, off, q_len);
    Spans own = spans_of(a, min(max(kw, first), keys - 1), min(max(kw + 31, first), keys - 1), off, q_len);
    Rows run = all.any;
    const Rows wrun = own.any;
    Rows mine = rows_of(a, ki, off, q_len);
    if (ki < first) mine.hi = mine.lo;  // another grid's
    if (kw < first) own.hi = own.lo;
    if (k0 > ktile) all.hi = all.lo;  // a tile with keys of the other grid
    const bool idle = kw >= keys || kw + 32 <= first;
    if (SINKS) {  // a part of the rows, in whole tiles for the four waves
      const int per = ((run.hi - run.lo + a.sink_parts - 1) / a.sink_parts + 127) / 128 * 128;
      run.lo = (int)min((int64_t)run.lo + (int64_t)part * per, (int64_t)run.hi);
      run.hi = (int)min((int64_t)run.lo + per, (int64_t)run.hi);
    }
    f32x16_t dk[MT], dv[MT];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
      clear(dk[mt]);
      clear(dv[mt]);
    }
    bool met = false;
    u32x4_t qr[NL], dr[NL];
    float sv = 0.f;
    constexpr int STEP = SHARE ? 4 * BQ : BQ;
    constexpr bool AHEAD = !SHARE;  // as there
    // Rows past the last one repeat it: they are masked.
    auto load = [&](int xb) {
      if (xb >= run.hi) return;
#pragma unroll
      for (int i = 0; i < NL; ++i) {
        const int id = tid + NT * i, x = min(xb + id / Ti::CPR, run.hi - 1), c = id % Ti::CPR * EPC;
        const int qi = query_of(a, x);
        const int64_t hd = (int64_t)(h * a.G + x - qi * a.G) * D + c;
        qr[i] = *(const u32x4_t*)(qbase + qi * a.ldq + hd);
        dr[i] = *(const u32x4_t*)(dbase + (int64_t)qi * H * D + hd);
      }
      if (tid < 64) {
        const int x = min(xb + (tid & 31), run.hi - 1);
        const int64_t at = q0 * (int64_t)H + row_at(a, H, h, x, 1);
        sv = tid < 32 ? a.lse[at] : a.r[at];
      }
    };
    int row = Ti::row_of(l32, hf), col = Ti::col_of(lane);
    auto step = [&](const unsigned char* qt, const unsigned char* dt, const float(*st2)[BQ], int xb, auto masked) __attribute__((always_inline)) {
      constexpr bool MASK = decltype(masked)::value;
      f32x16_t c, dp;
      clear(c);
      clear(dp);
#pragma unroll
      for (int st = 0; st < KS; ++st) {
        F::mma(Ti::row_at(qt, 0, row, st), kf[st], c);
        F::mma(Ti::row_at(dt, 0, row, st), vf[st], dp);
      }
      auto see = [&](int e) { return (uint32_t)(xb + e - mine.lo) < (uint32_t)(mine.hi - mine.lo); };
      float p[16], d[16];
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        const int e = 8 * (j >> 2) + 4 * hf + (j & 3);
        p[j] = fast_exp2(fmaf(c[j], a.sl2, -st2[0][e]));
        d[j] = p[j] * (dp[j] - st2[1][e]);
        if (MASK && !see(e)) p[j] = d[j] = 0.f;
      }
      const Fr pf[2] = {F::pack(p), F::pack(p + 8)};
      add_rows<T, D, MASK>(dt, col, pf, dv, met);
      const Fr df[2] = {F::pack(d), F::pack(d + 8)};
      add_rows<T, D, MASK>(qt, col, df, dk, met);
    };
    int xb = run.lo + (SHARE ? w * BQ : 0), buf = 0;
    if (AHEAD) load(xb);
    // As there: tiles with masks, those that all keys see, and again with masks.
    const int run_lo = SHARE ? own.lo : all.lo, run_hi = SHARE ? own.hi : all.hi;
    auto tiles = [&](auto masked, auto more) __attribute__((always_inline)) {
      for (; xb < run.hi && more(); xb += STEP, buf ^= 1) {
        asm volatile("" : "+v"(row), "+v"(col));
        unsigned char *qt = lds + (SHARE ? w : buf) * 2 * TB, *dt = qt + TB;
        float(*st2)[BQ] = stats[SHARE ? w : buf];
        if (!AHEAD) load(xb);
        if (SHARE) tile_sync<SHARE>();
#pragma unroll
        for (int i = 0; i < NL; ++i) {
          const int id = tid + NT * i;
          Ti::put(qt, id / Ti::CPR, id % Ti::CPR, qr[i]);
          Ti::put(dt, id / Ti::CPR, id % Ti::CPR, dr[i]);
        }
        if (tid < 64) st2[tid >> 5][tid & 31] = sv;
        tile_sync<SHARE>();
        if (AHEAD) load(xb + STEP);
        if (idle || (decltype(masked)::value && (xb >= wrun.hi || xb + BQ <= wrun.lo))) continue;
        step(qt, dt, st2, xb, masked);
      }
    };
    auto full = [&] { return xb >= run_lo && xb + BQ <= min(run_hi, run.hi); };
    tiles(std::true_type(), [&] { return !full(); });
    tiles(std::false_type(), full);
    tiles(std::true_type(), [&] { return true; });
    if (met)
      for (int x = max(wrun.lo, run.lo); x < min(wrun.hi, run.hi); ++x) {
        const bool seen = x >= mine.lo && x < mine.hi;
        add_odd<T, D, true>(qbase + row_at(a, a.ldq, h, x, D), hf, seen, dk);
        add_odd<T, D, false>(dbase + row_at(a, (int64_t)H * D, h, x, D), hf, seen, dv);
      }
    if (SHARE) {
      join_waves<MT>((float*)lds, w, lane, dk);
      join_waves<MT>((float*)lds, w, lane, dv);
    } else {
      __syncthreads();  // every wave has left the buffers
    }
    if (kw + l32 < keys && kw + l32 >= first && (!SHARE || w == 0)) {
      const int64_t at = (krow * a.Hk + h) * D;
      if constexpr (SINKS) {
        float* p = a.sink_sums + ((((int64_t)part * gridDim.z + bb) * a.Hk + h) * a.sink_keys + ki) * 2 * D;
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
          store_dims(p + 32 * mt, hf, dk[mt], 1.f);
          store_dims(p + D + 32 * mt, hf, dv[mt], 1.f);
        }
        continue;
      }
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) {
        store_dims((T*)a.dk + at + 32 * mt, hf, dk[mt], scale);
        store_dims((T*)a.dv + at + 32 * mt, hf, dv[mt], 1.f);
      }
    }
  }
}

// dk and dv of 128 keys at D = 128 in 16 bits: two waves to 32 keys.  With the sums of both gradients, k and v a wave
// has the registers of its SIMD for itself, and the matrix cores wait for its exponentials and LDS reads (16384
// tokens, 12 x 128, window 256 / 1024: 321 / 903 us).  Here one wave makes the scores, P and dv, and hands P on
// through LDS, in fp32; the other makes dP and, a tile of rows later, dS and dk.  The same products, 16 a tile for
// each, and none is made twice.  Tiles of 32 rows come through three buffers (q, read a tile later) and two.
// Measured: 274 / 692 us there (64 rows a tile, which spill 72 registers: 338 / 799); 275 for 9000 + 6143 tokens, window 256,
// matrix cores busy 15 %, VALU 39 %, waiting 41 %: a barrier a tile, and both waves of a pair wait for the longer half.
template <typename T>
__global__ void __launch_bounds__(512, 2) wa_dkv_pair_kernel(const WaArgs a) {
  constexpr int D = 128, KS = D / 16, MT = D / 32, BQ = 32, ROWS = 128;
  typedef Frag<T> F;
  typedef Tile<T, D> Ti;
  constexpr int TB = BQ * Ti::ROWB;
  static_assert(BQ * Ti::CPR == 512, "a chunk a thread");
  __shared__ __attribute__((aligned(16))) unsigned char qbuf[3][TB], dbuf[2][TB];
  __shared__ __attribute__((aligned(16))) float pbuf[2][4][16 * 64];
  __shared__ __attribute__((aligned(16))) float stats[3][2][BQ];
  int bx, h, bb;
  block_tile(a.cu_q, &bx, &h, &bb);
  int q0, q_len, kv0, kv_len;
  segment(a.cu_q, bb, a.total_q, &q0, &q_len);
  segment(a.cu_kv, bb, a.total_kv, &kv0, &kv_len);
  const int tid = threadIdx.x, lane = tid & 63, l32 = lane & 31, hf = lane >> 5;
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6), pair = w & 3;
  const bool of_k = w >= 4;  // the wave of dP and dk
  const int H = a.Hk * a.G, off = kv_len - q_len, first = a.own_sinks ? a.sinks : 0;
  if (a.rest) {
    zero_rest((T*)a.dk, a.cu_kv, a.total_kv, bb, a.Hk, D, h, bx, gridDim.x, 1);
    zero_rest((T*)a.dv, a.cu_kv, a.total_kv, bb, a.Hk, D, h, bx, gridDim.x, 1);
  }
  const T* qbase = (const T*)a.q + (int64_t)q0 * a.ldq;
  const T* dbase = (const T*)a.dout + (int64_t)q0 * H * D;
  const float scale = a.sl2 / kLog2e;

  for (int64_t ktile = (int64_t)bx * ROWS; ktile < kv_len; ktile += (int64_t)gridDim.x * ROWS) {
    if (ktile + ROWS <= first) continue;
    const int k0 = max((int)ktile, first), kw = (int)ktile + pair * 32, ki = min(kw + l32, kv_len - 1);
    const int64_t krow = kv0 + ki;
    u32x4_t kv[KS];  // k of the wave's keys, or v
    {
      const T* p = (of_k ? (const T*)a.v + krow * a.ldv : (const T*)a.k + krow * a.ldk) + (int64_t)h * D + 8 * hf;
#pragma unroll
      for (int st = 0; st < KS; ++st) kv[st] = F::load(p + 16 * st);
    }
    const Spans all = spans_of(a, k0, (int)min(ktile + ROWS, (int64_t)kv_len) - 1, off, q_len);
    Spans own = spans_of(a, min(max(kw, first), kv_len - 1), min(max(kw + 31, first), kv_len - 1), off, q_len);
    if (kw < first) own.hi = own.lo;
    Rows mine = rows_of(a, ki, off, q_len);
    if (ki < first) mine.hi = mine.lo;  // another grid's
    const Rows run = all.any;
    const bool idle = kw >= kv_len || kw + 32 <= first;
    const int nt = (run.hi - run.lo + BQ - 1) / BQ;
    f32x16_t acc[MT], dp;
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) clear(acc[mt]);
    bool met = false;
    u32x4_t qr, dr;
    float sv = 0.f;
    auto load = [&](int i) {  // rows past the last one repeat it: they are masked
      const int x = min(run.lo + BQ * i + tid / Ti::CPR, run.hi - 1), qi = query_of(a, x);
      const int64_t hd = (int64_t)(h * a.G + x - qi * a.G) * D + tid % Ti::CPR * 8;
      qr = *(const u32x4_t*)(qbase + qi * a.ldq + hd);
      dr = *(const u32x4_t*)(dbase + (int64_t)qi * H * D + hd);
      if (tid < 64) {
        const int64_t at = q0 * (int64_t)H + row_at(a, H, h, min(run.lo + BQ * i + (tid & 31), run.hi - 1), 1);
        sv = tid < 32 ? a.lse[at] : a.r[at];
      }
    };
    auto at_work = [&](int i) {
      const int xb = run.lo + BQ * i;
      return i >= 0 && i < nt && !idle && xb < own.any.hi && xb + BQ > own.any.lo;
    };
    auto masked = [&](int i) { return run.lo + BQ * i < own.lo || run.lo + BQ * i + BQ > own.hi; };
    auto see = [&](int i, int e) { return (uint32_t)(run.lo + BQ * i + e - mine.lo) < (uint32_t)(mine.hi - mine.lo); };
    int row = Ti::row_of(l32, hf), col = Ti::col_of(lane);
    // acc += rows of t weighted with s (rounded to T), what is not finite left out of tiles with masks.
    auto add = [&](const unsigned char* t, const float(&s)[16], bool mask) __attribute__((always_inline)) {
#pragma unroll
      for (int g = 0; g < 2; ++g) {
        const u32x4_t sf = F::pack(s + 8 * g);
        u32x4_t v[MT];
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) v[mt] = Ti::col_at(t, 0, col, g, mt);
        if (mask) {
          uint32_t bad = 0;
#pragma unroll
          for (int mt = 0; mt < MT; ++mt) bad |= odd<T>(v[mt]);
          if (__builtin_amdgcn_ballot_w64(bad != 0)) {
            met = true;
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) v[mt] = finite<T>(v[mt]);
          }
        }
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) F::mma(v[mt], sf, acc[mt]);
      }
    };
    if (nt > 0) load(0);
    for (int i = 0; i <= nt; ++i) {
      asm volatile("" : "+v"(row), "+v"(col));  // no address made from them is kept from tile to tile
      if (i < nt) {
        Ti::put(qbuf[i % 3], tid / Ti::CPR, tid % Ti::CPR, qr);
        Ti::put(dbuf[i & 1], tid / Ti::CPR, tid % Ti::CPR, dr);
        if (tid < 64) stats[i % 3][tid >> 5][tid & 31] = sv;
      }
      // What a buffer held before was last read one barrier ago at least: q and r of tile i - 3 and d and P of tile
      // i - 2 in step i - 2 or (P) i - 1, whose readers have passed the last barrier or will pass this one first.
      __syncthreads();
      if (i + 1 < nt) load(i + 1);
      if (!of_k) {
        if (!at_work(i)) continue;
        f32x16_t c;
        clear(c);
#pragma unroll
        for (int st = 0; st < KS; ++st) F::mma(Ti::row_at(qbuf[i % 3], 0, row, st), kv[st], c);
        const bool mask = masked(i);
        float p[16];
#pragma unroll
        for (int j = 0; j < 16; ++j) p[j] = fast_exp2(fmaf(c[j], a.sl2, -stats[i % 3][0][8 * (j >> 2) + 4 * hf + (j & 3)]));
        if (mask) {
#pragma unroll
          for (int j = 0; j < 16; ++j)
            if (!see(i, 8 * (j >> 2) + 4 * hf + (j & 3))) p[j] = 0.f;
        }
#pragma unroll
        for (int g = 0; g < 4; ++g)
          *(float4*)&pbuf[i & 1][pair][(g * 64 + lane) * 4] = make_float4(p[4 * g], p[4 * g + 1], p[4 * g + 2], p[4 * g + 3]);
        add(dbuf[i & 1], p, mask);
      } else {
        if (at_work(i - 1)) {
          const bool mask = masked(i - 1);
          float d[16];
#pragma unroll
          for (int g = 0; g < 4; ++g) {
            const float4 p = *(const float4*)&pbuf[(i - 1) & 1][pair][(g * 64 + lane) * 4];
            d[4 * g] = p.x, d[4 * g + 1] = p.y, d[4 * g + 2] = p.z, d[4 * g + 3] = p.w;
          }
#pragma unroll
          for (int j = 0; j < 16; ++j) d[j] *= dp[j] - stats[(i + 2) % 3][1][8 * (j >> 2) + 4 * hf + (j & 3)];
          if (mask) {
#pragma unroll
            for (int j = 0; j < 16; ++j)
              if (!see(i - 1, 8 * (j >> 2) + 4 * hf + (j & 3))) d[j] = 0.f;
          }
          add(qbuf[(i + 2) % 3], d, mask);
        }
        if (at_work(i)) {
          clear(dp);
#pragma unroll
          for (int st = 0; st < KS; ++st) F::mma(Ti::row_at(dbuf[i & 1], 0, row, st), kv[st], dp);
        }
      }
    }
    if (met)
      for (int x = own.any.lo; x < own.any.hi; ++x) {
        const bool seen = x >= mine.lo && x < mine.hi;
        if (of_k) add_odd<T, D, true>(qbase + row_at(a, a.ldq, h, x, D), hf, seen, acc);
        else add_odd<T, D, false>(dbase + row_at(a, (int64_t)H * D, h, x, D), hf, seen, acc);
      }
    if (kw + l32 < kv_len && kw + l32 >= first) {
      T* p = (T*)(of_k ? a.dk : a.dv) + (krow * a.Hk + h) * D;
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) store_dims(p + 32 * mt, hf, acc[mt], of_k ? scale : 1.f);
    }
    __syncthreads();  // the next keys' rows go into these buffers
  }
}

// Adds up the parts of the sinks' gradients: a block for four sinks of a key head, a wave each.
template <typename T, int D>
__global__ void __launch_bounds__(kNT) wa_sinks_kernel(const WaArgs a) {
  const int lane = threadIdx.x & 63, k = blockIdx.x * 4 + (threadIdx.x >> 6), h = blockIdx.y, bb = blockIdx.z;
  int kv0, kv_len;
  segment(a.cu_kv, bb, a.total_kv, &kv0, &kv_len);
  if (k >= min(kv_len, a.sinks)) return;
  const float scale = a.sl2 / kLog2e;
  const float* p = a.sink_sums + (((int64_t)bb * a.Hk + h) * a.sink_keys + k) * 2 * D;
  const int64_t step = (int64_t)gridDim.z * a.Hk * a.sink_keys * 2 * D, at = ((int64_t)(kv0 + k) * a.Hk + h) * D;
  float s[2 * D / 64] = {};
#pragma unroll 4
  for (int i = 0; i < a.sink_parts; ++i)
#pragma unroll
    for (int e = 0; e < 2 * D / 64; ++e) s[e] += p[i * step + lane + 64 * e];
#pragma unroll
  for (int e = 0; e < D / 64; ++e) {
    ((T*)a.dk)[at + lane + 64 * e] = (T)(s[e] * scale);
    ((T*)a.dv)[at + lane + 64 * e] = (T)s[D / 64 + e];
  }
}

// ------------------------------------------------------------------------------- host
constexpr int64_t kCUs = 256;

// Tiles of `rows` rows that the grid gives a sequence; the kernels' loops cover longer ones.
unsigned tiles_of(int64_t longest, int64_t hb, int rows) {
  return (unsigned)std::max<int64_t>(
      1, std::min<int64_t>(std::min<int64_t>((longest + rows - 1) / rows, 65535), (INT32_MAX / 1024) / hb));
}

// Blocks of the forward pass: rows of each, and the parts of their keys.
struct Plan {
  int rows, splits;  // 32: wa_few_kernel
};
constexpr int64_t kScratchInputs = 4, kScratchLeast = 64 << 20;
int64_t part_bytes(int64_t total_q, int32_t H, int32_t D) { return 4 * total_q * H * (D + 2); }
Plan wa_plan(const WindowAttnSizes& z) {
  const int64_t hb = (int64_t)z.Hk * z.B, G = z.H / z.Hk;
  const int64_t max_q = std::max<int64_t>(z.max_q, (z.total_q + z.B - 1) / z.B);
  Plan p = {z.dtype == TSC_F32 ? kBQ : kBQ16, 1};
  // Blocks of 32 rows, whose waves share their keys, while there are too few of the wide ones.  Measured, us, wide /
  // 32 rows, window 256: 12 x 128 bf16, 2048 tokens 50 / 37, 3000 42 / 53; 16 x 64, 2048 tokens 38 / 30, 3000 37 / 43.
  const int64_t wide = z.dtype != TSC_F32 && z.D == 64 ? 320 : kCUs;
  if ((int64_t)tiles_of(max_q * G, hb, kBQ) * hb >= wide) return p;
  p.rows = 32;
  const int64_t blocks = (int64_t)tiles_of(max_q * G, hb, 32) * hb;
  if (blocks >= 2 * kCUs) return p;
  // Parts of 512 keys at least, four tiles a wave.  (us, 256 / 512 / 1024: one token on 33 to 20011 keys, 16 / 4 x 128 bf16,
  // window 4095: 23.2 / 21.1 / 23.1; x 64 fp32 25.0 / 25.0 / 33.7; 1000 tokens of 8 / 2 x 64 fp32, window 256: 25 / 20 / 20.)
  const int64_t span = std::min<int64_t>(z.max_kv, (z.causal ? 1 : 2) * (int64_t)z.window + 32 + z.sinks);
  const int64_t es = z.dtype == TSC_F32 ? 4 : 2;
  const int64_t io = 2 * z.D * es * (z.total_q * z.H + z.total_kv * z.Hk);
  const int64_t room = std::max(kScratchLeast, kScratchInputs * io) / std::max<int64_t>(1, part_bytes(z.total_q, z.H, z.D));
  p.splits = (int)std::max<int64_t>(1, std::min({span / 512, 2 * kCUs / blocks, room}));
  return p;
}

// The blocks that share the rows of a tile of sinks: a block on each CU, of four waves' tiles of rows at least, in
// scratch as above; 1: sinks are keys like others, whose blocks would not have twice the rows of another's.
// (16384 tokens, 12 x 128 bf16, window 256, 4 sinks: 30 us in 21 parts, 39 in 30, 52 in 7, and 4 to 5 to add them up.)
struct SinkPlan {
  int parts, keys;
  int64_t bytes;
};
SinkPlan sink_plan(const WindowAttnSizes& z) {
  SinkPlan p = {1, 0, 0};
  const int64_t sinks = std::min<int64_t>(z.sinks, z.max_kv);
  const int64_t rows = std::min<int64_t>(z.max_q, (z.causal ? 1 : 2) * (int64_t)z.window + 32);
  if (z.B == 0 || sinks == 0 || 2 * sinks > z.max_kv || z.max_q < 2 * rows) return p;
  p.keys = (int)((sinks + 31) / 32 * 32);
  const int64_t part = (int64_t)z.B * z.Hk * p.keys * 2 * z.D * 4;
  const int64_t es = z.dtype == TSC_F32 ? 4 : 2;
  const int64_t io = 2 * z.D * es * (z.total_q * z.H + z.total_kv * z.Hk);
  const int64_t blocks = (int64_t)p.keys / 32 * z.Hk * z.B, most = (int64_t)z.max_q * (z.H / z.Hk) / 128;
  p.parts = (int)std::min({std::max<int64_t>(2, kCUs / blocks), most, std::max(kScratchLeast, kScratchInputs * io) / part});
  if (p.parts < 2) return {1, 0, 0};
  p.bytes = p.parts * part;
  return p;
}

template <typename F>
int by_type(int32_t dtype, int32_t D, F f) {
  constexpr std::integral_constant<int, 64> D64{};
  constexpr std::integral_constant<int, 128> D128{};
  auto dims = [&](auto t) { D == 64 ? f(t, D64) : f(t, D128); };
  if (dtype == TSC_BF16) dims(__bf16());
  else if (dtype == TSC_F16) dims(_Float16());
  else dims(float());
  return check_hip(hipGetLastError(), "window_attention launch");
}

WaArgs wa_args(const WindowAttnArgs& x) {
  const WindowAttnSizes& z = x.z;
  WaArgs a = {};
  a.q = x.q;
  a.k = x.k;
  a.v = x.v;
  a.ldq = x.ldq;
  a.ldk = x.ldk;
  a.ldv = x.ldv;
  a.cu_q = x.cu_q;
  a.cu_kv = x.cu_kv;
  a.total_q = z.total_q;
  a.total_kv = z.total_kv;
  a.Hk = z.Hk;
  a.G = z.H / z.Hk;
  a.shift = -1;
  for (int s = 0; s < 16; ++s)
    if (a.G == 1 << s) a.shift = s;
  a.sl2 = x.scale * kLog2e;
  a.window = z.window;
  a.sinks = z.sinks;
  a.causal = z.causal;
  a.rest = x.rest;
  a.splits = 1;
  return a;
}
int too_many(const WindowAttnSizes& z) {
  const int64_t hb = (int64_t)z.Hk * z.B, G = z.H / z.Hk;
  if (hb > (int64_t)(INT32_MAX / 1024))
    return fail(TSC_ERR_UNSUPPORTED, "window_attention: %lld (key head, sequence) pairs", (long long)hb);
  if (z.total_q * G > INT32_MAX - 1024)
    return fail(TSC_ERR_UNSUPPORTED, "window_attention: %lld queries with %lld heads to a key head",
                (long long)z.total_q, (long long)G);
  return TSC_OK;
}

}  // namespace

int64_t window_attention_workspace_bytes(const WindowAttnSizes& z, int32_t backward) {
  if (z.B == 0 || z.total_q == 0) return 0;
  if (backward) return (int64_t)align_up(4 * z.total_q * z.H, 16) + sink_plan(z).bytes;
  const int s = wa_plan(z).splits;
  return s > 1 ? s * part_bytes(z.total_q, z.H, z.D) : 0;
}

int window_attention_launch(tsc_ctx* ctx, const WindowAttnArgs& x, void* out, void* out_lo, float* lse, void* ws) {
  const WindowAttnSizes& z = x.z;
  if (int st = too_many(z)) return st;
  WaArgs a = wa_args(x);
  a.out = out;
  a.lo = out_lo;
  a.lse = lse;
  a.part = (float*)ws;
  const Plan plan = wa_plan(z);
  a.splits = plan.splits;
  const int64_t hb = (int64_t)z.Hk * z.B;
  const dim3 grid(tiles_of((int64_t)z.max_q * a.G, hb, plan.rows) * a.splits, (unsigned)z.Hk, (unsigned)z.B);
  return by_type(z.dtype, z.D, [&](auto t, auto d) {
    using T = decltype(t);
    constexpr int D = decltype(d)::value;
    {
      ProfScope p(ctx, "window_attention");
      if (plan.rows == 32) wa_few_kernel<T, D><<<grid, kNT, 0, ctx->stream>>>(a);
      else if constexpr (sizeof(T) == 4) wa_forward32_kernel<D><<<grid, kNT, 0, ctx->stream>>>(a);
      else {
        constexpr int QT = D == 64 ? 2 : 1, NW = kBQ16 / 32 / QT;
        if (a.lse) wa_forward16_kernel<T, D, QT, NW, true><<<grid, 64 * NW, 0, ctx->stream>>>(a);
        else wa_forward16_kernel<T, D, QT, NW, false><<<grid, 64 * NW, 0, ctx->stream>>>(a);
      }
    }
    if (a.splits > 1) {
      ProfScope p(ctx, "window_attention_join");
      wa_join_kernel<T, D><<<(unsigned)((z.total_q * z.H + 3) / 4), kNT, 0, ctx->stream>>>(a, z.B);
    }
  });
}

int window_attention_backward_launch(tsc_ctx* ctx, const WindowAttnArgs& x, const void* out, const void* out_lo,
                                     const float* lse, const void* dout, void* ws, void* dq, void* dk, void* dv) {
  const WindowAttnSizes& z = x.z;
  if (int st = too_many(z)) return st;
  WaArgs a = wa_args(x);
  a.lse = (float*)lse;
  a.out = (void*)out;
  a.lo = (void*)out_lo;
  a.dout = dout;
  a.r = (float*)ws;
  a.dq = dq;
  a.dk = dk;
  a.dv = dv;
  const int64_t hb = (int64_t)z.Hk * z.B, rows = z.total_q * z.H;
  // SHARE where blocks of 128 would leave CUs idle; in 16 bits where they would half of them, a wave's own tiles being quick
  // and the joint at the end not.  Both gradients, us, 128 / 32: 192 tiles of 12 x 128 bf16, 2048 tokens 81 / 119; 128 of
  // 16 x 64, 1000 tokens 49 / 68; 96 of 12 x 128, 1000 tokens 80 / 72; fp32, 8 / 2 x 64, 2048 tokens 154 / 133.
  const int64_t few = z.dtype == TSC_F32 ? kCUs : kCUs / 2;
  const bool few_q = (int64_t)tiles_of((int64_t)z.max_q * a.G, hb, kBQ) * hb < few;
  const bool few_k = (int64_t)tiles_of(z.max_kv, hb, kBQ) * hb < few;
  const dim3 gq(tiles_of((int64_t)z.max_q * a.G, hb, few_q ? 32 : kBQ), (unsigned)z.Hk, (unsigned)z.B);
  const dim3 gk(tiles_of(z.max_kv, hb, few_k ? 32 : kBQ), (unsigned)z.Hk, (unsigned)z.B);
  const SinkPlan sinks = rows > 0 ? sink_plan(z) : SinkPlan{1, 0, 0};
  a.own_sinks = sinks.parts > 1;
  a.sink_parts = sinks.parts;
  a.sink_keys = sinks.keys;
  a.sink_sums = (float*)((char*)ws + align_up(4 * rows, 16));
  return by_type(z.dtype, z.D, [&](auto t, auto d) {
    using T = decltype(t);
    constexpr int D = decltype(d)::value;
    if (rows > 0) {
      ProfScope p(ctx, "window_attention_dq");
      if (few_q) wa_dq_kernel<T, D, true><<<gq, kNT, 0, ctx->stream>>>(a);
      else wa_dq_kernel<T, D, false><<<gq, kNT, 0, ctx->stream>>>(a);
    }
    {
      ProfScope p(ctx, "window_attention_dkv");
      if (few_k) wa_dkv_kernel<T, D, true, false><<<gk, kNT, 0, ctx->stream>>>(a);
      else if constexpr (sizeof(T) == 2 && D == 128) wa_dkv_pair_kernel<T><<<gk, 512, 0, ctx->stream>>>(a);
      else wa_dkv_kernel<T, D, false, false><<<gk, kNT, 0, ctx->stream>>>(a);
    }
    if (a.own_sinks) {
      ProfScope p(ctx, "window_attention_sinks");
      const dim3 gs((unsigned)(sinks.keys / 32 * sinks.parts), (unsigned)z.Hk, (unsigned)z.B);
      wa_dkv_kernel<T, D, true, true><<<gs, kNT, 0, ctx->stream>>>(a);
      wa_sinks_kernel<T, D><<<dim3((unsigned)(sinks.keys / 4), (unsigned)z.Hk, (unsigned)z.B), kNT, 0, ctx->stream>>>(a);
    }
  });
}

}  // namespace tsc
