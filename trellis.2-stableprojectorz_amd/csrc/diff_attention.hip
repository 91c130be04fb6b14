// Differential attention over packed sequences, and its gradient: the difference of two softmax maps,
// each over half of a head's dimensions.
//
//   q = [q1 | q2], k = [k1 | k2] per head (halves of D), z = scale
//   P1 = softmax(q1 k1^T z), P2 = softmax(q2 k2^T z);   out = (P1 - lambda_h P2) v
//   n in [cu_q[b], cu_q[b+1]), m in [cu_kv[b], cu_kv[b+1]);  no keys: zeros
// Gradient, with do = d out, dP = do v^T, r_i = do . (P_i v) per query:
//   dv = (P1 - lambda P2)^T do;  dS1 = P1 (dP - r1);  dS2 = -lambda P2 (dP - r2)
//   dq_i = z dS_i k_i;  dk_i = z dS_i^T q_i;  dlambda_h = - sum over queries of r2
//
// The tensors are those of tsc_attention (rows of H heads of D = 64 or 128), so a fragment of k or q
// feeds one map or the other by its dimensions, and one walk over the keys serves both.  The two
// maps' weighted sums of v stay apart until their denominators are known: 6 D flops a pair.  (A second walk
// with known denominators would multiply only the difference with v, 2 D instead of 4 D, but make the
// scores again, 2 D, and the exponentials.)  For the gradient the forward pass keeps
// P1 v and P2 v in fp32 and the two log-sum-exps, from which the probabilities are made again.
//
// Scores are computed in 32 x 32 tiles whose result layout (lane: one column, 16 rows 8(j/4) +
// 4(lane/32) + j%4) is the operand layout of the next product, contracted over those rows: transposed
// (keys x queries) where a wave owns queries (forward, dq), plain (queries x keys) where it owns keys
// (dk, dv).  The other operand of that product is read transposed from the row-major tile in LDS.
// All three types run the same code on fragments of 8 elements: one 32x32x16 product in 16 bits,
// eight 32x32x2 products of the same elements in fp32.  P and dS are rounded to the input type for the
// second products (as v and k are stored); softmax, sums and accumulators are fp32.
// No atomics: dq and (dk, dv) come from two kernels, each owning its rows, which costs the scores and
// dP twice (14 D instead of 10 D flops a pair; 18 D where a wave has one map, D = 128 in 16 bits) and
// keeps the bits of a result fixed.

#include <float.h>

#include <algorithm>
#include <type_traits>

#include "attention_common.h"
#include "tsc_internal.h"

namespace tsc {
namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLazy = 8.f;  // log2 headroom before a running maximum is raised (16 bits)

// ---- fragments: 8 elements of a lane --------------------------------------------------------
struct F32x8 {
  float v[8];
};
template <typename T>
struct Frag {
  typedef u32x4_t type;
  static __device__ __forceinline__ void mma(const u32x4_t& a, const u32x4_t& b, f32x16_t& c) {
    Mma<T>::run(a, b, c);
  }
  // Elements 8 g .. 8 g + 7 of a score tile.
  static __device__ __forceinline__ u32x4_t pack(const float* s) {
    u32x4_t r;
#pragma unroll
    for (int i = 0; i < 4; ++i) r[i] = Mma<T>::pack(s[2 * i], s[2 * i + 1]);
    return r;
  }
  static __device__ __forceinline__ u32x4_t load(const T* p) { return *(const u32x4_t*)p; }
};
template <>
struct Frag<float> {
  typedef F32x8 type;
  static __device__ __forceinline__ void mma(const F32x8& a, const F32x8& b, f32x16_t& c) {
#pragma unroll
    for (int i = 0; i < 8; ++i) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a.v[i], b.v[i], c, 0, 0, 0);
  }
  static __device__ __forceinline__ F32x8 pack(const float* s) {
    F32x8 r;
#pragma unroll
    for (int i = 0; i < 8; ++i) r.v[i] = s[i];
    return r;
  }
  static __device__ __forceinline__ F32x8 load(const float* p) {
    F32x8 r;
    *(float4*)&r.v[0] = *(const float4*)p;
    *(float4*)&r.v[4] = *(const float4*)(p + 4);
    return r;
  }
};

// ---- row-major tiles in LDS -----------------------------------------------------------------
// 16 bits: 16-byte chunks XOR-swizzled by row, so that 16 rows of one chunk column (row fragments)
// and 64 bytes of 4 consecutive rows (transposed reads) both fall into distinct banks.
// fp32: rows padded by 4 floats.
template <typename T, int D>
struct Tile {
  static constexpr int CPR = D / 8;  // 16-byte chunks of a row
  static constexpr int ROWB = 2 * D;
  static __device__ __forceinline__ int swz(int row) {
    return D == 128 ? ((row & 3) << 2) | ((row >> 2) & 3) : ((row & 2) << 1) | ((row >> 2) & 3);
  }
  static __device__ __forceinline__ void put(unsigned char* t, int row, int c, u32x4_t v) {
    *(u32x4_t*)(t + row * ROWB + ((c ^ swz(row)) << 4)) = v;
  }
  // Dims 16 st + 8 hf .. + 7 of row l32 (r0 a multiple of 16).
  static __device__ __forceinline__ u32x4_t row(const unsigned char* t, int r0, int l32, int hf, int st) {
    const int r = r0 + l32;
    return *(const u32x4_t*)(t + r * ROWB + (((2 * st + hf) ^ swz(r)) << 4));
  }
  // Column 32 mt + l32; rows r0 + 16 g + 8 (e / 4) + 4 hf + e % 4, e = 0 .. 7.
  static __device__ __forceinline__ u32x4_t col(const unsigned char* t, int r0, int lane, int g, int mt) {
    const int vr = 4 * (lane >> 5) + ((lane & 15) >> 2);
    const int c = 4 * mt + 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1);
    u32x4_t r;
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      const int rr = r0 + 16 * g + 8 * x + vr;
      const uint2 h = lds_read_tr(t + rr * ROWB + ((c ^ swz(rr)) << 4) + (lane & 1) * 8);
      r[2 * x] = h.x;
      r[2 * x + 1] = h.y;
    }
    return r;
  }
};
template <int D>
struct Tile<float, D> {
  static constexpr int CPR = D / 4;
  static constexpr int ROWB = 4 * (D + 4);
  static __device__ __forceinline__ void put(unsigned char* t, int row, int c, u32x4_t v) {
    *(u32x4_t*)(t + row * ROWB + 16 * c) = v;
  }
  static __device__ __forceinline__ F32x8 row(const unsigned char* t, int r0, int l32, int hf, int st) {
    return Frag<float>::load((const float*)(t + (r0 + l32) * ROWB) + 16 * st + 8 * hf);
  }
  static __device__ __forceinline__ F32x8 col(const unsigned char* t, int r0, int lane, int g, int mt) {
    F32x8 r;
#pragma unroll
    for (int e = 0; e < 8; ++e)
      r.v[e] = ((const float*)(t + (r0 + 16 * g + 8 * (e >> 2) + 4 * (lane >> 5) + (e & 3)) * ROWB))
          [32 * mt + (lane & 31)];
    return r;
  }
};

// Rows on their way from global memory into a tile: ROWS rows by NT threads.
template <typename T, int D, int ROWS, int NT>
struct Stage {
  typedef Tile<T, D> Ti;
  static constexpr int NL = ROWS * Ti::CPR / NT;
  static_assert(NL >= 1 && NL * NT == ROWS * Ti::CPR, "tile shape");
  u32x4_t r[NL];
  int last;  // the last row of the tile that there is
  // Rows first .. first + ROWS - 1 of base (row stride ld elements); nothing if first >= end.
  // No lane branches: rows from `end` on repeat the last one, and with CLEAR are cleared on their way into
  // LDS (at the load the compiler would wait for it to do so).
  __device__ __forceinline__ void load(const T* base, int64_t ld, int first, int end, int tid) {
    if (first >= end) return;
    const uint32_t rb = (uint32_t)ld * sizeof(T);
    const char* p = (const char*)base + (int64_t)first * rb;
    last = min(end - 1 - first, ROWS - 1);
#pragma unroll
    for (int i = 0; i < NL; ++i) {
      const int id = tid + NT * i;
      r[i] = *(const u32x4_t*)(p + ((uint32_t)min(id / Ti::CPR, last) * rb + 16u * (id % Ti::CPR)));
    }
  }
  template <bool CLEAR = true>
  __device__ __forceinline__ void store(unsigned char* t, int tid) {
#pragma unroll
    for (int i = 0; i < NL; ++i) {
      const int id = tid + NT * i;
      if (CLEAR && id / Ti::CPR > last) r[i] = u32x4_t{0, 0, 0, 0};
      Ti::put(t, id / Ti::CPR, id % Ti::CPR, r[i]);
    }
  }
};

__device__ __forceinline__ void clear(f32x16_t& c) {
#pragma unroll
  for (int j = 0; j < 16; ++j) c[j] = 0.f;
}

// Writes f times a transposed result (lane: one row; dims 8(j/4) + 4 hf + j%4 of each 32) to that row.
template <typename T>
__device__ __forceinline__ void store_dims(T* p, int hf, const f32x16_t& c, float f) {
#pragma unroll
  for (int g = 0; g < 4; ++g) {
    const float a = c[4 * g] * f, b = c[4 * g + 1] * f, d = c[4 * g + 2] * f, e = c[4 * g + 3] * f;
    if constexpr (sizeof(T) == 4)
      *(float4*)(p + 8 * g + 4 * hf) = make_float4(a, b, d, e);
    else
      *(uint2*)(p + 8 * g + 4 * hf) = make_uint2(Mma<T>::pack(a, b), Mma<T>::pack(d, e));
  }
}

// Zeros in head h of the rows [r0, r1), shared by the gx blocks of index bx.
template <typename T>
__device__ __forceinline__ void zero_rows(T* p, int64_t r0, int64_t r1, int H, int D, int h, int bx,
                                          int gx) {
  const int per = D * (int)sizeof(T) / 16;
  for (int64_t i = threadIdx.x + (int64_t)bx * blockDim.x; i < (r1 - r0) * per;
       i += (int64_t)gx * blockDim.x)
    *(uint4*)((char*)(p + ((r0 + i / per) * H + h) * D) + 16 * (i % per)) = make_uint4(0, 0, 0, 0);
}
// ... of the rows outside every sequence, by the blocks of the first and the last sequence.
template <typename T>
__device__ __forceinline__ void zero_rest(T* p, const int32_t* cu, int64_t total, int bb, int H, int D,
                                          int h, int bx, int gx) {
  int b0, n;
  if (bb == 0) {
    segment(cu, 0, total, &b0, &n);
    zero_rows(p, 0, b0, H, D, h, bx, gx);
  }
  if (bb == (int)gridDim.z - 1) {
    segment(cu, bb, total, &b0, &n);
    zero_rows(p, b0 + n, total, H, D, h, bx, gx);
  }
}

// Adds up the 4 waves' sums through LDS (2 N x 4 KB at lds, which every wave has left): wave 0 has them.
template <int N>
__device__ __forceinline__ void join_waves(float* lds, int w, int lane, f32x16_t (&c)[N]) {
  __syncthreads();
#pragma unroll
  for (int half = 2; half > 0; half >>= 1) {  // waves half .. 2 half - 1 hand theirs on
    float* meet = lds + (w % half) * N * 1024 + lane;
    if (w >= half && w < 2 * half)
#pragma unroll
      for (int i = 0; i < N; ++i)
#pragma unroll
        for (int j = 0; j < 16; ++j) meet[(16 * i + j) * 64] = c[i][j];
    __syncthreads();
    if (w < half)
#pragma unroll
      for (int i = 0; i < N; ++i)
#pragma unroll
        for (int j = 0; j < 16; ++j) c[i][j] += meet[(16 * i + j) * 64];
    __syncthreads();
  }
}

struct DaArgs {
  const void *q, *k, *v;
  int64_t ldq, ldk, ldv;
  const float* lambda;
  const int32_t *cu_q, *cu_kv;
  int64_t total_q, total_kv;
  int32_t H;
  float sl2;     // scale * log2(e)
  int32_t rest;  // zero the rows outside every sequence
  // forward
  void* out;
  float* maps;       // (total_q, H, 2, D): P1 v, P2 v, or null
  float* lse;        // (2, H, total_q): log2 of the sum of 2^(score sl2), or null
  int32_t splits, part_keys;  // small grids: blocks that share a sequence's keys, keys of each
  float* part;       // splits > 1: (splits, total_q, H, 2, D) sums, then (splits, total_q, H, 2, 4)
  // backward
  const void* dout;
  const float* r12;  // (2, H, total_q)
  float* lam_part;   // (H, B, dk / dv blocks of a sequence)
  int32_t lam_parts;
  void *dq, *dk, *dv;
  float* dlambda;
};

// ------------------------------------------------------------------------------- forward
constexpr int kNT = 256;  // 4 waves of 32 queries (or keys, in dk / dv)
constexpr int kBQ = 128;

// Small grids share a sequence's keys out over a.splits blocks.  Keys of a part of a sequence: more than
// part_keys where the splits would not reach over it.
__device__ __forceinline__ int64_t part_of(const DaArgs& a, int kv_len) {
  return max((int64_t)a.part_keys, ((int64_t)(kv_len + a.splits - 1) / a.splits + 63) / 64 * 64);
}
// Narrows a sequence's keys to those of part sp.
__device__ __forceinline__ void take_part(const DaArgs& a, int sp, int* kv0, int* kv_len) {
  const int64_t per = part_of(a, *kv_len);
  const int lo = (int)min(per * sp, (int64_t)*kv_len);
  *kv0 += lo;
  *kv_len = (int)min(per, (int64_t)(*kv_len - lo));
}
// Where part sp of a.part has map i of (row, head) number at: D weighted sums, and the maximum (times
// sl2), the denominator and the sum of the unrounded probabilities.
__device__ __forceinline__ float* part_sums(const DaArgs& a, int sp, int64_t at, int i, int D) {
  return a.part + (((int64_t)sp * a.total_q * a.H + at) * 2 + i) * D;
}
__device__ __forceinline__ float4* part_stat(const DaArgs& a, int sp, int64_t at, int i, int D) {
  return (float4*)part_sums(a, a.splits, 0, 0, D) + ((int64_t)sp * a.total_q * a.H + at) * 2 + i;
}

// One 32-key step of both maps for a wave's 32 queries: k and v in LDS rows r0 .. r0 + 31, the keys
// k0 .. of which those below k_hi count.
template <typename T, int D>
__device__ __forceinline__ void forward_step(const unsigned char* kt, const unsigned char* vt, int r0,
                                             int lane, int k0, int k_hi, float sl2,
                                             const typename Frag<T>::type (&qf)[D / 16],
                                             float (&m)[2], float (&l)[2],
                                             f32x16_t (&o)[2][D / 32]) {
  typedef Frag<T> F;
  typedef typename F::type Fr;
  typedef Tile<T, D> Ti;
  constexpr int KS = D / 16, MT = D / 32;
  const int l32 = lane & 31, hf = lane >> 5;
  Fr pf[2][2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    f32x16_t s;
    clear(s);
#pragma unroll
    for (int st = i * KS / 2; st < (i + 1) * KS / 2; ++st)
      F::mma(Ti::row(kt, r0, l32, hf, st), qf[st], s);
    if (k0 + 32 > k_hi) {  // uniform; the asm keeps it a branch
      asm volatile("");
#pragma unroll
      for (int j = 0; j < 16; ++j)
        if (k0 + 8 * (j >> 2) + 4 * hf + (j & 3) >= k_hi) s[j] = -INFINITY;
    }
    float mx = s[0], p[16];
#pragma unroll
    for (int j = 1; j < 16; ++j) mx = fmaxf(mx, s[j]);
    mx = pair_max(mx) * sl2;
    if (__builtin_amdgcn_ballot_w64(mx > m[i])) {
      const float mn = fmaxf(m[i], mx), f = fast_exp2(m[i] - mn);
      m[i] = mn;
      l[i] *= f;
#pragma unroll
      for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int j = 0; j < 16; ++j) o[i][mt][j] *= f;
    }
#pragma unroll
    for (int j = 0; j < 16; ++j) {
      p[j] = fast_exp2(fmaf(s[j], sl2, -m[i]));
      l[i] += p[j];
    }
    pf[i][0] = F::pack(p);
    pf[i][1] = F::pack(p + 8);
  }
#pragma unroll
  for (int g = 0; g < 2; ++g)
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
      const Fr vf = Ti::col(vt, r0, lane, g, mt);
      F::mma(vf, pf[0][g], o[0][mt]);
      F::mma(vf, pf[1][g], o[1][mt]);
    }
}

// Writes a wave's finished rows: qi the lane's query of q_len, l summed over both halves.
template <typename T, int D>
__device__ __forceinline__ void forward_store(const DaArgs& a, int h, int64_t row, int hf, bool keys,
                                              const float (&m)[2], const float (&l)[2],
                                              f32x16_t (&o)[2][D / 32]) {
  const float i1 = keys ? 1.f / l[0] : 0.f, i2 = keys ? 1.f / l[1] : 0.f, f2 = a.lambda[h] * i2;
  const int64_t at = (row * a.H + h) * D;
#pragma unroll
  for (int mt = 0; mt < D / 32; ++mt) {
    if (a.maps) {
      store_dims(a.maps + 2 * at + 32 * mt, hf, o[0][mt], i1);
      store_dims(a.maps + 2 * at + D + 32 * mt, hf, o[1][mt], i2);
    }
#pragma unroll
    for (int j = 0; j < 16; ++j) o[0][mt][j] = fmaf(-f2, o[1][mt][j], o[0][mt][j] * i1);
    store_dims((T*)a.out + at + 32 * mt, hf, o[0][mt], 1.f);
  }
  if (a.lse && hf == 0) {
    a.lse[(int64_t)h * a.total_q + row] = keys ? m[0] + log2f(l[0]) : INFINITY;
    a.lse[(int64_t)(a.H + h) * a.total_q + row] = keys ? m[1] + log2f(l[1]) : INFINITY;
  }
}

// fp32, whole sequences: a block of 4 waves owns 128 queries and walks the keys in tiles of 32.  Bound by
// the fp32 matrix cores: 4096 tokens, 8 x 64, 471 us or 109 TFLOP/s of the 154 a large product reaches.
// At D = 64 two waves per SIMD fill each other's waits; at D = 128 the registers hold one.
template <int D>
__global__ void __launch_bounds__(kNT, D == 64 ? 2 : 1) da_forward32_kernel(const DaArgs a) {
  typedef float T;
  typedef Frag<T> F;
  typedef Tile<T, D> Ti;
  constexpr int BK = 32;
  constexpr int KS = D / 16, MT = D / 32;
  __shared__ __attribute__((aligned(16))) unsigned char kt[BK * Ti::ROWB], vt[BK * Ti::ROWB];
  int bx, h, bb;
  block_tile(a.cu_kv, &bx, &h, &bb);
  int q0, q_len, kv0, kv_len;
  segment(a.cu_q, bb, a.total_q, &q0, &q_len);
  segment(a.cu_kv, bb, a.total_kv, &kv0, &kv_len);
  const int tid = threadIdx.x, lane = tid & 63, w = tid >> 6, l32 = lane & 31, hf = lane >> 5;
  if (a.rest) zero_rest((T*)a.out, a.cu_q, a.total_q, bb, a.H, D, h, bx, gridDim.x);
  const T* kbase = (const T*)a.k + (int64_t)kv0 * a.ldk + (int64_t)h * D;
  const T* vbase = (const T*)a.v + (int64_t)kv0 * a.ldv + (int64_t)h * D;

  for (int qt = bx * kBQ; qt < q_len; qt += gridDim.x * kBQ) {
    const int qi = qt + w * 32 + l32;
    typename F::type qf[KS];
    {
      const T* p = (const T*)a.q + (int64_t)(q0 + min(qi, q_len - 1)) * a.ldq + (int64_t)h * D + 8 * hf;
#pragma unroll
      for (int st = 0; st < KS; ++st) qf[st] = F::load(p + 16 * st);
    }
    float m[2] = {-FLT_MAX, -FLT_MAX}, l[2] = {0.f, 0.f};  // a finite start: a tile of scores of -inf
    f32x16_t o[2][MT];                                     // then adds nothing
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
      clear(o[0][mt]);
      clear(o[1][mt]);
    }
    Stage<T, D, BK, kNT> ks, vs;
    ks.load(kbase, a.ldk, 0, kv_len, tid);
    vs.load(vbase, a.ldv, 0, kv_len, tid);
    for (int kb = 0; kb < kv_len; kb += BK) {
      __syncthreads();
      ks.store(kt, tid);
      vs.store(vt, tid);
      __syncthreads();
      ks.load(kbase, a.ldk, kb + BK, kv_len, tid);
      vs.load(vbase, a.ldv, kb + BK, kv_len, tid);
      forward_step<T, D>(kt, vt, 0, lane, kb, kv_len, a.sl2, qf, m, l, o);
    }
    l[0] = pair_sum(l[0]);
    l[1] = pair_sum(l[1]);
    if (qi < q_len) forward_store<T, D>(a, h, q0 + qi, hf, kv_len > 0, m, l, o);
  }
}

// fp32, small grids: a block owns 32 queries, and its waves and the blocks of a.splits
// parts share out the keys, 32 at a time.  Each wave brings its own keys through its own piece of LDS,
// so none waits for another until the end, where their maxima, denominators and sums are joined.
// 1024 tokens, 8 x 64 (256 blocks): 50 us, and 124 in the 64 blocks of 128 queries.
template <int D>
__global__ void __launch_bounds__(kNT) da_few32_kernel(const DaArgs a) {
  typedef float T;
  typedef Frag<T> F;
  typedef Tile<T, D> Ti;
  constexpr int KS = D / 16, MT = D / 32, NW = kNT / 64;
  constexpr int TB = 32 * Ti::ROWB;  // bytes of a tile
  __shared__ __attribute__((aligned(16))) unsigned char lds[NW][2 * TB];
  __shared__ float sm[NW][2][32], sl[NW][2][32];
  int bx, h, bb;
  block_tile(a.cu_kv, &bx, &h, &bb);
  int q0, q_len, kv0, kv_len;
  segment(a.cu_q, bb, a.total_q, &q0, &q_len);
  segment(a.cu_kv, bb, a.total_kv, &kv0, &kv_len);
  const int lane = threadIdx.x & 63, l32 = lane & 31, hf = lane >> 5;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);  // uniform: its keys are scalars
  const int sp = bx % a.splits, tile = bx / a.splits, tiles = gridDim.x / a.splits;
  if (a.rest && sp == 0) zero_rest((T*)a.out, a.cu_q, a.total_q, bb, a.H, D, h, tile, tiles);
  if (a.splits > 1) {
    take_part(a, sp, &kv0, &kv_len);
    if (kv_len == 0) return;  // the join passes over it
  }
  const T* kbase = (const T*)a.k + (int64_t)kv0 * a.ldk + (int64_t)h * D;
  const T* vbase = (const T*)a.v + (int64_t)kv0 * a.ldv + (int64_t)h * D;
  unsigned char *kt = lds[w], *vt = lds[w] + TB;

  for (int qt = tile * 32; qt < q_len; qt += tiles * 32) {
    const int qi = qt + l32;
    typename F::type qf[KS];
    {
      const T* p = (const T*)a.q + (int64_t)(q0 + min(qi, q_len - 1)) * a.ldq + (int64_t)h * D + 8 * hf;
#pragma unroll
      for (int st = 0; st < KS; ++st) qf[st] = F::load(p + 16 * st);
    }
    float m[2] = {-FLT_MAX, -FLT_MAX}, l[2] = {0.f, 0.f};
    f32x16_t o[2][MT];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
      clear(o[0][mt]);
      clear(o[1][mt]);
    }
    // The next keys come in during a step, but at D = 128: no registers are left to hold them, and a
    // step there takes ten times as long as they do.
    constexpr bool AHEAD = D == 64;
    Stage<T, D, 32, 64> ks, vs;
    int k0 = 32 * w;
    auto load = [&](int k) {
      ks.load(kbase, a.ldk, k, kv_len, lane);
      vs.load(vbase, a.ldv, k, kv_len, lane);
    };
    if (AHEAD) load(k0);
    for (; k0 < kv_len; k0 += 32 * NW) {
      if (!AHEAD) load(k0);
      // A wave's LDS operations are carried out in order; the compiler has to keep that order.
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      ks.store(kt, lane);
      vs.store(vt, lane);
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      if (AHEAD) load(k0 + 32 * NW);
      forward_step<T, D>(kt, vt, 0, lane, k0, kv_len, a.sl2, qf, m, l, o);
    }
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      l[i] = pair_sum(l[i]);
      if (hf == 0) {
        sm[w][i][l32] = m[i];
        sl[w][i][l32] = l[i];
      }
    }
    __syncthreads();  // every wave has left its tiles
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const float own = m[i];
      m[i] = sm[0][i][l32];
#pragma unroll
      for (int x = 1; x < NW; ++x) m[i] = fmaxf(m[i], sm[x][i][l32]);
      l[i] = 0.f;
#pragma unroll
      for (int x = 0; x < NW; ++x) l[i] = fmaf(sl[x][i][l32], fast_exp2(sm[x][i][l32] - m[i]), l[i]);
      const float f = fast_exp2(own - m[i]);
#pragma unroll
      for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int j = 0; j < 16; ++j) o[i][mt][j] *= f;
    }
    join_waves<MT>((float*)lds[0], w, lane, o[0]);
    join_waves<MT>((float*)lds[0], w, lane, o[1]);
    if (w != 0 || qi >= q_len) continue;
    if (a.splits == 1) {
      forward_store<T, D>(a, h, q0 + qi, hf, kv_len > 0, m, l, o);
    } else {
      const int64_t at = (int64_t)(q0 + qi) * a.H + h;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) store_dims(part_sums(a, sp, at, i, D) + 32 * mt, hf, o[i][mt], 1.f);
        if (hf == 0) *part_stat(a, sp, at, i, D) = make_float4(m[i], l[i], l[i], 0.f);
      }
    }
  }
}

// 16 bits: the two maps' softmax beside the matrix products.  As in attention.hip's
// kernel of this kind a step of 32 keys has two phases, pinned in program order:
//   A  the next step's scores (matrix) beside the rest of this step's exponentials (VALU) and the
//      transposed reads of v
//   B  both maps' sums += V^T P^T beside the next step's row maxima, the first half of its
//      exponentials and the reads of k for the step after
// The exponentials bound it: twice those of one map, a quarter of the VALU's rate each.
// A wave has NM maps of its 32 queries: both at D = 64; one at D = 128, where the sums of both would
// leave one wave per SIMD, whose stalls nothing fills (9000 + 6143 tokens, 12 x 128 bf16: 1500 us that way,
// 1260 us or 870 TFLOP/s now).  The two waves of a query tile then meet in LDS at the end.
// Counted there: matrix cores busy 38 % and VALU 50 % of the cycles, the clock down to 1.8 - 2.0 GHz; at
// D = 64 (36011 queries on 7 x 1374 keys, 16 heads, f16: 455 us) 29 % and 70 %.
// A wave has 256 registers.  Spilled to scratch: with KEEP 12 at D = 64, at D = 128 2 in blocks of eight
// waves and 47 in blocks of four; without it 14 in the latter and none in the others.
// The sums of v are divided by the sum of the rounded P that they were made of.  KEEP (for the backward
// pass) also adds up the unrounded P: the log-sum-exps have to be those of the fp32 probabilities.
template <typename T, int D, int NM, int NW, bool KEEP>
__global__ void __launch_bounds__(64 * NW, 2) da_forward16_kernel(const DaArgs a) {
  typedef Tile<T, D> Ti;
  constexpr int BK = 64;             // keys per staged block: two steps of 32
  constexpr int CPR = Ti::CPR, ROWB = Ti::ROWB;
  constexpr int KH = D / 32, KS = NM * KH, MT = D / 32;  // k-steps of a map's scores, of the wave's
  constexpr int NT = 64 * NW, QW = NW * NM / 2, BQ = 32 * QW;  // query tiles of the block
  constexpr int RI = NT / CPR, NL = BK / RI;  // rows a load of the block covers; loads of a thread
  constexpr int NA = KS, NB = 2 * MT * NM;    // products of the two phases
  static_assert(NL >= 1, "tile shape");
  __shared__ __attribute__((aligned(16))) unsigned char lds[4][BK * ROWB];
  static_assert(NM == 2 || QW * 32 * D * 4 <= 4 * BK * ROWB, "the second map's sums fit");
  unsigned char(*kbuf)[BK * ROWB] = lds, (*vbuf)[BK * ROWB] = lds + 2;
  int bx, h, bb;
  block_tile(a.cu_kv, &bx, &h, &bb);
  int q0, q_len, kv0, kv_len;
  segment(a.cu_q, bb, a.total_q, &q0, &q_len);
  segment(a.cu_kv, bb, a.total_kv, &kv0, &kv_len);
  const int sp = bx % a.splits, qtile = bx / a.splits, qtiles = gridDim.x / a.splits;
  if (a.rest && sp == 0) zero_rest((T*)a.out, a.cu_q, a.total_q, bb, a.H, D, h, qtile, qtiles);
  if (a.splits > 1) {
    take_part(a, sp, &kv0, &kv_len);
    if (kv_len == 0) return;  // the join passes over it
  }
  const T* kbase = (const T*)a.k + (int64_t)kv0 * a.ldk + (int64_t)h * D;
  const T* vbase = (const T*)a.v + (int64_t)kv0 * a.ldv + (int64_t)h * D;
  const float sl2 = a.sl2;

  for (int qt = qtile * BQ; qt < q_len; qt += qtiles * BQ) {
    int tid = threadIdx.x;
    asm volatile("" : "+v"(tid));  // nothing derived from it is kept across q tiles
    const int lane = tid & 63, w = tid >> 6, l32 = lane & 31, hf = lane >> 5;
    const int map = NM == 2 ? 0 : w & 1, tile = NM == 2 ? w : w >> 1;  // the wave's first map
    const int qi = qt + tile * 32 + l32;
    // A wave without queries brings its share of the keys and does no more.
    const bool idle = __builtin_amdgcn_readfirstlane(qt + tile * 32) >= q_len;
    const int64_t at = (int64_t)(q0 + qi) * a.H + h;
    if (kv_len == 0) {  // uniform over the block
      if (map == 0 && qi < q_len) {
        for (int c = hf; c < CPR; c += 2) *(uint4*)((T*)a.out + at * D + 8 * c) = make_uint4(0, 0, 0, 0);
        if (a.maps)
          for (int c = hf; c < D / 2; c += 2) *(uint4*)(a.maps + at * 2 * D + 4 * c) = make_uint4(0, 0, 0, 0);
        if (a.lse && hf == 0) {
          a.lse[(int64_t)h * a.total_q + q0 + qi] = INFINITY;
          a.lse[(int64_t)(a.H + h) * a.total_q + q0 + qi] = INFINITY;
        }
      }
      continue;
    }
    const int srow = tid / CPR, sc = tid % CPR;  // staging: chunk sc of rows srow + RI * i
    const uint32_t kst = (uint32_t)(2 * a.ldk), vst = (uint32_t)(2 * a.ldv);  // row bytes
    u32x4_t qf[KS];
    {
      const T* p = (const T*)a.q + (int64_t)(q0 + min(qi, q_len - 1)) * a.ldq + (int64_t)h * D + map * 16 * KH + 8 * hf;
#pragma unroll
      for (int st = 0; st < KS; ++st) qf[st] = *(const u32x4_t*)(p + 16 * st);
    }
    // Block kb's rows; rows past the last key repeat it, a block past the end is block 0.  The scores
    // of such keys are masked, and their v is stored as zeros.
    u32x4_t kr[NL], vr[NL];
    auto load = [&](const T* base, uint32_t rb, int kb, u32x4_t(&r)[NL]) {
      if (kb >= kv_len) kb = 0;
      const char* p = (const char*)base + (int64_t)kb * rb;
      const uint32_t lim = (uint32_t)min(kv_len - 1 - kb, BK - 1) * rb + 16u * sc;
      const uint32_t off = (uint32_t)srow * rb + 16u * sc;
#pragma unroll
      for (int i = 0; i < NL; ++i) r[i] = *(const u32x4_t*)(p + min(off + (uint32_t)(RI * i) * rb, lim));
    };
    auto store = [&](int vb, int kb, auto masked, int v0) {  // v0: first key of the v block
#pragma unroll
      for (int i = 0; i < NL; ++i) {
        if (decltype(masked)::value && v0 + srow + RI * i >= kv_len) vr[i] = u32x4_t{0, 0, 0, 0};
        Ti::put(vbuf[vb], srow + RI * i, sc, vr[i]);
      }
#pragma unroll
      for (int i = 0; i < NL; ++i) Ti::put(kbuf[kb], srow + RI * i, sc, kr[i]);
    };
    constexpr std::true_type Y{};
    constexpr std::false_type N{};
    float mc[NM], l[NM], lu[NM], alpha[NM];  // mc: running maxima, times sl2
    f32x16_t o[NM][MT], sa[NM], sb[NM];
#pragma unroll
    for (int i = 0; i < NM; ++i) {
      mc[i] = -FLT_MAX;
      l[i] = lu[i] = 0.f;
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) clear(o[i][mt]);
    }
    u32x4_t kf[KS], vf[2][MT], pf[NM][2];
    float pr[16 * NM];
    auto read_k = [&](int buf, int half, int st) { kf[st] = Ti::row(kbuf[buf], half * 32, l32, hf, map * KH + st); };
    auto read_v = [&](int buf, int half, int n) {
      vf[n / MT][n % MT] = Ti::col(vbuf[buf], half * 32, lane, n / MT, n % MT);
    };
    auto score = [&](const f32x16_t(&s)[NM], int i, int j, auto masked, int k0) {
      return decltype(masked)::value && k0 + 8 * (j >> 2) + 4 * hf + (j & 3) >= kv_len ? -INFINITY
                                                                                        : s[i][j];
    };
    auto exp_one = [&](const f32x16_t(&s)[NM], int e, auto masked, int k0) {
      pr[e] = fast_exp2(fmaf(score(s, e / 16, e % 16, masked, k0), sl2, -mc[e / 16]));
      if (KEEP) lu[e / 16] += pr[e];
    };
    auto pack_one = [&](int n) {  // n-th of 8 NM pairs -> rounded P and the denominator
      const int i = n / 8, e = 2 * (n % 8);
      const uint32_t p = Mma<T>::pack(pr[2 * n], pr[2 * n + 1]);
      pf[i][e / 8][(e / 2) % 4] = p;
      l[i] = Mma<T>::add2(p, l[i]);
    };
    auto max_part = [&](const f32x16_t(&s)[NM], int i, int part, float mx, auto masked, int k0) {
#pragma unroll
      for (int j = 4 * part; j < 4 * part + 4; ++j) mx = fmaxf(mx, score(s, i, j, masked, k0));
      return mx;
    };
    // Raises map i's running maxima where a score exceeds one by more than 2^kLazy.
    auto raise = [&](int i, float mx) {
      mx *= sl2;
      const bool up = __builtin_amdgcn_ballot_w64(mx > mc[i] + kLazy) != 0;
      if (up) {
        const float mn = fmaxf(mc[i], mx);
        alpha[i] = fast_exp2(mc[i] - mn);
        mc[i] = mn;
        if (KEEP) lu[i] *= alpha[i];  // the next exponentials are already added to it
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
    // n-th product of a step's scores: the maps in turn.
    auto qk = [&](int n, f32x16_t(&s)[NM]) {
      const int i = n % NM, st = i * KH + n / NM;
      if (n < NM) clear(s[i]);
      Mma<T>::run(kf[st], qf[st], s[i]);
    };
    auto pv = [&](int n) {
      const int g = n / (MT * NM), mt = (n / NM) % MT, i = n % NM;
      Mma<T>::run(vf[g][mt], pf[i][g], o[i][mt]);
    };
    auto step = [&](f32x16_t(&cur)[NM], f32x16_t(&nxt)[NM], int vb, int vhalf, int kb, int khalf,
                    auto masked, int k0, auto stage) {
      constexpr int EA = 8 * NM / NA;               // exponentials and packed pairs per A group
      constexpr int VA = (2 * MT + NA - 1) / NA;    // v reads per A group
#pragma unroll
      for (int n = 0; n < NA; ++n) {
        qk(n, nxt);
#pragma unroll
        for (int x = 0; x < VA; ++x)
          if (n * VA + x < 2 * MT) read_v(vb, vhalf, n * VA + x);
#pragma unroll
        for (int x = 0; x < EA; ++x) exp_one(cur, 8 * NM + n * EA + x, masked, k0);
#pragma unroll
        for (int x = 0; x < EA; ++x) pack_one(n * EA + x);  // those made longest ago first
        __builtin_amdgcn_sched_barrier(0);
      }
      constexpr int KB = (KS + NB - 1) / NB;
      constexpr int M0 = NB / 8;             // groups before the row maxima (matrix latency)
      constexpr int MG = NB / 4;             // groups of the row maxima
      constexpr int E0 = M0 + MG;
      constexpr int EB = (8 * NM + NB - E0 - 1) / (NB - E0);
      float mx[NM];
#pragma unroll
      for (int n = 0; n < E0; ++n) {
        pv(n);
#pragma unroll
        for (int x = 0; x < KB; ++x)
          if (n * KB + x < KS) read_k(kb, khalf, n * KB + x);
        if (n == M0) {
#pragma unroll
          for (int i = 0; i < NM; ++i) mx[i] = score(nxt, i, 0, masked, k0 + 32);
        }
        if (n >= M0) {
#pragma unroll
          for (int x = (n - M0) * 4 * NM / MG; x < (n - M0 + 1) * 4 * NM / MG; ++x)
            mx[x / 4] = max_part(nxt, x / 4, x % 4, mx[x / 4], masked, k0 + 32);
        }
        __builtin_amdgcn_sched_barrier(0);
      }
      bool up[NM];
#pragma unroll
      for (int i = 0; i < NM; ++i) up[i] = raise(i, pair_max(mx[i]));
#pragma unroll
      for (int n = E0; n < NB; ++n) {
        pv(n);
#pragma unroll
        for (int x = 0; x < KB; ++x)
          if (n * KB + x < KS) read_k(kb, khalf, n * KB + x);
#pragma unroll
        for (int x = 0; x < EB; ++x)
          if ((n - E0) * EB + x < 8 * NM) exp_one(nxt, (n - E0) * EB + x, masked, k0 + 32);
        if (decltype(stage)::value && n == NB - NB / 4) store(kb, kb ^ 1, masked, k0 + 32);
        __builtin_amdgcn_sched_barrier(0);
      }
#pragma unroll
      for (int i = 0; i < NM; ++i)
        if (up[i]) rescale(i);
    };
    {
      u32x4_t k1[NL];
      load(kbase, kst, 0, kr);
      load(vbase, vst, 0, vr);
      load(kbase, kst, BK, k1);
      store(0, 0, Y, 0);
#pragma unroll
      for (int i = 0; i < NL; ++i) kr[i] = k1[i];
      store(0, 1, Y, 0);
    }
    __syncthreads();
    if (idle) {  // the same copies and barriers
      __syncthreads();
      for (int jb = 0; jb * BK < kv_len; ++jb) {
        load(vbase, vst, jb * BK + BK, vr);
        load(kbase, kst, jb * BK + 2 * BK, kr);
        store(~jb & 1, jb & 1, Y, jb * BK + BK);
        __syncthreads();
      }
      if (NM == 1 && a.splits == 1) __syncthreads();
      if (a.splits == 1) __syncthreads();
      continue;
    }
#pragma unroll
    for (int st = 0; st < KS; ++st) read_k(0, 0, st);
#pragma unroll
    for (int n = 0; n < KS; ++n) qk(n, sa);
#pragma unroll
    for (int st = 0; st < KS; ++st) read_k(0, 1, st);
#pragma unroll
    for (int i = 0; i < NM; ++i) {
      float mx = -INFINITY;
#pragma unroll
      for (int part = 0; part < 4; ++part) mx = max_part(sa, i, part, mx, Y, 0);
      raise(i, pair_max(mx));  // the sums are still zero
    }
#pragma unroll
    for (int e = 0; e < 8 * NM; ++e) exp_one(sa, e, Y, 0);
    __syncthreads();  // block 0's k has been read by every wave: kbuf[0] may be refilled
    // Block jb: its v and the next block's k are in LDS; meanwhile the v of the next block and the k of
    // the one after come in through registers, into the buffers that the block before used.
    int jb = 0;
    auto block = [&](auto masked) {
      const int b = jb & 1, kb = jb * BK;
      load(vbase, vst, kb + BK, vr);
      load(kbase, kst, kb + 2 * BK, kr);
      step(sa, sb, b, 0, b ^ 1, 0, masked, kb, N);
      step(sb, sa, b, 1, b ^ 1, 1, masked, kb + 32, Y);
      __syncthreads();
    };
    const int nfull = max(0, kv_len / BK - 1), nblk = (kv_len + BK - 1) / BK;
    for (; jb < nfull; ++jb) block(N);
    for (; jb < nblk; ++jb) block(Y);
    if (a.splits > 1) {
#pragma unroll
      for (int i = 0; i < NM; ++i) {
        l[i] = pair_sum(l[i]);
        lu[i] = pair_sum(lu[i]);
        if (qi < q_len) {
#pragma unroll
          for (int mt = 0; mt < MT; ++mt)
            store_dims(part_sums(a, sp, at, map + i, D) + 32 * mt, hf, o[i][mt], 1.f);
          if (hf == 0) *part_stat(a, sp, at, map + i, D) = make_float4(mc[i], l[i], lu[i], 0.f);
        }
      }
      continue;  // the last block of keys ended with a barrier
    }
#pragma unroll
    for (int i = 0; i < NM; ++i) {
      const float inv = 1.f / pair_sum(l[i]);
#pragma unroll
      for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int j = 0; j < 16; ++j) o[i][mt][j] *= inv;
      if (KEEP) {
        lu[i] = pair_sum(lu[i]);
        if (qi < q_len && hf == 0)
          a.lse[(int64_t)((map + i) * a.H + h) * a.total_q + q0 + qi] = mc[i] + log2f(lu[i]);
        if (qi < q_len)
#pragma unroll
          for (int mt = 0; mt < MT; ++mt)
            store_dims(a.maps + (2 * at + map + i) * D + 32 * mt, hf, o[i][mt], 1.f);
      }
    }
    const float lam = a.lambda[h];
    if constexpr (NM == 1) {  // the last block ended with a barrier: its buffers are free
      float* meet = (float*)lds + tile * 32 * D + lane;
      if (map == 1)
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
          for (int j = 0; j < 16; ++j) meet[(16 * mt + j) * 64] = lam * o[0][mt][j];
      __syncthreads();
      if (map == 0)
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
          for (int j = 0; j < 16; ++j) o[0][mt][j] -= meet[(16 * mt + j) * 64];
    } else {
#pragma unroll
      for (int mt = 0; mt < MT; ++mt)
#pragma unroll
        for (int j = 0; j < 16; ++j) o[0][mt][j] = fmaf(-lam, o[NM - 1][mt][j], o[0][mt][j]);
    }
    if (map == 0 && qi < q_len)
#pragma unroll
      for (int mt = 0; mt < MT; ++mt) store_dims((T*)a.out + at * D + 32 * mt, hf, o[0][mt], 1.f);
    __syncthreads();  // the next q tile of this block stages over these buffers
  }
}

// Joins the parts of the keys: one wave for a (query, head), D / 64 dims a lane.
template <typename T, int D>
__global__ void __launch_bounds__(kNT) da_join_kernel(const DaArgs a, int32_t B) {
  const int64_t at = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (at >= a.total_q * a.H) return;
  const int lane = threadIdx.x & 63, h = (int)(at % a.H);
  const int64_t row = at / a.H;
  // The sequence of the row, and its keys.
  bool in = false;
  int kv_len = 0;
  for (int b = lane; b < B; b += 64) {
    int q0, ql, k0, kl;
    segment(a.cu_q, b, a.total_q, &q0, &ql);
    segment(a.cu_kv, b, a.total_kv, &k0, &kl);
    if (row >= q0 && row < (int64_t)q0 + ql) {
      in = true;
      kv_len = kl;
    }
  }
  const uint64_t who = __builtin_amdgcn_ballot_w64(in);
  if (who == 0) return;
  kv_len = __shfl(kv_len, __builtin_ctzll(who), 64);
  const int64_t per = part_of(a, kv_len);
  const int parts = (int)((kv_len + per - 1) / per);
  float m[2], l[2] = {0.f, 0.f}, lu[2] = {0.f, 0.f}, o[2][D / 64] = {};
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    m[i] = -FLT_MAX;
    for (int p = lane; p < parts; p += 64) m[i] = fmaxf(m[i], part_stat(a, p, at, i, D)->x);
    for (int off = 32; off > 0; off >>= 1) m[i] = fmaxf(m[i], __shfl_xor(m[i], off, 64));
#pragma unroll 4
    for (int p = 0; p < parts; ++p) {  // independent loads, one order of the sums
      const float4 st = *part_stat(a, p, at, i, D);
      const float* po = part_sums(a, p, at, i, D);
      const float f = fast_exp2(st.x - m[i]);
      l[i] = fmaf(st.y, f, l[i]);
      lu[i] = fmaf(st.z, f, lu[i]);
#pragma unroll
      for (int e = 0; e < D / 64; ++e) o[i][e] = fmaf(po[lane + 64 * e], f, o[i][e]);
    }
  }
  const float i1 = parts ? 1.f / l[0] : 0.f, i2 = parts ? 1.f / l[1] : 0.f, lam = a.lambda[h];
#pragma unroll
  for (int e = 0; e < D / 64; ++e) {
    const int64_t p = at * D + lane + 64 * e;
    const float o1 = o[0][e] * i1, o2 = o[1][e] * i2;
    ((T*)a.out)[p] = (T)fmaf(-lam, o2, o1);  // one form, whether the maps are stored or not
    if (a.maps) {
      a.maps[at * 2 * D + lane + 64 * e] = o1;
      a.maps[at * 2 * D + D + lane + 64 * e] = o2;
    }
  }
  if (a.lse && lane == 0) {
    a.lse[(int64_t)h * a.total_q + row] = parts ? m[0] + log2f(lu[0]) : INFINITY;
    a.lse[(int64_t)(a.H + h) * a.total_q + row] = parts ? m[1] + log2f(lu[1]) : INFINITY;
  }
}

// ------------------------------------------------------------------------------- backward
// r_i = do . (P_i v) per query, from the sums in fp32: dS_i = P_i (dP - r_i) cancels where one key has most
// of a map, and out's rounding would be most of what is left (scores of standard deviation 4: dq off by 0.0042
// of its norm in bf16 instead of 0.0028).
// Block: one head, the rows of one sequence in steps of 256 / (D / 8) per grid column.
// Bound by memory: 20 us for the 117 MB of 7607 queries, 12 x 128 bf16, 5.8 TB/s.
template <typename T, int D>
__global__ void __launch_bounds__(kNT) da_rowdot_kernel(const DaArgs a, float* r12) {
  constexpr int LPR = D / 8;  // lanes of a row, 8 elements each
  constexpr int RPB = kNT / LPR;
  const int h = blockIdx.y, bb = blockIdx.z, e0 = threadIdx.x % LPR * 8;
  int q0, q_len;
  segment(a.cu_q, bb, a.total_q, &q0, &q_len);
  for (int64_t r = (int64_t)blockIdx.x * RPB + threadIdx.x / LPR; r < q_len;
       r += (int64_t)gridDim.x * RPB) {
    const int64_t at = ((q0 + r) * a.H + h) * D + e0;
    const T* d = (const T*)a.dout + at;
    const float* o = a.maps + 2 * (at - e0) + e0;
    float x[8], r1 = 0.f, r2 = 0.f;
#pragma unroll
    for (int c = 0; c < 8; c += 16 / sizeof(T)) {
      const u32x4_t w = *(const u32x4_t*)(d + c);
#pragma unroll
      for (int e = 0; e < (int)(16 / sizeof(T)); ++e) x[c + e] = (float)((const T*)&w)[e];
    }
#pragma unroll
    for (int c = 0; c < 8; c += 4) {
      const float4 y = *(const float4*)(o + c), z = *(const float4*)(o + D + c);
      r1 = fmaf(x[c + 3], y.w, fmaf(x[c + 2], y.z, fmaf(x[c + 1], y.y, fmaf(x[c], y.x, r1))));
      r2 = fmaf(x[c + 3], z.w, fmaf(x[c + 2], z.z, fmaf(x[c + 1], z.y, fmaf(x[c], z.x, r2))));
    }
#pragma unroll
    for (int off = LPR / 2; off > 0; off >>= 1) {
      r1 += __shfl_xor(r1, off, 64);
      r2 += __shfl_xor(r2, off, 64);
    }
    if (e0 == 0) {
      r12[(int64_t)h * a.total_q + q0 + r] = r1;
      r12[(int64_t)(a.H + h) * a.total_q + q0 + r] = r2;
    }
  }
}

// Both gradient kernels: a block's waves own 32 rows each and share the tiles of the other side, through
// two buffers in LDS; or, where that leaves CUs idle (SHARE), all own the same 32 rows and take the
// tiles in turn, each through its own piece of LDS, and their sums are joined at the end.
// Two waves per SIMD in 16 bits: with one, whose products, exponentials and LDS reads wait for each
// other, the matrix cores were busy 15 % of the time in dk / dv at D = 128, now 37 %.
// 4096 tokens: 12 x 128 bf16, dk and dv 410 us, dq 217 (755 and 715 TFLOP/s executed); 16 x 64 bf16 203
// and 155 (675 and 665); 8 x 64 fp32 640 and 500 (107 and 103 of the 154 that a large product reaches).
template <bool SHARE>
__device__ __forceinline__ void tile_sync() {
  // A wave's own LDS operations are carried out in order; the compiler has to keep that order.
  if (SHARE) __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  else __syncthreads();
}

// dq of 128 (32) queries; one block of each head also adds up dlambda.
template <typename T, int D, bool SHARE>
__global__ void __launch_bounds__(kNT, sizeof(T) == 2 && !SHARE ? 2 : 1) da_dq_kernel(const DaArgs a) {
  typedef Frag<T> F;
  typedef typename F::type Fr;
  typedef Tile<T, D> Ti;
  constexpr int BK = 32;
  constexpr int KS = D / 16, MT = D / 32;
  constexpr int TB = BK * Ti::ROWB, ROWS = SHARE ? 32 : kBQ, NT = SHARE ? 64 : kNT;
  __shared__ __attribute__((aligned(16))) unsigned char lds[SHARE ? 4 : 2][2 * TB];
  int bx, h, bb;
  block_tile(a.cu_kv, &bx, &h, &bb);
  int q0, q_len, kv0, kv_len;
  segment(a.cu_q, bb, a.total_q, &q0, &q_len);
  segment(a.cu_kv, bb, a.total_kv, &kv0, &kv_len);
  const int lane = threadIdx.x & 63, l32 = lane & 31, hf = lane >> 5;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), tid = SHARE ? lane : threadIdx.x;
  if (a.rest) zero_rest((T*)a.dq, a.cu_q, a.total_q, bb, a.H, D, h, bx, gridDim.x);
  if (bx == 0 && bb == 0 && w == 0 && a.dlambda) {
    double s = 0.;
    for (int i = lane; i < a.lam_parts; i += 64) s += (double)a.lam_part[(int64_t)h * a.lam_parts + i];
    for (int off = 32; off > 0; off >>= 1) s += __shfl_xor(s, off, 64);
    if (lane == 0) a.dlambda[h] = (float)s;
  }
  const T* kbase = (const T*)a.k + (int64_t)kv0 * a.ldk + (int64_t)h * D;
  const T* vbase = (const T*)a.v + (int64_t)kv0 * a.ldv + (int64_t)h * D;
  const float nlam = -a.lambda[h], scale = kv_len > 1 ? a.sl2 / kLog2e : 0.f;  // one key: P is constant

  for (int qt = bx * ROWS; qt < q_len; qt += gridDim.x * ROWS) {
    const int qi = qt + (SHARE ? 0 : w * 32) + l32;
    const int64_t qrow = q0 + min(qi, q_len - 1), stat = (int64_t)h * a.total_q + qrow;
    const int64_t map2 = (int64_t)a.H * a.total_q;
    Fr qf[KS], df[KS];
    {
      const T* p = (const T*)a.q + qrow * a.ldq + (int64_t)h * D + 8 * hf;
      const T* d = (const T*)a.dout + (qrow * a.H + h) * D + 8 * hf;
#pragma unroll
      for (int st = 0; st < KS; ++st) {
        qf[st] = F::load(p + 16 * st);
        df[st] = F::load(d + 16 * st);
      }
    }
    const float l1 = a.lse[stat], l2 = a.lse[map2 + stat], r1 = a.r12[stat], r2 = a.r12[map2 + stat];
    f32x16_t acc[MT];
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) clear(acc[mt]);
    Stage<T, D, BK, NT> ks, vs;
    constexpr int STEP = SHARE ? 4 * BK : BK;
    constexpr bool AHEAD = !SHARE || sizeof(T) == 2 || D == 64;  // registers for the next tile's rows
    int kb = SHARE ? w * BK : 0;
    auto load = [&](int k) {
      ks.load(kbase, a.ldk, k, kv_len, tid);
      vs.load(vbase, a.ldv, k, kv_len, tid);
    };
    if (AHEAD) load(kb);
    for (int buf = 0; kb < kv_len; kb += STEP, buf ^= 1) {
      unsigned char *kt = lds[SHARE ? w : buf], *vt = kt + TB;
      if (!AHEAD) load(kb);
      if (SHARE) tile_sync<SHARE>();
      ks.store(kt, tid);
      vs.store(vt, tid);
      tile_sync<SHARE>();
      if (AHEAD) load(kb + STEP);
      f32x16_t s1, s2, dp;
      clear(s1);
      clear(s2);
      clear(dp);
#pragma unroll
      for (int st = 0; st < KS; ++st) {
        F::mma(Ti::row(kt, 0, l32, hf, st), qf[st], st < KS / 2 ? s1 : s2);
        F::mma(Ti::row(vt, 0, l32, hf, st), df[st], dp);
      }
      if (kb + BK > kv_len) {  // uniform; the asm keeps it a branch, 48 instructions that no other tile needs
        asm volatile("");
#pragma unroll
        for (int j = 0; j < 16; ++j)
          if (kb + 8 * (j >> 2) + 4 * hf + (j & 3) >= kv_len) s1[j] = s2[j] = -INFINITY;
      }
      float d1[16], d2[16];
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        const float p1 = fast_exp2(fmaf(s1[j], a.sl2, -l1));
        const float p2 = fast_exp2(fmaf(s2[j], a.sl2, -l2));
        d1[j] = p1 * (dp[j] - r1);
        d2[j] = p2 * (dp[j] - r2);
      }
      const Fr f1[2] = {F::pack(d1), F::pack(d1 + 8)}, f2[2] = {F::pack(d2), F::pack(d2 + 8)};
#pragma unroll
      for (int g = 0; g < 2; ++g)
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
          F::mma(Ti::col(kt, 0, lane, g, mt), mt < MT / 2 ? f1[g] : f2[g], acc[mt]);
    }
    if (SHARE) join_waves<MT>((float*)lds, w, lane, acc);
    else __syncthreads();  // the next tile's rows go into these buffers
    if (qi < q_len && (!SHARE || w == 0)) {
      T* p = (T*)a.dq + ((int64_t)(q0 + qi) * a.H + h) * D;
#pragma unroll
      for (int mt = 0; mt < MT; ++mt)
        store_dims(p + 32 * mt, hf, acc[mt], mt < MT / 2 ? scale : nlam * scale);
    }
  }
}

// dk and dv of 128 (32) keys, and the block's part of dlambda = - sum P2 dP, from the unrounded fp32
// probabilities (do . (P2 v) with P2 v in 16 bits is off by 2^-9 of it).  The sequence ranking of
// block_tile goes by the queries here.
// A wave has NM maps of its 32 keys: both, or one where the registers of both (dk, dv, k and v: 192 at
// D = 128) leave one wave per SIMD.  Then dP is made twice, P1 and P2 are multiplied with do one by one
// (12 D flops a pair instead of 8 D), and the two waves' parts of dv meet in LDS at the end; 13 of the 256
// registers are spilled.
template <typename T, int D, bool SHARE, int NM>
__global__ void __launch_bounds__(SHARE ? kNT : 512 / NM, sizeof(T) == 2 && !SHARE ? 2 : 1)
    da_dkv_kernel(const DaArgs a) {
  typedef Frag<T> F;
  typedef typename F::type Fr;
  typedef Tile<T, D> Ti;
  constexpr int BQ = 32;
  constexpr int KS = D / 16, KH = KS / 2 * NM, MT = D / 32, MH = MT / 2 * NM;  // of the wave's maps
  constexpr int NW = SHARE ? 4 : 8 / NM, ROWS = SHARE ? 32 : 128, NT = SHARE ? 64 : 64 * NW;
  constexpr int TB = BQ * Ti::ROWB, MEET = NM == 1 ? 4 * 32 * D * 4 : 0;
  static_assert(!SHARE || NM == 2, "shared tiles: both maps");
  constexpr int BUFS = SHARE ? 4 : 2;
  __shared__ __attribute__((aligned(16))) unsigned char lds[BUFS * 2 * TB > MEET ? BUFS * 2 * TB : MEET];
  __shared__ __attribute__((aligned(16))) float stats[BUFS][4][BQ];  // log-sum-exps and r
  __shared__ float lam_sum[NW];
  int bx, h, bb;
  block_tile(a.cu_q, &bx, &h, &bb);
  int q0, q_len, kv0, kv_len;
  segment(a.cu_q, bb, a.total_q, &q0, &q_len);
  segment(a.cu_kv, bb, a.total_kv, &kv0, &kv_len);
  const int lane = threadIdx.x & 63, l32 = lane & 31, hf = lane >> 5;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), tid = SHARE ? lane : threadIdx.x;
  const int map = NM == 1 ? w & 1 : 0, tile = SHARE ? 0 : NM == 1 ? w >> 1 : w;  // first map; key tile
  if (a.rest) {
    zero_rest((T*)a.dk, a.cu_kv, a.total_kv, bb, a.H, D, h, bx, gridDim.x);
    zero_rest((T*)a.dv, a.cu_kv, a.total_kv, bb, a.H, D, h, bx, gridDim.x);
  }
  const T* qbase = (const T*)a.q + (int64_t)q0 * a.ldq + (int64_t)h * D;
  const T* dbase = (const T*)a.dout + ((int64_t)q0 * a.H + h) * D;
  const int64_t ldd = (int64_t)a.H * D;
  const float lam = a.lambda[h], scale = kv_len > 1 ? a.sl2 / kLog2e : 0.f;  // one key: P is constant
  // Thread tid < 128 brings statistic tid / 32 of query tid % 32; of one wave, each lane two.
  float dlam = 0.f;
  const int64_t sbase = ((int64_t)(tid & 32 ? a.H : 0) + h) * a.total_q + q0;

  for (int kt = bx * ROWS; kt < kv_len; kt += gridDim.x * ROWS) {
    const int ki = kt + tile * 32 + l32;
    const int64_t krow = kv0 + min(ki, kv_len - 1);
    Fr kf[KH], vf[KS];
    {
      const T* p = (const T*)a.k + krow * a.ldk + (int64_t)h * D + 8 * hf;
      const T* d = (const T*)a.v + krow * a.ldv + (int64_t)h * D + 8 * hf;
#pragma unroll
      for (int st = 0; st < KH; ++st) kf[st] = F::load(p + 16 * (map * KH + st));
#pragma unroll
      for (int st = 0; st < KS; ++st) vf[st] = F::load(d + 16 * st);
    }
    f32x16_t dk[MH], dv[MT];
#pragma unroll
    for (int mt = 0; mt < MH; ++mt) clear(dk[mt]);
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) clear(dv[mt]);
    Stage<T, D, BQ, NT> qs, ds;
    float sv[2] = {0.f, 0.f};
    constexpr int STEP = SHARE ? 4 * BQ : BQ;
    constexpr bool AHEAD = !SHARE || sizeof(T) == 2 || D == 64;
    auto load = [&](int qb) {
      qs.load(qbase, a.ldq, qb, q_len, tid);
      ds.load(dbase, ldd, qb, q_len, tid);
      const int r = qb + (tid & 31);
      if (SHARE || tid < 64) sv[0] = r < q_len ? a.lse[sbase + r] : INFINITY;
      if (SHARE || (tid >= 64 && tid < 128)) sv[1] = r < q_len ? a.r12[sbase + r] : 0.f;
    };
    int qb = SHARE ? w * BQ : 0;
    if (AHEAD) load(qb);
    for (int buf = 0; qb < q_len; qb += STEP, buf ^= 1) {
      unsigned char *qt = lds + (SHARE ? w : buf) * 2 * TB, *dt = qt + TB;
      float(*st4)[BQ] = stats[SHARE ? w : buf];
      if (!AHEAD) load(qb);
      if (SHARE) tile_sync<SHARE>();
      // Past the last query P = 2^(score - inf) = 0 and the row there is the last query's once more: a row of
      // zeros would make NaN of an infinite key, whose scores of -inf are 0 to every query.
      qs.template store<false>(qt, tid);
      ds.template store<false>(dt, tid);
      if (SHARE || tid < 64) st4[(tid >> 5) & 1][tid & 31] = sv[0];
      if (SHARE || (tid >= 64 && tid < 128)) st4[2 + ((tid >> 5) & 1)][tid & 31] = sv[1];
      tile_sync<SHARE>();
      if (AHEAD) load(qb + STEP);
      f32x16_t s[NM], dp;
#pragma unroll
      for (int i = 0; i < NM; ++i) clear(s[i]);
      clear(dp);
#pragma unroll
      for (int st = 0; st < KS; ++st) {
        F::mma(Ti::row(dt, 0, l32, hf, st), vf[st], dp);
        if (st < KH) F::mma(Ti::row(qt, 0, l32, hf, map * KH + st), kf[st], s[st / (KS / 2)]);
      }
      float p[16], d[NM][16], lsum = 0.f;
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        const int r = 8 * (j >> 2) + 4 * hf + (j & 3);
        if constexpr (NM == 2) {
          const float p1 = fast_exp2(fmaf(s[0][j], a.sl2, -st4[0][r]));
          const float q2 = fast_exp2(fmaf(s[1][j], a.sl2, -st4[1][r])), p2 = lam * q2;
          lsum = fmaf(q2, dp[j], lsum);
          p[j] = p1 - p2;
          d[0][j] = p1 * (dp[j] - st4[2][r]);
          d[1][j] = p2 * (st4[3][r] - dp[j]);
        } else {
          p[j] = fast_exp2(fmaf(s[0][j], a.sl2, -st4[map][r]));
          lsum = fmaf(p[j], dp[j], lsum);
          d[0][j] = p[j] * (dp[j] - st4[2 + map][r]);
        }
      }
      if (ki < kv_len && (NM == 2 || map == 1)) dlam -= lsum;  // lanes past the last key repeat it
#pragma unroll
      for (int g = 0; g < 2; ++g) {
        const Fr pf = F::pack(p + 8 * g);
        Fr df[NM];
#pragma unroll
        for (int i = 0; i < NM; ++i) df[i] = F::pack(d[i] + 8 * g);
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) {
          F::mma(Ti::col(dt, 0, lane, g, mt), pf, dv[mt]);
          if (mt < MH) F::mma(Ti::col(qt, 0, lane, g, map * MH + mt), df[mt / (MT / 2)], dk[mt]);
        }
      }
    }
    if (SHARE) {
      join_waves<MH>((float*)lds, w, lane, dk);
      join_waves<MT>((float*)lds, w, lane, dv);
    } else {
      __syncthreads();  // every wave has left the buffers
    }
    if constexpr (NM == 1) {
      float* meet = (float*)lds + tile * 32 * D + lane;
      if (map == 1)
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
          for (int j = 0; j < 16; ++j) meet[(16 * mt + j) * 64] = lam * dv[mt][j];
      __syncthreads();
      if (map == 0)
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
          for (int j = 0; j < 16; ++j) dv[mt][j] -= meet[(16 * mt + j) * 64];
      __syncthreads();
    }
    if (ki < kv_len && (!SHARE || w == 0)) {
      const int64_t at = ((int64_t)(kv0 + ki) * a.H + h) * D;
#pragma unroll
      for (int mt = 0; mt < MH; ++mt)
        store_dims((T*)a.dk + at + 32 * (map * MH + mt), hf, dk[mt], map == 1 ? -lam * scale : scale);
      if (map == 0)
#pragma unroll
        for (int mt = 0; mt < MT; ++mt) store_dims((T*)a.dv + at + 32 * mt, hf, dv[mt], 1.f);
    }
  }
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) dlam += __shfl_xor(dlam, off, 64);
  if (lane == 0) lam_sum[w] = dlam;
  __syncthreads();
  if (threadIdx.x == 0) {
    float t = lam_sum[0];
    for (int i = 1; i < NW; ++i) t += lam_sum[i];
    a.lam_part[((int64_t)h * gridDim.z + bb) * gridDim.x + bx] = t;
  }
}

// ------------------------------------------------------------------------------- host
constexpr int64_t kCUs = 256;

// Tiles of `rows` rows that the grid gives a sequence; the kernels' loops cover longer ones.
unsigned tiles_of(int64_t longest, int64_t hb, int rows = kBQ) {
  return (unsigned)std::max<int64_t>(
      1, std::min<int64_t>(std::min<int64_t>((longest + rows - 1) / rows, 65535), (INT32_MAX / 16) / hb));
}
// Rows of a block: 128, or 32 that its waves share.  Blocks of 32 are a quarter of the work each, and
// waste less of the last round over the CUs, but take longer for the joining and for copies that no other
// wave shares: `cost` tenths of a quarter of the other's time.  Measured, us, in blocks of 128 / of 32
// rows (the number of 128): fp32 8 x 64, dk and dv, 1024 tokens (64) 164 / 59, 2900 (184) 455 / 388,
// 4096 (256) 640 / 707, 5000 (320) 1538 / 1088; bf16 12 x 128, dk and dv, 512 (48) 37 / 25, 768 (72)
// 50 / 54, 1024 (96) 61 / 62, 4096 (384) 408 / 482; bf16 16 x 64, dq, 1024 (128) 29 / 22, 1536 (192)
// 41 / 41, 4096 (512) 156 / 218, its dk and dv 38 / 39, 54 / 75 and 202 / 432.
constexpr int kCostF32 = 12, kCost16 = 25, kCost16Dq64 = 15;
int block_rows(int cost, int64_t longest, int64_t hb) {
  const int64_t b = (int64_t)tiles_of(longest, hb) * hb, rounds = (b + kCUs - 1) / kCUs;
  return cost * ((4 * b + kCUs - 1) / kCUs) < 40 * rounds ? 32 : kBQ;
}
int dkv_rows(int32_t dtype, int64_t max_kv, int64_t hb) {
  return block_rows(dtype == TSC_F32 ? kCostF32 : kCost16, max_kv, hb);
}
int dq_rows(int32_t dtype, int32_t D, int64_t max_q, int64_t hb) {
  return block_rows(dtype == TSC_F32 ? kCostF32 : D == 64 ? kCost16Dq64 : kCost16, max_q, hb);
}

// The forward pass' blocks: query rows of each, and the parts of the keys.  Fewer blocks than CUs take
// the keys in parts, which da_join_kernel adds up, as many as run at once: two blocks of four waves on a
// CU (one query on 30000 keys, 16 x 64: 36 us, and 50 with one; 128 and 70 on 20000 and 9000: 53, 83), or
// one of eight at D = 128 in 16 bits.  There up to 32 queries have blocks of 64 rows and four waves (one
// query on each of 4 sequences, 32071 keys, 12 x 128: 43 us instead of 52; 33 rows: 41 instead of 32), in
// parts of 1024 keys or more (16 and 9 queries on 20000 and 9000 keys, 8 x 128: 32 us, 39 from 512 on).
// Grids of kCUs blocks are not split (900 + 700 tokens, 16 x 64, 256 blocks: 25 us, and 55 in two parts).
// Every query has scratch for as many parts as the longest sequence, so there are no more of them than fit
// four times what q, k, v and out take, or 64 MB (8192 queries on 64 sequences of which one has 220000 of
// 229376 keys, 1 x 64 f16: 54 parts in 241 MB, 103 us; 430 in 1.9 GB, 143 us; 14 in 67 MB, 293 us).
constexpr int64_t kScratchInputs = 4, kScratchLeast = 64 << 20;
// Scratch of a part: sums of D values and four statistics for each query, head and map.
int64_t part_bytes(int64_t total_q, int32_t H, int32_t D) { return 4 * total_q * H * 2 * (D + 4); }
struct Plan {
  int rows, splits, part_keys;
};
Plan da_plan(int32_t dtype, int32_t B, int64_t total_q, int64_t total_kv, int32_t H, int32_t D,
             int64_t max_q, int64_t max_kv) {
  const int64_t hb = (int64_t)H * B;
  max_q = std::max(max_q, (total_q + B - 1) / B);  // whatever the caller thinks: parts x rows of scratch
  Plan p = {kBQ, 1, INT32_MAX};
  int64_t slots = kCUs, least = 512;  // blocks that run at once, keys a part has at least
  if (dtype == TSC_F32) {
    p.rows = block_rows(kCostF32, max_q, hb);
    if (p.rows == kBQ) return p;  // 193 blocks of 128 and more: that kernel takes whole sequences
    least = 256;
  } else if (D == 64) {
    slots = 2 * kCUs;
  } else if (max_q <= 32) {  // four waves instead of eight
    p.rows = 64;
    slots = 2 * kCUs;
    least = 1024;
  }
  const int64_t blocks = (int64_t)tiles_of(max_q, hb, p.rows) * hb;
  if (blocks >= kCUs) return p;
  // Parts of one size, so that long sequences get more of them, and no more blocks than run at once: of
  // n a sequence's query tiles and heads can have, sum ceil(keys / part) <= total / part + B.
  const int64_t n = slots / (blocks / B) - B;
  if (n <= 0) return p;
  const int64_t part = std::max<int64_t>(least, ((total_kv + n - 1) / n + 63) / 64 * 64);
  const int64_t es = dtype == TSC_F32 ? 4 : 2, io = 2 * (total_q + total_kv) * H * D * es;
  const int64_t room = std::max(kScratchLeast, kScratchInputs * io) / part_bytes(total_q, H, D);
  p.splits = (int)std::max<int64_t>(1, std::min({(max_kv + part - 1) / part, slots, room}));
  if (p.splits > 1) p.part_keys = (int)std::min<int64_t>(part, INT32_MAX);
  return p;
}

// Blocks of the r kernel for a (head, sequence).
int rowdot_blocks(int64_t max_q) { return (int)std::min<int64_t>(std::max<int64_t>(1, (max_q + 63) / 64), 256); }

template <typename F>
int by_type(int32_t dtype, int32_t D, F f) {
  constexpr std::integral_constant<int, 64> D64{};
  constexpr std::integral_constant<int, 128> D128{};
  auto dims = [&](auto t) { D == 64 ? f(t, D64) : f(t, D128); };
  if (dtype == TSC_BF16) dims(__bf16());
  else if (dtype == TSC_F16) dims(_Float16());
  else dims(float());
  return check_hip(hipGetLastError(), "diff_attention launch");
}

DaArgs da_args(const DiffAttnArgs& x) {
  DaArgs a = {};
  a.q = x.q;
  a.k = x.k;
  a.v = x.v;
  a.ldq = x.ldq;
  a.ldk = x.ldk;
  a.ldv = x.ldv;
  a.lambda = x.lambda;
  a.cu_q = x.cu_q;
  a.cu_kv = x.cu_kv;
  a.total_q = x.total_q;
  a.total_kv = x.total_kv;
  a.H = x.H;
  a.sl2 = x.scale * kLog2e;
  a.rest = x.rest;
  a.splits = 1;
  return a;
}

}  // namespace

int64_t diff_attention_workspace_bytes(int32_t dtype, int32_t B, int64_t total_q, int64_t total_kv, int32_t H,
                                       int32_t D, int32_t max_q, int32_t max_kv, int32_t backward) {
  const int64_t hb = (int64_t)H * B;
  if (B == 0 || (total_q == 0 && !backward)) return 0;
  if (backward) return 4 * (2 * (int64_t)H * total_q + hb * tiles_of(max_kv, hb, dkv_rows(dtype, max_kv, hb)));
  const int s = da_plan(dtype, B, total_q, total_kv, H, D, max_q, max_kv).splits;
  return s > 1 ? s * part_bytes(total_q, H, D) : 0;
}

int diff_attention_launch(tsc_ctx* ctx, const DiffAttnArgs& x, void* out, float* maps, float* lse,
                          void* ws) {
  const int64_t hb = (int64_t)x.H * x.B;
  if (hb > (int64_t)(INT32_MAX / 1024))
    return fail(TSC_ERR_UNSUPPORTED, "diff_attention: %lld (head, sequence) pairs", (long long)hb);
  DaArgs a = da_args(x);
  a.out = out;
  a.maps = maps;
  a.lse = lse;
  const Plan plan = da_plan(x.dtype, x.B, x.total_q, x.total_kv, x.H, x.D, x.max_q, x.max_kv);
  a.splits = plan.splits;
  a.part_keys = plan.part_keys;
  a.part = (float*)ws;
  const unsigned gx = tiles_of(x.max_q, hb, plan.rows) * a.splits;
  const dim3 grid(gx, (unsigned)x.H, (unsigned)x.B);
  return by_type(x.dtype, x.D, [&](auto t, auto d) {
    using T = decltype(t);
    constexpr int D = decltype(d)::value;
    {
      ProfScope p(ctx, "diff_attention");
      if constexpr (sizeof(T) == 4) {
        if (plan.rows == 32) da_few32_kernel<D><<<grid, kNT, 0, ctx->stream>>>(a);
        else da_forward32_kernel<D><<<grid, kNT, 0, ctx->stream>>>(a);
      } else {
        auto run = [&](auto nm, auto nw) {
          constexpr int NM = decltype(nm)::value, NW = decltype(nw)::value;
          if (a.lse) da_forward16_kernel<T, D, NM, NW, true><<<grid, 64 * NW, 0, ctx->stream>>>(a);
          else da_forward16_kernel<T, D, NM, NW, false><<<grid, 64 * NW, 0, ctx->stream>>>(a);
        };
        constexpr std::integral_constant<int, 1> I1{};
        constexpr std::integral_constant<int, 2> I2{};
        constexpr std::integral_constant<int, 4> I4{};
        constexpr std::integral_constant<int, 8> I8{};
        if constexpr (D == 64) run(I2, I4);
        else if (plan.rows == 64) run(I1, I4);
        else run(I1, I8);
      }
    }
    if (a.splits > 1) {
      ProfScope p(ctx, "diff_attention_join");
      da_join_kernel<T, D><<<(unsigned)((x.total_q * x.H + 3) / 4), kNT, 0, ctx->stream>>>(a, x.B);
    }
  });
}

int diff_attention_backward_launch(tsc_ctx* ctx, const DiffAttnArgs& x, const float* maps,
                                   const float* lse, const void* dout, void* ws, void* dq, void* dk,
                                   void* dv, float* dlambda) {
  const int64_t hb = (int64_t)x.H * x.B;
  if (hb > (int64_t)(INT32_MAX / 1024))
    return fail(TSC_ERR_UNSUPPORTED, "diff_attention: %lld (head, sequence) pairs", (long long)hb);
  DaArgs a = da_args(x);
  a.maps = (float*)maps;
  a.lse = (float*)lse;
  a.dout = dout;
  a.dq = dq;
  a.dk = dk;
  a.dv = dv;
  a.dlambda = dlambda;
  float* r12 = (float*)ws;
  float* lam_part = r12 + 2 * (int64_t)x.H * x.total_q;
  a.r12 = r12;
  a.lam_part = lam_part;
  const int rq = dq_rows(x.dtype, x.D, x.max_q, hb), rk = dkv_rows(x.dtype, x.max_kv, hb);
  const dim3 gq(tiles_of(x.max_q, hb, rq), (unsigned)x.H, (unsigned)x.B);
  const dim3 gk(tiles_of(x.max_kv, hb, rk), (unsigned)x.H, (unsigned)x.B);
  a.lam_parts = (int)gk.x * x.B;
  return by_type(x.dtype, x.D, [&](auto t, auto d) {
    using T = decltype(t);
    constexpr int D = decltype(d)::value;
    {
      ProfScope p(ctx, "diff_attention_rowdot");
      da_rowdot_kernel<T, D><<<dim3((unsigned)rowdot_blocks(x.max_q), (unsigned)x.H, (unsigned)x.B),
                               kNT, 0, ctx->stream>>>(a, r12);
    }
    {
      ProfScope p(ctx, "diff_attention_dkv");
      constexpr int NM = sizeof(T) == 2 && D == 128 ? 1 : 2;
      if (rk == 32) da_dkv_kernel<T, D, true, 2><<<gk, kNT, 0, ctx->stream>>>(a);
      else da_dkv_kernel<T, D, false, NM><<<gk, 512 / NM, 0, ctx->stream>>>(a);
    }
    ProfScope p(ctx, "diff_attention_dq");
    if (rq == 32) da_dq_kernel<T, D, true><<<gq, kNT, 0, ctx->stream>>>(a);
    else da_dq_kernel<T, D, false><<<gq, kNT, 0, ctx->stream>>>(a);
  });
}

}  // namespace tsc
