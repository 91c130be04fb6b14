// Group norm over the rows of each sample, channels last, with an optional SiLU, and its gradient.
//
//   sample b = rows [cu[b], cu[b+1]) of x (N, C); its group g = channels [g C/G, (g+1) C/G); n values
//   mean = sum x / n;  var = sum (x - mean)^2 / n;  rstd = 1 / sqrt(var + eps)
//   xh = (x - mean) rstd;  h = xh gamma + beta;  y = h, or h s with s = 1 / (1 + exp(-h))
//   dh = dy, or dy s (1 + h (1 - s));  dbeta = sum dh;  dgamma = sum dh xh   (over all samples)
//   dx = rstd (gamma dh - A / n - xh B / n),  A = sum gamma dh, B = sum gamma dh xh  (sample, group)
//
// Bound by memory: the statistics need all of a sample before its first output, so x (and dy) is
// read twice, the second time from the 256 MB memory-side cache as far as it fits.  64304 x 1024 bf16
// with SiLU: 78 us, its three passes over 132 MB at 5.1 TB/s, the rate of a large copy.  Forward and gradient
// of 243547 x 512 bf16: 350 us, 8 passes over 249 MB at 5.7 TB/s.  In the gradient's sums, whose exponential
// and reciprocal per value take 40 % of the VALU's time, the VALU is busy 68 %.
// Two launches each way.  The rows are cut into T tiles and the channels into slabs
// of whole vectors; a block has one slab of the rows that a tile and a sample share, each thread one
// vector column and every TY-th row.  The first kernel leaves one partial result per (tile, sample,
// granule) - a granule is the largest run of channels that lies in one group and one slab - and each
// block of the second kernel adds up those of its own groups: a few KB from the L2, and no launch or
// atomic in between, so that the sums have one order.  Tile t and sample b meet in slot t + b: along
// the rows one of the two grows at each step, so slots are distinct; those in which a tile and a sample
// only touch, and those past the last, hold zeros, so that all T + B of them are written.
// Statistics are fp32 (mean, M2) pairs about their own means, merged pairwise, and merged over tiles
// in fp64 about the first one's mean: no sum of squares of raw values, which would lose a spread
// that is small beside the mean.

#include <algorithm>
#include <initializer_list>
#include <type_traits>

#include "rownorm.h"
#include "tsc_internal.h"

namespace tsc {
namespace {

constexpr int kNT = 512;       // threads of a block, two of which fill a CU (128 registers)
constexpr int kParamCh = 8;    // channels of a block that adds up dgamma and dbeta
constexpr int kSlab = 256;     // channels of a slab, at most

struct GnShape {
  const int32_t* cu;  // null: B samples of N / B rows
  int64_t N, each;    // each = N / B
  int32_t B, C, groups, cpg;  // cpg = C / groups
  int32_t nvec, TX, TY, slabs;
  int32_t T;           // row tiles
  int64_t R;           // rows of a tile
  int32_t gran, NG, GP;  // channels of a granule, granules in all, granules of a group
  int32_t sub, lsub;     // channels of one granule that a vector holds side by side, a power of 2; its log
};

template <typename T, int VN>
struct __attribute__((aligned(VN * sizeof(T)))) Pack {
  T v[VN];
};
template <int BYTES>
struct Word;
template <>
struct Word<16> { typedef uint32_t type __attribute__((ext_vector_type(4))); };
template <>
struct Word<8> { typedef uint32_t type __attribute__((ext_vector_type(2))); };
template <>
struct Word<4> { typedef uint32_t type; };
template <>
struct Word<2> { typedef uint16_t type; };

// Outputs are next read by another layer's kernel; x is what the second pass wants kept.
template <typename T, int VN>
__device__ __forceinline__ void store_nt(T* p, const float (&f)[VN]) {
  Pack<T, VN> o;
#pragma unroll
  for (int e = 0; e < VN; ++e) o.v[e] = (T)f[e];
  typedef typename Word<VN * sizeof(T)>::type W;
  __builtin_nontemporal_store(__builtin_bit_cast(W, o), (W*)p);
}

__device__ __forceinline__ void gn_segment(const GnShape& s, int b, int64_t* lo, int64_t* hi) {
  if (!s.cu) {
    *lo = b * s.each;
    *hi = *lo + s.each;
    return;
  }
  *lo = min<int64_t>(max<int64_t>(s.cu[b], 0), s.N);
  *hi = min<int64_t>(max<int64_t>(s.cu[b + 1], *lo), s.N);
}

__device__ __forceinline__ int tile_of(const GnShape& s, int64_t row) {  // rows and R fit 31 bits
  return (int)((uint32_t)row / (uint32_t)s.R);
}

// The sample of a slot: the last one whose first slot, tile_of(its first row) + its number, is not past
// it.  Every lane of the wave takes part.
__device__ __forceinline__ int slot_sample(const GnShape& s, int slot) {
  if (s.B == 1) return 0;
  auto starts = [&](int b) {
    const int64_t row = s.cu ? min<int64_t>(max<int64_t>(s.cu[b], 0), s.N) : b * s.each;
    return tile_of(s, row) + b <= slot;
  };
  int lo = 0, n = min(s.B, 64);
  if (s.B > 64) {  // until 64 are left
    int hi = s.B;  // it is in [lo, hi)
    while (hi - lo > 64) {
      const int mid = (lo + hi) >> 1;
      if (starts(mid)) lo = mid;
      else hi = mid;
    }
    n = hi - lo;
  }
  const int k = threadIdx.x & 63;
  return lo + max(0, __popcll(__builtin_amdgcn_ballot_w64(k < n && starts(lo + min(k, n - 1)))) - 1);
}

// What a block does: a slot's tile and sample, their common rows, and the thread's place in a slab.
struct Where {
  int slot, slab, col, ty, c0;  // vector column, first row's lane, first channel
  bool live;
  int b;
  int64_t r0, r1;    // the tile's rows
  int64_t beg, end;  // the sample's
  int64_t lo, hi;    // both
};
template <int VN>
__device__ __forceinline__ Where columns(const GnShape& s, int slab) {
  Where w;
  w.slab = slab;
  w.col = threadIdx.x % s.TX;
  w.ty = threadIdx.x / s.TX;
  const int vec = slab * s.TX + w.col;
  w.live = w.ty < s.TY && vec < s.nvec;
  w.c0 = vec * VN;
  return w;
}
template <int VN>
__device__ __forceinline__ Where where(const GnShape& s, int slot, int slab) {
  Where w = columns<VN>(s, slab);
  w.slot = slot;
  w.b = slot_sample(s, slot);
  gn_segment(s, w.b, &w.beg, &w.end);
  w.r0 = min<int64_t>(max(slot - w.b, 0) * s.R, s.N);
  w.r1 = min<int64_t>(w.r0 + s.R, s.N);
  w.lo = max(w.beg, w.r0);
  w.hi = min(w.end, w.r1);
  return w;
}

// Zeros for the tile's rows before the first sample and after the last one, by the slots of those.
template <typename T, int VN>
__device__ __forceinline__ void zero_rest(const GnShape& s, const Where& w, T* y) {
  if (!s.cu || !w.live || (w.b != 0 && w.b != s.B - 1)) return;
  const int64_t before = w.b == 0 ? w.beg : 0, after = w.b == s.B - 1 ? w.end : s.N;
  const float z[VN] = {};
  for (int64_t r = w.r0 + w.ty; r < w.r1; r += s.TY)
    if (r < before || r >= after) store_nt<T, VN>(y + r * s.C + w.c0, z);
}

// Merges elements e and e + STEP of n values each (e a multiple of 2 STEP) into e; the count doubles for
// all of them, which the caller's n, a count of rows, leaves out.
template <int STEP, int VN>
__device__ __forceinline__ void pair_up(float (&mean)[VN], float (&m2)[VN], float rows) {
#pragma unroll
  for (int e = 0; e + STEP < VN; e += 2 * STEP) {
    const float d = mean[e + STEP] - mean[e];
    mean[e] = fmaf(0.5f, d, mean[e]);
    m2[e] = fmaf(d * d, 0.5f * STEP * rows, m2[e] + m2[e + STEP]);
  }
}

// ------------------------------------------------------------------------------- forward
// Mean and M2 of rows lo .. hi - 1 for each unit (the channels of a granule within a vector) of every
// vector column, in order, in smean and sm2 (kNT VN floats each; scnt: kNT).
template <typename T, int VN>
__device__ __forceinline__ void tile_stats(const GnShape& s, const Where& w, int64_t lo, int64_t hi,
                                           const T* __restrict__ x, float* smean, float* sm2,
                                           float* scnt) {
  constexpr int KR = 4;  // rows in flight per thread (8: 128 registers do not hold them)
  const int tid = threadIdx.x;
  float cnt = 0.f, mean[VN], m2[VN];
#pragma unroll
  for (int e = 0; e < VN; ++e) mean[e] = m2[e] = 0.f;
  if (w.live) {
    const T* p = x + w.c0;
    auto chunk = [&](int64_t r, int k, auto whole) {  // rows r, r + TY, ..., k of them
      Pack<T, VN> v[KR];
#pragma unroll
      for (int i = 0; i < KR; ++i)
        if (decltype(whole)::value || i < k)
          v[i] = *(const Pack<T, VN>*)(p + (r + (int64_t)i * s.TY) * s.C);
      const float kf = decltype(whole)::value ? (float)KR : (float)k, ik = 1.f / kf;
      const float f = kf / (cnt + kf);
#pragma unroll
      for (int e = 0; e < VN; ++e) {
        float a = 0.f, q = 0.f;
#pragma unroll
        for (int i = 0; i < KR; ++i)
          if (decltype(whole)::value || i < k) a += (float)v[i].v[e];
        a *= ik;
#pragma unroll
        for (int i = 0; i < KR; ++i)
          if (decltype(whole)::value || i < k) {
            const float d = (float)v[i].v[e] - a;
            q = fmaf(d, d, q);
          }
        const float d = a - mean[e];
        mean[e] = fmaf(d, f, mean[e]);
        m2[e] += fmaf(d * d, f * cnt, q);
      }
      cnt += kf;
    };
    int64_t r = lo + w.ty;
    for (; r + (int64_t)(KR - 1) * s.TY < hi; r += (int64_t)KR * s.TY) chunk(r, KR, std::true_type());
    if (r < hi) chunk(r, (int)((hi - r + s.TY - 1) / s.TY), std::false_type());
  }
  // The channels of a granule within the thread's vector: equal counts.
  if (VN >= 2 && s.sub >= 2) pair_up<1>(mean, m2, cnt);
  if (VN >= 4 && s.sub >= 4) pair_up<2>(mean, m2, cnt);
  if (VN >= 8 && s.sub >= 8) pair_up<4>(mean, m2, cnt);
  const int units = VN >> s.lsub;  // unit i is element i * sub
#pragma unroll
  for (int e = 0; e < VN; ++e)
    if ((e & (s.sub - 1)) == 0) {
      smean[tid * units + (e >> s.lsub)] = mean[e];
      sm2[tid * units + (e >> s.lsub)] = m2[e];
    }
  scnt[tid] = cnt;
  __syncthreads();
  int half = 1;
  while (2 * half < s.TY) half *= 2;
  for (; half > 0 && s.TY > 1; half >>= 1) {
    if (w.ty < half && w.ty + half < s.TY) {
      const int o = tid + half * s.TX;
      const float nb = scnt[o];
      if (nb > 0.f) {
        const float f = nb / (cnt + nb);
#pragma unroll
        for (int e = 0; e < VN; ++e)
          if ((e & (s.sub - 1)) == 0) {
            const int u = e >> s.lsub;
            const float d = smean[o * units + u] - mean[e];
            mean[e] = fmaf(d, f, mean[e]);
            m2[e] += fmaf(d * d, f * cnt * (float)s.sub, sm2[o * units + u]);
            smean[tid * units + u] = mean[e];
            sm2[tid * units + u] = m2[e];
          }
        cnt += nb;
        scnt[tid] = cnt;
      }
    }
    __syncthreads();
  }
}

// Granule i's mean and M2 from tile_stats' units.
__device__ __forceinline__ float2 granule(const GnShape& s, int i, int64_t rows, const float* smean,
                                          const float* sm2) {
  const int per = s.gran >> s.lsub;
  const float* mc = smean + i * per;
  const float* qc = sm2 + i * per;
  float a = 0.f, q = 0.f;
  for (int c = 1; c < per; ++c) a += mc[c] - mc[0];
  a = mc[0] + a / (float)per;
  for (int c = 0; c < per; ++c) {
    const float d = mc[c] - a;
    q += fmaf(d * d, (float)(rows * s.sub), qc[c]);
  }
  return make_float2(a, q);
}

// How many of rows lo .. hi - 1 are the thread's: lo + ty and every TY-th one from there.
__device__ __forceinline__ int64_t thread_rows(const GnShape& s, const Where& w, int64_t lo, int64_t hi) {
  return hi - lo > w.ty ? (hi - lo - w.ty + s.TY - 1) / s.TY : 0;
}

// The second pass goes from the last rows on: they were read last and are still in the memory-side cache.
// Its first whole chunk is fetched ahead, before the sums that everything else waits for.
constexpr int kApplyRows = 4;
template <typename T, int VN>
struct ApplyRows {
  Pack<T, VN> v[kApplyRows];
  __device__ __forceinline__ void fetch(const T* x, int64_t at, int64_t step) {
#pragma unroll
    for (int k = 0; k < kApplyRows; ++k) v[k] = *(const Pack<T, VN>*)(x + at + k * step);
  }
  __device__ __forceinline__ void ahead(const GnShape& s, const Where& w, int64_t lo, int64_t hi,
                                        const T* x) {
    const int64_t whole = thread_rows(s, w, lo, hi) / kApplyRows * kApplyRows;
    if (w.live && whole > 0)
      fetch(x, (lo + w.ty + (whole - kApplyRows) * s.TY) * s.C + w.c0, (int64_t)s.TY * s.C);
  }
};

// y of rows lo .. hi - 1 from the groups' (mean, rstd) in sg (group gl first).
template <typename T, int VN>
__device__ __forceinline__ void apply_rows(const GnShape& s, const Where& w, int64_t lo, int64_t hi,
                                           const float2* sg, int gl, const T* x,
                                           const T* __restrict__ gamma, const T* __restrict__ beta,
                                           int32_t silu, T* y, ApplyRows<T, VN>& rows) {
  if (!w.live) return;
  float mean[VN], a[VN], c[VN];
#pragma unroll
  for (int e = 0; e < VN; ++e) {
    const float2 m = sg[(w.c0 + e) / s.cpg - gl];
    mean[e] = m.x;
    a[e] = m.y * (gamma ? (float)gamma[w.c0 + e] : 1.f);
    c[e] = beta ? (float)beta[w.c0 + e] : 0.f;
  }
  const int64_t n = thread_rows(s, w, lo, hi), whole = n / kApplyRows * kApplyRows;
  const int64_t step = (int64_t)s.TY * s.C, at0 = (lo + w.ty) * s.C + w.c0;
  auto one = [&](int64_t i, const Pack<T, VN>& v) {
    float o[VN];
#pragma unroll
    for (int e = 0; e < VN; ++e) {
      const float h = fmaf((float)v.v[e] - mean[e], a[e], c[e]);
      o[e] = silu ? h * __builtin_amdgcn_rcpf(1.f + __expf(-h)) : h;
    }
    store_nt<T, VN>(y + at0 + i * step, o);
  };
  for (int64_t i = whole; i > 0; i -= kApplyRows) {
    if (i < whole) rows.fetch(x, at0 + (i - kApplyRows) * step, step);
#pragma unroll
    for (int k = 0; k < kApplyRows; ++k) one(i - kApplyRows + k, rows.v[k]);
  }
  for (int64_t i = whole; i < n; ++i) one(i, *(const Pack<T, VN>*)(x + at0 + i * step));
}

// Partial statistics: part[slot * NG + granule] = (mean, M2).
template <typename T, int VN>
__global__ void __launch_bounds__(kNT, 4)
    gn_stats_kernel(GnShape s, const T* __restrict__ x, float2* __restrict__ part) {
  __shared__ float smean[kNT * VN], sm2[kNT * VN], scnt[kNT];
  const Where w = where<VN>(s, blockIdx.x, blockIdx.y);
  const int tid = threadIdx.x, SC = s.TX * VN;
  const int g0 = w.slab * SC / s.gran, ng = min(SC / s.gran, s.NG - g0);
  float2* dst = part + (int64_t)w.slot * s.NG + g0;
  if (w.hi <= w.lo) {  // uniform over the block
    for (int i = tid; i < ng; i += kNT) dst[i] = make_float2(0.f, 0.f);
    return;
  }
  tile_stats<T, VN>(s, w, w.lo, w.hi, x, smean, sm2, scnt);
  for (int i = tid; i < ng; i += kNT) dst[i] = granule(s, i, w.hi - w.lo, smean, sm2);
}

// Columns of threads, a power of two: thread tid adds up group tid % columns, so that neighbors read
// neighboring partials.
__device__ __forceinline__ int sum_columns(int ng) {
  int c = 1;
  while (c < ng) c <<= 1;
  return c;
}

// Adds a pair of doubles over the threads of each column; those of the first row have the sums.
__device__ __forceinline__ void column_sum(double* sa, double* sb, int columns, double* a, double* b) {
  const int tid = threadIdx.x;
  sa[tid] = *a;
  sb[tid] = *b;
  __syncthreads();
  for (int half = kNT / 2; half >= columns; half >>= 1) {
    if (tid < half) {
      *a += sa[tid + half];
      *b += sb[tid + half];
      sa[tid] = *a;
      sb[tid] = *b;
    }
    __syncthreads();
  }
}

template <typename T, int VN>
__global__ void __launch_bounds__(kNT, 4)
    gn_apply_kernel(GnShape s, const T* x, const float2* __restrict__ part,
                    const T* __restrict__ gamma, const T* __restrict__ beta, float eps,
                    int32_t silu, int32_t rest, float* __restrict__ stats, T* y) {
  __shared__ double sa[kNT], sb[kNT];
  __shared__ float2 sg[kSlab];
  const Where w = where<VN>(s, blockIdx.x, blockIdx.y);
  const int tid = threadIdx.x, SC = s.TX * VN;
  const int gl = w.slab * SC / s.cpg, gh = (min((w.slab + 1) * SC, s.C) - 1) / s.cpg;
  const int ng = gh - gl + 1, cols = sum_columns(ng), P = kNT / cols;
  if (rest) zero_rest<T, VN>(s, w, y);
  if (w.hi <= w.lo) return;  // uniform over the block
  ApplyRows<T, VN> rows;
  rows.ahead(s, w, w.lo, w.hi, x);
  const int64_t beg = w.beg, end = w.end;
  {
    const int t0 = tile_of(s, beg), nt = tile_of(s, end - 1) - t0 + 1;
    const int g = gl + (tid & (cols - 1)), j = tid / cols;
    double n = 0., d1 = 0., d2 = 0.;
    float m0 = 0.f;
    if (g <= gh) {
      const float2* src = part + (int64_t)(t0 + w.b) * s.NG + (int64_t)g * s.GP;
      m0 = src->x;
      for (int k = 0; k < s.GP; ++k)
#pragma unroll 4
        for (int i = j; i < nt; i += P) {
          const float2 p = src[(int64_t)i * s.NG + k];
          const int64_t a0 = max(beg, (t0 + i) * s.R), a1 = min(end, (t0 + i + 1) * s.R);
          const double c = (double)((a1 - a0) * s.gran), d = (double)p.x - (double)m0;
          d1 += c * d;
          d2 += (double)p.y + c * d * d;
        }
    }
    column_sum(sa, sb, cols, &d1, &d2);
    if (g <= gh && j == 0) {
      n = (double)(end - beg) * s.cpg;
      const double mean = (double)m0 + d1 / n;
      const double q = d2 - d1 * d1 / n;
      const double var = q < 0. ? 0. : q / n;  // NaN stays
      const float2 r = make_float2((float)mean, (float)(1. / sqrt(var + (double)eps)));
      sg[g - gl] = r;
      if (stats && w.r0 <= beg && g * s.cpg >= w.slab * SC)
        *(float2*)(stats + 2 * ((int64_t)w.b * s.groups + g)) = r;
    }
    __syncthreads();
  }
  apply_rows<T, VN>(s, w, w.lo, w.hi, sg, gl, x, gamma, beta, silu, y, rows);
}

// ------------------------------------------------------------------------------- backward
// dh of one value, from x - mean: h = (x - mean) rstd gamma + beta.
__device__ __forceinline__ float grad_one(float xm, float dy, float a, float beta, int silu) {
  if (!silu) return dy;
  const float h = fmaf(xm, a, beta);
  const float sg = __builtin_amdgcn_rcpf(1.f + __expf(-h));
  return dy * sg * fmaf(h, 1.f - sg, 1.f);
}

// The thread's per-channel constants of sample b: mean, rstd, rstd gamma, beta.
template <typename T, int VN>
__device__ __forceinline__ void channel_consts(const GnShape& s, int b, int c0, const float* stats,
                                               const T* gamma, const T* beta, float (&mean)[VN],
                                               float (&rstd)[VN], float (&a)[VN], float (&be)[VN]) {
#pragma unroll
  for (int e = 0; e < VN; ++e) {
    const float2 m = *(const float2*)(stats + 2 * ((int64_t)b * s.groups + (c0 + e) / s.cpg));
    mean[e] = m.x;
    rstd[e] = m.y;
    a[e] = m.y * (gamma ? (float)gamma[c0 + e] : 1.f);
    be[e] = beta ? (float)beta[c0 + e] : 0.f;
  }
}

// Sums over a tile's rows of one sample: pc[slot * C + channel] = (sum dh, sum dh xh), and
// pg[slot * NG + granule] the same weighted with gamma and summed over the granule.
template <typename T, int VN>
__global__ void __launch_bounds__(kNT, 4)
    gn_grad_sums_kernel(GnShape s, const T* __restrict__ dy, const T* __restrict__ x,
                        const float* __restrict__ stats, const T* __restrict__ gamma,
                        const T* __restrict__ beta, int32_t silu, float2* __restrict__ pc,
                        float2* __restrict__ pg) {
  constexpr int KR = 2;
  __shared__ float s1[kNT * VN], s2[kNT * VN];
  const Where w = where<VN>(s, blockIdx.x, blockIdx.y);
  const int tid = threadIdx.x, SC = s.TX * VN;
  const int g0 = w.slab * SC / s.gran, ng = min(SC / s.gran, s.NG - g0);
  const int ch0 = w.slab * SC, nch = min(SC, s.C - ch0);
  const int b = w.b;
  const int64_t lo = w.lo, hi = w.hi;
  float2* dc = pc + (int64_t)w.slot * s.C + ch0;
  float2* dg = pg + (int64_t)w.slot * s.NG + g0;
  if (hi <= lo) {
    for (int i = tid; i < nch; i += kNT) dc[i] = make_float2(0.f, 0.f);
    for (int i = tid; i < ng; i += kNT) dg[i] = make_float2(0.f, 0.f);
    return;
  }
  float a1[VN], a2[VN];
#pragma unroll
  for (int e = 0; e < VN; ++e) a1[e] = a2[e] = 0.f;
  if (w.live) {
    float mean[VN], rstd[VN], a[VN], be[VN];
    channel_consts<T, VN>(s, b, w.c0, stats, gamma, beta, mean, rstd, a, be);
    auto chunk = [&](int64_t r, int k, auto whole) {
      Pack<T, VN> vx[KR], vy[KR];
#pragma unroll
      for (int i = 0; i < KR; ++i)
        if (decltype(whole)::value || i < k) {
          const int64_t at = (r + (int64_t)i * s.TY) * s.C + w.c0;
          vx[i] = *(const Pack<T, VN>*)(x + at);
          vy[i] = *(const Pack<T, VN>*)(dy + at);
        }
#pragma unroll
      for (int i = 0; i < KR; ++i)
        if (decltype(whole)::value || i < k)
#pragma unroll
          for (int e = 0; e < VN; ++e) {
            const float xm = (float)vx[i].v[e] - mean[e];
            const float dh = grad_one(xm, (float)vy[i].v[e], a[e], be[e], silu);
            a1[e] += dh;
            a2[e] = fmaf(dh, xm, a2[e]);
            if (e & 1) __builtin_amdgcn_sched_barrier(0);
          }
    };
    int64_t r = lo + w.ty;
    for (; r + (int64_t)(KR - 1) * s.TY < hi; r += (int64_t)KR * s.TY) chunk(r, KR, std::true_type());
    if (r < hi) chunk(r, (int)((hi - r + s.TY - 1) / s.TY), std::false_type());
#pragma unroll
    for (int e = 0; e < VN; ++e)
      a2[e] *= stats[2 * ((int64_t)b * s.groups + (w.c0 + e) / s.cpg) + 1];
  }
  __syncthreads();
#pragma unroll
  for (int e = 0; e < VN; ++e) {
    s1[tid * VN + e] = a1[e];
    s2[tid * VN + e] = a2[e];
  }
  __syncthreads();
  int half = 1;
  while (2 * half < s.TY) half *= 2;
  for (; half > 0 && s.TY > 1; half >>= 1) {
    if (w.ty < half && w.ty + half < s.TY) {
      const int o = tid + half * s.TX;
#pragma unroll
      for (int e = 0; e < VN; ++e) {
        a1[e] += s1[o * VN + e];
        a2[e] += s2[o * VN + e];
        s1[tid * VN + e] = a1[e];
        s2[tid * VN + e] = a2[e];
      }
    }
    __syncthreads();
  }
  for (int i = tid; i < nch; i += kNT) dc[i] = make_float2(s1[i], s2[i]);
  // The first TX threads have the totals: weighted with gamma, and the granules joined in LDS.
  __syncthreads();
  if (w.ty == 0 && w.live) {
    float u = 0.f, v = 0.f;
#pragma unroll
    for (int e = 0; e < VN; ++e) {
      const float g = gamma ? (float)gamma[w.c0 + e] : 1.f;
      u = fmaf(g, a1[e], u);
      v = fmaf(g, a2[e], v);
      if (((e + 1) & (s.sub - 1)) == 0) {
        s1[(w.col * VN + e) >> s.lsub] = u;
        s2[(w.col * VN + e) >> s.lsub] = v;
        u = v = 0.f;
      }
    }
  }
  __syncthreads();
  const int per = s.gran >> s.lsub;
  for (int i = tid; i < ng; i += kNT) {
    float u = 0.f, v = 0.f;
    for (int c = i * per; c < (i + 1) * per; ++c) {
      u += s1[c];
      v += s2[c];
    }
    dg[i] = make_float2(u, v);
  }
}

// dx; the first pblocks blocks add up dgamma and dbeta instead, 8 channels each, in the grid's first
// prows rows, whose other blocks have nothing to do.  A row holds the slots of a slab: along one axis of a
// launch there may be 2^32 - 1 threads only, which 2^20 samples would pass with 8 slabs.
template <typename T, int VN>
__global__ void __launch_bounds__(kNT, 4)
    gn_grad_kernel(GnShape s, const T* dy, const T* x, const float* __restrict__ stats,
                   const T* __restrict__ gamma, const T* __restrict__ beta, int32_t silu,
                   int32_t rest, int32_t pblocks, int32_t prows, const float2* __restrict__ pc,
                   const float2* __restrict__ pg, T* dx, T* dgamma, T* dbeta) {
  constexpr int KR = 2;
  __shared__ double sa[kNT], sb[kNT];
  __shared__ float2 sg[kSlab];
  const int tid = threadIdx.x;
  if ((int)blockIdx.y < prows) {
    const int pb = blockIdx.y * gridDim.x + blockIdx.x;
    if (pb >= pblocks) return;  // uniform over the block
    const int e = tid % kParamCh, j = tid / kParamCh, c = pb * kParamCh + e;
    double u = 0., v = 0.;
    if (c < s.C)
      for (int i = j; i < s.T + s.B; i += kNT / kParamCh) {
        const float2 p = pc[(int64_t)i * s.C + c];
        u += (double)p.x;
        v += (double)p.y;
      }
    sa[tid] = u;
    sb[tid] = v;
    __syncthreads();
    for (int half = kNT / 2; half >= kParamCh; half >>= 1) {
      if (tid < half) {
        sa[tid] += sa[tid + half];
        sb[tid] += sb[tid + half];
      }
      __syncthreads();
    }
    if (tid < kParamCh && c < s.C) {
      if (dbeta) dbeta[c] = (T)(float)sa[tid];
      if (dgamma) dgamma[c] = (T)(float)sb[tid];
    }
    return;
  }
  const Where w = where<VN>(s, blockIdx.x, blockIdx.y - prows);
  const int SC = s.TX * VN;
  const int gl = w.slab * SC / s.cpg, gh = (min((w.slab + 1) * SC, s.C) - 1) / s.cpg;
  const int ng = gh - gl + 1, cols = sum_columns(ng), P = kNT / cols;
  if (rest) zero_rest<T, VN>(s, w, dx);
  if (w.hi <= w.lo) return;  // uniform over the block
  const int b = w.b;
  const int64_t beg = w.beg, end = w.end, lo = w.lo, hi = w.hi;
  const int64_t n = thread_rows(s, w, lo, hi), whole = n / KR * KR;
  const int64_t step = (int64_t)s.TY * s.C, at0 = (lo + w.ty) * s.C + w.c0;
  Pack<T, VN> vx[KR], vy[KR];  // from the last rows on, the first whole chunk ahead of the sums
  auto fetch = [&](int64_t i) {
#pragma unroll
    for (int k = 0; k < KR; ++k) {
      vx[k] = *(const Pack<T, VN>*)(x + at0 + (i + k) * step);
      vy[k] = *(const Pack<T, VN>*)(dy + at0 + (i + k) * step);
    }
  };
  if (w.live && whole > 0) fetch(whole - KR);
  {
    const int t0 = tile_of(s, beg), nt = tile_of(s, end - 1) - t0 + 1;
    const int g = gl + (tid & (cols - 1)), j = tid / cols;
    double u = 0., v = 0.;
    if (g <= gh) {
      const float2* src = pg + (int64_t)(t0 + b) * s.NG + (int64_t)g * s.GP;
      for (int k = 0; k < s.GP; ++k)
#pragma unroll 4
        for (int i = j; i < nt; i += P) {
          const float2 p = src[(int64_t)i * s.NG + k];
          u += (double)p.x;
          v += (double)p.y;
        }
    }
    column_sum(sa, sb, cols, &u, &v);
    if (g <= gh && j == 0) {
      const double n = (double)(end - beg) * s.cpg;
      sg[g - gl] = make_float2((float)(u / n), (float)(v / n));
    }
    __syncthreads();
  }
  if (w.live) {
    // dx = rstd gamma dh - rstd A / n - (x - mean) rstd^2 B / n
    float mean[VN], rstd[VN], a[VN], be[VN], ma[VN], mb[VN];
    const bool alone = (end - beg) * s.cpg == 1;  // a single value's norm is 0 whatever it is: so is dx
    channel_consts<T, VN>(s, b, w.c0, stats, gamma, beta, mean, rstd, a, be);
#pragma unroll
    for (int e = 0; e < VN; ++e) {
      const float2 m = sg[(w.c0 + e) / s.cpg - gl];
      ma[e] = m.x * rstd[e];
      mb[e] = m.y * rstd[e] * rstd[e];
      if (alone) a[e] = ma[e] = 0.f;
    }
    auto one = [&](int64_t i, const Pack<T, VN>& px, const Pack<T, VN>& py) {
      float o[VN];
#pragma unroll
      for (int e = 0; e < VN; ++e) {
        const float xm = (float)px.v[e] - mean[e];
        const float dh = grad_one(xm, (float)py.v[e], a[e], be[e], silu);
        o[e] = fmaf(-xm, mb[e], fmaf(a[e], dh, -ma[e]));
      }
      store_nt<T, VN>(dx + at0 + i * step, o);
    };
    for (int64_t i = whole; i > 0; i -= KR) {
      if (i < whole) fetch(i - KR);
#pragma unroll
      for (int k = 0; k < KR; ++k) one(i - KR + k, vx[k], vy[k]);
    }
    for (int64_t i = whole; i < n; ++i)
      one(i, *(const Pack<T, VN>*)(x + at0 + i * step), *(const Pack<T, VN>*)(dy + at0 + i * step));
  }
}

// ------------------------------------------------------------------------------- host
int gcd(int a, int b) {
  while (b) {
    const int r = a % b;
    a = b;
    b = r;
  }
  return a;
}

constexpr int kTargetBlocks = 512;  // two per CU: few partial sums for every block to add up

GnShape gn_shape(const int32_t* cu, int32_t B, int64_t N, int32_t C, int32_t groups, int vn) {
  GnShape s;
  s.cu = cu;
  s.N = N;
  s.each = N / B;
  s.B = B;
  s.C = C;
  s.groups = groups;
  s.cpg = C / groups;
  s.nvec = C / vn;
  const int cols = std::min(kSlab / vn, 64);
  s.slabs = (s.nvec + cols - 1) / cols;
  s.TX = (s.nvec + s.slabs - 1) / s.slabs;
  s.slabs = (s.nvec + s.TX - 1) / s.TX;
  s.TY = kNT / s.TX;
  // No more slots than there is room for at once: 520 blocks instead of 512 for 243547 x 512 bf16 in four
  // samples took 164 us instead of 143.
  const int64_t room = kTargetBlocks / s.slabs, most = std::max<int64_t>({1, room - B, room / 2});
  const int64_t want = (N + (int64_t)s.TY * 8 - 1) / ((int64_t)s.TY * 8);
  s.T = (int32_t)std::max<int64_t>(1, std::min(most, want));
  s.R = std::max<int64_t>(1, (N + s.T - 1) / s.T);
  s.T = (int32_t)std::max<int64_t>(1, (N + s.R - 1) / s.R);
  s.gran = gcd(s.cpg, s.TX * vn);
  s.sub = 1;
  s.lsub = 0;
  for (; s.sub < vn && s.gran % (2 * s.sub) == 0; s.sub *= 2) ++s.lsub;
  s.NG = C / s.gran;
  s.GP = s.cpg / s.gran;
  return s;
}

// Elements per load: 16 bytes where the rows and every buffer allow it, else 8, else one element.
int vec_elems(int es, int32_t C, std::initializer_list<const void*> bufs) {
  for (int bytes = 16; bytes >= 8; bytes /= 2) {
    bool ok = ((int64_t)C * es) % bytes == 0;
    for (const void* p : bufs) ok = ok && ((uintptr_t)p % bytes) == 0;
    if (ok) return bytes / es;
  }
  return 1;
}

// f(T value, integral_constant VN) for the runtime type and vector length.
template <int MOST, typename F>
void by_type(int32_t dtype, int vn, F f) {
  constexpr std::integral_constant<int, 4> I4{};
  constexpr std::integral_constant<int, 2> I2{};
  constexpr std::integral_constant<int, 1> I1{};
  if (dtype == TSC_F32) {
    if (vn == 4) f(float(), I4);
    else if (vn == 2) f(float(), I2);
    else f(float(), I1);
  } else if (dtype == TSC_F16) {
    if (MOST == 8 && vn == 8) f(_Float16(), std::integral_constant<int, MOST>());
    else if (vn == 4) f(_Float16(), I4);
    else f(_Float16(), I1);
  } else {
    if (MOST == 8 && vn == 8) f(__bf16(), std::integral_constant<int, MOST>());
    else if (vn == 4) f(__bf16(), I4);
    else f(__bf16(), I1);
  }
}

}  // namespace

int64_t groupnorm_workspace_bytes(int32_t dtype, int32_t B, int64_t N, int32_t C, int32_t groups,
                                  int32_t backward) {
  if (B == 0) return 0;
  // the buffers' alignment decides the vector length only at the call: the largest of the lengths
  const int es = dtype == TSC_F32 ? 4 : 2;
  int64_t most = 0;
  for (int vn : {16 / es, 8 / es, 1}) {
    if (C % vn) continue;
    const GnShape s = gn_shape(nullptr, B, N, C, groups, vn);
    const int64_t slots = (int64_t)s.T + B;
    most = std::max(most, slots * 8 * ((int64_t)s.NG + (backward ? C : 0)));
  }
  return most;
}

int groupnorm_launch(tsc_ctx* ctx, int32_t dtype, const void* x, const int32_t* cu, int32_t B,
                     int64_t N, int32_t C, int32_t groups, const void* gamma, const void* beta,
                     float eps, int32_t silu, int32_t rest, float* stats, void* ws, void* y) {
  const int es = dtype == TSC_F32 ? 4 : 2;
  const int vn = vec_elems(es, C, {x, y});
  const GnShape s = gn_shape(cu, B, N, C, groups, vn);
  const dim3 grid((unsigned)(s.T + s.B), (unsigned)s.slabs);
  by_type<8>(dtype, vn, [&](auto t, auto v) {
    using T = decltype(t);
    constexpr int VN = decltype(v)::value;
    {
      ProfScope p(ctx, "groupnorm_stats");
      gn_stats_kernel<T, VN><<<grid, kNT, 0, ctx->stream>>>(s, (const T*)x, (float2*)ws);
    }
    ProfScope p(ctx, silu ? "groupnorm_silu" : "groupnorm");
    gn_apply_kernel<T, VN><<<grid, kNT, 0, ctx->stream>>>(
        s, (const T*)x, (const float2*)ws, (const T*)gamma, (const T*)beta, eps, silu, rest,
        stats, (T*)y);
  });
  return check_hip(hipGetLastError(), "groupnorm launch");
}

int groupnorm_backward_launch(tsc_ctx* ctx, int32_t dtype, const void* dy, const void* x,
                              const int32_t* cu, int32_t B, int64_t N, int32_t C, int32_t groups,
                              const void* gamma, const void* beta, int32_t silu, int32_t rest,
                              const float* stats, void* ws, void* dx, void* dgamma, void* dbeta) {
  const int es = dtype == TSC_F32 ? 4 : 2;
  // 16 bits: 8-byte loads, half the per-channel constants, none of which spill (step of 243547 x 512
  // bf16: 263 us with 16-byte loads, 247 so)
  const int vn = std::min(4, vec_elems(es, C, {x, dy, dx}));
  const GnShape s = gn_shape(cu, B, N, C, groups, vn);
  const int pblocks = dgamma || dbeta ? (C + kParamCh - 1) / kParamCh : 0;
  const int slots = s.T + s.B, prows = (pblocks + slots - 1) / slots;
  float2* pc = (float2*)ws;
  float2* pg = pc + ((int64_t)s.T + B) * C;
  by_type<4>(dtype, vn, [&](auto t, auto v) {
    using T = decltype(t);
    constexpr int VN = decltype(v)::value;
    {
      ProfScope p(ctx, "groupnorm_grad_sums");
      gn_grad_sums_kernel<T, VN><<<dim3((unsigned)slots, (unsigned)s.slabs), kNT, 0, ctx->stream>>>(
          s, (const T*)dy, (const T*)x, stats, (const T*)gamma, (const T*)beta, silu, pc, pg);
    }
    ProfScope p(ctx, "groupnorm_grad");
    gn_grad_kernel<T, VN>
        <<<dim3((unsigned)slots, (unsigned)(s.slabs + prows)), kNT, 0, ctx->stream>>>(
            s, (const T*)dy, (const T*)x, stats, (const T*)gamma, (const T*)beta, silu, rest,
            pblocks, prows, pc, pg, (T*)dx, (T*)dgamma, (T*)dbeta);
  });
  return check_hip(hipGetLastError(), "groupnorm backward launch");
}

}  // namespace tsc
