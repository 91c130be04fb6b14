// The norms before and after a transformer block, fused with its gate, its residual scale and its
// samples' modulation, and their gradients.  Per row of C values, sample b of the row:
//
//   v = norm(y) pw + pb               the block's output, after its norm (or y itself)
//   r = rs x + gate_b v               the residual stream
//   h = (norm(r) w + bias)(1 + scale_b) + shift_b     the next block's input
//   norm(t) = (t - mean) rstd, rstd = 1 / sqrt(var + eps)   (layer), or t / sqrt(mean(t^2) + eps)  (rms)
// without y: r = x, and without h: only r.  Gradient, with rh = norm(r), yh = norm(y):
//   drh = dh (1 + scale) w;   dr += rstd_r (drh - m1 - rh mean(drh rh)),  m1 = mean(drh) (layer) or 0
//   dx = rs dr;   dyh = gate pw dr;   dy = rstd_y (dyh - m2 - yh mean(dyh yh))
//   per sample P = sum dh rh, Q = sum dh, P' = sum dr yh, Q' = sum dr:
//   dscale = w P + bias Q, dshift = Q, dgate = pw P' + pb Q';   dw = sum_b (1 + scale) P,
//   dbias = sum_b (1 + scale) Q, dpw = sum_b gate P', dpb = sum_b gate Q'
//
// Bound by memory: a row stays in registers between its reads and its writes, and what is the same for
// all rows of a sample (modulation and weights, folded) is in registers for a run of rows.
// A row belongs to G lanes of a wave (a power of 2) or to a whole block; a block has R
// rows one after the other, through as many samples as those rows touch.  Means and variances are taken
// in two steps from the registers, so that a spread beside a large mean keeps its bits.  r is not
// rounded before its own norm, and the gradient makes it again from x and y instead of reading it
// (the same bytes), so that both are those of the unrounded sum.
// The samples' sums have one order: a block adds up its rows of a sample in slot t + b of the scratch
// (block t and sample b; along the rows one of the two grows at each step, so slots are distinct),
// and a second kernel adds up each sample's slots.
//
// Measured (each kernel by itself in a trace, us; TB/s of what the pass has to read and write; a copy of 1 GiB reaches
// 5.1), bf16 in two samples with a norm after (rms) and a norm before (layer), weights and biases of both: forward, r and h,
// 243547 x 512 206 (4.8), 64304 x 1024 133 (4.0), 60000 x 1536 170 (4.3); gradient and, behind the +, the kernel of its sums,
// 243547 x 512 321 (4.7) + 10, 64304 x 1024 174 (4.5) + 28, 60000 x 1024 fp32 324 (4.6) + 30, 60000 x 1536 297 (3.7) + 20: with the
// sums of both norms two waves a SIMD are left to wait for memory and for each row's two reductions.  Without weights and
// biases, and without a norm after: r and h of 64304 x 1024 110 (4.8), h of 15143 x 1536 23 (4.1).  The kernel figures at the
// constants are of the same inputs unless they say otherwise.

#include <algorithm>
#include <initializer_list>
#include <type_traits>

#include "tsc_internal.h"

namespace tsc {
namespace {

// Most values of a wave's lane, forward and backward: wider rows have a block.  (64304 x 1024 bf16 with 16 in the
// gradient 199 + 9 us, in blocks 174 + 28; 60000 x 1024 fp32 667 + 10, its registers spill, and 324 + 30.)
constexpr int kLaneF = 16, kLaneB = 8;
// Threads of a block of the gradient, where a row has lanes of a wave: its waves add up their sums in LDS.  (400000 x 256
// bf16 in 256 threads 273 + 19 us, in 512 275 + 10.)
constexpr int kBackThreads = 512;
constexpr int kMaxC = 8192;     // widest row of a block of 16 waves
constexpr int kSumCols = 16, kSumRows = 64, kSumWaves = kSumCols * kSumRows / 64;  // of a block that adds up slots
// Rows on their way where a block of 16-byte vectors has both norms' gradients and two waves a SIMD: of few bytes each.
// us, bf16, 1 / 2 / 3 / 4: 60000 x 1536 350 / 325 / 297 / 316, 30000 x 4096 491 / 431 / 398 / 407.  Others have more waves
// (modulated_norm, 60000 x 1536: 131 with 1, 163 with 3) or no registers (16000 x 8192: 745, 1398).
constexpr int kAhead = 3;
constexpr int kLoopB = 16;      // samples that one block of that kernel walks

struct GnArgs {
  const void *x, *y;
  const int32_t* cu;  // null: B samples of `each` rows
  int64_t N, each, R;
  int32_t B, C, G, post, norm, rest;
  const void *pw, *pb, *w, *bias, *gate, *scale, *shift;
  int64_t ldg, lds, ldt;
  float rs, eps, inv_c;
  float2 *ystat, *rstat;  // mean, rstd of each row, or null
  void *r, *h;
  // backward
  const void *dr, *dh;
  void *dx, *dy;
  float* part;  // (slots, sums, C)
  int32_t sums;
};

template <typename T, int VN>
struct __attribute__((aligned(VN * sizeof(T)))) Pack {
  T v[VN];
};

// The sample of a row and the end of its run of rows with the same sample, both uniform; -1 outside.
// Every lane of the wave takes part.  `row` < N; the run ends past row whatever cu holds.
__device__ __forceinline__ int sample_of(const GnArgs& a, int64_t row, int64_t* stop) {
  if (!a.cu) {
    const int b = (int)(row / a.each);
    *stop = (int64_t)(b + 1) * a.each;
    return b;
  }
  const int lane = threadIdx.x & 63;
  int base = 0, len = a.B + 1, count = 0;  // count: offsets at or below row, searched 64 at a time
  while (true) {
    const int stride = (len + 63) / 64, at = lane * stride;
    const bool in = at < len && (int64_t)a.cu[base + min(at, len - 1)] <= row;
    const int c = __popcll(__builtin_amdgcn_ballot_w64(in));
    if (stride == 1) {
      count = base + c;
      break;
    }
    if (c == 0) {
      count = base;
      break;
    }
    base += (c - 1) * stride;
    len = min(stride, len - (c - 1) * stride);
  }
  count = __builtin_amdgcn_readfirstlane(count);
  const int64_t next = count <= a.B ? (int64_t)a.cu[count] : a.N;
  *stop = min(a.N, max(row + 1, next));
  return count >= 1 && count <= a.B ? count - 1 : -1;
}

// A row's lanes: G of a wave, or the block.
template <int MAXV, bool BLOCK>
struct Team {
  int G, lane, first, step;  // lanes of a row, this one's number, first row slot, rows a step covers
  int phase = 0;
  __device__ explicit Team(int g) {
    if (BLOCK) {
      G = blockDim.x;
      lane = threadIdx.x;
      first = 0;
      step = 1;
    } else {
      G = g;
      lane = threadIdx.x & (g - 1);
      first = threadIdx.x / g;
      step = blockDim.x / g;
    }
  }
  // Sums of N values over the row's lanes.
  template <int N>
  __device__ __forceinline__ void sum(float (&v)[N]) {
#pragma unroll
    for (int off = 32; off > 0; off >>= 1)
      if (BLOCK || off < G)
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] += __shfl_xor(v[i], off, 64);
    if constexpr (BLOCK) {  // two rounds of slots, so that one barrier keeps a round from the next
      __shared__ float meet[2][16][2];
      static_assert(N <= 2, "slots");
      const int nw = blockDim.x >> 6, w = threadIdx.x >> 6;
      if ((threadIdx.x & 63) == 0)
#pragma unroll
        for (int i = 0; i < N; ++i) meet[phase][w][i] = v[i];
      __syncthreads();
#pragma unroll
      for (int i = 0; i < N; ++i) {
        float t = 0.f;
        for (int x = 0; x < nw; ++x) t += meet[phase][x][i];
        v[i] = t;
      }
      phase ^= 1;
    }
  }
};

// The lane's values of a row: vectors lane + G k, k < MAXV.
template <typename T, int VN, int MAXV>
struct Cols {
  Pack<T, VN> v[MAXV];
  __device__ __forceinline__ void load(const T* row, int lane, int G, int nvec) {
#pragma unroll
    for (int k = 0; k < MAXV; ++k)
      if (lane + G * k < nvec) v[k] = *(const Pack<T, VN>*)(row + (int64_t)(lane + G * k) * VN);
  }
};
template <typename T, int VN, int MAXV>
__device__ __forceinline__ void store_row(T* row, int lane, int G, int nvec, const float (&f)[MAXV][VN]) {
#pragma unroll
  for (int k = 0; k < MAXV; ++k)
    if (lane + G * k < nvec) {
      Pack<T, VN> o;
#pragma unroll
      for (int e = 0; e < VN; ++e) o.v[e] = (T)f[k][e];
      *(Pack<T, VN>*)(row + (int64_t)(lane + G * k) * VN) = o;
    }
}
// A vector of C parameters in fp32, `none` where there is none.
template <typename T, int VN, int MAXV>
__device__ __forceinline__ void params(const void* p, int64_t at, int lane, int G, int nvec, float none,
                                       float (&f)[MAXV][VN]) {
  Cols<T, VN, MAXV> c;
  if (p) c.load((const T*)p + at, lane, G, nvec);
#pragma unroll
  for (int k = 0; k < MAXV; ++k)
#pragma unroll
    for (int e = 0; e < VN; ++e) f[k][e] = p && lane + G * k < nvec ? (float)c.v[k].v[e] : none;
}

// Normalizes t in place; lanes past the row's end hold zeros before and after.
template <int VN, int MAXV, typename Tm>
__device__ __forceinline__ float2 normalize(Tm& team, int kind, float inv_c, float eps, int nvec,
                                            float (&t)[MAXV][VN]) {
  float mean = 0.f;
  if (kind == TSC_NORM_LAYER) {
    float s[1] = {0.f};
#pragma unroll
    for (int k = 0; k < MAXV; ++k)
#pragma unroll
      for (int e = 0; e < VN; ++e) s[0] += t[k][e];
    team.sum(s);
    mean = s[0] * inv_c;
  }
  float q[1] = {0.f};
#pragma unroll
  for (int k = 0; k < MAXV; ++k)
    if (team.lane + team.G * k < nvec)
#pragma unroll
      for (int e = 0; e < VN; ++e) {
        t[k][e] -= mean;
        q[0] = fmaf(t[k][e], t[k][e], q[0]);
      }
  team.sum(q);
  const float rstd = 1.f / sqrtf(fmaf(q[0], inv_c, eps));
#pragma unroll
  for (int k = 0; k < MAXV; ++k)
#pragma unroll
    for (int e = 0; e < VN; ++e) t[k][e] *= rstd;
  return make_float2(mean, rstd);
}

// A row's block is bounded by the widest rows' 1024 threads whatever its own: rows in single values, of widths that nothing
// wider divides or that are not aligned, spill for it (88 to 90 registers with both parts), and fp32 ones of both parts 6.
template <typename T, int VN, int MAXV, bool BLOCK, bool Y, bool H>
__global__ void __launch_bounds__(BLOCK ? 1024 : 256) gated_norm_kernel(const GnArgs a) {
  Team<MAXV, BLOCK> team(a.G);
  const int lane = team.lane, G = team.G, C = a.C, nvec = C / VN;
  const int64_t end = min(a.N, ((int64_t)blockIdx.x + 1) * a.R);
  for (int64_t row0 = (int64_t)blockIdx.x * a.R; row0 < end;) {
    int64_t stop;
    const int b = sample_of(a, row0, &stop);
    stop = min(stop, end);
    if (b < 0) {  // outside every sample
      if (a.rest) {
        float zero[MAXV][VN] = {};
        for (int64_t row = row0 + team.first; row < stop; row += team.step) {
          if (Y) store_row<T, VN, MAXV>((T*)a.r + row * C, lane, G, nvec, zero);
          if (H) store_row<T, VN, MAXV>((T*)a.h + row * C, lane, G, nvec, zero);
        }
      }
      row0 = stop;
      continue;
    }
    // v's factor and summand with the gate; h's factor and summand with the modulation.
    float gf[MAXV][VN], gs[MAXV][VN], hf[MAXV][VN], hs[MAXV][VN], t[MAXV][VN];
    if (Y) {
      params<T, VN, MAXV>(a.gate, b * a.ldg, lane, G, nvec, 1.f, gf);
      params<T, VN, MAXV>(a.pb, 0, lane, G, nvec, 0.f, gs);
      params<T, VN, MAXV>(a.pw, 0, lane, G, nvec, 1.f, t);
#pragma unroll
      for (int k = 0; k < MAXV; ++k)
#pragma unroll
        for (int e = 0; e < VN; ++e) {
          if (a.pb) gs[k][e] *= gf[k][e];  // uniform: without one it is 0, whatever the gate
          gf[k][e] *= t[k][e];
        }
    }
    if (H) {
      params<T, VN, MAXV>(a.scale, b * a.lds, lane, G, nvec, 0.f, hf);
      params<T, VN, MAXV>(a.bias, 0, lane, G, nvec, 0.f, hs);
      params<T, VN, MAXV>(a.shift, b * a.ldt, lane, G, nvec, 0.f, t);
#pragma unroll
      for (int k = 0; k < MAXV; ++k)
#pragma unroll
        for (int e = 0; e < VN; ++e) {
          hf[k][e] += 1.f;
          hs[k][e] = a.bias ? fmaf(hs[k][e], hf[k][e], t[k][e]) : t[k][e];
        }
      params<T, VN, MAXV>(a.w, 0, lane, G, nvec, 1.f, t);
#pragma unroll
      for (int k = 0; k < MAXV; ++k)
#pragma unroll
        for (int e = 0; e < VN; ++e) hf[k][e] *= t[k][e];
    }
    Cols<T, VN, MAXV> xn, yn;  // the next row's, on their way
    int64_t row = row0 + team.first;
    if (row < stop) {
      xn.load((const T*)a.x + row * C, lane, G, nvec);
      if (Y) yn.load((const T*)a.y + row * C, lane, G, nvec);
    }
    // Lanes of a wave whose row is past the run still take part in the sums.
    for (int64_t lead = row0; lead < stop; lead += team.step, row += team.step) {
      const bool live = row < stop;
      float x[MAXV][VN], y[MAXV][VN];
#pragma unroll
      for (int k = 0; k < MAXV; ++k)
#pragma unroll
        for (int e = 0; e < VN; ++e) {
          const bool in = live && lane + G * k < nvec;
          x[k][e] = in ? (float)xn.v[k].v[e] : 0.f;
          if (Y) y[k][e] = in ? (float)yn.v[k].v[e] : 0.f;
        }
      if (row + team.step < stop) {
        xn.load((const T*)a.x + (row + team.step) * C, lane, G, nvec);
        if (Y) yn.load((const T*)a.y + (row + team.step) * C, lane, G, nvec);
      }
      if (Y) {
        if (a.post != TSC_NORM_NONE) {
          const float2 st = normalize<VN, MAXV>(team, a.post, a.inv_c, a.eps, nvec, y);
          if (a.ystat && live && lane == 0) a.ystat[row] = st;
        }
#pragma unroll
        for (int k = 0; k < MAXV; ++k)
          if (lane + G * k < nvec)
#pragma unroll
            for (int e = 0; e < VN; ++e) x[k][e] = fmaf(a.rs, x[k][e], fmaf(gf[k][e], y[k][e], gs[k][e]));
        if (live) store_row<T, VN, MAXV>((T*)a.r + row * C, lane, G, nvec, x);
      }
      if (H) {
        const float2 st = normalize<VN, MAXV>(team, a.norm, a.inv_c, a.eps, nvec, x);
        if (a.rstat && live && lane == 0) a.rstat[row] = st;
#pragma unroll
        for (int k = 0; k < MAXV; ++k)
#pragma unroll
          for (int e = 0; e < VN; ++e) x[k][e] = fmaf(x[k][e], hf[k][e], hs[k][e]);
        if (live) store_row<T, VN, MAXV>((T*)a.h + row * C, lane, G, nvec, x);
      }
    }
    row0 = stop;
  }
}

// Adds up the block's lanes that hold the same columns and leaves the sums of a sample's rows in their slot.
template <int VN, int MAXV, bool BLOCK>
__device__ __forceinline__ void flush(const GnArgs& a, const Team<MAXV, BLOCK>& team, int64_t slot, int which,
                                      float (&s)[MAXV][VN]) {
  const int nvec = a.C / VN;
  float* out = a.part + (slot * a.sums + which) * a.C;
  if constexpr (BLOCK) {
#pragma unroll
    for (int k = 0; k < MAXV; ++k)
      if (team.lane + team.G * k < nvec)
#pragma unroll
        for (int e = 0; e < VN; ++e) out[(team.lane + team.G * k) * VN + e] = s[k][e];
  } else {
    constexpr int NW = kBackThreads / 64;
    __shared__ float meet[NW][64 * MAXV * VN];
    for (int off = 32; off >= team.G; off >>= 1)
#pragma unroll
      for (int k = 0; k < MAXV; ++k)
#pragma unroll
        for (int e = 0; e < VN; ++e) s[k][e] += __shfl_xor(s[k][e], off, 64);
    const int w = threadIdx.x >> 6, l = threadIdx.x & 63;
    __syncthreads();  // the last sums have been read
    if (l < team.G)
#pragma unroll
      for (int k = 0; k < MAXV; ++k)
#pragma unroll
        for (int e = 0; e < VN; ++e) meet[w][(k * VN + e) * 64 + l] = s[k][e];
    __syncthreads();
    for (int c = threadIdx.x; c < a.C; c += kBackThreads) {
      const int vec = c / VN, at = (vec / team.G * VN + c % VN) * 64 + vec % team.G;
      float t = meet[0][at];
#pragma unroll
      for (int x = 1; x < NW; ++x) t += meet[x][at];
      out[c] = t;
    }
  }
}

// NT: threads of a block at most.  Rows of more than 4096 values, whose blocks have 1024 threads of 128 registers, spill:
// with both norms 55 registers in 16 bits, 103 in fp32, 192 in single values; so do single values with both norms at 512
// threads, 28 to 36.
template <typename T, int VN, int MAXV, bool BLOCK, int NT, bool Y, bool H>
__global__ void __launch_bounds__(NT) gated_norm_backward_kernel(const GnArgs a) {
  constexpr int AHEAD = sizeof(T) == 2 && VN == 8 && BLOCK && NT == 512 && Y && H ? kAhead : 1;  // rows on their way
  Team<MAXV, BLOCK> team(a.G);
  const int lane = team.lane, G = team.G, C = a.C, nvec = C / VN;
  const int64_t end = min(a.N, ((int64_t)blockIdx.x + 1) * a.R);
  for (int64_t row0 = (int64_t)blockIdx.x * a.R; row0 < end;) {
    int64_t stop;
    const int b = sample_of(a, row0, &stop);
    stop = min(stop, end);
    if (b < 0) {
      if (a.rest) {
        float zero[MAXV][VN] = {};
        for (int64_t row = row0 + team.first; row < stop; row += team.step) {
          store_row<T, VN, MAXV>((T*)a.dx + row * C, lane, G, nvec, zero);
          if (Y) store_row<T, VN, MAXV>((T*)a.dy + row * C, lane, G, nvec, zero);
        }
      }
      row0 = stop;
      continue;
    }
    float hf[MAXV][VN], gf[MAXV][VN], gs[MAXV][VN];  // (1 + scale) w, gate pw, gate pb
    {
      float t[MAXV][VN];
      if (H) {
        params<T, VN, MAXV>(a.scale, b * a.lds, lane, G, nvec, 0.f, hf);
        params<T, VN, MAXV>(a.w, 0, lane, G, nvec, 1.f, t);
#pragma unroll
        for (int k = 0; k < MAXV; ++k)
#pragma unroll
          for (int e = 0; e < VN; ++e) hf[k][e] = (1.f + hf[k][e]) * t[k][e];
      }
      if (Y) {
        params<T, VN, MAXV>(a.gate, b * a.ldg, lane, G, nvec, 1.f, gf);
        params<T, VN, MAXV>(a.pw, 0, lane, G, nvec, 1.f, t);
        params<T, VN, MAXV>(a.pb, 0, lane, G, nvec, 0.f, gs);
#pragma unroll
        for (int k = 0; k < MAXV; ++k)
#pragma unroll
          for (int e = 0; e < VN; ++e) {
            if (a.pb) gs[k][e] *= gf[k][e];
            gf[k][e] *= t[k][e];
          }
      }
    }
    float P[MAXV][VN] = {}, Q[MAXV][VN] = {}, Py[MAXV][VN] = {}, Qy[MAXV][VN] = {};
    struct Ahead {  // a row's, on their way
      Cols<T, VN, MAXV> x, y, dh, dr;
      float2 ys = make_float2(0.f, 1.f), rs = make_float2(0.f, 1.f);
    } ahead[AHEAD];
    auto load = [&](Ahead& n, int64_t row) {
      if (row >= stop) return;
      if (H) n.x.load((const T*)a.x + row * C, lane, G, nvec);
      if (Y) n.y.load((const T*)a.y + row * C, lane, G, nvec);
      if (H) n.dh.load((const T*)a.dh + row * C, lane, G, nvec);
      if (a.dr) n.dr.load((const T*)a.dr + row * C, lane, G, nvec);
      if (Y && a.post != TSC_NORM_NONE) n.ys = a.ystat[row];
      if (H) n.rs = a.rstat[row];
    };
    auto step = [&](Ahead& n, int64_t row) __attribute__((always_inline)) {
      const bool live = row < stop;
      const float2 ys = n.ys, rst = n.rs;
      const Cols<T, VN, MAXV> dr = n.dr;
      float y[MAXV][VN], x[MAXV][VN], d[MAXV][VN], s2[2] = {0.f, 0.f};
#pragma unroll
      for (int k = 0; k < MAXV; ++k) {
        const bool in = live && lane + G * k < nvec;
#pragma unroll
        for (int e = 0; e < VN; ++e) {
          y[k][e] = Y && in ? ((float)n.y.v[k].v[e] - ys.x) * ys.y : 0.f;
          d[k][e] = 0.f;
          if (H) {
            float r = in ? (float)n.x.v[k].v[e] : 0.f;
            if (Y) r = fmaf(a.rs, r, fmaf(gf[k][e], y[k][e], gs[k][e]));
            x[k][e] = in ? (r - rst.x) * rst.y : 0.f;
            const float dh = in ? (float)n.dh.v[k].v[e] : 0.f;
            P[k][e] = fmaf(dh, x[k][e], P[k][e]);
            Q[k][e] += dh;
            d[k][e] = dh * hf[k][e];
            s2[0] += d[k][e];
            s2[1] = fmaf(d[k][e], x[k][e], s2[1]);
          }
        }
      }
      load(n, row + AHEAD * team.step);
      if (H) {
        team.sum(s2);
        const float m1 = a.norm == TSC_NORM_LAYER ? s2[0] * a.inv_c : 0.f, m2 = s2[1] * a.inv_c;
#pragma unroll
        for (int k = 0; k < MAXV; ++k)
#pragma unroll
          for (int e = 0; e < VN; ++e) d[k][e] = rst.y * (d[k][e] - fmaf(x[k][e], m2, m1));
      }
      if (a.dr) {
#pragma unroll
        for (int k = 0; k < MAXV; ++k)
#pragma unroll
          for (int e = 0; e < VN; ++e)
            if (live && lane + G * k < nvec) d[k][e] += (float)dr.v[k].v[e];
      }
      // d: the gradient of r
      if (live) {
        if (Y) {
#pragma unroll
          for (int k = 0; k < MAXV; ++k)
#pragma unroll
            for (int e = 0; e < VN; ++e) x[k][e] = a.rs * d[k][e];
          store_row<T, VN, MAXV>((T*)a.dx + row * C, lane, G, nvec, x);
        } else {
          store_row<T, VN, MAXV>((T*)a.dx + row * C, lane, G, nvec, d);
        }
      }
      if (Y) {
        float e2[2] = {0.f, 0.f};
#pragma unroll
        for (int k = 0; k < MAXV; ++k)
          if (live && lane + G * k < nvec)
#pragma unroll
            for (int e = 0; e < VN; ++e) {
              Py[k][e] = fmaf(d[k][e], y[k][e], Py[k][e]);
              Qy[k][e] += d[k][e];
              d[k][e] *= gf[k][e];
              e2[0] += d[k][e];
              e2[1] = fmaf(d[k][e], y[k][e], e2[1]);
            }
        if (a.post != TSC_NORM_NONE) {
          team.sum(e2);
          const float m1 = a.post == TSC_NORM_LAYER ? e2[0] * a.inv_c : 0.f, m2 = e2[1] * a.inv_c;
#pragma unroll
          for (int k = 0; k < MAXV; ++k)
#pragma unroll
            for (int e = 0; e < VN; ++e) d[k][e] = ys.y * (d[k][e] - fmaf(y[k][e], m2, m1));
        }
        if (live) store_row<T, VN, MAXV>((T*)a.dy + row * C, lane, G, nvec, d);
      }
    };
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) load(ahead[i], row0 + team.first + i * team.step);
    for (int64_t lead = row0; lead < stop; lead += AHEAD * team.step) {
#pragma unroll
      for (int i = 0; i < AHEAD; ++i)
        if (i == 0 || lead + i * team.step < stop) step(ahead[i], lead + team.first + i * team.step);
    }
    if (a.sums) {
      const int64_t slot = (int64_t)blockIdx.x + b;
      int which = 0;
      if (H) {
        flush<VN, MAXV, BLOCK>(a, team, slot, which++, P);
        flush<VN, MAXV, BLOCK>(a, team, slot, which++, Q);
      }
      if (Y) {
        flush<VN, MAXV, BLOCK>(a, team, slot, which++, Py);
        if (a.sums > which) flush<VN, MAXV, BLOCK>(a, team, slot, which, Qy);
      }
    }
    row0 = stop;
  }
}

struct SumArgs {
  const float* part;
  double* total;  // (B, 4, C): what the weights' gradients add up, where blocks have one sample each
  const int32_t* cu;
  int64_t N, each, R;
  int32_t B, C, sums, h, y;  // h, y: whether those parts have sums
  const void *w, *bias, *scale, *pw, *pb, *gate;
  int64_t lds, ldg;
  void *dscale, *dshift, *dgate, *dw, *dbias, *dpw, *dpb;
};

template <typename T>
__device__ __forceinline__ float at_or(const void* p, int64_t i, float none) {
  return p ? (float)((const T*)p)[i] : none;
}
template <typename T>
__device__ __forceinline__ void put(void* p, int64_t i, double v) {
  if (p) ((T*)p)[i] = (T)(float)v;
}

// Adds up v over a block's rows of threads: in a wave, then over the waves.  Row 0 of threads has the sums.
template <int N>
__device__ __forceinline__ void sum_rows(double (&v)[N], double (*meet)[kSumWaves][kSumCols], int tc) {
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
#pragma unroll
  for (int off = 32; off >= kSumCols; off >>= 1)
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] += __shfl_xor(v[i], off, 64);
  __syncthreads();  // the last sums have been read
  if (lane < kSumCols)
#pragma unroll
    for (int i = 0; i < N; ++i) meet[i][w][tc] = v[i];
  __syncthreads();
  if (w == 0)
#pragma unroll
    for (int i = 0; i < N; ++i) {
      double t = 0.;
#pragma unroll
      for (int x = 0; x < kSumWaves / 4; ++x) t += meet[i][4 * x + lane / kSumCols][tc];
#pragma unroll
      for (int off = 32; off >= kSumCols; off >>= 1) t += __shfl_xor(t, off, 64);
      v[i] = t;
    }
}

// Sums over a sample's slots, 16 columns by 64 slots at a time, merged in fp64.  Grid y = 1: all samples,
// one after the other, and the weights' gradients; else one sample each, whose parts of those go to `total`.
// NS: a.sums.
template <typename T, int NS>
__global__ void __launch_bounds__(kSumCols* kSumRows) gated_norm_sums_kernel(const SumArgs a) {
  __shared__ double meet[NS][kSumWaves][kSumCols];
  const int tc = threadIdx.x % kSumCols, tr = threadIdx.x / kSumCols, c = blockIdx.x * kSumCols + tc;
  const bool in = c < a.C, alone = gridDim.y == 1;
  double weights[4] = {0., 0., 0., 0.};
  for (int b = blockIdx.y; b < a.B; b += gridDim.y) {
    int64_t lo = b * a.each, hi = lo + a.each;
    if (a.cu) {
      lo = min<int64_t>(max<int64_t>(a.cu[b], 0), a.N);
      hi = min<int64_t>(max<int64_t>(a.cu[b + 1], lo), a.N);
    }
    const int64_t t0 = lo / a.R, t1 = hi > lo ? (hi - 1) / a.R + 1 : t0;  // blocks of these rows
    double s[NS] = {};
    if (in)
#pragma unroll 4
      for (int64_t t = t0 + tr; t < t1; t += kSumRows)
#pragma unroll
        for (int i = 0; i < NS; ++i) s[i] += (double)a.part[((t + b) * NS + i) * a.C + c];
    sum_rows<NS>(s, meet, tc);
    if (!in || tr) continue;
    const int64_t at = (int64_t)b * a.C + c;
    double part[4] = {0., 0., 0., 0.};
    if (NS > 1 && a.h) {
      const double P = s[0], Q = s[NS > 1], f = 1. + (double)at_or<T>(a.scale, b * a.lds + c, 0.f);
      put<T>(a.dscale, at, (double)at_or<T>(a.w, c, 1.f) * P + (a.bias ? (double)at_or<T>(a.bias, c, 0.f) * Q : 0.));
      put<T>(a.dshift, at, Q);
      part[0] = f * P;
      part[1] = f * Q;
    }
    if (a.y) {
      constexpr int A = NS > 2 ? 2 : 0;  // with h's two sums before them
      const double P = s[A], Q = NS % 2 ? 0. : s[NS - 1];
      const double gate = at_or<T>(a.gate, b * a.ldg + c, 1.f);
      put<T>(a.dgate, at, (double)at_or<T>(a.pw, c, 1.f) * P + (a.pb ? (double)at_or<T>(a.pb, c, 0.f) * Q : 0.));
      part[2] = gate * P;
      part[3] = gate * Q;
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (alone) weights[j] += part[j];
      else if (a.total) a.total[((int64_t)b * 4 + j) * a.C + c] = part[j];
    }
  }
  if (alone && in && tr == 0) {
    put<T>(a.dw, c, weights[0]);
    put<T>(a.dbias, c, weights[1]);
    put<T>(a.dpw, c, weights[2]);
    put<T>(a.dpb, c, weights[3]);
  }
}

// The weights' gradients of more than kLoopB samples.
template <typename T>
__global__ void __launch_bounds__(kSumCols* kSumRows) gated_norm_weights_kernel(const SumArgs a) {
  __shared__ double meet[4][kSumWaves][kSumCols];
  const int tc = threadIdx.x % kSumCols, tr = threadIdx.x / kSumCols, c = blockIdx.x * kSumCols + tc;
  double v[4] = {0., 0., 0., 0.};
  if (c < a.C)
    for (int b = tr; b < a.B; b += kSumRows)
#pragma unroll
      for (int j = 0; j < 4; ++j) v[j] += a.total[((int64_t)b * 4 + j) * a.C + c];
  sum_rows<4>(v, meet, tc);
  if (c < a.C && tr == 0) {
    put<T>(a.dw, c, v[0]);
    put<T>(a.dbias, c, v[1]);
    put<T>(a.dpw, c, v[2]);
    put<T>(a.dpb, c, v[3]);
  }
}

// ------------------------------------------------------------------------------- host
struct Shape {
  bool block;
  int vn, maxv;          // values of a vector, vectors of a lane
  int G, threads, rows;  // lanes of a row, threads of a block, rows a step of it covers
};
Shape shape_of(int32_t C, int vn, int lane_values, int threads) {
  const int nvec = C / vn;
  if (C <= 64 * lane_values) {
    int g = 1;
    while (g < 64 && g < nvec) g *= 2;
    return {false, vn, nvec <= 64 ? 1 : lane_values / vn, g, threads, threads / g};
  }
  const int maxv = 8 / vn;
  threads = ((nvec + maxv - 1) / maxv + 63) / 64 * 64;
  return {true, vn, maxv, threads, threads, 1};
}
// Rows of a block: as many blocks as `most` where there are enough rows.
int64_t rows_of(const Shape& s, int64_t N, int64_t most) {
  const int64_t steps = (N + s.rows - 1) / s.rows;
  return s.rows * std::max<int64_t>(1, (steps + most - 1) / most);
}
// Blocks of the forward pass: enough that those at work at one time are near each other in memory, and rows enough in
// each for its sample's parameters.  us, r and h of bf16: 243547 x 512 in 2048 blocks 210, 8192 206, 16384 233; 60000 x
// 1536 (rows of a block) in 2048 177, 4096 170, 8192 172; 16000 x 8192 in 2000 340, 4096 371.  64304 x 1024 (two vectors a lane) in
// 2048 119, 4096 133; without weights, biases and a norm after (timed among others, not in a trace) 110, 108.
int64_t forward_blocks(const Shape& s, int64_t N) {
  if (!s.block) return s.maxv == 1 ? 8192 : 4096;
  return std::min<int64_t>(4096, std::max<int64_t>(1, N / 8));
}
// Waves of a CU in the gradient, by its registers: with the sums of r's norm and of y's (176 to 256), of one (92 to 128).
constexpr int kBothWaves = 8, kOneWaves = 16;
// Blocks of the gradient: as many as run at once; more of them leave more sums to add up.  us, both norms and the sums' kernel,
// bf16, with 8 / 12 / 16 waves a CU: 64304 x 1024 174 + 28, 214 + 47, 228 + 58; 60000 x 1536 297 + 20, 307 + 36, 348 + 37; 243547 x
// 512 321 + 10, 319 + 10, 321 + 24.
int64_t back_blocks(const Shape& s, bool both) {
  return 256 * std::max(1, (both ? kBothWaves : kOneWaves) * 64 / s.threads);
}

// A step's rows and with them the slots do not depend on the alignment: the scratch has room for both.
int64_t slots_of(int32_t dtype, int32_t B, int64_t N, int32_t C) {
  int64_t most = 0;
  for (int v : {8, 4, 1}) {
    if (C % v || (v == 8 && dtype == TSC_F32)) continue;
    const Shape s = shape_of(C, v, kLaneB, kBackThreads);
    const int64_t r = rows_of(s, N, back_blocks(s, false));
    most = std::max(most, (N + r - 1) / r);
  }
  return most + B;
}

GnArgs args_of(const GatedNormArgs& x) {
  GnArgs a = {};
  a.x = x.x;
  a.y = x.y;
  a.cu = x.cu;
  a.N = x.N;
  a.each = x.cu || x.B == 0 ? 0 : x.N / x.B;
  a.B = x.B;
  a.C = x.C;
  a.post = x.post_norm;
  a.norm = x.norm;
  a.rest = x.rest;
  a.pw = x.post_weight;
  a.pb = x.post_bias;
  a.w = x.weight;
  a.bias = x.bias;
  a.gate = x.gate;
  a.scale = x.scale;
  a.shift = x.shift;
  a.ldg = x.ld_gate;
  a.lds = x.ld_scale;
  a.ldt = x.ld_shift;
  a.rs = x.residual_scale;
  a.eps = x.eps;
  a.inv_c = 1.f / (float)x.C;
  return a;
}
// The widest vectors that rows and parameters divide into and are aligned to: 16 bytes, 8 in 16 bits, or one value.
Shape shape_for(const GatedNormArgs& x, int lane_values, int threads,
                std::initializer_list<const void*> rows) {
  const int es = x.dtype == TSC_F32 ? 4 : 2;
  for (int vn : {8, 4}) {
    if (x.C % vn || vn * es > 16) continue;
    bool fits = !((x.gate && x.ld_gate % vn) || (x.scale && x.ld_scale % vn) || (x.shift && x.ld_shift % vn));
    for (const void* p : rows) fits &= (uintptr_t)p % (vn * es) == 0;
    for (const void* p : {x.x, x.y, x.post_weight, x.post_bias, x.weight, x.bias, x.gate, x.scale, x.shift})
      fits &= (uintptr_t)p % (vn * es) == 0;
    if (fits) return shape_of(x.C, vn, lane_values, threads);
  }
  return shape_of(x.C, 1, lane_values, threads);
}

// Calls f(type, VN, MAXV, BLOCK) with the kernel's shape.
template <int LANE, typename F>
void by_shape(int32_t dtype, const Shape& s, F f) {
  auto with = [&](auto t, auto vn) {
    constexpr int VN = decltype(vn)::value;
    if (s.block) f(t, vn, std::integral_constant<int, 8 / VN>(), std::true_type());
    else if (s.maxv == 1) f(t, vn, std::integral_constant<int, 1>(), std::false_type());
    else f(t, vn, std::integral_constant<int, LANE / VN>(), std::false_type());
  };
  auto types = [&](auto t) {
    if constexpr (sizeof(decltype(t)) == 2)
      if (s.vn == 8) return with(t, std::integral_constant<int, 8>());
    if (s.vn == 4) with(t, std::integral_constant<int, 4>());
    else with(t, std::integral_constant<int, 1>());
  };
  if (dtype == TSC_BF16) types(__bf16());
  else if (dtype == TSC_F16) types(_Float16());
  else types(float());
}

}  // namespace

int32_t gated_norm_max_channels() { return kMaxC; }

int gated_norm_launch(tsc_ctx* ctx, const GatedNormArgs& x, float* stats, void* r, void* h) {
  GnArgs a = args_of(x);
  a.r = r;
  a.h = h;
  if (stats) {
    const bool post = x.y && x.post_norm != TSC_NORM_NONE;
    a.ystat = post ? (float2*)stats : nullptr;
    a.rstat = h ? (float2*)stats + (post ? x.N : 0) : nullptr;
  }
  const Shape s = shape_for(x, kLaneF, 256, {r, h});
  a.G = s.G;
  a.R = rows_of(s, x.N, forward_blocks(s, x.N));
  const unsigned grid = (unsigned)((x.N + a.R - 1) / a.R);
  ProfScope p(ctx, "gated_norm");
  by_shape<kLaneF>(x.dtype, s, [&](auto t, auto v, auto m, auto blk) {
    using T = decltype(t);
    constexpr int VN = decltype(v)::value, MAXV = decltype(m)::value;
    constexpr bool BLOCK = decltype(blk)::value;
    if (x.y && h) gated_norm_kernel<T, VN, MAXV, BLOCK, true, true><<<grid, s.threads, 0, ctx->stream>>>(a);
    else if (x.y) gated_norm_kernel<T, VN, MAXV, BLOCK, true, false><<<grid, s.threads, 0, ctx->stream>>>(a);
    else gated_norm_kernel<T, VN, MAXV, BLOCK, false, true><<<grid, s.threads, 0, ctx->stream>>>(a);
  });
  return check_hip(hipGetLastError(), "gated_norm launch");
}

int64_t gated_norm_workspace_bytes(int32_t dtype, int32_t B, int64_t N, int32_t C) {
  if (B == 0) return 0;
  const int64_t part = align_up((size_t)slots_of(dtype, B, N, C) * 4 * C * 4, 16);
  return part + (B > kLoopB ? (int64_t)B * 4 * C * 8 : 0);
}

int gated_norm_backward_launch(tsc_ctx* ctx, const GatedNormArgs& x, const float* stats, const void* dr,
                               const void* dh, void* ws, const GatedNormGrads& g) {
  GnArgs a = args_of(x);
  const bool post = x.y && x.post_norm != TSC_NORM_NONE;
  a.ystat = (float2*)stats;
  a.rstat = (float2*)stats + (post ? x.N : 0);
  a.dr = dr;
  a.dh = dh;
  a.dx = g.dx;
  a.dy = g.dy;
  const bool want_h = dh && (g.dscale || g.dshift || g.dweight || g.dbias);
  const bool want_y = x.y && (g.dgate || g.dpost_weight || g.dpost_bias);
  // Either part's sums where any is wanted: the kernel makes them all the same.  Q' is for the bias, its own gradient
  // and its part of the gate's.
  a.sums = want_h || want_y ? (dh ? 2 : 0) + (x.y ? (x.post_bias || g.dpost_bias ? 2 : 1) : 0) : 0;
  a.part = (float*)ws;
  const Shape s = shape_for(x, kLaneB, kBackThreads, {dr, dh, g.dx, g.dy});
  a.G = s.G;
  a.R = rows_of(s, std::max<int64_t>(x.N, 1), back_blocks(s, x.y && dh));
  if (x.N > 0) {
    const unsigned grid = (unsigned)((x.N + a.R - 1) / a.R);
    ProfScope p(ctx, "gated_norm_backward");
    by_shape<kLaneB>(x.dtype, s, [&](auto t, auto v, auto m, auto blk) {
      using T = decltype(t);
      constexpr int VN = decltype(v)::value, MAXV = decltype(m)::value;
      constexpr bool BLOCK = decltype(blk)::value;
      auto run = [&](auto nt) {
        constexpr int NT = decltype(nt)::value;
        auto with = [&](auto y, auto hh) {
          gated_norm_backward_kernel<T, VN, MAXV, BLOCK, NT, decltype(y)::value, decltype(hh)::value>
              <<<grid, s.threads, 0, ctx->stream>>>(a);
        };
        if (x.y && dh) with(std::true_type(), std::true_type());
        else if (x.y) with(std::true_type(), std::false_type());
        else with(std::false_type(), std::true_type());
      };
      if constexpr (!BLOCK) run(std::integral_constant<int, kBackThreads>());
      else if (s.threads <= 512) run(std::integral_constant<int, 512>());
      else run(std::integral_constant<int, 1024>());
    });
  }
  if (a.sums) {
    SumArgs q = {};
    q.part = a.part;
    q.cu = a.cu;
    q.N = a.N;
    q.each = a.each;
    q.R = a.R;
    q.B = a.B;
    q.C = a.C;
    q.sums = a.sums;
    q.h = dh != nullptr;
    q.y = x.y != nullptr;
    q.w = x.weight;
    q.bias = x.bias;
    q.scale = x.scale;
    q.pw = x.post_weight;
    q.pb = x.post_bias;
    q.gate = x.gate;
    q.lds = x.ld_scale;
    q.ldg = x.ld_gate;
    q.dscale = g.dscale;
    q.dshift = g.dshift;
    q.dgate = g.dgate;
    q.dw = g.dweight;
    q.dbias = g.dbias;
    q.dpw = g.dpost_weight;
    q.dpb = g.dpost_bias;
    const bool weights = g.dweight || g.dbias || g.dpost_weight || g.dpost_bias;
    const bool loop = x.B <= kLoopB;
    if (!loop && weights)
      q.total = (double*)((char*)ws + align_up((size_t)slots_of(x.dtype, x.B, x.N, x.C) * 4 * x.C * 4, 16));
    const unsigned gx = (unsigned)((x.C + kSumCols - 1) / kSumCols);
    const dim3 grid(gx, loop ? 1u : (unsigned)std::min(x.B, 65535));
    auto run = [&](auto t) {
      using T = decltype(t);
      {
        ProfScope p(ctx, "gated_norm_sums");
        auto sums = [&](auto ns) {
          gated_norm_sums_kernel<T, decltype(ns)::value><<<grid, kSumCols * kSumRows, 0, ctx->stream>>>(q);
        };
        if (q.sums == 1) sums(std::integral_constant<int, 1>());
        else if (q.sums == 2) sums(std::integral_constant<int, 2>());
        else if (q.sums == 3) sums(std::integral_constant<int, 3>());
        else sums(std::integral_constant<int, 4>());
      }
      if (!loop && weights) {
        ProfScope p(ctx, "gated_norm_weights");
        gated_norm_weights_kernel<T><<<gx, kSumCols * kSumRows, 0, ctx->stream>>>(q);
      }
    };
    if (x.dtype == TSC_BF16) run(__bf16());
    else if (x.dtype == TSC_F16) run(_Float16());
    else run(float());
  }
  return check_hip(hipGetLastError(), "gated_norm_backward launch");
}

}  // namespace tsc
