// Device helpers shared by the attention kernels that train (diff_attention.hip, window_attention.hip):
// fragments of 8 elements of each type, row-major tiles in LDS with row and transposed reads, rows on
// their way into them, and a wave's results out of its registers.
//
// Scores are computed in 32 x 32 tiles whose result layout (lane: one column, 16 rows 8(j/4) +
// 4(lane/32) + j%4) is the operand layout of the next product, contracted over those rows.  The other
// operand of that product is read transposed from the row-major tile in LDS.  All types run the same code
// on fragments of 8 elements: one 32x32x16 product in 16 bits, eight 32x32x2 products in fp32.
#pragma once

#include "attention_common.h"

namespace tsc {
namespace {

constexpr float kLog2e = 1.4426950408889634f;

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
  // The same with addresses made from one register each, so that a loop keeps that and no more.  row_of: chunk
  // 2 st + hf of row l32 is at it ^ 32 st; col_of: the piece of dim tile mt in rows 8 x + .. at it ^ (64 mt ^ 32 x).
  static __device__ __forceinline__ int row_of(int l32, int hf) { return l32 * ROWB + ((hf ^ swz(l32)) << 4); }
  static __device__ __forceinline__ int col_of(int lane) {
    const int vr = 4 * (lane >> 5) + ((lane & 15) >> 2);
    return vr * ROWB + (((2 * ((lane >> 4) & 1) + ((lane & 3) >> 1)) ^ swz(vr)) << 4) + (lane & 1) * 8;
  }
  static __device__ __forceinline__ u32x4_t row_at(const unsigned char* t, int r0, int it, int st) {
    return *(const u32x4_t*)(t + ((it ^ (32 * st)) + r0 * ROWB));
  }
  static __device__ __forceinline__ u32x4_t col_at(const unsigned char* t, int r0, int it, int g, int mt) {
    u32x4_t r;
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      const uint2 h = lds_read_tr(t + ((it ^ (64 * mt ^ 32 * x)) + (r0 + 16 * g + 8 * x) * ROWB));
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
  static __device__ __forceinline__ int row_of(int l32, int hf) { return l32 * ROWB + 32 * hf; }
  static __device__ __forceinline__ int col_of(int lane) { return 4 * (lane >> 5) * ROWB + 4 * (lane & 31); }
  static __device__ __forceinline__ F32x8 row_at(const unsigned char* t, int r0, int it, int st) {
    return Frag<float>::load((const float*)(t + (it + r0 * ROWB + 64 * st)));
  }
  static __device__ __forceinline__ F32x8 col_at(const unsigned char* t, int r0, int it, int g, int mt) {
    F32x8 r;
#pragma unroll
    for (int e = 0; e < 8; ++e)
      r.v[e] = *(const float*)(t + (it + (r0 + 16 * g + 8 * (e >> 2) + (e & 3)) * ROWB + 128 * mt));
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

// Zeros in `heads` heads from h on of the rows [r0, r1), shared by the gx blocks of index bx.
template <typename T>
__device__ __forceinline__ void zero_rows(T* p, int64_t r0, int64_t r1, int H, int D, int h, int bx,
                                          int gx, int heads) {
  const int per = heads * D * (int)sizeof(T) / 16;
  for (int64_t i = threadIdx.x + (int64_t)bx * blockDim.x; i < (r1 - r0) * per;
       i += (int64_t)gx * blockDim.x)
    *(uint4*)((char*)(p + ((r0 + i / per) * H + h) * D) + 16 * (i % per)) = make_uint4(0, 0, 0, 0);
}
// ... of the rows outside every sequence, by the blocks of the first and the last sequence.
template <typename T>
__device__ __forceinline__ void zero_rest(T* p, const int32_t* cu, int64_t total, int bb, int H, int D,
                                          int h, int bx, int gx, int heads = 1) {
  int b0, n;
  if (bb == 0) {
    segment(cu, 0, total, &b0, &n);
    zero_rows(p, 0, b0, H, D, h, bx, gx, heads);
  }
  if (bb == (int)gridDim.z - 1) {
    segment(cu, bb, total, &b0, &n);
    zero_rows(p, b0 + n, total, H, D, h, bx, gx, heads);
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

}  // namespace
}  // namespace tsc
