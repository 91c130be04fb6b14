// Device helpers shared by the attention kernels (attention.hip, diff_attention.hip): the matrix
// products of 16-bit fragments, exchanges between a wave's halves, sequence bounds, the block ->
// tile mapping and transposed LDS reads.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace tsc {
namespace {

typedef __bf16 bf16x8_t __attribute__((__vector_size__(8 * sizeof(__bf16))));
typedef _Float16 f16x8_t __attribute__((__vector_size__(8 * sizeof(_Float16))));
typedef float f32x16_t __attribute__((__vector_size__(16 * sizeof(float))));
typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));
typedef float f32x2_t __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));
typedef _Float16 f16x2_t __attribute__((ext_vector_type(2)));

template <typename T>
struct Mma;
template <>
struct Mma<__bf16> {
  static __device__ __forceinline__ void run(u32x4_t a, u32x4_t b, f32x16_t& c) {
    c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_t, a),
                                                __builtin_bit_cast(bf16x8_t, b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ uint32_t pack(float lo, float hi) {  // RNE, one cvt_pk
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2_t{lo, hi}, bf16x2_t));
  }
  // acc + the two packed values (v_dot2 with (1, 1)): the softmax denominator is summed over the
  // same rounded P that the second product uses.
  static __device__ __forceinline__ float add2(uint32_t packed, float acc) {
    return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2_t, packed),
                                          __builtin_bit_cast(bf16x2_t, 0x3f803f80u), acc, false);
  }
};
template <>
struct Mma<_Float16> {
  static __device__ __forceinline__ void run(u32x4_t a, u32x4_t b, f32x16_t& c) {
    c = __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8_t, a),
                                               __builtin_bit_cast(f16x8_t, b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ uint32_t pack(float lo, float hi) {
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2_t{lo, hi}, f16x2_t));
  }
  static __device__ __forceinline__ float add2(uint32_t packed, float acc) {
    return __builtin_amdgcn_fdot2(__builtin_bit_cast(f16x2_t, packed),
                                  __builtin_bit_cast(f16x2_t, 0x3c003c00u), acc, false);
  }
};

__device__ __forceinline__ float fast_exp2(float x) { return __builtin_amdgcn_exp2f(x); }

// Max / sum of a value and the one held by lane l ^ 32 (both halves of the wave hold the same
// query): v_permlane32_swap exchanges the wave halves in registers (no LDS round trip).
__device__ __forceinline__ float pair_max(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float pair_sum(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// Segment b's [begin, end) clamped into [0, total] (a malformed cu_seqlens cannot index outside).
__device__ __forceinline__ void segment(const int32_t* cu, int b, int64_t total, int* begin,
                                        int* len) {
  const int64_t s = min<int64_t>(max<int64_t>(cu[b], 0), total);
  const int64_t e = min<int64_t>(max<int64_t>(cu[b + 1], s), total);
  *begin = (int)s;
  *len = (int)(e - s);
}

// Block -> (q tile, head, sequence).  Blocks start in the order of their index and go to the 8 XCDs
// round robin.  Every XCD gets the same share of every sequence, whatever the sequences' lengths:
// of each eight heads XCD x takes one, so that a head's K and V come into one L2 only, and the q
// tiles of the heads past a multiple of eight are spread over all XCDs.  (Contiguous runs of
// blocks per XCD left the XCDs of the short sequences idle: 21.1 ms against 14.2 ms for sequences
// of 24.7 k and 39.6 k tokens, 12 x 128 bf16, MFMAs and softmax still in turn.)
// Sequences with more keys go first, so that the launch ends on its shortest blocks; past
// kMaxRanked sequences the ranking would cost more than the tail it saves, and they keep their
// order.
constexpr int kMaxRanked = 8;

__device__ __forceinline__ void block_tile(const int32_t* cu_kv, int* bx, int* bh, int* bb) {
  const int gx = gridDim.x, H = gridDim.y, B = gridDim.z;
  const int per_seq = gx * H;
  const int lin = blockIdx.x + gx * (blockIdx.y + H * blockIdx.z);
  const int slot = blockIdx.z, u = lin - slot * per_seq;
  const int whole = H & ~7;  // heads dealt one per XCD
  if (u < gx * whole) {      // a run of eight blocks holds every XCD once, so (u / 8, lin % 8) is
    const int i = u >> 3;    // another numbering of the same blocks
    *bx = i % gx;
    *bh = (i / gx) * 8 + (lin & 7);
  } else {
    *bx = blockIdx.x;
    *bh = blockIdx.y;
  }
  int seq = slot;
  if (B > 1 && B <= kMaxRanked) {  // lane 8 b + c: does sequence c come before sequence b?
    const int lane = threadIdx.x & 63, b = min(lane >> 3, B - 1), c = min(lane & 7, B - 1);
    const uint32_t len = (uint32_t)cu_kv[b + 1] - (uint32_t)cu_kv[b];
    const uint32_t other = (uint32_t)cu_kv[c + 1] - (uint32_t)cu_kv[c];
    const bool before = (lane & 7) < B && (other > len || (other == len && c < b));
    const uint64_t all = __builtin_amdgcn_ballot_w64(before);
    const bool mine = lane < B && __popc((uint32_t)(all >> (8 * (lane & 7))) & 0xffu) == slot;
    seq = __builtin_ctzll(__builtin_amdgcn_ballot_w64(mine));  // exactly one lane
  }
  *bb = seq;
}

typedef short s16x4_t __attribute__((ext_vector_type(4)));
// Lane i of each 16 gets column i of the 4 rows x 16 columns whose row r the lanes 4r..4r+3
// address (8 bytes each).
__device__ __forceinline__ uint2 lds_read_tr(const unsigned char* p) {
#if defined(__HIP_DEVICE_COMPILE__)
  return __builtin_bit_cast(
      uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                 (__attribute__((address_space(3))) s16x4_t*)(__attribute__((address_space(3))) void*)p));
#else
  return make_uint2(0, 0);
#endif
}

}  // namespace
}  // namespace tsc
