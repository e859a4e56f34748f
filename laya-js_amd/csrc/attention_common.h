// Device helpers of the 16-bit attention kernels with 32 queries per wave: the
// operand layouts of v_mfma_f32_32x32x16 over 64-key, 64-column tiles of K and V
// in LDS, the loads that fill them, and the exchanges between the lanes of a
// query.
#pragma once
#include "common.h"

namespace hb {

struct S4 {
  int64_t s[4];
};

static S4 s4(const int64_t* p) {
  S4 r;
  for (int i = 0; i < 4; i++) r.s[i] = p ? p[i] : 0;
  return r;
}

template <bool BF16>
__device__ __forceinline__ float tof(uint32_t h) {
  return BF16 ? bf16_to_f32((uint16_t)h) : f16_bits_to_f32((uint16_t)h);
}
template <bool BF16>
__device__ __forceinline__ uint32_t fromf(float v) {
  return BF16 ? f32_to_bf16(v) : f32_to_f16_bits(v);
}

// Two f32 values packed as 16-bit (v_cvt_pk_f16_f32 / v_cvt_pk_bf16_f32: RNE).
template <bool BF16>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  typedef float float2v __attribute__((ext_vector_type(2)));
  if constexpr (BF16) {
    typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(uint32_t, __builtin_convertvector((float2v){a, b}, bf16x2));
  } else {
    return __builtin_bit_cast(uint32_t, __builtin_convertvector((float2v){a, b}, half2v));
  }
}

// Cross-lane exchanges for the 4 lanes that hold one query (lane, lane ^ 16,
// lane ^ 32, lane ^ 48): ds_swizzle in bit-mask mode (and 0x1f, xor 0x10)
// reads lane ^ 16 within each half-wave; v_permlane32_swap exchanges the
// two halves, returning (per lane) its own value and the one of lane ^ 32.
__device__ __forceinline__ float from_xor16(float x) {
  return __builtin_bit_cast(float, __builtin_amdgcn_ds_swizzle(__builtin_bit_cast(int, x), 0x401F));
}
__device__ __forceinline__ float max_xor32(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(uint32_t, x), __builtin_bit_cast(uint32_t, x),
                                                  false, false);
  return fmaxf(__builtin_bit_cast(float, (uint32_t)r[0]), __builtin_bit_cast(float, (uint32_t)r[1]));
}
__device__ __forceinline__ float sum_xor32(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(uint32_t, x), __builtin_bit_cast(uint32_t, x),
                                                  false, false);
  return __builtin_bit_cast(float, (uint32_t)r[0]) + __builtin_bit_cast(float, (uint32_t)r[1]);
}

typedef short short4t __attribute__((ext_vector_type(4)));
// Transposing LDS read: within 16 lanes, lanes 4r .. 4r + 3 point at 4 x 4
// consecutive values of row r; lane c gets column c's 4 rows.
__device__ __forceinline__ uint2v lds_tr16(const uint16_t* p) {
  const short4t v = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) short4t*)p);
  return __builtin_bit_cast(uint2v, v);
}
template <bool BF16>
__device__ __forceinline__ float16v mfma32x16(const uint4v& a, const uint4v& b, float16v c) {
  if constexpr (BF16)
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0,
                                                   0, 0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(half8, a), __builtin_bit_cast(half8, b), c, 0, 0,
                                                  0);
}

// chunk c (8 values) of row r of a [64][64] K or V tile sits at c ^ kv_f(r): a
// 16-lane pass of the K fragment reads (16 rows, one chunk) and of the V
// transpose reads (4 rows, 4 chunks) covers all 64 banks
__device__ __forceinline__ int kv_f(int r) { return (((r >> 1) & 1) << 2) | ((r >> 2) & 3); }

// LDS element offsets of a lane's fragment reads within a [64][64] tile: K
// chunk 2 s + lg of row l32 (+ 2048 for the second 32 keys); V transpose
// read of keys 16 t + 8 u + 4 lg .., columns 32 d .. (+ 1024 t).
struct Frag32 {
  int ka[4], va[2][2];
};
__device__ __forceinline__ Frag32 frag32(int lane) {
  Frag32 f;
  const int l32 = lane & 31, lg = lane >> 5, j16 = lane & 15, vrow = 4 * lg + (j16 >> 2);
#pragma unroll
  for (int s = 0; s < 4; s++) f.ka[s] = l32 * 64 + (((2 * s + lg) ^ kv_f(l32)) << 3);
#pragma unroll
  for (int u = 0; u < 2; u++)
#pragma unroll
    for (int d = 0; d < 2; d++) {
      const int r = 8 * u + vrow, c = 4 * d + 2 * ((lane >> 4) & 1) + ((j16 & 3) >> 1);
      f.va[u][d] = r * 64 + ((c ^ kv_f(r)) << 3) + 4 * (j16 & 1);
    }
  return f;
}

// A K or V tile by direct-to-LDS loads: 8 pieces of 1 KB (8 rows); a piece's
// lane l fills slot l % 8 of row l / 8, so it fetches chunk (l % 8) ^
// kv_f(row).  Rows past Lk become zeros (an offset past the buffer's records).
// The caller waits for the loads (vmcnt(0)).
__device__ __forceinline__ void dma_piece(const uint16_t* base, int64_t stride, int k0, int piece, int Lk, uint16_t* dst,
                                          int lane) {
  const uint64_t a = (uint64_t)(base + (int64_t)k0 * stride);
  const uint4v rs = {(uint32_t)__builtin_amdgcn_readfirstlane((uint32_t)a),
                     (uint32_t)__builtin_amdgcn_readfirstlane((uint32_t)(a >> 32) & 0xffffu), 0x80000000u, 0x00020000u};
  const int r = piece * 8 + (lane >> 3);
  const uint32_t off = __umul24(r, (uint32_t)stride) * 2u + (((lane & 7) ^ kv_f(r)) << 4);
  const uint32_t lds = (uint32_t)__builtin_amdgcn_readfirstlane(
      (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint16_t*)(dst + piece * 512));
  buffer_lds16(rs, k0 + r < Lk ? off : 0xfffffff0u, lds);
}

}  // namespace hb
