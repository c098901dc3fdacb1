// bank8.h -- the paged 8-bit bank: storage, code conversions and argument checks, shared by bank8.hip (plan, append, gather) and
// bank8_attn.hip (the read).
//
// A page holds `page` tokens of every head, one byte per element, laid out for the read's MFMA operands:
//   keys    [page][head][dim/16][token][16]             a lane's 16 bytes = 16 dims of one token (A operand of S^T = K . Q^T)
//   values  [page][head][token/32][half][dim][16]       a lane's 16 bytes = 16 tokens of one dim (A operand of O^T = V^T . P^T):
//                                                       byte 4 m + r of half h is token 8 m + 4 h + r of its 32-token tile --
//                                                       the order in which the accumulators of S^T hold a lane's 16 tokens
// so that every operand load is one contiguous 1 KB per wave and the weights never cross lanes between the two products.
#pragma once
#include "../../include/rmem_hip.h"
#include "rmem_common.h"

namespace bank8 {

constexpr int INT8 = 0, E4M3 = 1;         // rmem_bank8.code
constexpr int FP32 = 0, FP16 = 1, BF16 = 2;   // dense tensors

typedef __attribute__((ext_vector_type(2))) unsigned int u32x2_t;
typedef __attribute__((ext_vector_type(4))) float f32x4_t;

// 4 codes -> 4 fp16 values, exact.  int8 codes are held as code + 128: v_perm puts the byte into the mantissa of 1024.0 and a
// packed fp16 subtraction takes 1024 + 128 off again; e4m3 has an instruction of its own.
template <int CODE>
__device__ __forceinline__ void decode4(uint32_t u, uint32_t& a, uint32_t& b) {
  if constexpr (CODE == INT8) {
    const f16x2_t off = {(_Float16)1152.f, (_Float16)1152.f};
    a = __builtin_bit_cast(uint32_t, __builtin_bit_cast(f16x2_t, __builtin_amdgcn_perm(0x64646464u, u, 0x04010400u)) - off);
    b = __builtin_bit_cast(uint32_t, __builtin_bit_cast(f16x2_t, __builtin_amdgcn_perm(0x64646464u, u, 0x04030402u)) - off);
  } else {
    a = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(u, 1.0f, false));
    b = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(u, 1.0f, true));
  }
}
// 8 codes (two dwords) -> one MFMA operand fragment
template <int CODE>
__device__ __forceinline__ frag8_t decode8(uint32_t u0, uint32_t u1) {
  uint32_t a, b, c, d;
  decode4<CODE>(u0, a, b);
  decode4<CODE>(u1, c, d);
  u32x4_t w;
  w[0] = a; w[1] = b; w[2] = c; w[3] = d;
  return __builtin_bit_cast(frag8_t, w);
}

// Four numbers in units of the scale -> four code bytes: round to nearest even, saturating, NaN -> 0.  int8: adding 1.5 * 2^23 + 128
// leaves the rounded number + 128 in the low byte.
__device__ __forceinline__ float clean(float x, float top) {
  x = x == x ? x : 0.f;
  return __builtin_amdgcn_fmed3f(x, -top, top);
}
// CLEAN false: the four are known to be finite and at most half a step beyond the largest code's value.
template <int CODE, bool CLEAN = true>
__device__ __forceinline__ uint32_t encode4(float a, float b, float c, float d) {
#pragma clang fp contract(off)             // (a product that comes in is rounded before it is rounded to a code)
  if constexpr (CLEAN) {
    constexpr float top = CODE == INT8 ? 127.f : 448.f;
    a = clean(a, top);
    b = clean(b, top);
    c = clean(c, top);
    d = clean(d, top);
  }
  if constexpr (CODE == INT8) {
    const uint32_t x = __float_as_uint(a + 12583040.f), y = __float_as_uint(b + 12583040.f),
                   z = __float_as_uint(c + 12583040.f), w = __float_as_uint(d + 12583040.f);
    return __builtin_amdgcn_perm(__builtin_amdgcn_perm(w, z, 0x0c0c0400u), __builtin_amdgcn_perm(y, x, 0x0c0c0400u), 0x05040100u);
  } else {
    const int lo = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, lo, true);
  }
}
// four code bytes -> their values
template <int CODE>
__device__ __forceinline__ f32x4_t values4(uint32_t u) {
  f32x4_t x;
  if constexpr (CODE == INT8) {
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = (float)((u >> (8 * i)) & 0xffu) - 128.f;
  } else {
    uint32_t a, b;
    decode4<CODE>(u, a, b);
    const f16x2_t p = __builtin_bit_cast(f16x2_t, a), q = __builtin_bit_cast(f16x2_t, b);
    x[0] = (float)p[0]; x[1] = (float)p[1]; x[2] = (float)q[0]; x[3] = (float)q[1];
  }
  return x;
}
template <int CODE>
__device__ __forceinline__ uint32_t recode4(uint32_t u, float ratio) {       // codes of a page whose scale has risen
  const f32x4_t x = values4<CODE>(u) * ratio;
  return encode4<CODE>(x[0], x[1], x[2], x[3]);
}
template <int CODE>
__device__ __forceinline__ uint32_t zeros4() { return CODE == INT8 ? 0x80808080u : 0u; }

// Argument checks shared by the entry points (no HIP call: they run without a GPU).
inline bool valid_bank(const rmem_bank8* b) {
  return b && b->k && b->v && b->k_scale && b->v_scale && b->pages > 0 && b->heads > 0 &&
         (b->page == 32 || b->page == 64 || b->page == 128) && (b->dim == 32 || b->dim == 64 || b->dim == 128) &&
         (b->code == INT8 || b->code == E4M3) && (int64_t)b->pages * b->page <= 0x7fffffff &&
         ((uintptr_t)b->k % 16) == 0 && ((uintptr_t)b->v % 16) == 0;
}
inline bool valid_type(int t) { return t == FP32 || t == FP16 || t == BF16; }
inline int log2_of(int x) { return x == 32 ? 5 : x == 64 ? 6 : 7; }

}  // namespace bank8
