// bank8.h -- the paged 8-bit bank: storage, code conversions and the division of a read into units, shared by
// bank8.hip (plan, append, gather) and bank8_attn.hip (the read).
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

__device__ __forceinline__ float decode1(uint32_t byte, int code) {
  if (code == INT8) return (float)(int)byte - 128.f;
  const f16x2_t h = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(byte, 1.0f, false);
  return (float)h[0];
}
// x in units of the scale -> code byte, round to nearest even, saturating; NaN -> 0
__device__ __forceinline__ uint32_t encode1(float x, int code) {
  x = x == x ? x : 0.f;
  if (code == INT8) return (uint32_t)((int)rintf(fminf(fmaxf(x, -127.f), 127.f)) + 128);
  x = fminf(fmaxf(x, -448.f), 448.f);
  return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(x, 0.f, 0, false) & 0xffu;
}
__device__ __forceinline__ uint32_t zero_code(int code) { return code == INT8 ? 128u : 0u; }
__device__ __forceinline__ float code_top(int code) { return code == INT8 ? 127.f : 448.f; }

template <int T>
struct Elem;
template <>
struct Elem<FP32> { typedef float type; };
template <>
struct Elem<FP16> { typedef _Float16 type; };
template <>
struct Elem<BF16> { typedef __bf16 type; };

__device__ __forceinline__ float load1(const void* p, long i, int type) {
  if (type == FP32) return static_cast<const float*>(p)[i];
  if (type == FP16) return (float)static_cast<const _Float16*>(p)[i];
  return (float)static_cast<const __bf16*>(p)[i];
}
__device__ __forceinline__ void store1(void* p, long i, float x, int type) {
  if (type == FP32) static_cast<float*>(p)[i] = x;
  else if (type == FP16) static_cast<_Float16*>(p)[i] = (_Float16)x;
  else static_cast<__bf16*>(p)[i] = (__bf16)x;
}

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
