// q8_core.h -- the 8-bit checkpoint format of include/csnet_hip.h: 32 elements share a power of two, one byte of code each.
//
// The block's exponent follows from the bits of its largest finite magnitude amax = 1.f 2^(E - 127).  With e = E - 127 - 6 the
// scaled maximum lies in [64, 128) and rounds to 128 (one too many for int8) from 127.5 on, that is from a fraction of 0x7f0000:
// adding 0x10000 to the bits carries into E exactly then.  For e4m3, e = E - 127 - 8 puts it into [256, 512); 464 is the last number
// that still rounds (to even) to 448, fraction 0x680000: adding 0x17ffff carries from 0x680001 on.
#pragma once
#include "csn_device.h"

enum { Q8_INT8 = 0, Q8_E4M3 = 1 };
#define Q8_MIN_EXP 32       // 2^-95: the smallest step; keeps every value a normal number in bfloat16 and float
#define Q8_NAN_INT8 0x80u
#define Q8_NAN_E4M3 0x7fu

template <int FMT>
__device__ __forceinline__ unsigned q8_exponent(float amax) {
  const unsigned b = csn_f_bits(amax);
  const int s = FMT == Q8_INT8 ? (int)((b + 0x10000u) >> 23) - 6 : (int)((b + 0x17ffffu) >> 23) - 8;
  return (unsigned)(s < Q8_MIN_EXP ? Q8_MIN_EXP : s);
}
__device__ __forceinline__ float q8_scale(unsigned s) { return csn_bits_f(s << 23); }             // 2^(s - 127)
__device__ __forceinline__ float q8_inv_scale(unsigned s) { return csn_bits_f((254u - s) << 23); }   // 2^(127 - s)
// what the codes can hold: not infinities, NaN or magnitudes that would round to 2^128 (they would unpack to an infinity)
template <int FMT>
__device__ __forceinline__ bool q8_in_range(float x) { return (csn_f_bits(x) & 0x7fffffffu) < (FMT == Q8_INT8 ? 0x7f7f0000u : 0x7f680001u); }
// |x| for the block maximum: values out of range do not take part
template <int FMT>
__device__ __forceinline__ float q8_mag(float x) { return q8_in_range<FMT>(x) ? fabsf(x) : 0.f; }

// the e4m3 number nearest to |v| <= 448 (3 fraction bits, exponents 2^-6 .. 2^8, subnormal step 2^-9), sign in bit 7
__device__ __forceinline__ unsigned q8_to_e4m3(float v) {
#ifdef CSN_CPU_EMU
  const unsigned b = csn_f_bits(v), sign = (b >> 24) & 0x80u;
  const float a = fabsf(v);
  if (a < 0.015625f) return sign | (unsigned)rintf(a * 512.f);           // (8 = the first normal number's code)
  const int ex = (int)((b >> 23) & 0xffu) - 127;
  return sign | (unsigned)(((ex + 7) << 3) + (int)rintf(a * csn_bits_f((unsigned)(127 + 3 - ex) << 23)) - 8);   // (16: carries)
#else
  return (unsigned)__builtin_amdgcn_cvt_pk_fp8_f32(v, v, 0, false) & 0xffu;
#endif
}
__device__ __forceinline__ float q8_from_e4m3(unsigned c) {
#ifdef CSN_CPU_EMU
  const unsigned ex = (c >> 3) & 15u, m = c & 7u;
  if ((c & 0x7fu) == 0x7fu) return csn_bits_f(0x7fc00000u);
  const float a = ex ? (float)(8u + m) * csn_bits_f((ex + 117u) << 23) : (float)m * 0.001953125f;   // (8 + m) 2^(ex - 10)
  return (c & 0x80u) ? -a : a;
#else
  return __builtin_amdgcn_cvt_f32_fp8((int)c, 0);
#endif
}

template <int FMT>
__device__ __forceinline__ unsigned q8_encode(float x, float inv) {
  if (FMT == Q8_INT8) return q8_in_range<FMT>(x) ? (unsigned)(int)rintf(x * inv) & 0xffu : Q8_NAN_INT8;
  return q8_in_range<FMT>(x) ? q8_to_e4m3(x * inv) : Q8_NAN_E4M3;
}
template <int FMT>
__device__ __forceinline__ float q8_decode(unsigned c, float scale) {
  if (FMT == Q8_INT8) return c == Q8_NAN_INT8 ? csn_bits_f(0x7fc00000u) : (float)(int)(signed char)c * scale;
  return q8_from_e4m3(c) * scale;
}

// E codes at once, packed in dwords
template <int FMT, int E>
__device__ __forceinline__ void q8_encode_vec(const float (&f)[E], float inv, unsigned (&w)[E / 4]) {
#pragma unroll
  for (int j = 0; j < E / 4; ++j)
    w[j] = q8_encode<FMT>(f[4 * j], inv) | q8_encode<FMT>(f[4 * j + 1], inv) << 8 | q8_encode<FMT>(f[4 * j + 2], inv) << 16 |
           q8_encode<FMT>(f[4 * j + 3], inv) << 24;
}
template <int FMT, int E>
__device__ __forceinline__ void q8_decode_vec(const unsigned (&w)[E / 4], float scale, float (&f)[E]) {
#pragma unroll
  for (int j = 0; j < E; ++j) f[j] = q8_decode<FMT>((w[j >> 2] >> (8 * (j & 3))) & 0xffu, scale);
}
#ifndef CSN_EMU_SEQ
// exponent of the block that the 32 / E neighbouring lanes hold together
template <int FMT, int E>
__device__ __forceinline__ unsigned q8_block_exponent(const float (&f)[E]) {
  float m = 0.f;
#pragma unroll
  for (int j = 0; j < E; ++j) m = fmaxf(m, q8_mag<FMT>(f[j]));
  m = fmaxf(m, csn_lane_xor_f32<1>(m));
  m = fmaxf(m, csn_lane_xor_f32<2>(m));
  if (E == 4) m = fmaxf(m, csn_lane_xor_f32<4>(m));
  return q8_exponent<FMT>(m);
}
#endif
