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
template <int FMT> struct Q8Limit { static constexpr unsigned bits = FMT == Q8_INT8 ? 0x7f7f0000u : 0x7f680001u; };
__device__ __forceinline__ unsigned q8_mag(float x) { return csn_f_bits(x) & 0x7fffffffu; }   // |x| as an integer of the same order
// ... for the block maximum: values out of range do not take part
template <int FMT>
__device__ __forceinline__ unsigned q8_mag_in_range(float x) { const unsigned m = q8_mag(x); return m < Q8Limit<FMT>::bits ? m : 0u; }

// four codes from four scaled values (|v| <= 127 / 448) in one dword.  int8: adding 1.5 2^23 leaves the rounded integer in the low
// bits of the sum
template <int FMT>
__device__ __forceinline__ unsigned q8_codes4(float a, float b, float c, float d) {
  if (FMT == Q8_INT8) {
    const float k = 12582912.f;
    const unsigned ua = csn_f_bits(a + k), ub = csn_f_bits(b + k), uc = csn_f_bits(c + k), ud = csn_f_bits(d + k);
#ifdef CSN_CPU_EMU
    return (ua & 0xffu) | (ub & 0xffu) << 8 | (uc & 0xffu) << 16 | ud << 24;
#else
    return __builtin_amdgcn_perm(__builtin_amdgcn_perm(ud, uc, 0x0c0c0400u), __builtin_amdgcn_perm(ub, ua, 0x0c0c0400u), 0x05040100u);
#endif
  }
#ifdef CSN_CPU_EMU
  // the e4m3 number nearest to |v| (3 fraction bits, exponents 2^-6 .. 2^8, subnormal step 2^-9), sign in bit 7
  const float v[4] = {a, b, c, d};
  unsigned w = 0;
  for (int j = 0; j < 4; ++j) {
    const unsigned u = csn_f_bits(v[j]), sign = (u >> 24) & 0x80u;
    const float m = fabsf(v[j]);
    const int ex = (int)((u >> 23) & 0xffu) - 127;
    const unsigned code = m < 0.015625f ? (unsigned)rintf(m * 512.f)      // (8 = the first normal number's code)
                                        : (unsigned)(((ex + 7) << 3) + (int)rintf(m * csn_bits_f((unsigned)(130 - ex) << 23)) - 8);
    w |= (sign | code) << (8 * j);
  }
  return w;
#else
  const int lo = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
  return (unsigned)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, lo, true);
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
__device__ __forceinline__ float q8_decode(unsigned c, float scale) {
  if (FMT == Q8_INT8) return c == Q8_NAN_INT8 ? csn_bits_f(0x7fc00000u) : (float)(int)(signed char)c * scale;
  return q8_from_e4m3(c) * scale;
}
// the values of E codes packed in dwords.  int8: the one code that is no number, 0x80, is looked for in four codes at a time
template <int FMT, int E>
__device__ __forceinline__ void q8_decode_vec(const unsigned (&w)[E / 4], float scale, float (&f)[E]) {
  if (FMT == Q8_INT8) {
    unsigned none = 0;
#pragma unroll
    for (int i = 0; i < E / 4; ++i) {
      const unsigned u = w[i] ^ 0x80808080u;
      none |= (u - 0x01010101u) & ~u & 0x80808080u;   // a zero byte
#pragma unroll
      for (int j = 0; j < 4; ++j) f[4 * i + j] = (float)(int)(signed char)(w[i] >> (8 * j)) * scale;
    }
    if (none) {
#pragma unroll
      for (int j = 0; j < E; ++j)
        if (((w[j >> 2] >> (8 * (j & 3))) & 0xffu) == Q8_NAN_INT8) f[j] = csn_bits_f(0x7fc00000u);
    }
  } else {
#ifdef CSN_CPU_EMU
    for (int j = 0; j < E; ++j) f[j] = q8_decode<FMT>((w[j >> 2] >> (8 * (j & 3))) & 0xffu, scale);
#else
    typedef float f2 __attribute__((ext_vector_type(2)));
#pragma unroll
    for (int i = 0; i < E / 4; ++i) {
      const f2 lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)w[i], false), hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)w[i], true);
      f[4 * i] = lo.x * scale; f[4 * i + 1] = lo.y * scale; f[4 * i + 2] = hi.x * scale; f[4 * i + 3] = hi.y * scale;
    }
#endif
  }
}

#ifndef CSN_EMU_SEQ
template <int LANES>
__device__ __forceinline__ unsigned q8_lanes_max(unsigned m) {   // over 2, 4 or 8 neighbouring lanes
  m = max(m, csn_f_bits(csn_lane_xor_f32<1>(csn_bits_f(m))));
  if (LANES >= 4) m = max(m, csn_f_bits(csn_lane_xor_f32<2>(csn_bits_f(m))));
  if (LANES >= 8) m = max(m, csn_f_bits(csn_lane_xor_f32<4>(csn_bits_f(m))));
  return m;
}
// Pack a block of 32 that 32 / L neighbouring lanes hold together, L elements each (zeros past a row's end): the exponent; codes in w.
// Values out of range are looked for once per block, in the maximum of everything.
template <int FMT, int L>
__device__ __forceinline__ unsigned q8_pack_block(const float (&f)[L], unsigned (&w)[L / 4]) {
  unsigned m = 0;
#pragma unroll
  for (int j = 0; j < L; ++j) m = max(m, q8_mag(f[j]));
  m = q8_lanes_max<32 / L>(m);
  const bool all = m < Q8Limit<FMT>::bits;
  if (!all) {
    m = 0;
#pragma unroll
    for (int j = 0; j < L; ++j) m = max(m, q8_mag_in_range<FMT>(f[j]));
    m = q8_lanes_max<32 / L>(m);
  }
  const unsigned s = q8_exponent<FMT>(csn_bits_f(m));
  const float inv = q8_inv_scale(s);
  if (all) {
#pragma unroll
    for (int j = 0; j < L / 4; ++j) w[j] = q8_codes4<FMT>(f[4 * j] * inv, f[4 * j + 1] * inv, f[4 * j + 2] * inv, f[4 * j + 3] * inv);
  } else {
#pragma unroll
    for (int j = 0; j < L / 4; ++j) {
      float g[4];
      unsigned none = 0;
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const bool in = q8_mag(f[4 * j + k]) < Q8Limit<FMT>::bits;
        g[k] = in ? f[4 * j + k] * inv : 0.f;
        none |= in ? 0u : (FMT == Q8_INT8 ? Q8_NAN_INT8 : Q8_NAN_E4M3) << (8 * k);   // (the code of 0 has no bits)
      }
      w[j] = q8_codes4<FMT>(g[0], g[1], g[2], g[3]) | none;
    }
  }
  return s;
}
#endif
