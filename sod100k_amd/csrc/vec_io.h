// vec_io.h -- 16 bytes of consecutive elements per lane, from and to any element address (training operators beside the plan).
//
// Rows and planes of odd sizes start anywhere, so the vector types below claim the alignment of one element only: the hardware takes
// 128-bit global accesses at any address and a misaligned wave touches one more line, where a loop over elements would take eight
// instructions.  The last piece of a row, n < E elements long, is loaded as the row's last E elements and shifted down; it is
// stored element by element.  Rows shorter than E are loaded element by element too (a form of its own: WIDE = false).
#pragma once
#include <type_traits>

#include "csn_device.h"

struct __attribute__((packed, aligned(2))) csn_raw16_a2 { unsigned w[4]; };
struct __attribute__((packed, aligned(2))) csn_raw8_a2 { unsigned w[2]; };
struct __attribute__((packed, aligned(4))) csn_raw16_a4 { unsigned w[4]; };
struct __attribute__((packed, aligned(1))) csn_raw16_a1 { unsigned w[4]; };
struct __attribute__((packed, aligned(1))) csn_raw8_a1 { unsigned w[2]; };
struct __attribute__((packed, aligned(1))) csn_raw4_a1 { unsigned w[1]; };

// The compiler may not reuse what it computed from w before this point: a second pass over loaded elements unpacks them again
// instead of keeping two to four times as many registers across the sum in between.
__device__ __forceinline__ void csn_pin(unsigned& w) {
#ifndef CSN_CPU_EMU
  asm volatile("" : "+v"(w));
#else
  (void)w;
#endif
}

// elements to step back so that E elements from there end at the row's end; n = elements of the row from here on
__device__ __forceinline__ int vec_back(int n, int E) { return n >= E ? 0 : E - n; }

// E elements of a tensor as they were loaded: 16 bytes, or four elements whatever their size
template <typename AT> struct VecElems { static constexpr int E = 16 / sizeof(AT); };
template <typename AT, int E_ = VecElems<AT>::E> struct VecIo;
template <int E_> struct VecIo<csn_bf16, E_> {
  static constexpr int E = E_, W = E / 2;
  unsigned w[W];
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int j = 0; j < W; ++j) w[j] = 0;
  }
  __device__ __forceinline__ void load(const csn_bf16* p) {
    if constexpr (E == 8) {
      const csn_raw16_a2 r = *reinterpret_cast<const csn_raw16_a2*>(p);
#pragma unroll
      for (int j = 0; j < W; ++j) w[j] = r.w[j];
    } else {
      const csn_raw8_a2 r = *reinterpret_cast<const csn_raw8_a2*>(p);
#pragma unroll
      for (int j = 0; j < W; ++j) w[j] = r.w[j];
    }
  }
  __device__ __forceinline__ void load_each(const csn_bf16* p, int n) {
#pragma unroll
    for (int j = 0; j < E; ++j)
      if (j < n) w[j >> 1] |= (unsigned)p[j].u << (16 * (j & 1));
  }
  __device__ __forceinline__ void shift(int s) {   // drop the first s < E elements
    if (E == 8 && (s & 4)) {
#pragma unroll
      for (int j = 0; j < W / 2; ++j) { w[j] = w[j + W / 2]; w[j + W / 2] = 0; }
    }
    if (s & 2) {
#pragma unroll
      for (int j = 0; j + 1 < W; ++j) w[j] = w[j + 1];
      w[W - 1] = 0;
    }
    if (s & 1) {
#pragma unroll
      for (int j = 0; j + 1 < W; ++j) w[j] = csn_alignbit(w[j + 1], w[j], 16);
      w[W - 1] >>= 16;
    }
  }
  __device__ __forceinline__ void pin() {
#pragma unroll
    for (int j = 0; j < W; ++j) csn_pin(w[j]);
  }
  __device__ __forceinline__ void get(float (&f)[E]) const {
#pragma unroll
    for (int j = 0; j < W; ++j) { f[2 * j] = csn_bits_f(w[j] << 16); f[2 * j + 1] = csn_bits_f(w[j] & 0xffff0000u); }
  }
  static __device__ __forceinline__ void store(csn_bf16* p, const float (&f)[E], int n) {
    if (n >= E) {
      typedef typename std::conditional<E == 8, csn_raw16_a2, csn_raw8_a2>::type raw;
      raw o;
#pragma unroll
      for (int j = 0; j < W; ++j) o.w[j] = csn_pack_bf2(f[2 * j], f[2 * j + 1]);
      *reinterpret_cast<raw*>(p) = o;
    } else {
#pragma unroll
      for (int j = 0; j < E; ++j)
        if (j < n) p[j].u = csn_f2bf(f[j]);
    }
  }
};
template <> struct VecIo<float, 4> {
  static constexpr int E = 4;
  unsigned w[4];
  __device__ __forceinline__ void zero() { w[0] = w[1] = w[2] = w[3] = 0; }
  __device__ __forceinline__ void load(const float* p) {
    const csn_raw16_a4 r = *reinterpret_cast<const csn_raw16_a4*>(p);
#pragma unroll
    for (int j = 0; j < 4; ++j) w[j] = r.w[j];
  }
  __device__ __forceinline__ void load_each(const float* p, int n) {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (j < n) w[j] = csn_f_bits(p[j]);
  }
  __device__ __forceinline__ void shift(int s) {
    if (s & 2) { w[0] = w[2]; w[1] = w[3]; w[2] = w[3] = 0; }
    if (s & 1) { w[0] = w[1]; w[1] = w[2]; w[2] = w[3]; w[3] = 0; }
  }
  __device__ __forceinline__ void pin() {
#pragma unroll
    for (int j = 0; j < 4; ++j) csn_pin(w[j]);
  }
  __device__ __forceinline__ void get(float (&f)[4]) const {
#pragma unroll
    for (int j = 0; j < 4; ++j) f[j] = csn_bits_f(w[j]);
  }
  static __device__ __forceinline__ void store(float* p, const float (&f)[4], int n) {
    if (n >= 4) {
      csn_raw16_a4 o;
#pragma unroll
      for (int j = 0; j < 4; ++j) o.w[j] = csn_f_bits(f[j]);
      *reinterpret_cast<csn_raw16_a4*>(p) = o;
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (j < n) p[j] = f[j];
    }
  }
};
// Load the piece of a row whose next element is p[0] and that has n more elements (n <= 0: nothing is read); WIDE: the row has at
// least E elements.  vec_end() after the loads of a batch drops what a stepped-back piece holds of its predecessor.
template <bool WIDE, typename AT, int E>
__device__ __forceinline__ void vec_load(VecIo<AT, E>& v, const AT* p, int n) {
  v.zero();
  if (WIDE) {
    if (n > 0) v.load(p - vec_back(n, E));
  } else {
    v.load_each(p, n);
  }
}
template <bool WIDE, typename AT, int E>
__device__ __forceinline__ void vec_end(VecIo<AT, E>& v, int n) {
  if (WIDE && n > 0 && n < E) v.shift(E - n);
}

// E codes (one byte each) of a checkpoint
template <int E> struct CodeRaw;
template <> struct CodeRaw<8> { typedef csn_raw8_a1 type; };
template <> struct CodeRaw<4> { typedef csn_raw4_a1 type; };
template <int E> struct CodeIo {
  static constexpr int W = E / 4;
  unsigned w[W];
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int j = 0; j < W; ++j) w[j] = 0;
  }
  __device__ __forceinline__ void load(const uint8_t* p) {
    const typename CodeRaw<E>::type r = *reinterpret_cast<const typename CodeRaw<E>::type*>(p);
#pragma unroll
    for (int j = 0; j < W; ++j) w[j] = r.w[j];
  }
  __device__ __forceinline__ void pin() {
#pragma unroll
    for (int j = 0; j < W; ++j) csn_pin(w[j]);
  }
};
template <bool WIDE, int E>
__device__ __forceinline__ void code_load(CodeIo<E>& v, const uint8_t* p, int n) {
  v.zero();
  if (WIDE) {
    if (n > 0) v.load(p - vec_back(n, E));
  } else {
#pragma unroll
    for (int j = 0; j < E; ++j)
      if (j < n) v.w[j >> 2] |= (unsigned)p[j] << (8 * (j & 3));
  }
}
template <bool WIDE, int E>
__device__ __forceinline__ void code_end(CodeIo<E>& v, int n) {
  if (WIDE && n > 0 && n < E) {
    if (E == 8) {
      const unsigned long long u = ((unsigned long long)v.w[E / 4 - 1] << 32 | v.w[0]) >> (8 * (E - n));
      v.w[0] = (unsigned)u; v.w[E / 4 - 1] = (unsigned)(u >> 32);
    } else {
      v.w[0] >>= 8 * (E - n);
    }
  }
}
template <int E>
__device__ __forceinline__ void code_store(uint8_t* p, const unsigned (&w)[E / 4], int n) {
  if (n >= E) {
    typename CodeRaw<E>::type r;
#pragma unroll
    for (int j = 0; j < E / 4; ++j) r.w[j] = w[j];
    *reinterpret_cast<typename CodeRaw<E>::type*>(p) = r;
  } else {
#pragma unroll
    for (int j = 0; j < E; ++j)
      if (j < n) p[j] = (uint8_t)(w[j >> 2] >> (8 * (j & 3)));
  }
}
