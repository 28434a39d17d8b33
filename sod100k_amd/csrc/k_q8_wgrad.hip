// k_q8_wgrad.hip -- weight and bias gradient of a product (1x1 convolution / linear layer) from the 8-bit checkpoint of its input.
//
//     dW[o][i] = sum_t dY[t][o] X[t][i],   db[o] = sum_t dY[t][o]        (X: the values of the checkpoint, q8_core.h)
//
// A matrix product whose reduction runs over the tokens.  A value of the checkpoint is a code of at most 8 significant bits times a
// power of two, that is a bfloat16 number, and the product of two bfloat16 numbers is exact in float: bfloat16 dY goes to
// v_mfma_f32_32x32x16_bf16 as it is.  A float dY is cut by truncation into three bfloat16 numbers of 8 bits each (exact), whose
// products with X go into the same accumulators: three matrix instructions, nothing lost but the accumulation's own rounding.
//
// Block = TM x TN of dW over a slab of the tokens.  64 tokens -- 128 of bfloat16 maps, whose codes then come by whole lines -- are staged at a
// time into two LDS buffers.
// Planar maps hold eight consecutive pixels of a channel together, an operand of the matrix instruction: LDS rows are channels,
// [row][tokens], operands are 128-bit reads.  The 16-byte piece c of row r lies at c ^ (r & 7), so that eight consecutive rows fall on eight
// different pieces.
// Token rows hold the channels of a token together: LDS rows are tokens, [64 tokens][row], as they come, and the operands -- eight
// tokens of a channel -- are formed by the transposing LDS read, four tokens of 16 channels per 16 lanes.  Its four rows' 32 bytes
// lie in different banks: the 16-byte pieces of token t are exchanged by an xor with 2 (t & 7).
//
// Few tiles and many tokens are the usual case (the channels of a map against its pixels), so the tokens are cut into slabs whose
// partial tiles a second kernel adds in order.
//
// Measured, us, with the sum of the slabs in brackets: 256 -> 128 channels over 32x88x88 bf16 47.9 (+5.5), 2.7 TB/s, where dY and the codes
// alone are 20.8 at the rate of a copy and the multiplications 14: no single part holds it (with steps of 64 tokens, 57 with the sum: 50
// without the exponents' loads, 45 without X's or without dY's, 53 without multiplying, 55 without decoding).  16384 tokens,
// 1024 -> 4096 channels, bf16: 177 (+15.7), 776 TFLOP/s of matrix instructions against 841 of the library's product of two bf16 tensors of
// these sizes.  37 -> 21 channels over 5x13x17 float 7.8 (+1.9).  float dY, with the sum, of the floor (three times the bf16 operations):
// 16384 tokens, 1024 -> 4096 632 of 347, 512 -> 512 50.6 of 21.7, 32x88x88, 256 -> 128 95.5 of 41.0: one wave per SIMD (the three parts fill
// the LDS), so that cutting and multiplying take turns.
#include "q8_core.h"
#include "slab_sum.h"
#include "train_ops.h"
#include "vec_io.h"

#ifdef CSN_EMU_SEQ
int csn_launch_q8_wgrad(const Q8WgradArgs&, int, int, int, void*) { return -1; }   // (matrix instructions: lane-exact mode only)
int64_t csn_q8_wgrad_partial_floats(int, int, int64_t, int64_t, int64_t, int64_t) { return 0; }
#else

template <int STEP>   // planar: channel rows of STEP tokens
__device__ __forceinline__ unsigned wg_piece(int row, int c) { return (unsigned)(row * (2 * STEP) + ((c ^ (row & 7)) << 4)); }
template <int C>   // token rows of C channels
__device__ __forceinline__ unsigned wg_token(int t, int piece) {
  constexpr int M = C >= 128 ? 7 : 3;
  return (unsigned)(t * (2 * C) + ((piece ^ ((t & M) << 1)) << 4));
}
__device__ __forceinline__ csn_u4 wg_u4(unsigned a, unsigned b, unsigned c, unsigned d) {
  csn_u4 r;
  r.x = a; r.y = b; r.z = c; r.w = d;
  return r;
}
// ds_read_b64_tr_b16: four 16-bit elements per lane from LDS, transposed within 16 lanes: result r of lane i is element i % 4 of lane
// 4 r + i / 4 of the 16.  Lanes 4 r .. 4 r + 3 point at 16 consecutive elements of row r; lane i ends with column i of the four rows.
__device__ __forceinline__ uint2 wg_read_tr16(const unsigned char* p) {
  uint2 r;
#ifdef CSN_EMU_LANES
  const unsigned lane = threadIdx.x & 63, i = lane & 15;
  const csn_emu::Xchg x = csn_emu::wave_xchg(11, nullptr, p, 8, true);
  unsigned short v[4];
  for (unsigned k = 0; k < 4; ++k) __builtin_memcpy(&v[k], x.tab + 64 * ((lane & ~15u) + 4 * k + (i >> 2)) + 2 * (i & 3), 2);
  __builtin_memcpy(&r, v, 8);
#else
  typedef short s4 __attribute__((ext_vector_type(4)));
  const s4 v = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s4*)(const_cast<unsigned char*>(p)));
  r = __builtin_bit_cast(uint2, v);
#endif
  return r;
}
// {the high halves of a and b}: two bfloat16 by truncation
__device__ __forceinline__ unsigned wg_hi2(float a, float b) {
#ifdef CSN_CPU_EMU
  return (csn_f_bits(a) >> 16) | (csn_f_bits(b) & 0xffff0000u);
#else
  return __builtin_amdgcn_perm(csn_f_bits(b), csn_f_bits(a), 0x07060302u);
#endif
}
// one of the three parts of a float and what is left of it
__device__ __forceinline__ float wg_cut(float& x) {
  const float h = csn_bits_f(csn_f_bits(x) & 0xffff0000u);
  x -= h;
  return h;
}

// eight consecutive elements of dY as they were loaded
template <typename AT> struct WgY;
template <> struct WgY<csn_bf16> {
  VecIo<csn_bf16> v;
  __device__ __forceinline__ void zero() { v.zero(); }
  __device__ __forceinline__ void load(const csn_bf16* p) { v.load(p); }
  __device__ __forceinline__ void load_each(const csn_bf16* p, int n) { v.load_each(p, n); }
  __device__ __forceinline__ void shift(int s) { v.shift(s); }
  __device__ __forceinline__ void get(float (&f)[8]) const { v.get(f); }
  __device__ __forceinline__ void put(unsigned char* lds, unsigned at, unsigned) const {
    *reinterpret_cast<csn_u4*>(lds + at) = wg_u4(v.w[0], v.w[1], v.w[2], v.w[3]);
  }
};
template <> struct WgY<float> {
  VecIo<float> a, b;
  __device__ __forceinline__ void zero() { a.zero(); b.zero(); }
  __device__ __forceinline__ void load(const float* p) { a.load(p); b.load(p + 4); }
  __device__ __forceinline__ void load_each(const float* p, int n) { a.load_each(p, n); b.load_each(p + 4, n - 4); }
  __device__ __forceinline__ void shift(int s) {   // drop the first s < 8 elements
    if (s & 4) { a = b; b.zero(); }
#pragma unroll
    for (int k = 2; k; k >>= 1)
      if (s & k) {
#pragma unroll
        for (int j = 0; j < 4; ++j) a.w[j] = j + k < 4 ? a.w[(j + k) & 3] : b.w[(j + k) & 3];
        b.shift(k);
      }
  }
  __device__ __forceinline__ void get(float (&f)[8]) const {
#pragma unroll
    for (int j = 0; j < 4; ++j) { f[j] = csn_bits_f(a.w[j]); f[4 + j] = csn_bits_f(b.w[j]); }
  }
  __device__ __forceinline__ void put(unsigned char* lds, unsigned at, unsigned part) const {
    float f[8];
    get(f);
#pragma unroll
    for (int q = 0; q < 3; ++q) {
      float h[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) h[j] = wg_cut(f[j]);
      *reinterpret_cast<csn_u4*>(lds + at + q * part) = wg_u4(wg_hi2(h[0], h[1]), wg_hi2(h[2], h[3]), wg_hi2(h[4], h[5]), wg_hi2(h[6], h[7]));
    }
  }
};

// tokens of a step; waves of a block and their grid over its tile
template <typename AT, bool ROWS, int TM, int TN> struct WgShape {
  static constexpr int STEP = !ROWS && sizeof(AT) == 2 ? 128 : 64;
  static constexpr int T = TM == 256 || (STEP == 128 && TM + TN > 128) ? 512 : 256;
  static constexpr int WM = T == 512 && TM > TN ? 4 : 2, WN = T / 64 / WM;
  static constexpr int MI = TM / WM / 32, NJ = TN / WN / 32;      // 32 x 32 tiles of a wave
  static constexpr int SMEM = 2 * ((sizeof(AT) == 4 ? 3 : 1) * TM + TN) * 2 * STEP;
};
// what a thread holds of a step in flight: pieces of eight elements of dY and of X (planar: n pixels of each are the map's)
template <typename AT, int NY, int NX> struct WgRegs {
  WgY<AT> y[NY];
  CodeIo<8> x[NX];
  unsigned s[NX];
  int n;
};

// WIDE: a plane / a token of either tensor has at least eight elements.  A piece that reaches past its end is then loaded stepped back
// and shifted (vec_io.h); channels past the last one are loaded from inside the tensor -- every entry of dW is a sum of its own and
// those are not stored -- and only tokens past the last one are cleared.
template <typename AT, int FMT, bool ROWS, bool WIDE, int TM, int TN>
__global__ __launch_bounds__((WgShape<AT, ROWS, TM, TN>::T)) void q8_wgrad_kernel(Q8WgradArgs a) {
  CSN_DYN_SMEM(unsigned char, sm);
  typedef WgShape<AT, ROWS, TM, TN> S;
  constexpr int PARTS = sizeof(AT) == 4 ? 3 : 1, T = S::T, MI = S::MI, NJ = S::NJ, STEP = S::STEP;
  constexpr unsigned YB = TM * 2 * STEP, BUF = PARTS * YB + TN * 2 * STEP;   // (STEP tokens x TM bfloat16 either way)
  constexpr int NY = TM * (STEP / 8) / T, NX = TN * (STEP / 8) / T;          // pieces per thread and step
  constexpr int PP = STEP / 8, PR = T / PP;                                  // planar: pieces of a channel, channels a load round covers
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  // (slab, tile) items in order over the XCDs (block b runs on XCD b % 8): the tiles of a slab read the same tokens, through one L2
  const int ntile = a.mtiles * a.ntiles, total = ntile * a.slabs, per = (total + 7) >> 3;
  const int item = (int)(blockIdx.x & 7u) * per + (int)(blockIdx.x >> 3);
  if (item >= total || (int)(blockIdx.x >> 3) >= per) return;
  const int slab = item / ntile, tile = item - slab * ntile;
  const int mt = tile / a.ntiles, nt = tile - mt * a.ntiles;
  const int o0 = mt * TM, i0 = nt * TN;
  const int s0 = slab * a.steps_per_slab, s1 = s0 + a.steps_per_slab;
  const bool bias = a.dbias != nullptr && nt == 0;

  float bsum[ROWS ? 8 : NY];
#pragma unroll
  for (int j = 0; j < (ROWS ? 8 : NY); ++j) bsum[j] = 0.f;
  WgRegs<AT, NY, NX> r0, r1;

  auto load = [&](WgRegs<AT, NY, NX>& rg, int step) {
    if constexpr (!ROWS) {   // piece j: channel tid / PP + j PR, eight pixels number tid % PP of the step
      const unsigned g = (unsigned)step * PP + (unsigned)(tid % PP);
      unsigned o = g / (unsigned)a.chunks, c = g - o * (unsigned)a.chunks;
      const bool in = (int64_t)o < a.outer;
      if (!in) { o = (unsigned)a.outer - 1; c = 0; }
      const int64_t p = (int64_t)c * 8;
      const int left = (int)min((int64_t)8, a.inner - p), n = in ? left : 0;
      rg.n = n;
      const AT* py = reinterpret_cast<const AT*>(a.dy) + (int64_t)o * a.dy_so + p;
      const int64_t row0 = (int64_t)o * a.cin;
      if constexpr (WIDE) {
        py -= 8 - left;
#pragma unroll
        for (int j = 0; j < NY; ++j) rg.y[j].load(py + (int64_t)min((int64_t)(o0 + tid / PP + PR * j), a.cout - 1) * a.dy_sc);
#pragma unroll
        for (int j = 0; j < NX; ++j) {
          const int64_t row = row0 + min((int64_t)(i0 + tid / PP + PR * j), a.cin - 1);
          rg.x[j].load(a.codes + row * a.inner + p - (8 - left));
          rg.s[j] = a.exps[row * a.nblk + (p >> 5)];
        }
      } else {
#pragma unroll
        for (int j = 0; j < NY; ++j) {
          const int r = o0 + tid / PP + PR * j;
          rg.y[j].zero();
          if (r < a.cout) rg.y[j].load_each(py + (int64_t)r * a.dy_sc, n);
        }
#pragma unroll
        for (int j = 0; j < NX; ++j) {
          const int r = i0 + tid / PP + PR * j;
          rg.x[j].zero();
          rg.s[j] = 127;
          if (r < a.cin && n > 0) {
            code_load<false, 8>(rg.x[j], a.codes + (row0 + r) * a.inner + p, n);
            rg.s[j] = a.exps[(row0 + r) * a.nblk + (p >> 5)];
          }
        }
      }
    } else {                 // piece j: token tid / (TM / 8) + j T / (TM / 8) of the step, eight channels number tid % (TM / 8)
      constexpr int GY = TM / 8, GX = TN / 8;
      const int64_t t0 = (int64_t)step * STEP;
      const int cy = o0 + 8 * (tid % GY), cx = i0 + 8 * (tid % GX);
      if constexpr (WIDE) {
        const int by = min(cy, (int)a.cout - 8), bx = min(cx, (int)a.cin - 8);   // (stepped back; wholly outside: anywhere)
        const int64_t last = a.outer - 1 - t0;
#pragma unroll
        for (int j = 0; j < NY; ++j)
          rg.y[j].load(reinterpret_cast<const AT*>(a.dy) + (t0 + min((int64_t)(tid / GY + T / GY * j), last)) * a.dy_so + by);
#pragma unroll
        for (int j = 0; j < NX; ++j) {
          const int64_t t = t0 + min((int64_t)(tid / GX + T / GX * j), last);
          rg.x[j].load(a.codes + t * a.cin + bx);
          rg.s[j] = a.exps[t * a.nblk + (min(cx, (int)a.cin - 1) >> 5)];
        }
      } else {
#pragma unroll
        for (int j = 0; j < NY; ++j) {
          const int64_t t = t0 + tid / GY + T / GY * j;
          rg.y[j].zero();
          if (t < a.outer) rg.y[j].load_each(reinterpret_cast<const AT*>(a.dy) + t * a.dy_so + cy, (int)min((int64_t)8, a.cout - cy));
        }
#pragma unroll
        for (int j = 0; j < NX; ++j) {
          const int64_t t = t0 + tid / GX + T / GX * j;
          rg.x[j].zero();
          rg.s[j] = 127;
          if (t < a.outer && cx < a.cin) {
            code_load<false, 8>(rg.x[j], a.codes + t * a.cin + cx, (int)min((int64_t)8, a.cin - cx));
            rg.s[j] = a.exps[t * a.nblk + (cx >> 5)];
          }
        }
      }
    }
  };
  // what the loads brought that is not the tensors': shifted down or cleared
  auto finish = [&](WgRegs<AT, NY, NX>& rg, int step) {
    if constexpr (WIDE && !ROWS) {
      if (rg.n < 8) {
#pragma unroll
        for (int j = 0; j < NY; ++j) {
          if (rg.n > 0) rg.y[j].shift(8 - rg.n);
          else rg.y[j].zero();
        }
#pragma unroll
        for (int j = 0; j < NX; ++j) {
          if (rg.n > 0) code_end<true, 8>(rg.x[j], rg.n);
          else rg.x[j].zero();
        }
      }
    }
    if constexpr (WIDE && ROWS) {
      constexpr int GY = TM / 8, GX = TN / 8;
      const int64_t t0 = (int64_t)step * STEP;
      const int cy = o0 + 8 * (tid % GY), cx = i0 + 8 * (tid % GX);
      if (o0 + TM > a.cout && cy < a.cout && cy + 8 > a.cout)
#pragma unroll
        for (int j = 0; j < NY; ++j) rg.y[j].shift(cy + 8 - (int)a.cout);
      if (i0 + TN > a.cin && cx < a.cin && cx + 8 > a.cin)
#pragma unroll
        for (int j = 0; j < NX; ++j) code_end<true, 8>(rg.x[j], (int)a.cin - cx);
      if (t0 + STEP > a.outer) {
#pragma unroll
        for (int j = 0; j < NY; ++j)
          if (t0 + tid / GY + T / GY * j >= a.outer) rg.y[j].zero();
#pragma unroll
        for (int j = 0; j < NX; ++j)
          if (t0 + tid / GX + T / GX * j >= a.outer) rg.x[j].zero();
      }
    }
  };

  auto store = [&](WgRegs<AT, NY, NX>& rg, int step, unsigned char* buf) {
    unsigned char* bx = buf + PARTS * YB;
    finish(rg, step);
#pragma unroll
    for (int j = 0; j < NY; ++j) {
      unsigned at;
      if constexpr (!ROWS) at = wg_piece<STEP>(tid / PP + PR * j, tid % PP);
      else at = wg_token<TM>(tid / (TM / 8) + T / (TM / 8) * j, tid % (TM / 8));
      rg.y[j].put(buf, at, YB);
      if (bias) {
        float f[8];
        rg.y[j].get(f);
        if constexpr (!ROWS) {
          bsum[j] += ((f[0] + f[1]) + (f[2] + f[3])) + ((f[4] + f[5]) + (f[6] + f[7]));
        } else {
#pragma unroll
          for (int q = 0; q < 8; ++q) bsum[q] += f[q];
        }
      }
    }
#pragma unroll
    for (int j = 0; j < NX; ++j) {
      unsigned at;
      if constexpr (!ROWS) at = wg_piece<STEP>(tid / PP + PR * j, tid % PP);
      else at = wg_token<TN>(tid / (TN / 8) + T / (TN / 8) * j, tid % (TN / 8));
      float f[8];
      q8_decode_vec<FMT, 8>(rg.x[j].w, q8_scale(rg.s[j]), f);
      *reinterpret_cast<csn_u4*>(bx + at) = wg_u4(wg_hi2(f[0], f[1]), wg_hi2(f[2], f[3]), wg_hi2(f[4], f[5]), wg_hi2(f[6], f[7]));
    }
  };

  csn_f16v acc[MI][NJ];
#pragma unroll
  for (int i = 0; i < MI; ++i)
#pragma unroll
    for (int j = 0; j < NJ; ++j)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.f;

  const int wr = (wave / S::WN) * (TM / S::WM), wc = (wave % S::WN) * (TN / S::WN);
  // Operand of 32 channels, tokens 16 kk + 8 (lane >> 5) .. + 7.  Of token rows: two transposing reads of four tokens each, whose addresses
  // in the first 16 tokens are kept (the pieces' exchange depends on the token modulo 8 alone).
  unsigned ya[ROWS ? MI : 1][2], xa[ROWS ? NJ : 1][2];
  if constexpr (ROWS) {
    const int t = 8 * (lane >> 5) + ((lane & 15) >> 2), ch = (lane & 16) + 4 * (lane & 3);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
#pragma unroll
      for (int i = 0; i < MI; ++i) ya[i][h] = wg_token<TM>(t + 4 * h, (wr + 32 * i + ch) >> 3) + 2u * (ch & 4);
#pragma unroll
      for (int j = 0; j < NJ; ++j) xa[j][h] = PARTS * YB + wg_token<TN>(t + 4 * h, (wc + 32 * j + ch) >> 3) + 2u * (ch & 4);
    }
  }
  auto read8 = [&](const unsigned char* p, const unsigned char* q) {
    const uint2 lo = wg_read_tr16(p), hi = wg_read_tr16(q);
    return wg_u4(lo.x, lo.y, hi.x, hi.y);
  };
  auto multiply = [&](const unsigned char* buf) {
#pragma unroll
    for (int kk = 0; kk < STEP / 16; ++kk) {
      csn_u4 b[NJ];
#pragma unroll
      for (int j = 0; j < NJ; ++j) {
        if constexpr (ROWS) b[j] = read8(buf + xa[j][0] + 32 * TN * kk, buf + xa[j][1] + 32 * TN * kk);
        else b[j] = *reinterpret_cast<const csn_u4*>(buf + PARTS * YB + wg_piece<STEP>(wc + 32 * j + (lane & 31), 2 * kk + (lane >> 5)));
      }
#pragma unroll
      for (int part = 0; part < PARTS; ++part)
#pragma unroll
        for (int i = 0; i < MI; ++i) {
          csn_u4 y;
          if constexpr (ROWS) y = read8(buf + part * YB + ya[i][0] + 32 * TM * kk, buf + part * YB + ya[i][1] + 32 * TM * kk);
          else y = *reinterpret_cast<const csn_u4*>(buf + part * YB + wg_piece<STEP>(wr + 32 * i + (lane & 31), 2 * kk + (lane >> 5)));
#pragma unroll
          for (int j = 0; j < NJ; ++j) acc[i][j] = csn_mfma_32x32x16_bf16(y, b[j], acc[i][j]);
        }
      if constexpr (TM == 256) CSN_SCHED_FENCE();   // (operands of one kk at a time: the accumulators take half of the registers)
    }
  };
  // The slab's steps in pairs (steps_per_slab is even, tokens behind the last read as zeros).  Two register sets: the registers of a step
  // are free again once it lies in its buffer, and hold the step two further on while the buffers are multiplied.  The large tile's
  // accumulators leave room for one set, one step ahead.
  // (The last pair stands by itself: loads behind a branch would be waited for where the paths join again.)
  constexpr bool TWO = TM < 256;
  load(r0, s0);
  if constexpr (TWO) load(r1, s0 + 1);
  store(r0, s0, sm);
#pragma unroll 1
  for (int s = s0; s + 2 < s1; s += 2) {
    load(r0, s + (TWO ? 2 : 1));
    __syncthreads();
    multiply(sm);
    if constexpr (TWO) store(r1, s + 1, sm + BUF);
    else store(r0, s + 1, sm + BUF);
    if constexpr (TWO) load(r1, s + 3);
    else load(r0, s + 2);
    __syncthreads();
    multiply(sm + BUF);
    store(r0, s + 2, sm);
  }
  if constexpr (!TWO) load(r0, s1 - 1);
  __syncthreads();
  multiply(sm);
  if constexpr (TWO) store(r1, s1 - 1, sm + BUF);
  else store(r0, s1 - 1, sm + BUF);
  __syncthreads();
  multiply(sm + BUF);

  float* out = a.slabs > 1 ? a.partial + (int64_t)slab * a.cout * (a.cin + 1) : a.dweight;
#pragma unroll
  for (int i = 0; i < MI; ++i)
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      const int64_t o = o0 + wr + 32 * i + 8 * (r >> 2) + 4 * (lane >> 5) + (r & 3);
      if (o < a.cout)
#pragma unroll
        for (int j = 0; j < NJ; ++j) {
          const int64_t c = i0 + wc + 32 * j + (lane & 31);
          if (c < a.cin) out[o * a.cin + c] = acc[i][j][r];
        }
    }
  if (bias) {   // the block's sums of dY: K threads hold a channel's
    constexpr int K = ROWS ? T / (TM / 8) : PP;
    __syncthreads();
    float* sb = reinterpret_cast<float*>(sm);   // [TM][K]
    if constexpr (!ROWS) {
#pragma unroll
      for (int j = 0; j < NY; ++j) sb[(tid / PP + PR * j) * K + tid % PP] = bsum[j];
    } else {
#pragma unroll
      for (int q = 0; q < 8; ++q) sb[(8 * (tid % (TM / 8)) + q) * K + tid / (TM / 8)] = bsum[q];
    }
    __syncthreads();
    if (tid < TM && o0 + tid < a.cout) {
      float v = 0.f;
      for (int j = 0; j < K; ++j) v += sb[tid * K + j];
      (a.slabs > 1 ? out + a.cout * a.cin : a.dbias)[o0 + tid] = v;   // (behind the slab's dW)
    }
  }
}

struct WgPlan { int tm, tn, mtiles, ntiles, steps_per_slab, slabs, chunks; };

// Tiles of 128 where the channels fill more than 64; of 256 x 256, whose operands are read from LDS half as often, where there are enough of
// them times steps for every CU (bfloat16 dY: the three parts of a float one do not fit).  Tiles of 128 / of 256, us with the sum of the
// slabs: 16384 tokens, 1024 -> 4096 245 / 172, 1024 -> 1024 72 / 64, 512 -> 512 32 / 36; 2048 tokens, 1024 -> 4096 50 / 46; 131072 tokens,
// 256 -> 256 45 / 46, 65536 tokens 32 / 37.  As many blocks as the CUs hold at a time, but at least 256 tokens each: a slab costs a partial
// tile written and read again.  A CU holds one block of eight waves or two of four, and one of four where the three parts of a float dY of
// 128 channels fill its LDS; two rounds of those / one, us: 16384 tokens, 512 -> 512 58.4 / 50.6, 32768 tokens, 256 -> 256 41.4 / 32.6,
// 32x44x44 maps, 256 -> 256 60.4 / 51.6, 32x88x88, 256 -> 128 101.2 / 95.5.
static bool wg_plan(int rows, int a16, int64_t outer, int64_t inner, int64_t cin, int64_t cout, WgPlan& p) {
  const int64_t chunks = rows ? 1 : (inner + 7) / 8, per_step = !rows && a16 ? 16 : 8;
  const int64_t all = rows ? (outer + 7) / 8 : outer * chunks, steps = (all + per_step - 1) / per_step;
  p.tm = cout > 64 ? 128 : 64;
  p.tn = cin > 64 ? 128 : 64;
  const bool big = rows && a16 && cout > 128 && cin > 128 && ((cout + 255) / 256) * ((cin + 255) / 256) * steps >= 256 * 8;
  if (big) p.tm = p.tn = 256;
  const int64_t mt = (cout + p.tm - 1) / p.tm, nt = (cin + p.tn - 1) / p.tn;
  if (mt * nt > (1 << 20) || all > 0x7ffffe00LL || chunks > 0x7ffffe00LL) return false;
  const bool one = big || (per_step == 16 && p.tm + p.tn > 128) || (!a16 && p.tm == 128);
  int64_t slabs = ((one ? 256 : 512) + mt * nt - 1) / (mt * nt);
  slabs = std::max(std::min(slabs, (steps * per_step + 31) / 32), (int64_t)1);
  p.mtiles = (int)mt; p.ntiles = (int)nt; p.chunks = (int)std::max(chunks, (int64_t)1);
  p.steps_per_slab = std::max(((int)((steps + slabs - 1) / slabs) + 1) & ~1, 2);
  p.slabs = std::max((int)((steps + p.steps_per_slab - 1) / p.steps_per_slab), 1);
  return true;
}

int64_t csn_q8_wgrad_partial_floats(int rows, int a16, int64_t outer, int64_t inner, int64_t cin, int64_t cout) {
  WgPlan p;
  if (!wg_plan(rows, a16, outer, inner, cin, cout, p) || p.slabs <= 1) return 0;
  return (int64_t)p.slabs * (cout * cin + cout);
}

template <typename AT, int FMT, bool ROWS, bool WIDE, int TM, int TN>
static int q8_wgrad_go(const Q8WgradArgs& a, void* stream) {
  typedef WgShape<AT, ROWS, TM, TN> S;
#ifndef CSN_CPU_EMU
  static CsnPerDeviceOnce once;
  const int st = once.run([] {
    return (int)hipFuncSetAttribute(reinterpret_cast<const void*>(&q8_wgrad_kernel<AT, FMT, ROWS, WIDE, TM, TN>),
                                    hipFuncAttributeMaxDynamicSharedMemorySize, S::SMEM);
  });
  if (st != 0) return st;
#endif
  const int total = a.mtiles * a.ntiles * a.slabs;
  CSN_LAUNCH((q8_wgrad_kernel<AT, FMT, ROWS, WIDE, TM, TN>), dim3((unsigned)((total + 7) / 8 * 8)), dim3(S::T), S::SMEM, stream, a);
  if (a.slabs > 1) {
    const int e = (int)hipGetLastError();
    if (e != 0) return e;
    SlabSumArgs r;
    r.partial = a.partial; r.out0 = a.dweight; r.out1 = a.dbias; r.n0 = a.cout * a.cin; r.n = r.n0 + a.cout; r.slabs = a.slabs;
    return csn_launch_slab_sum(r, stream);
  }
  return (int)hipGetLastError();
}

template <typename AT, int FMT, bool ROWS, int TM, int TN>
static int q8_wgrad_run(const Q8WgradArgs& a, void* stream) {
  if (ROWS ? a.cin >= 8 && a.cout >= 8 : a.inner >= 8) return q8_wgrad_go<AT, FMT, ROWS, true, TM, TN>(a, stream);
  if constexpr (TM == 256) return -1;   // (never: that tile is for more channels)
  else return q8_wgrad_go<AT, FMT, ROWS, false, TM, TN>(a, stream);
}
template <typename AT, int FMT, bool ROWS>
static int q8_wgrad_tile(const Q8WgradArgs& a, const WgPlan& p, void* stream) {
  if constexpr (ROWS && sizeof(AT) == 2)
    if (p.tm == 256) return q8_wgrad_run<AT, FMT, ROWS, 256, 256>(a, stream);
  if (p.tm == 128) return p.tn == 128 ? q8_wgrad_run<AT, FMT, ROWS, 128, 128>(a, stream) : q8_wgrad_run<AT, FMT, ROWS, 128, 64>(a, stream);
  return p.tn == 128 ? q8_wgrad_run<AT, FMT, ROWS, 64, 128>(a, stream) : q8_wgrad_run<AT, FMT, ROWS, 64, 64>(a, stream);
}

int csn_launch_q8_wgrad(const Q8WgradArgs& a0, int rows, int a16, int fmt, void* stream) {
  Q8WgradArgs a = a0;
  WgPlan p;
  if (!wg_plan(rows, a16, a.outer, a.inner, a.cin, a.cout, p)) return -1;
  a.mtiles = p.mtiles; a.ntiles = p.ntiles; a.steps_per_slab = p.steps_per_slab; a.slabs = p.slabs; a.chunks = p.chunks;
  if (a.outer * a.inner == 0) {   // no tokens: the gradients are zero
    SlabSumArgs r;
    r.partial = nullptr; r.out0 = a.dweight; r.out1 = a.dbias; r.n0 = a.cout * a.cin; r.n = r.n0 + a.cout; r.slabs = 0;
    return csn_launch_slab_sum(r, stream);
  }
  if (fmt == Q8_INT8) {
    if (rows) return a16 ? q8_wgrad_tile<csn_bf16, Q8_INT8, true>(a, p, stream) : q8_wgrad_tile<float, Q8_INT8, true>(a, p, stream);
    return a16 ? q8_wgrad_tile<csn_bf16, Q8_INT8, false>(a, p, stream) : q8_wgrad_tile<float, Q8_INT8, false>(a, p, stream);
  }
  if (rows) return a16 ? q8_wgrad_tile<csn_bf16, Q8_E4M3, true>(a, p, stream) : q8_wgrad_tile<float, Q8_E4M3, true>(a, p, stream);
  return a16 ? q8_wgrad_tile<csn_bf16, Q8_E4M3, false>(a, p, stream) : q8_wgrad_tile<float, Q8_E4M3, false>(a, p, stream);
}
#endif  // CSN_EMU_SEQ
