// k_norm.hip -- layer norm over the channels of a token, forward and backward, for planar maps and for rows of tokens.
//
//     mean = sum_c x / C,  var = sum_c (x - mean)^2 / C,  rstd = (var + eps)^(-1/2),  y = (x - mean) rstd w + b
//     g = dy w,  c1 = sum_c g / C,  c2 = sum_c g xh / C,  dx = rstd (g - c1 - xh c2),  dw = sum_t dy xh,  db = sum_t dy
//
// with xh = (x - mean) rstd; in the backward x may be the 8-bit checkpoint that the forward left (q8_core.h).
//
// Bound by bytes: forward x and y, backward x, dy and dx, each once, at the 6.2 TB/s of a large copy.  A token's channels therefore stay in
// registers over the passes that the formulas make (sum, sum of squares, output; the two sums of the backward, output), which are
// lane exchanges and one trip through LDS.  Kernel times against that floor, us (cold caches):
//   25088 x 512 float         forward 22.7 of 16.6   backward 28.8 of 24.8, sum of the slabs 4.0
//   16384 x 1024 bf16         forward 17.2 of 10.8   backward 23.7 of 16.2, sum of the slabs 4.0
//   16384 x 1024 bf16, int8 checkpoint    forward 21.9 of 13.6   backward 25.6 of 13.6, sum of the slabs 4.0
//   32x256x88x88 bf16         forward 48.7 of 40.9   backward 98.5 of 61.3, sum of the slabs 4.7
//   32x256x88x88 float        forward 101.5 of 81.8  backward 158.5 of 123, sum of the slabs 4.8
//   16x512x44x44 float, e4m3 checkpoint   forward 36.6 of 23.1   backward 42.2 of 23.1, sum of the slabs 4.0
// The forward of maps waits for its loads between blocks (no room for the next tile beside 16 channels); the backward has the next tile
// in flight, and what is left is the arithmetic and the exchanges between a tile's loads and its stores, two waves per SIMD.
#include "csn_reduce.h"
#include "q8_core.h"
#include "slab_sum.h"
#include "train_ops.h"
#include "vec_io.h"

// channel c of token (o, p), from x or from its checkpoint
template <typename AT, int FMT, bool ROWS>
__device__ __forceinline__ float norm_x(const NormArgs& a, int64_t o, int64_t p, int64_t c) {
  if (a.x) return act_ld(reinterpret_cast<const AT*>(a.x) + o * a.x_so + (ROWS ? c : c * a.x_sc + p));
  const int64_t row = ROWS ? o : o * a.C + c, col = ROWS ? c : p, cols = ROWS ? a.C : a.inner;
  return q8_decode<FMT>(a.codes_in[row * cols + col], q8_scale(a.exps_in[row * a.nblk + col / 32]));
}
template <typename AT, bool ROWS>
__device__ __forceinline__ float norm_dy(const NormArgs& a, int64_t o, int64_t p, int64_t c) {
  return act_ld(reinterpret_cast<const AT*>(a.dy) + o * a.dy_so + (ROWS ? c : c * a.dy_sc + p));
}

// ---- simple forms, for tokens of more channels than the register forms below hold: one block per token / per channel
template <typename AT, bool ROWS>
__global__ __launch_bounds__(CSN_BLOCK) void norm_fwd_kernel(NormArgs a) {
  CSN_DYN_SMEM(double, sm);
  const int64_t tokens = a.outer * a.inner;
  for (int64_t t = blockIdx.x; t < tokens; t += gridDim.x) {
    const int64_t o = t / a.inner, p = t - o * a.inner;
    double s = 0.0;
    for (int64_t c = threadIdx.x; c < a.C; c += CSN_BLOCK) s += norm_x<AT, 0, ROWS>(a, o, p, c);
    const float mean = (float)(bn_block_sum(s, sm) / (double)a.C);
    double q = 0.0;
    for (int64_t c = threadIdx.x; c < a.C; c += CSN_BLOCK) {
      const float d = norm_x<AT, 0, ROWS>(a, o, p, c) - mean;
      q += d * d;
    }
    const float rstd = (float)(1.0 / sqrt(bn_block_sum(q, sm) / (double)a.C + (double)a.eps));
    for (int64_t c = threadIdx.x; c < a.C; c += CSN_BLOCK) {
      const float xh = (norm_x<AT, 0, ROWS>(a, o, p, c) - mean) * rstd;
      const float v = fmaf(xh, a.weight ? a.weight[c] : 1.f, a.bias ? a.bias[c] : 0.f);
      act_st(reinterpret_cast<AT*>(a.y) + (ROWS ? o * a.C + c : (o * a.C + c) * a.inner + p), v);
    }
    if (threadIdx.x == 0) {
      if (a.mean) a.mean[t] = mean;
      if (a.rstd) a.rstd[t] = rstd;
    }
  }
}

template <typename AT, int FMT, bool ROWS>
__global__ __launch_bounds__(CSN_BLOCK) void norm_bwd_kernel(NormArgs a) {
  CSN_DYN_SMEM(double, sm);
  const int64_t tokens = a.outer * a.inner;
  for (int64_t t = blockIdx.x; t < tokens; t += gridDim.x) {
    const int64_t o = t / a.inner, p = t - o * a.inner;
    const float mean = a.mean[t], rstd = a.rstd[t];
    double s1 = 0.0, s2 = 0.0;
    for (int64_t c = threadIdx.x; c < a.C; c += CSN_BLOCK) {
      const float xh = (norm_x<AT, FMT, ROWS>(a, o, p, c) - mean) * rstd;
      const float g = norm_dy<AT, ROWS>(a, o, p, c) * (a.weight ? a.weight[c] : 1.f);
      s1 += g; s2 += g * xh;
    }
    const float c1 = (float)(bn_block_sum(s1, sm) / (double)a.C), c2 = (float)(bn_block_sum(s2, sm) / (double)a.C);
    for (int64_t c = threadIdx.x; c < a.C; c += CSN_BLOCK) {
      const float xh = (norm_x<AT, FMT, ROWS>(a, o, p, c) - mean) * rstd;
      const float g = norm_dy<AT, ROWS>(a, o, p, c) * (a.weight ? a.weight[c] : 1.f);
      act_st(reinterpret_cast<AT*>(a.y) + (ROWS ? o * a.C + c : (o * a.C + c) * a.inner + p), rstd * (g - c1 - xh * c2));
    }
  }
}

template <typename AT, int FMT, bool ROWS>
__global__ __launch_bounds__(CSN_BLOCK) void norm_dw_kernel(NormArgs a) {
  CSN_DYN_SMEM(double, sm);
  const int64_t tokens = a.outer * a.inner;
  for (int64_t c = blockIdx.x; c < a.C; c += gridDim.x) {
    double s1 = 0.0, s2 = 0.0;
    for (int64_t t = threadIdx.x; t < tokens; t += CSN_BLOCK) {
      const int64_t o = t / a.inner, p = t - o * a.inner;
      const float dy = norm_dy<AT, ROWS>(a, o, p, c);
      s1 += dy;
      s2 += dy * ((norm_x<AT, FMT, ROWS>(a, o, p, c) - a.mean[t]) * a.rstd[t]);
    }
    const float db = (float)bn_block_sum(s1, sm), dw = (float)bn_block_sum(s2, sm);
    if (threadIdx.x == 0) {
      if (a.dweight) a.dweight[c] = dw;
      if (a.dbias) a.dbias[c] = db;
    }
  }
}


static unsigned norm_grid(int64_t items) { return (unsigned)(items < 16384 ? items : 16384); }

#ifndef CSN_EMU_SEQ
// ---- the fast forms: a token's channels stay in registers -----------------------------------------------------------------
enum { NORM_X = -1 };   // input of the backward: x itself (else a checkpoint format); forward: no checkpoint is written

// sums over G lanes (a power of two): a butterfly inside the wave, then the block's waves in order through LDS (two buffers of
// [2][16] floats in turn: one barrier per sum)
template <int G, int N>
__device__ __forceinline__ void norm_sum(float (&v)[N], float* sm, int& turn) {
#pragma unroll
  for (int i = 0; i < N; ++i) {
    if (G >= 64) v[i] += csn_lane_xor_f32<32>(v[i]);
    if (G >= 32) v[i] += csn_lane_xor_f32<16>(v[i]);
    if (G >= 16) v[i] += csn_lane_xor_f32<8>(v[i]);
    if (G >= 8) v[i] += csn_lane_xor_f32<4>(v[i]);
    v[i] += csn_lane_xor_f32<2>(v[i]);
    v[i] += csn_lane_xor_f32<1>(v[i]);
  }
  if (G > 64) {
    static_assert(N <= 2, "a buffer holds two sums");
    float* b = sm + turn * 32;
    turn ^= 1;
    if ((threadIdx.x & 63) == 0)
#pragma unroll
      for (int i = 0; i < N; ++i) b[i * 16 + (threadIdx.x >> 6)] = v[i];
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; ++i) {
      float s = 0.f;
#pragma unroll
      for (int w = 0; w < G / 64; ++w) s += b[i * 16 + w];
      v[i] = s;
    }
  }
}

// where the block's sums of dy xh (q = 0) / of dy (q = 1) go: its slab, or the gradient itself where there is one block; null: not wanted
__device__ __forceinline__ float* norm_slab(const NormArgs& a, int q) {
  if (gridDim.x == 1) return q ? a.dbias : a.dweight;
  return a.partial ? a.partial + ((int64_t)blockIdx.x * 2 + q) * a.C : nullptr;
}

// E weights (or biases) of a piece, `none` past the row's end or without a tensor
template <int E>
__device__ __forceinline__ void norm_param(float (&f)[E], const float* p, int n, float none) {
#pragma unroll
  for (int h = 0; h < E; h += 4) {
    VecIo<float> v;
    v.zero();
    if (p && n - h >= 4) v.load(p + h);
    else if (p) v.load_each(p + h, n - h);
#pragma unroll
    for (int j = 0; j < 4; ++j) f[h + j] = p && h + j < n ? csn_bits_f(v.w[j]) : none;
  }
}

// The mean m of float channels, from a sum that rounds, is off by some of the last places of the largest; where the channels are close
// together that shows.  The second pass, over x - m, finds out by how much.  (bfloat16 channels that are close together have an exact sum.)
// The product that gives m must not be contracted with the subtraction: what is taken off would not be m.
__device__ __forceinline__ float norm_first_mean(float sum, float inv_c) {
  unsigned m = csn_f_bits(sum * inv_c);
  csn_pin(m);
  return csn_bits_f(m);
}
// From the sums of (x - m)^2 and of x - m: the variance, and m becomes the mean where it is off by more than the second sum's own rounding,
// counted as 2^-21 of the spread.  (Equal channels: x - m is the same few last places of x for all of them; sums, the quotient --
// corrected once, a division at less cost -- and the difference are exact: mean x, variance 0.)
__device__ __forceinline__ float norm_correct(float& m, float sq, float sum, float channels, float inv_c) {
  const float q = sum * inv_c, off = fmaf(fmaf(-q, channels, sum), inv_c, q), far = off * 2097152.f;
  if (!(far * far > sq * inv_c)) return sq * inv_c;
  m += off;
  return fmaxf(fmaf(-off, sum, sq) * inv_c, 0.f);
}

template <int G> struct NormRowsBlock { static constexpr int T = G > CSN_BLOCK ? G : CSN_BLOCK; };

// Rows of tokens: G lanes per token, NV pieces of E elements (16 bytes) per lane.  A block walks tokens, its weights in registers.
// W: a token has at least E channels
template <typename AT, int G, int NV, bool W, int CK>
__global__ __launch_bounds__(NormRowsBlock<G>::T) void norm_rows_fwd_kernel(NormArgs a) {
  constexpr int E = VecIo<AT>::E, T = NormRowsBlock<G>::T, R = T / G;
  CSN_DYN_SMEM(float, sm);
  const int l = threadIdx.x % G, C = (int)a.C;
  const float inv_c = 1.f / (float)C;
  float w[NV][E], b[NV][E];
  int n[NV];
#pragma unroll
  for (int v = 0; v < NV; ++v) {
    const int c0 = E * (l + G * v);
    n[v] = C - c0;
    norm_param<E>(w[v], a.weight ? a.weight + c0 : nullptr, n[v], 1.f);
    norm_param<E>(b[v], a.bias ? a.bias + c0 : nullptr, n[v], 0.f);
  }
  int turn = 0;
  const int64_t step = (int64_t)gridDim.x * R;
  int64_t t = (int64_t)blockIdx.x * R + threadIdx.x / G;
  VecIo<AT> nx[NV];
  auto load = [&](int64_t row) {
    const AT* x = reinterpret_cast<const AT*>(a.x) + row * a.x_so;
#pragma unroll
    for (int v = 0; v < NV; ++v) vec_load<W>(nx[v], x + E * (l + G * v), n[v]);
  };
  load(t < a.outer ? t : a.outer - 1);
  for (; t < a.outer; t += step) {
    VecIo<AT> r[NV];
#pragma unroll
    for (int v = 0; v < NV; ++v) r[v] = nx[v];
    load(t + step < a.outer ? t + step : a.outer - 1);   // (in flight while this token is worked on; a branch around it would be a wait)
    float s[1] = {0.f};
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      float f[E];
      vec_end<W>(r[v], n[v]);
      r[v].get(f);
#pragma unroll
      for (int j = 0; j < E; ++j) s[0] += f[j];
    }
    norm_sum<G, 1>(s, sm, turn);
    constexpr bool FIX = sizeof(AT) == 4;
    float mean = FIX ? norm_first_mean(s[0], inv_c) : s[0] / (float)C, d2[FIX ? 2 : 1];   // (divided: equal channels have no variance at all)
    d2[0] = d2[FIX] = 0.f;
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      float f[E];
      r[v].pin();
      r[v].get(f);
#pragma unroll
      for (int j = 0; j < E; ++j) {
        const float d = j < n[v] ? f[j] - mean : 0.f;
        d2[0] = fmaf(d, d, d2[0]);
        if (FIX) d2[FIX] += d;
      }
    }
    norm_sum<G, FIX ? 2 : 1>(d2, sm, turn);
    const float var = FIX ? norm_correct(mean, d2[0], d2[FIX], (float)C, inv_c) : d2[0] * inv_c;
    const float rstd = 1.f / sqrtf(var + a.eps);
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      const int c0 = E * (l + G * v);
      float f[E], y[E];
      r[v].pin();
      r[v].get(f);
#pragma unroll
      for (int j = 0; j < E; ++j) y[j] = fmaf((f[j] - mean) * rstd, w[v][j], b[v][j]);
      VecIo<AT>::store(reinterpret_cast<AT*>(a.y) + t * C + c0, y, n[v]);
      if (CK >= 0) {
        unsigned c[E / 4];
        const unsigned e = q8_pack_block<CK, E>(f, c);
        code_store<E>(a.codes + t * C + c0, c, n[v]);
        if ((l & (32 / E - 1)) == 0 && n[v] > 0) a.exps[t * a.nblk + (c0 >> 5)] = (uint8_t)e;
      }
    }
    if (l == 0) {
      if (a.mean) a.mean[t] = mean;
      if (a.rstd) a.rstd[t] = rstd;
    }
  }
}

// one piece of the backward's input, the tensor or its checkpoint
template <typename AT, int E, int SRC> struct NormIn {
  CodeIo<E> c;
  unsigned e;
  template <bool W> __device__ __forceinline__ void end(int n) { code_end<W, E>(c, n); }
  __device__ __forceinline__ void pin() { c.pin(); }
  __device__ __forceinline__ void get(float (&f)[E]) const { q8_decode_vec<SRC, E>(c.w, q8_scale(e), f); }
};
template <typename AT, int E> struct NormIn<AT, E, NORM_X> {
  VecIo<AT, E> v;
  template <bool W> __device__ __forceinline__ void end(int n) { vec_end<W>(v, n); }
  __device__ __forceinline__ void pin() { v.pin(); }
  __device__ __forceinline__ void get(float (&f)[E]) const { v.get(f); }
};

template <typename AT, int G, int NV, bool W, int SRC>
__global__ __launch_bounds__(NormRowsBlock<G>::T) void norm_rows_bwd_kernel(NormArgs a) {
  constexpr int E = VecIo<AT>::E, T = NormRowsBlock<G>::T, R = T / G;
  CSN_DYN_SMEM(float, sm);
  const int l = threadIdx.x % G, C = (int)a.C;
  const float inv_c = 1.f / (float)C;
  float w[NV][E], dw[NV][E], db[NV][E];
  int n[NV];
#pragma unroll
  for (int v = 0; v < NV; ++v) {
    const int c0 = E * (l + G * v);
    n[v] = C - c0;
    norm_param<E>(w[v], a.weight ? a.weight + c0 : nullptr, n[v], 1.f);
#pragma unroll
    for (int j = 0; j < E; ++j) dw[v][j] = db[v][j] = 0.f;
  }
  int turn = 0;
  const int64_t step = (int64_t)gridDim.x * R;
  int64_t t = (int64_t)blockIdx.x * R + threadIdx.x / G;
  NormIn<AT, E, SRC> nx[NV];
  VecIo<AT> nd[NV];
  float nmean = 0.f, nrstd = 0.f;
  auto load = [&](int64_t row) {
    const AT* dy = reinterpret_cast<const AT*>(a.dy) + row * a.dy_so;
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      const int c0 = E * (l + G * v);
      if constexpr (SRC == NORM_X) {
        vec_load<W>(nx[v].v, reinterpret_cast<const AT*>(a.x) + row * a.x_so + c0, n[v]);
      } else {
        code_load<W, E>(nx[v].c, a.codes_in + row * C + c0, n[v]);
        nx[v].e = n[v] > 0 ? a.exps_in[row * a.nblk + (c0 >> 5)] : 127;
      }
      vec_load<W>(nd[v], dy + c0, n[v]);
    }
    nmean = a.mean[row]; nrstd = a.rstd[row];
  };
  load(t < a.outer ? t : a.outer - 1);
  for (; t < a.outer; t += step) {
    NormIn<AT, E, SRC> rx[NV];
    VecIo<AT> rd[NV];
#pragma unroll
    for (int v = 0; v < NV; ++v) { rx[v] = nx[v]; rd[v] = nd[v]; }
    const float mean = nmean, rstd = nrstd;
    load(t + step < a.outer ? t + step : a.outer - 1);   // (in flight while this token is worked on; a branch around it would be a wait)
    float s[2] = {0.f, 0.f};
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      float f[E], d[E];
      rx[v].template end<W>(n[v]);
      vec_end<W>(rd[v], n[v]);
      rx[v].get(f);
      rd[v].get(d);
#pragma unroll
      for (int j = 0; j < E; ++j) {   // (past the end: d = 0)
        const float xh = (f[j] - mean) * rstd, g = d[j] * w[v][j];
        s[0] += g;
        s[1] = j < n[v] ? fmaf(g, xh, s[1]) : s[1];
        dw[v][j] = fmaf(d[j], xh, dw[v][j]);
        db[v][j] += d[j];
      }
    }
    norm_sum<G, 2>(s, sm, turn);
    const float c1 = s[0] * inv_c, c2 = s[1] * inv_c;
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      float f[E], d[E], o[E];
      rx[v].pin();
      rd[v].pin();
      rx[v].get(f);
      rd[v].get(d);
#pragma unroll
      for (int j = 0; j < E; ++j) o[j] = rstd * (fmaf(d[j], w[v][j], -c1) - (f[j] - mean) * rstd * c2);
      VecIo<AT>::store(reinterpret_cast<AT*>(a.y) + t * C + E * (l + G * v), o, n[v]);
    }
  }
  // the block's R tokens at a time share columns: added in order, one slab per block (a lone block: the gradients themselves)
#pragma unroll
  for (int q = 0; q < 2; ++q) {
    float* p = norm_slab(a, q);
    if (!p) continue;
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      const int c0 = E * (l + G * v);
      float o[E];
#pragma unroll
      for (int j = 0; j < E; ++j) o[j] = q ? db[v][j] : dw[v][j];
      if (R > 1) {
        __syncthreads();
#pragma unroll
        for (int j = 0; j < E; ++j) sm[threadIdx.x * E + j] = o[j];
        __syncthreads();
        if (threadIdx.x < G) {
#pragma unroll 1
          for (int k = 1; k < R; ++k)
#pragma unroll
            for (int j = 0; j < E; ++j) o[j] += sm[(k * G + threadIdx.x) * E + j];
        }
      }
      if (threadIdx.x < G)
#pragma unroll
        for (int h = 0; h < E; h += 4) {
          const float four[4] = {o[h], o[h + 1], o[h + 2], o[h + 3]};
          VecIo<float>::store(p + c0 + h, four, n[v] - h);
        }
    }
  }
}

// Planar maps: PX lanes along the pixels (four consecutive pixels of a channel per lane: eight would double the statistics that
// every lane carries), T / PX groups of lanes over the channels, NC channels per lane in registers.  Sums over a pixel's channels: butterfly over the groups of a wave, then the waves in
// order through LDS (two buffers of [waves][N][PX * E] floats in turn).
#define NORM_PE 4
template <int T, int PX, int E, int N>
__device__ __forceinline__ void norm_planar_sum(float (&v)[N][E], float* sm, int& turn) {
  constexpr int W = T / 64, TP = PX * E;
#pragma unroll
  for (int i = 0; i < N; ++i)
#pragma unroll
    for (int j = 0; j < E; ++j) {
      v[i][j] += csn_lane_xor_f32<32>(v[i][j]);
      if (PX <= 16) v[i][j] += csn_lane_xor_f32<16>(v[i][j]);
      if (PX <= 8) v[i][j] += csn_lane_xor_f32<8>(v[i][j]);
      if (PX <= 4) v[i][j] += csn_lane_xor_f32<4>(v[i][j]);
      if (PX <= 2) v[i][j] += csn_lane_xor_f32<2>(v[i][j]);
    }
  if (W == 1) return;
  float* b = sm + turn * (W * N * TP);
  turn ^= 1;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, px = lane % PX;
  if (lane < PX)
#pragma unroll
    for (int i = 0; i < N; ++i)
#pragma unroll
      for (int j = 0; j < E; ++j) b[(wave * N + i) * TP + px * E + j] = v[i][j];
  __syncthreads();
#pragma unroll
  for (int i = 0; i < N; ++i)
#pragma unroll
    for (int j = 0; j < E; ++j) v[i][j] = 0.f;
#pragma unroll 2
  for (int k = 0; k < W; ++k)
#pragma unroll
    for (int i = 0; i < N; ++i)
#pragma unroll
      for (int j = 0; j < E; ++j) v[i][j] += b[(k * N + i) * TP + px * E + j];
}

// (image, pixel tile) items of a persistent launch.  Addresses are a uniform base -- image, group of channels k -- plus one 32-bit
// byte offset per lane that all of its channels share (64-bit addresses per channel would cost two registers each).
template <typename T>
__device__ __forceinline__ T* norm_at(T* base, unsigned bytes) {
  return reinterpret_cast<T*>(reinterpret_cast<typename std::conditional<std::is_const<T>::value, const char, char>::type*>(base) + bytes);
}
// A block's items: first, first + step, ... below end.  Where tiles are not whole cache lines of the map, each XCD (block b runs on XCD b % 8, the
// grid is a multiple of 8) takes a run of neighbouring tiles, so that the lines that their edges cut are read once into one L2; whole lines
// lose a few percent that way.  Round robin / runs, us, backward: 16x512x44x44 bf16 40.5 / 29.4, 16x2048x28x28 bf16 158 / 68, 32x256x57x57
// bf16 60.2 / 45.6; of whole lines 32x256x88x88 bf16 94.2 / 97.2, 32x128x88x88 float 81.3 / 85.4.  Forward: 16x512x44x44 bf16 18.2 / 16.1, float
// 30.0 / 29.4, 16x2048x28x28 bf16 41.6 / 35.7, 32x256x57x57 bf16 40.7 / 29.3, float with a checkpoint 87.4 / 64.8.
struct NormItems { int first, step, end; };
__device__ __forceinline__ NormItems norm_items(const NormArgs& a) {
  const int b = blockIdx.x, grid = gridDim.x;
  if (!a.runs) return NormItems{b, grid, a.items};
  const int per = (a.items + 7) >> 3, r0 = (b & 7) * per;
  return NormItems{r0 + (b >> 3), grid >> 3, min(r0 + per, a.items)};
}
// n pixels (n <= 0: none) of a lane whose byte offset is that of its piece stepped back as far as vec_load would
template <typename AT, int E>
__device__ __forceinline__ void norm_load(VecIo<AT, E>& v, const AT* base, unsigned bytes, int n) {
  v.zero();
  if (n > 0) v.load(norm_at(base, bytes));
}
// (Four waves per SIMD: a float form with a checkpoint gives up ten registers for a second block of 512 threads on the CU, 16x512x44x44
// 37.5 -> 34.1 us, 32x256x57x57 61.2 -> 58.9.)
template <typename AT, int T, int PX, int NC, int CK>
__global__ __launch_bounds__(T, 4) void norm_planar_fwd_kernel(NormArgs a) {
  constexpr int E = NORM_PE, CG = T / PX, TP = PX * E;
  CSN_DYN_SMEM(float, sm);
  const int px = threadIdx.x % PX, cg = threadIdx.x / PX, C = (int)a.C, P = (int)a.inner;
  const float inv_c = 1.f / (float)C;
  float w[NC], b[NC];
#pragma unroll
  for (int k = 0; k < NC; ++k) {
    const int c = cg + CG * k;
    w[k] = a.weight && c < C ? a.weight[c] : 1.f;
    b[k] = a.bias && c < C ? a.bias[c] : 0.f;
  }
  constexpr unsigned ES = sizeof(AT);
  const unsigned xlane = (unsigned)cg * (unsigned)a.x_sc + px * E, ylane = (unsigned)cg * (unsigned)P + px * E;
  int turn = 0;
  const NormItems my = norm_items(a);
  for (int it = my.first; it < my.end; it += my.step) {
    const int o = it / a.tiles, t0 = (it - o * a.tiles) * TP;
    const int n = P - t0 - px * E;
    const AT* x = reinterpret_cast<const AT*>(a.x) + o * a.x_so;
    const unsigned xoff = (xlane + t0 - vec_back(n > 0 ? n : E, E)) * ES, yoff = ylane + t0;
    VecIo<AT, E> r[NC];
#pragma unroll
    for (int k = 0; k < NC; ++k) norm_load(r[k], x + (int64_t)(CG * k) * a.x_sc, xoff, cg + CG * k < C ? n : 0);
    if (t0 + TP > P)   // (the image's last tile, one branch for all channels: the sums below stay one straight block)
#pragma unroll
      for (int k = 0; k < NC; ++k) vec_end<true>(r[k], n);
    float s[1][E];
#pragma unroll
    for (int j = 0; j < E; ++j) s[0][j] = 0.f;
#pragma unroll
    for (int k = 0; k < NC; ++k) {
      float f[E];
      r[k].pin();
      r[k].get(f);
#pragma unroll
      for (int j = 0; j < E; ++j) s[0][j] += f[j];
      CSN_SCHED_FENCE();   // one channel's floats at a time in registers
    }
    norm_planar_sum<T, PX, E, 1>(s, sm, turn);
    // (As above; float channels leave no registers for both sums of the second pass at once, so the mean is corrected in a pass of its own:
    // at once / in turn, us, 16x2048x28x28 57.2 / 51.9, 16x1024x32x32 34.0 / 29.9, 32x256x88x88 107.6 / 105.4.)
    constexpr bool FIX = sizeof(AT) == 4;
    float mean[E], rstd[E];
#pragma unroll
    for (int j = 0; j < E; ++j) { mean[j] = FIX ? norm_first_mean(s[0][j], inv_c) : s[0][j] / (float)C; s[0][j] = 0.f; }
    if constexpr (FIX) {
#pragma unroll
      for (int k = 0; k < NC; ++k) {
        float f[E];
        r[k].pin();
        r[k].get(f);
#pragma unroll
        for (int j = 0; j < E; ++j) s[0][j] += cg + CG * k < C ? f[j] - mean[j] : 0.f;
        CSN_SCHED_FENCE();
      }
      norm_planar_sum<T, PX, E, 1>(s, sm, turn);
#pragma unroll
      for (int j = 0; j < E; ++j) { mean[j] = fmaf(s[0][j], inv_c, mean[j]); s[0][j] = 0.f; }
    }
#pragma unroll
    for (int k = 0; k < NC; ++k) {
      float f[E];
      r[k].pin();
      r[k].get(f);
#pragma unroll
      for (int j = 0; j < E; ++j) {
        const float d = cg + CG * k < C ? f[j] - mean[j] : 0.f;
        s[0][j] = fmaf(d, d, s[0][j]);
      }
      CSN_SCHED_FENCE();
    }
    norm_planar_sum<T, PX, E, 1>(s, sm, turn);
#pragma unroll
    for (int j = 0; j < E; ++j) rstd[j] = 1.f / sqrtf(fmaf(s[0][j], inv_c, a.eps));
    const int64_t row0 = (int64_t)o * C;
#pragma unroll
    for (int k = 0; k < NC; ++k) {
      const int c = cg + CG * k;
      float f[E], y[E];
      r[k].pin();
      r[k].get(f);
#pragma unroll
      for (int j = 0; j < E; ++j) y[j] = fmaf((f[j] - mean[j]) * rstd[j], w[k], b[k]);
      const int64_t base = (row0 + CG * k) * P;
      if (c < C) VecIo<AT, E>::store(norm_at(reinterpret_cast<AT*>(a.y) + base, yoff * ES), y, n);
      if (CK >= 0) {
        unsigned q[E / 4];
        const unsigned e = q8_pack_block<CK, E>(f, q);
        if (c < C) {
          code_store<E>(norm_at(a.codes + base, yoff), q, n);
          if ((px & (32 / E - 1)) == 0 && n > 0)
            *norm_at(a.exps + (row0 + CG * k) * a.nblk, (unsigned)cg * (unsigned)a.nblk + ((t0 + px * E) >> 5)) = (uint8_t)e;
        }
      }
      CSN_SCHED_FENCE();
    }
    if (cg == 0) {
      const int64_t st = (int64_t)o * P + t0 + px * E;
      if (a.mean)
#pragma unroll
        for (int j = 0; j < E; ++j)
          if (j < n) a.mean[st + j] = mean[j];
      if (a.rstd)
#pragma unroll
        for (int j = 0; j < E; ++j)
          if (j < n) a.rstd[st + j] = rstd[j];
    }
  }
}

template <typename AT, int T, int PX, int NC, int SRC>
__global__ __launch_bounds__(T) void norm_planar_bwd_kernel(NormArgs a) {
  constexpr int E = NORM_PE, CG = T / PX, TP = PX * E;
  CSN_DYN_SMEM(float, sm);
  const int px = threadIdx.x % PX, cg = threadIdx.x / PX, C = (int)a.C, P = (int)a.inner;
  const float inv_c = 1.f / (float)C;
  float w[NC], dw[NC], db[NC];
#pragma unroll
  for (int k = 0; k < NC; ++k) {
    w[k] = a.weight && cg + CG * k < C ? a.weight[cg + CG * k] : 1.f;
    dw[k] = db[k] = 0.f;
  }
  constexpr unsigned ES = sizeof(AT);
  const unsigned xlane = (unsigned)cg * (unsigned)a.x_sc + px * E, dlane = (unsigned)cg * (unsigned)a.dy_sc + px * E;
  const unsigned ylane = (unsigned)cg * (unsigned)P + px * E;
  int turn = 0;
  NormIn<AT, E, SRC> nx[NC];
  VecIo<AT, E> nd[NC];
  VecIo<float> nm, nr;   // mean, rstd of the lane's pixels
  auto load = [&](int it) {
    const int o = it / a.tiles, t0 = (it - o * a.tiles) * TP;
    const int n = P - t0 - px * E;
    const int64_t row0 = (int64_t)o * C;
    const AT* x = reinterpret_cast<const AT*>(a.x) + o * a.x_so;
    const AT* dy = reinterpret_cast<const AT*>(a.dy) + o * a.dy_so;
    const int tb = t0 - vec_back(n > 0 ? n : E, E);
    const unsigned xoff = (xlane + tb) * ES, doff = (dlane + tb) * ES, coff = ylane + tb;
    const unsigned eoff = (unsigned)cg * (unsigned)a.nblk + ((t0 + px * E) >> 5);
#pragma unroll
    for (int k = 0; k < NC; ++k) {
      const int m = cg + CG * k < C ? n : 0;
      if constexpr (SRC == NORM_X) {
        norm_load(nx[k].v, x + (int64_t)(CG * k) * a.x_sc, xoff, m);
      } else {
        nx[k].c.zero();
        nx[k].e = 127;
        if (m > 0) {
          nx[k].c.load(norm_at(a.codes_in + (row0 + CG * k) * P, coff));
          nx[k].e = *norm_at(a.exps_in + (row0 + CG * k) * a.nblk, eoff);
        }
      }
      norm_load(nd[k], dy + (int64_t)(CG * k) * a.dy_sc, doff, m);
    }
    const int64_t st = (int64_t)o * P + t0 + px * E;
    vec_load<true>(nm, a.mean + st, n);
    vec_load<true>(nr, a.rstd + st, n);
  };
  const NormItems my = norm_items(a);
  load(min(my.first, my.end - 1));
  for (int it = my.first; it < my.end; it += my.step) {
    const int o = it / a.tiles, t0 = (it - o * a.tiles) * TP;
    const int n = P - t0 - px * E;
    const int64_t row0 = (int64_t)o * C;
    const unsigned yoff = (ylane + t0) * ES;
    NormIn<AT, E, SRC> rx[NC];
    VecIo<AT, E> rd[NC];
    VecIo<float> cm = nm, cr = nr;
#pragma unroll
    for (int k = 0; k < NC; ++k) { rx[k] = nx[k]; rd[k] = nd[k]; }
    load(min(it + my.step, my.end - 1));   // (in flight while this tile is worked on; a branch around it would be a wait)
    if (t0 + TP > P) {   // (the image's last tile, one branch for all channels: the sums below stay one straight block)
      vec_end<true>(cm, n);
      vec_end<true>(cr, n);
#pragma unroll
      for (int k = 0; k < NC; ++k) {
        rx[k].template end<true>(n);
        vec_end<true>(rd[k], n);
      }
    }
    float mean[E], rstd[E], s[2][E];
    cm.get(mean);
    cr.get(rstd);
#pragma unroll
    for (int j = 0; j < E; ++j) s[0][j] = s[1][j] = 0.f;
#pragma unroll
    for (int k = 0; k < NC; ++k) {
      float f[E], d[E];
      rx[k].pin();
      rd[k].pin();
      rx[k].get(f);
      rd[k].get(d);
#pragma unroll
      for (int j = 0; j < E; ++j) {   // (channels and pixels past the end: f = d = 0)
        const float xh = (f[j] - mean[j]) * rstd[j], g = d[j] * w[k];
        s[0][j] += g;
        s[1][j] = fmaf(g, xh, s[1][j]);
        dw[k] = fmaf(d[j], xh, dw[k]);
        db[k] += d[j];
      }
      CSN_SCHED_FENCE();   // one channel's floats at a time in registers
    }
    norm_planar_sum<T, PX, E, 2>(s, sm, turn);
#pragma unroll
    for (int j = 0; j < E; ++j) { s[0][j] *= inv_c; s[1][j] *= inv_c * rstd[j]; }
#pragma unroll
    for (int k = 0; k < NC; ++k) {
      float f[E], d[E], y[E];
      rx[k].pin();
      rd[k].pin();
      rx[k].get(f);
      rd[k].get(d);
#pragma unroll
      for (int j = 0; j < E; ++j) y[j] = rstd[j] * (fmaf(d[j], w[k], -s[0][j]) - (f[j] - mean[j]) * s[1][j]);
      if (cg + CG * k < C) VecIo<AT, E>::store(norm_at(reinterpret_cast<AT*>(a.y) + (row0 + CG * k) * P, yoff), y, n);
      CSN_SCHED_FENCE();
    }
  }
  float* pw = norm_slab(a, 0);
  float* pb = norm_slab(a, 1);
#pragma unroll
  for (int k = 0; k < NC; ++k) {
    float u = dw[k], v = db[k];
    if (PX >= 16) { u += csn_lane_xor_f32<8>(u); v += csn_lane_xor_f32<8>(v); }
    if (PX >= 8) { u += csn_lane_xor_f32<4>(u); v += csn_lane_xor_f32<4>(v); }
    if (PX >= 4) { u += csn_lane_xor_f32<2>(u); v += csn_lane_xor_f32<2>(v); }
    u += csn_lane_xor_f32<1>(u); v += csn_lane_xor_f32<1>(v);
    const int c = cg + CG * k;
    if (px == 0 && c < C) {
      if (pw) pw[c] = u;
      if (pb) pb[c] = v;
    }
  }
}

// Blocks of a persistent launch on 256 CUs, as waves per SIMD: about what the registers of the form let a CU hold, so that the last
// blocks do not run alone, and in the backward, whose blocks leave a slab of weight gradients each, no more than keep the loads in
// flight (with the next token's loads ahead of the sums, two waves are enough where a lane holds much).  Measured, us (backward with
// the sum of the slabs):
//   rows of one piece: forward 8 / 6 / 4 waves 19.2 / 17.7 / 18.4 (65536 x 256 bf16, checkpoint); backward 4 / 3 / 2 waves 58.3 / 56.7 / 60.3
//     (200704 x 128 float);
//   rows of two: forward 18.3 / 16.8 / 16.6 (16384 x 1024 bf16); backward 29.5 / 26.6 / 25.8, at 16384 x 4096 107 / 91 / 92;
//   planar: forward 43.6 / 44.9 / 46.2 (32x256x88x88 bf16); backward 95.9 / 94.1 / 94.2, at 64x40x112x112 bf16 70.7 / 71.4 / 56.3.
static int64_t norm_blocks(int threads, int waves) { return 256 * (int64_t)std::max(256 * waves / threads, 1); }

// The register forms: which one takes a case, what its grid is.  slabs = 0: none.
struct NormPlan { int G, NV; int T, PX, NC, runs; int64_t slabs, tiles, items; };
static NormPlan norm_plan(int rows, int a16, bool bwd, int64_t outer, int64_t C, int64_t inner, int64_t x_sc, int64_t dy_sc) {
  NormPlan p{};
  if (outer * inner == 0) return p;
  if (rows) {   // NV counts pieces of 8 elements
    if (C > 16384) return p;
    p.G = C <= 64 ? 8 : C <= 128 ? 16 : C <= 256 ? 32 : C <= 1024 ? 64 : C <= 4096 ? 256 : 1024;
    p.NV = C <= (int64_t)p.G * 8 ? 1 : 2;
    p.T = std::max(p.G, CSN_BLOCK);
    const int r = p.T / p.G;
    p.slabs = std::min(norm_blocks(p.T, p.NV == 1 ? (bwd ? 3 : 6) : (bwd ? 2 : 4)), (outer + r - 1) / r);
    return p;
  }
  if (C > 2048 || inner < NORM_PE) return p;
  // The forward does best with the most channels per lane that fit its registers and 16 lanes (128 / 256 bytes of a channel) across the
  // pixels: 16 channels 46 us, 8 channels 52 us (32x256x88x88 bf16), 36 against 50 us (16x512x44x44 float with a checkpoint).  The backward
  // holds two tensors, the next tile of both and two sums per channel: 8 channels 94 us, 16 channels 120 us (32x256x88x88 bf16); 4 channels in
  // blocks of 1024 threads, whose registers are half as many, lose in float (16x1024x32x32 80 against 63 us, 16x2048x28x28 171 against
  // 145) and are as good in bf16 (58 against 60, 159 against 159).  Wider tokens than that narrow the tile.
  if (!bwd) {
    p.T = C <= 64 ? 128 : C <= 128 ? 128 : C <= 256 ? 256 : C <= 512 ? 512 : 1024;
    p.PX = C <= 1024 ? 16 : 8;
    p.NC = C <= 64 ? 8 : 16;
  } else {
    p.T = C <= 64 ? 128 : C <= 128 ? 256 : C <= 256 && !a16 ? 256 : 512;
    p.PX = C <= 128 ? 16 : C <= 256 ? (a16 ? 16 : 8) : C <= 512 ? 8 : C <= 1024 ? 4 : 2;
    p.NC = 8;
  }
  const int cg = p.T / p.PX;
  const int64_t tile = (int64_t)p.PX * NORM_PE, lim = (int64_t)1 << 29;
  const int64_t es = a16 ? 2 : 4;
  p.tiles = (inner + tile - 1) / tile;
  p.items = outer * p.tiles;
  p.runs = p.items > 8 && (inner * es % 128 != 0 || tile * es % 128 != 0);
  // 32-bit byte offsets of a lane and 32-bit item counts
  if (inner > lim || p.items > lim || cg * std::max(inner, std::max(x_sc, dy_sc)) + inner + tile > lim) { p.slabs = 0; return p; }
  p.slabs = std::min(norm_blocks(p.T, bwd ? 2 : 8), p.runs ? (p.items + 7) & ~(int64_t)7 : p.items);
  return p;
}

template <typename AT, int G, int NVB, int CK, bool W = true>
static int norm_rows_go(const NormArgs& a, bool bwd, void* stream) {
  constexpr int NV = NVB * (8 / VecIo<AT>::E), T = NormRowsBlock<G>::T;
  const dim3 g((unsigned)a.slabs), b(T);
  const size_t sm = std::max((size_t)64 * sizeof(float), T / G > 1 ? (size_t)T * VecIo<AT>::E * sizeof(float) : (size_t)0);
  if (bwd) CSN_LAUNCH((norm_rows_bwd_kernel<AT, G, NV, W, CK>), g, b, sm, stream, a);
  else CSN_LAUNCH((norm_rows_fwd_kernel<AT, G, NV, W, CK>), g, b, sm, stream, a);
  return (int)hipGetLastError();
}
template <typename AT, int CK>
static int norm_rows_run(const NormArgs& a, const NormPlan& p, bool bwd, void* stream) {
  switch (p.G) {
    case 8: return a.C >= VecIo<AT>::E ? norm_rows_go<AT, 8, 1, CK>(a, bwd, stream) : norm_rows_go<AT, 8, 1, CK, false>(a, bwd, stream);
    case 16: return norm_rows_go<AT, 16, 1, CK>(a, bwd, stream);
    case 32: return norm_rows_go<AT, 32, 1, CK>(a, bwd, stream);
    case 64: return p.NV == 1 ? norm_rows_go<AT, 64, 1, CK>(a, bwd, stream) : norm_rows_go<AT, 64, 2, CK>(a, bwd, stream);
    case 256: return p.NV == 1 ? norm_rows_go<AT, 256, 1, CK>(a, bwd, stream) : norm_rows_go<AT, 256, 2, CK>(a, bwd, stream);
  }
  return p.NV == 1 ? norm_rows_go<AT, 1024, 1, CK>(a, bwd, stream) : norm_rows_go<AT, 1024, 2, CK>(a, bwd, stream);
}
template <typename AT, int T, int PX, int NC, int CK>
static int norm_planar_fwd(const NormArgs& a, void* stream) {
  const size_t sm = (size_t)2 * (T / 64) * PX * NORM_PE * sizeof(float);
  CSN_LAUNCH((norm_planar_fwd_kernel<AT, T, PX, NC, CK>), dim3((unsigned)a.slabs), dim3(T), sm, stream, a);
  return (int)hipGetLastError();
}
template <typename AT, int T, int PX, int NC, int CK>
static int norm_planar_bwd(const NormArgs& a, void* stream) {
  const size_t sm = (size_t)2 * (T / 64) * 2 * PX * NORM_PE * sizeof(float);
  CSN_LAUNCH((norm_planar_bwd_kernel<AT, T, PX, NC, CK>), dim3((unsigned)a.slabs), dim3(T), sm, stream, a);
  return (int)hipGetLastError();
}
template <typename AT, int CK>
static int norm_planar_run(const NormArgs& a, const NormPlan& p, bool bwd, void* stream) {
  if (!bwd) {
    if (p.NC == 8) return norm_planar_fwd<AT, 128, 16, 8, CK>(a, stream);
    if (p.T == 128) return norm_planar_fwd<AT, 128, 16, 16, CK>(a, stream);
    if (p.T == 256) return norm_planar_fwd<AT, 256, 16, 16, CK>(a, stream);
    if (p.T == 512) return norm_planar_fwd<AT, 512, 16, 16, CK>(a, stream);
    return p.PX == 16 ? norm_planar_fwd<AT, 1024, 16, 16, CK>(a, stream) : norm_planar_fwd<AT, 1024, 8, 16, CK>(a, stream);
  }
  if (p.T == 128) return norm_planar_bwd<AT, 128, 16, 8, CK>(a, stream);
  if (p.T == 256) return p.PX == 16 ? norm_planar_bwd<AT, 256, 16, 8, CK>(a, stream) : norm_planar_bwd<AT, 256, 8, 8, CK>(a, stream);
  if (p.PX == 16) return norm_planar_bwd<AT, 512, 16, 8, CK>(a, stream);
  if (p.PX == 8) return norm_planar_bwd<AT, 512, 8, 8, CK>(a, stream);
  return p.PX == 4 ? norm_planar_bwd<AT, 512, 4, 8, CK>(a, stream) : norm_planar_bwd<AT, 512, 2, 8, CK>(a, stream);
}
template <int CK>
static int norm_fast(const NormArgs& a, const NormPlan& p, int rows, int a16, bool bwd, void* stream) {
  if (rows) return a16 ? norm_rows_run<csn_bf16, CK>(a, p, bwd, stream) : norm_rows_run<float, CK>(a, p, bwd, stream);
  return a16 ? norm_planar_run<csn_bf16, CK>(a, p, bwd, stream) : norm_planar_run<float, CK>(a, p, bwd, stream);
}
static int norm_fast(NormArgs a, const NormPlan& p, int rows, int a16, int ck, bool bwd, void* stream) {
  a.slabs = (int32_t)p.slabs; a.tiles = (int32_t)p.tiles; a.items = (int32_t)p.items; a.runs = p.runs;
  if (ck == NORM_X) return norm_fast<NORM_X>(a, p, rows, a16, bwd, stream);
  return ck == Q8_INT8 ? norm_fast<Q8_INT8>(a, p, rows, a16, bwd, stream) : norm_fast<Q8_E4M3>(a, p, rows, a16, bwd, stream);
}
#else
struct NormPlan { int64_t slabs; };
static NormPlan norm_plan(int, int, bool, int64_t, int64_t, int64_t, int64_t, int64_t) { return NormPlan{0}; }
#endif  // CSN_EMU_SEQ

template <typename AT, bool ROWS>
static int norm_fwd(const NormArgs& a, void* stream) {
  const int64_t tokens = a.outer * a.inner;
  CSN_LAUNCH((norm_fwd_kernel<AT, ROWS>), dim3(norm_grid(tokens)), dim3(CSN_BLOCK), CSN_BLOCK * sizeof(double), stream, a);
  return (int)hipGetLastError();
}

// (maps of one pixel with consecutive channels are rows, but for the blocks of a checkpoint)
static bool norm_one_pixel(const NormArgs& a, bool bwd) {
  return a.inner == 1 && !a.codes_in && (a.x_sc == 1 || a.C == 1) && (!bwd || a.dy_sc == 1 || a.C == 1);
}

int csn_launch_norm_fwd(const NormArgs& a0, int rows, int a16, int fmt, void* stream) {
  NormArgs a = a0;
  if (a.outer * a.inner <= 0) return 0;
  const bool one = !rows && norm_one_pixel(a, false);
  const NormPlan p = norm_plan(rows || one, a16, false, a.outer, a.C, a.inner, a.x_sc, 0);
  if (a.codes && (p.slabs == 0 || one)) {   // the checkpoint of x as a pass of its own
    Q8PackArgs q;
    q.x = a.x; q.codes = a.codes; q.exps = a.exps; q.nblk = a.nblk;
    q.outer = rows ? 1 : a.outer; q.rows = rows ? a.outer : a.C; q.cols = rows ? a.C : a.inner;
    q.so = rows ? 0 : a.x_so; q.sr = rows ? a.x_so : a.x_sc;
    const int e = csn_launch_q8_pack(q, a16, fmt, stream);
    if (e != 0) return e;
    a.codes = nullptr;
  }
  if (one) rows = 1;
#ifndef CSN_EMU_SEQ
  if (p.slabs > 0) return norm_fast(a, p, rows, a16, a.codes ? fmt : NORM_X, false, stream);
#endif
  if (rows) return a16 ? norm_fwd<csn_bf16, true>(a, stream) : norm_fwd<float, true>(a, stream);
  return a16 ? norm_fwd<csn_bf16, false>(a, stream) : norm_fwd<float, false>(a, stream);
}

template <typename AT, int FMT, bool ROWS>
static int norm_bwd(const NormArgs& a, void* stream) {
  const int64_t tokens = a.outer * a.inner;
  const size_t sm = CSN_BLOCK * sizeof(double);
  if (tokens > 0) CSN_LAUNCH((norm_bwd_kernel<AT, FMT, ROWS>), dim3(norm_grid(tokens)), dim3(CSN_BLOCK), sm, stream, a);
  if (a.dweight || a.dbias) CSN_LAUNCH((norm_dw_kernel<AT, FMT, ROWS>), dim3(norm_grid(a.C)), dim3(CSN_BLOCK), sm, stream, a);
  return (int)hipGetLastError();
}

int csn_launch_norm_bwd(const NormArgs& a0, int rows, int a16, int fmt, void* stream) {
  NormArgs a = a0;
  if (!rows && norm_one_pixel(a, true)) rows = 1;
  const NormPlan p = norm_plan(rows, a16, true, a.outer, a.C, a.inner, a.x_sc, a.dy_sc);
#ifndef CSN_EMU_SEQ
  if (p.slabs > 0) {
    if (!a.dweight && !a.dbias) a.partial = nullptr;
    const int e = norm_fast(a, p, rows, a16, a.x ? NORM_X : fmt, true, stream);
    if (e != 0 || !a.partial || p.slabs == 1) return e;
    SlabSumArgs r;
    r.partial = a.partial; r.out0 = a.dweight; r.out1 = a.dbias; r.n0 = a.C; r.n = 2 * a.C; r.slabs = (int32_t)p.slabs;
    return csn_launch_slab_sum(r, stream);
  }
#endif
  if (fmt == Q8_INT8) {
    if (rows) return a16 ? norm_bwd<csn_bf16, Q8_INT8, true>(a, stream) : norm_bwd<float, Q8_INT8, true>(a, stream);
    return a16 ? norm_bwd<csn_bf16, Q8_INT8, false>(a, stream) : norm_bwd<float, Q8_INT8, false>(a, stream);
  }
  if (rows) return a16 ? norm_bwd<csn_bf16, Q8_E4M3, true>(a, stream) : norm_bwd<float, Q8_E4M3, true>(a, stream);
  return a16 ? norm_bwd<csn_bf16, Q8_E4M3, false>(a, stream) : norm_bwd<float, Q8_E4M3, false>(a, stream);
}

int64_t csn_norm_partial_floats(int rows, int a16, int64_t outer, int64_t C, int64_t inner) {
  // (strides decide between the forms, never for more slabs; maps of one pixel may run as rows)
  const int64_t slabs = norm_plan(rows || inner == 1, a16, true, outer, C, inner, 0, 0).slabs;
  return slabs > 1 ? slabs * 2 * C : 0;
}
