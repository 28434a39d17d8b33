// k_norm.hip -- layer norm over the channels of a token, forward and backward, for planar maps and for rows of tokens.
//
//     mean = sum_c x / C,  var = sum_c (x - mean)^2 / C,  rstd = (var + eps)^(-1/2),  y = (x - mean) rstd w + b
//     g = dy w,  c1 = sum_c g / C,  c2 = sum_c g xh / C,  dx = rstd (g - c1 - xh c2),  dw = sum_t dy xh,  db = sum_t dy
//
// with xh = (x - mean) rstd; in the backward x may be the 8-bit checkpoint that the forward left (q8_core.h).
#include "csn_reduce.h"
#include "q8_core.h"
#include "train_ops.h"

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

// one block per token
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

// one block per channel
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

template <typename AT, bool ROWS>
static int norm_fwd(const NormArgs& a, void* stream) {
  const int64_t tokens = a.outer * a.inner;
  CSN_LAUNCH((norm_fwd_kernel<AT, ROWS>), dim3(norm_grid(tokens)), dim3(CSN_BLOCK), CSN_BLOCK * sizeof(double), stream, a);
  return (int)hipGetLastError();
}

int csn_launch_norm_fwd(const NormArgs& a, int rows, int a16, int fmt, void* stream) {
  if (a.outer * a.inner <= 0) return 0;
  if (a.codes) {   // the checkpoint of x as a pass of its own
    Q8PackArgs q;
    q.x = a.x; q.codes = a.codes; q.exps = a.exps; q.nblk = a.nblk;
    q.outer = rows ? 1 : a.outer; q.rows = rows ? a.outer : a.C; q.cols = rows ? a.C : a.inner;
    q.so = rows ? 0 : a.x_so; q.sr = rows ? a.x_so : a.x_sc;
    const int e = csn_launch_q8_pack(q, a16, fmt, stream);
    if (e != 0) return e;
  }
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

int csn_launch_norm_bwd(const NormArgs& a, int rows, int a16, int fmt, void* stream) {
  if (fmt == Q8_INT8) {
    if (rows) return a16 ? norm_bwd<csn_bf16, Q8_INT8, true>(a, stream) : norm_bwd<float, Q8_INT8, true>(a, stream);
    return a16 ? norm_bwd<csn_bf16, Q8_INT8, false>(a, stream) : norm_bwd<float, Q8_INT8, false>(a, stream);
  }
  if (rows) return a16 ? norm_bwd<csn_bf16, Q8_E4M3, true>(a, stream) : norm_bwd<float, Q8_E4M3, true>(a, stream);
  return a16 ? norm_bwd<csn_bf16, Q8_E4M3, false>(a, stream) : norm_bwd<float, Q8_E4M3, false>(a, stream);
}

int64_t csn_norm_partial_floats(int, int, int64_t, int64_t, int64_t) { return 0; }
