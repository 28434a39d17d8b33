// k_q8_wgrad.hip -- weight and bias gradient of a product (1x1 convolution / linear layer) from the 8-bit checkpoint of its input.
//
//     dW[o][i] = sum_t dY[t][o] X[t][i],   db[o] = sum_t dY[t][o]        (X: the values of the checkpoint, q8_core.h)
#include "csn_reduce.h"
#include "q8_core.h"
#include "train_ops.h"

// a 16 x 16 tile of dW per block, 16 tokens at a time through LDS
template <typename AT, int FMT, bool ROWS>
__global__ __launch_bounds__(CSN_BLOCK) void q8_wgrad_kernel(Q8WgradArgs a) {
  CSN_DYN_SMEM(float, sm);
  float* sy = sm;               // [16 tokens][17]
  float* sx = sm + 16 * 17;
  const int ti = threadIdx.x & 15, to = threadIdx.x >> 4;
  const int64_t tokens = a.outer * a.inner, i0 = (int64_t)blockIdx.x * 16, o0 = (int64_t)blockIdx.y * 16;
  double acc = 0.0, bias = 0.0;
  for (int64_t t0 = 0; t0 < tokens; t0 += 16) {
    const int64_t t = t0 + (ROWS ? to : ti), ch = ROWS ? ti : to;   // consecutive threads on consecutive elements
    const int64_t o = t / a.inner, p = t - o * a.inner;
    float vy = 0.f, vx = 0.f;
    if (t < tokens && o0 + ch < a.cout)
      vy = act_ld(reinterpret_cast<const AT*>(a.dy) + o * a.dy_so + (ROWS ? o0 + ch : (o0 + ch) * a.dy_sc + p));
    if (t < tokens && i0 + ch < a.cin) {
      const int64_t row = ROWS ? o : o * a.cin + i0 + ch, col = ROWS ? i0 + ch : p, cols = ROWS ? a.cin : a.inner;
      vx = q8_decode<FMT>(a.codes[row * cols + col], q8_scale(a.exps[row * a.nblk + col / 32]));
    }
    __syncthreads();
    sy[(t - t0) * 17 + ch] = vy;
    sx[(t - t0) * 17 + ch] = vx;
    __syncthreads();
    float s = 0.f, sb = 0.f;
    for (int k = 0; k < 16; ++k) {
      s = fmaf(sy[k * 17 + to], sx[k * 17 + ti], s);
      sb += sy[k * 17 + to];
    }
    acc += s; bias += sb;
  }
  if (o0 + to < a.cout && i0 + ti < a.cin) a.dweight[(o0 + to) * a.cin + i0 + ti] = (float)acc;
  if (a.dbias && blockIdx.x == 0 && ti == 0 && o0 + to < a.cout) a.dbias[o0 + to] = (float)bias;
}

template <typename AT, int FMT, bool ROWS>
static int q8_wgrad(const Q8WgradArgs& a, void* stream) {
  const dim3 g((unsigned)((a.cin + 15) / 16), (unsigned)((a.cout + 15) / 16));
  CSN_LAUNCH((q8_wgrad_kernel<AT, FMT, ROWS>), g, dim3(CSN_BLOCK), 2 * 16 * 17 * sizeof(float), stream, a);
  return (int)hipGetLastError();
}

int csn_launch_q8_wgrad(const Q8WgradArgs& a, int rows, int a16, int fmt, void* stream) {
  if (a.cout > 65535 * 16) return -1;
  if (fmt == Q8_INT8) {
    if (rows) return a16 ? q8_wgrad<csn_bf16, Q8_INT8, true>(a, stream) : q8_wgrad<float, Q8_INT8, true>(a, stream);
    return a16 ? q8_wgrad<csn_bf16, Q8_INT8, false>(a, stream) : q8_wgrad<float, Q8_INT8, false>(a, stream);
  }
  if (rows) return a16 ? q8_wgrad<csn_bf16, Q8_E4M3, true>(a, stream) : q8_wgrad<float, Q8_E4M3, true>(a, stream);
  return a16 ? q8_wgrad<csn_bf16, Q8_E4M3, false>(a, stream) : q8_wgrad<float, Q8_E4M3, false>(a, stream);
}

int64_t csn_q8_wgrad_partial_floats(int, int, int64_t, int64_t, int64_t, int64_t) { return 0; }
