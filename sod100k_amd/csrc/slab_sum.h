// slab_sum.h -- the sum of per-block partial results in a fixed order (training operators beside the plan).
//
// partial is [slabs][n]; column e goes to out0[e] for e < n0, to out1[e - n0] behind that (null: not wanted).  A block of 1024 threads takes
// 1024 / W columns; W groups of its threads add every W-th slab in double, then the groups are added in order.  W grows
// with the slabs so that no thread walks more than a few dozen: 2048 slabs of 1024 columns 12.3 us with W = 16 (16 blocks of 64
// columns), see csn_launch_slab_sum.
#pragma once
#include "csn_device.h"

struct SlabSumArgs {
  const float* partial;
  float* out0;
  float* out1;
  int64_t n0, n;
  int32_t slabs;
};

template <int W>
__global__ __launch_bounds__(1024) void slab_sum_kernel(SlabSumArgs a) {
  CSN_DYN_SMEM(double, sd);   // [W][1024 / W]
  constexpr int L = 1024 / W;
  const int l = threadIdx.x % L, w = threadIdx.x / L;
  const int64_t e = (int64_t)blockIdx.x * L + l;
  double v = 0.0;
  if (e < a.n) {
#pragma unroll 4
    for (int s = w; s < a.slabs; s += W) v += a.partial[(int64_t)s * a.n + e];
  }
  if (W > 1) {
    sd[threadIdx.x] = v;
    __syncthreads();
    if (w == 0)
      for (int q = 1; q < W; ++q) v += sd[q * L + l];
  }
  if (w == 0 && e < a.n) {
    float* out = e < a.n0 ? a.out0 : a.out1;
    if (out) out[e < a.n0 ? e : e - a.n0] = (float)v;
  }
}

static int csn_launch_slab_sum(const SlabSumArgs& a, void* stream) {
  const int w = a.slabs <= 8 ? 1 : a.slabs <= 64 ? 4 : a.n >= 32768 ? 16 : 64;
  const dim3 g((unsigned)((a.n + 1024 / w - 1) / (1024 / w))), b(1024);
  const size_t sm = 1024 * sizeof(double);
  if (w == 1) CSN_LAUNCH((slab_sum_kernel<1>), g, b, sm, stream, a);
  else if (w == 4) CSN_LAUNCH((slab_sum_kernel<4>), g, b, sm, stream, a);
  else if (w == 16) CSN_LAUNCH((slab_sum_kernel<16>), g, b, sm, stream, a);
  else CSN_LAUNCH((slab_sum_kernel<64>), g, b, sm, stream, a);
  return (int)hipGetLastError();
}
