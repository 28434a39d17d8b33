// k_q8.hip -- 8-bit checkpoints of activations: pack and unpack (format and decisions: q8_core.h).
//
// Both are streams: pack reads 4 or 2 bytes an element and writes 1 + 1/32, unpack the reverse.
#include "q8_core.h"
#include "train_ops.h"

// one thread per block of 32 elements
template <typename AT, int FMT>
__global__ __launch_bounds__(CSN_BLOCK) void q8_pack_kernel(Q8PackArgs a) {
  const int64_t n = a.outer * a.rows * a.nblk;
  for (int64_t i = (int64_t)blockIdx.x * CSN_BLOCK + threadIdx.x; i < n; i += (int64_t)gridDim.x * CSN_BLOCK) {
    const int64_t row = i / a.nblk, blk = i - row * a.nblk;
    const int64_t o = row / a.rows, r = row - o * a.rows;
    const int64_t c0 = blk * 32;
    const int m = (int)min((int64_t)32, a.cols - c0);
    const AT* x = reinterpret_cast<const AT*>(a.x) + o * a.so + r * a.sr + c0;
    float amax = 0.f;
    for (int j = 0; j < m; ++j) amax = fmaxf(amax, q8_mag<FMT>(act_ld(x + j)));
    const unsigned s = q8_exponent<FMT>(amax);
    const float inv = q8_inv_scale(s);
    uint8_t* c = a.codes + row * a.cols + c0;
    for (int j = 0; j < m; ++j) c[j] = (uint8_t)q8_encode<FMT>(act_ld(x + j), inv);
    a.exps[i] = (uint8_t)s;
  }
}

template <typename AT, int FMT>
__global__ __launch_bounds__(CSN_BLOCK) void q8_unpack_kernel(Q8UnpackArgs a) {
  const int64_t n = a.rows * a.cols;
  for (int64_t i = (int64_t)blockIdx.x * CSN_BLOCK + threadIdx.x; i < n; i += (int64_t)gridDim.x * CSN_BLOCK) {
    const int64_t row = i / a.cols, col = i - row * a.cols;
    act_st(reinterpret_cast<AT*>(a.y) + i, q8_decode<FMT>(a.codes[i], q8_scale(a.exps[row * a.nblk + col / 32])));
  }
}

static unsigned q8_grid(int64_t items) {
  const int64_t g = (items + CSN_BLOCK - 1) / CSN_BLOCK;
  return (unsigned)(g < 16384 ? g : 16384);
}

int csn_launch_q8_pack(const Q8PackArgs& a, int a16, int fmt, void* stream) {
  const int64_t n = a.outer * a.rows * a.nblk;
  if (n <= 0) return 0;
  const dim3 g(q8_grid(n)), b(CSN_BLOCK);
  if (a16) {
    if (fmt == Q8_INT8) CSN_LAUNCH((q8_pack_kernel<csn_bf16, Q8_INT8>), g, b, 0, stream, a);
    else CSN_LAUNCH((q8_pack_kernel<csn_bf16, Q8_E4M3>), g, b, 0, stream, a);
  } else {
    if (fmt == Q8_INT8) CSN_LAUNCH((q8_pack_kernel<float, Q8_INT8>), g, b, 0, stream, a);
    else CSN_LAUNCH((q8_pack_kernel<float, Q8_E4M3>), g, b, 0, stream, a);
  }
  return (int)hipGetLastError();
}

int csn_launch_q8_unpack(const Q8UnpackArgs& a, int a16, int fmt, void* stream) {
  const int64_t n = a.rows * a.cols;
  if (n <= 0) return 0;
  const dim3 g(q8_grid(n)), b(CSN_BLOCK);
  if (a16) {
    if (fmt == Q8_INT8) CSN_LAUNCH((q8_unpack_kernel<csn_bf16, Q8_INT8>), g, b, 0, stream, a);
    else CSN_LAUNCH((q8_unpack_kernel<csn_bf16, Q8_E4M3>), g, b, 0, stream, a);
  } else {
    if (fmt == Q8_INT8) CSN_LAUNCH((q8_unpack_kernel<float, Q8_INT8>), g, b, 0, stream, a);
    else CSN_LAUNCH((q8_unpack_kernel<float, Q8_E4M3>), g, b, 0, stream, a);
  }
  return (int)hipGetLastError();
}
