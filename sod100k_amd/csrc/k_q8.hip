// k_q8.hip -- 8-bit checkpoints of activations: pack and unpack (format and decisions: q8_core.h).
//
// Both are streams: pack reads 4 or 2 bytes an element and writes 1 + 1/32, unpack the reverse.
//
// A lane takes a piece of 16 (bfloat16) or 8 (float) consecutive elements, so that codes move 16 or 8 bytes at a time; the two or four lanes of
// a block exchange its maximum.  Pieces are counted through rows of `per_row` pieces each, a row's last block being short; rows
// whose length is a multiple of 32 and that follow each other without a gap are one long row.  128-bit accesses at any
// address: vec_io.h.
#include "q8_core.h"
#include "train_ops.h"
#include "vec_io.h"

#ifdef CSN_EMU_SEQ
int csn_launch_q8_pack(const Q8PackArgs&, int, int, void*) { return -1; }   // (lane exchange: lane-exact mode only)
int csn_launch_q8_unpack(const Q8UnpackArgs&, int, int, void*) { return -1; }
#else

#define Q8_VECS 2    // 16-byte vectors of the tensor per piece

template <typename AT, int FMT, bool W>
__global__ __launch_bounds__(CSN_BLOCK) void q8_pack_kernel(Q8PackArgs a) {
  constexpr int E = VecIo<AT>::E, L = Q8_VECS * E;   // elements of a piece; 32 / L lanes hold a block
  const int64_t stride = (int64_t)gridDim.x * CSN_BLOCK;
  for (int64_t i = (int64_t)blockIdx.x * CSN_BLOCK + threadIdx.x; i < a.items; i += stride) {
    // (a wave's pieces of one block never part: items is a multiple of 32 / L lanes)
    int64_t row = 0, pos = i * L, o = 0;
    if (a.nrows > 1) {
      if (a.items <= 0x7fffffff) {
        const unsigned r = (unsigned)i / (unsigned)a.per_row;
        row = r;
        o = r / (unsigned)a.rows;
      } else {
        row = i / a.per_row;
        o = row / a.rows;
      }
      pos = (i - row * a.per_row) * L;
    }
    const int64_t left = a.cols - pos;
    const int n = (int)(left < L ? left : L);
    const AT* x = reinterpret_cast<const AT*>(a.x) + o * a.so + (row - o * a.rows) * a.sr + pos;
    VecIo<AT> v[Q8_VECS];
#pragma unroll
    for (int q = 0; q < Q8_VECS; ++q) vec_load<W>(v[q], x + q * E, n - q * E);
    float f[L];
#pragma unroll
    for (int q = 0; q < Q8_VECS; ++q) {
      float g[E];
      vec_end<W>(v[q], n - q * E);
      v[q].get(g);
#pragma unroll
      for (int j = 0; j < E; ++j) f[q * E + j] = g[j];
    }
    unsigned w[L / 4];
    const unsigned s = q8_pack_block<FMT, L>(f, w);
    uint8_t* c = a.codes + row * a.cols + pos;
    if (n >= L) {
      if (L == 16) {
        csn_raw16_a1 r;
#pragma unroll
        for (int j = 0; j < 4; ++j) r.w[j] = w[j];
        *reinterpret_cast<csn_raw16_a1*>(c) = r;
      } else {
        csn_raw8_a1 r;
#pragma unroll
        for (int j = 0; j < 2; ++j) r.w[j] = w[j];
        *reinterpret_cast<csn_raw8_a1*>(c) = r;
      }
    } else {
#pragma unroll
      for (int j = 0; j < L; ++j)
        if (j < n) c[j] = (uint8_t)(w[j >> 2] >> (8 * (j & 3)));
    }
    if ((i & (32 / L - 1)) == 0) a.exps[i / (32 / L)] = (uint8_t)s;   // (a row's pieces are whole blocks, the last one in part empty)
  }
}

template <typename AT, int FMT, bool W>
__global__ __launch_bounds__(CSN_BLOCK) void q8_unpack_kernel(Q8UnpackArgs a) {
  constexpr int E = VecIo<AT>::E, L = Q8_VECS * E;
  const int64_t stride = (int64_t)gridDim.x * CSN_BLOCK;
  for (int64_t i = (int64_t)blockIdx.x * CSN_BLOCK + threadIdx.x; i < a.items; i += stride) {
    int64_t row = 0, pos = i * L;
    if (a.rows > 1) {
      row = a.items <= 0x7fffffff ? (int64_t)((unsigned)i / (unsigned)a.per_row) : i / a.per_row;
      pos = (i - row * a.per_row) * L;
    }
    const int64_t left = a.cols - pos;
    const int n = (int)(left < L ? left : L);
    const uint8_t* c = a.codes + row * a.cols + pos;
    CodeIo<E> v[Q8_VECS];
    if (n >= L) {
      if (L == 16) {
        const csn_raw16_a1 r = *reinterpret_cast<const csn_raw16_a1*>(c);
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j / (E / 4)].w[j % (E / 4)] = r.w[j];
      } else {
        const csn_raw8_a1 r = *reinterpret_cast<const csn_raw8_a1*>(c);
#pragma unroll
        for (int j = 0; j < 2; ++j) v[j / (E / 4)].w[j % (E / 4)] = r.w[j];
      }
    } else {
#pragma unroll
      for (int q = 0; q < Q8_VECS; ++q) {
        code_load<W, E>(v[q], c + q * E, n - q * E);
        code_end<W, E>(v[q], n - q * E);
      }
    }
    const float sc = q8_scale(a.exps[i / (32 / L)]);
    AT* y = reinterpret_cast<AT*>(a.y) + row * a.cols + pos;
#pragma unroll
    for (int q = 0; q < Q8_VECS; ++q) {
      float f[E];
      q8_decode_vec<FMT, E>(v[q].w, sc, f);
      VecIo<AT>::store(y + q * E, f, n - q * E);
    }
  }
}

static unsigned q8_grid(int64_t items) {
  const int64_t g = (items + CSN_BLOCK - 1) / CSN_BLOCK;
  return (unsigned)(g < 65536 ? g : 65536);
}

template <typename AT, int FMT>
static int q8_pack_run(const Q8PackArgs& a, void* stream) {
  const dim3 g(q8_grid(a.items)), b(CSN_BLOCK);
  if (a.cols >= VecIo<AT>::E) CSN_LAUNCH((q8_pack_kernel<AT, FMT, true>), g, b, 0, stream, a);
  else CSN_LAUNCH((q8_pack_kernel<AT, FMT, false>), g, b, 0, stream, a);
  return (int)hipGetLastError();
}
template <typename AT, int FMT>
static int q8_unpack_run(const Q8UnpackArgs& a, void* stream) {
  const dim3 g(q8_grid(a.items)), b(CSN_BLOCK);
  if (a.cols >= VecIo<AT>::E) CSN_LAUNCH((q8_unpack_kernel<AT, FMT, true>), g, b, 0, stream, a);
  else CSN_LAUNCH((q8_unpack_kernel<AT, FMT, false>), g, b, 0, stream, a);
  return (int)hipGetLastError();
}

int csn_launch_q8_pack(const Q8PackArgs& a0, int a16, int fmt, void* stream) {
  Q8PackArgs a = a0;
  if (a.outer * a.rows * a.cols <= 0) return 0;
  if (a.cols % 32 == 0 && (a.rows == 1 || a.sr == a.cols) && (a.outer == 1 || a.so == a.rows * a.cols)) {
    a.cols *= a.outer * a.rows;
    a.outer = a.rows = 1;
  }
  a.nrows = a.outer * a.rows;
  a.nblk = (a.cols + 31) / 32;
  a.per_row = a.nblk * (a16 ? 2 : 4);
  a.items = a.nrows * a.per_row;
  if (a16) return fmt == Q8_INT8 ? q8_pack_run<csn_bf16, Q8_INT8>(a, stream) : q8_pack_run<csn_bf16, Q8_E4M3>(a, stream);
  return fmt == Q8_INT8 ? q8_pack_run<float, Q8_INT8>(a, stream) : q8_pack_run<float, Q8_E4M3>(a, stream);
}

int csn_launch_q8_unpack(const Q8UnpackArgs& a0, int a16, int fmt, void* stream) {
  Q8UnpackArgs a = a0;
  if (a.rows * a.cols <= 0) return 0;
  if (a.cols % 32 == 0) { a.cols *= a.rows; a.rows = 1; }
  a.nblk = (a.cols + 31) / 32;
  a.per_row = a.nblk * (a16 ? 2 : 4);
  a.items = a.rows * a.per_row;
  if (a16) return fmt == Q8_INT8 ? q8_unpack_run<csn_bf16, Q8_INT8>(a, stream) : q8_unpack_run<csn_bf16, Q8_E4M3>(a, stream);
  return fmt == Q8_INT8 ? q8_unpack_run<float, Q8_INT8>(a, stream) : q8_unpack_run<float, Q8_E4M3>(a, stream);
}
#endif  // CSN_EMU_SEQ
