// k_q8.hip -- 8-bit checkpoints of activations: pack and unpack (format and decisions: q8_core.h).
//
// Both are streams: pack reads 4 or 2 bytes an element and writes 1 + 1/32, unpack the reverse.  64x40x224x224 bf16, int8: pack
// 78 us (5.0 TB/s; with the tensor in the cache of the device 69), unpack 66 us (5.9 TB/s) where a plain copy moves 6.2 TB/s; small tensors
// (40x56x56) 2.8 us each, what a launch costs.
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
int csn_launch_q8_segments(Q8Seg*, int, bool, int, int, void*) { return -1; }
#else

#define Q8_VECS 2    // 16-byte vectors of the tensor per piece

// piece of n <= L elements at x -> codes at c, and the block's exponent at e from its first lane (32 / L neighbouring lanes, all of
// them here)
template <typename AT, int FMT, bool W>
__device__ __forceinline__ void q8_pack_piece(const AT* x, uint8_t* c, uint8_t* e, int n, bool first) {
  constexpr int E = VecIo<AT>::E, L = Q8_VECS * E;
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
  if (n >= L) {
    if (L == 16) {
      csn_raw16_a1 r;
#pragma unroll
      for (int j = 0; j < 4; ++j) r.w[j] = w[j % (L / 4)];
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
  if (first) *e = (uint8_t)s;
}

template <typename AT, int FMT, bool W>
__device__ __forceinline__ void q8_unpack_piece(const uint8_t* c, unsigned e, AT* y, int n) {
  constexpr int E = VecIo<AT>::E, L = Q8_VECS * E;
  CodeIo<E> v[Q8_VECS];
  if (n >= L) {
    if (L == 16) {
      const csn_raw16_a1 r = *reinterpret_cast<const csn_raw16_a1*>(c);
#pragma unroll
      for (int j = 0; j < 4; ++j) v[j / (E / 4) % Q8_VECS].w[j % (E / 4)] = r.w[j];
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
  const float sc = q8_scale(e);
#pragma unroll
  for (int q = 0; q < Q8_VECS; ++q) {
    float f[E];
    q8_decode_vec<FMT, E>(v[q].w, sc, f);
    VecIo<AT>::store(y + q * E, f, n - q * E);
  }
}

template <typename AT, int FMT, bool W>
__global__ __launch_bounds__(CSN_BLOCK) void q8_pack_kernel(Q8PackArgs a) {
  constexpr int L = Q8_VECS * VecIo<AT>::E;   // elements of a piece; 32 / L lanes hold a block
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
    const AT* x = reinterpret_cast<const AT*>(a.x) + o * a.so + (row - o * a.rows) * a.sr + pos;
    // (a row's pieces are whole blocks, the last one in part empty)
    q8_pack_piece<AT, FMT, W>(x, a.codes + row * a.cols + pos, a.exps + i / (32 / L), (int)(left < L ? left : L), (i & (32 / L - 1)) == 0);
  }
}

template <typename AT, int FMT, bool W>
__global__ __launch_bounds__(CSN_BLOCK) void q8_unpack_kernel(Q8UnpackArgs a) {
  constexpr int L = Q8_VECS * VecIo<AT>::E;
  const int64_t stride = (int64_t)gridDim.x * CSN_BLOCK;
  for (int64_t i = (int64_t)blockIdx.x * CSN_BLOCK + threadIdx.x; i < a.items; i += stride) {
    int64_t row = 0, pos = i * L;
    if (a.rows > 1) {
      row = a.items <= 0x7fffffff ? (int64_t)((unsigned)i / (unsigned)a.per_row) : i / a.per_row;
      pos = (i - row * a.per_row) * L;
    }
    const int64_t left = a.cols - pos, at = row * a.cols + pos;
    q8_unpack_piece<AT, FMT, W>(a.codes + at, a.exps[i / (32 / L)], reinterpret_cast<AT*>(a.y) + at, (int)(left < L ? left : L));
  }
}

// Many tensors of one type in one launch (the saved tensors of a plan): a block finds its segment among the launch's by its number
// and takes Q8_SEG_PIECES pieces of it.
#define Q8_SEG_PIECES (4 * CSN_BLOCK)
template <typename AT, int FMT, bool W, bool PACK>
__device__ __forceinline__ void q8_segment(const Q8Seg& g, int64_t first) {
  constexpr int L = Q8_VECS * VecIo<AT>::E;
  for (int r = 0; r < 4; ++r) {
    const int64_t i = first + r * CSN_BLOCK + threadIdx.x;
    if (i >= g.items) return;
    const int64_t row = g.items <= 0x7fffffff ? (int64_t)((unsigned)i / (unsigned)g.per_row) : i / g.per_row;
    const int64_t pos = (i - row * g.per_row) * L, left = g.cols - pos, at = row * g.cols + pos;
    const int n = (int)(left < L ? left : L);
    AT* x = reinterpret_cast<AT*>(g.x) + at;
    if (PACK) q8_pack_piece<AT, FMT, W>(x, g.codes + at, g.exps + i / (32 / L), n, (i & (32 / L - 1)) == 0);
    else q8_unpack_piece<AT, FMT, W>(g.codes + at, g.exps[i / (32 / L)], x, n);
  }
}
template <typename AT, int FMT, bool PACK>
__global__ __launch_bounds__(CSN_BLOCK) void q8_segments_kernel(Q8SegArgs a) {
  int s = 0;
  while (s + 1 < a.n && (int)blockIdx.x >= a.seg[s + 1].block0) ++s;
  const Q8Seg& g = a.seg[s];
  const int64_t first = (int64_t)((int)blockIdx.x - g.block0) * Q8_SEG_PIECES;
  if (g.cols >= VecIo<AT>::E) q8_segment<AT, FMT, true, PACK>(g, first);
  else q8_segment<AT, FMT, false, PACK>(g, first);
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

template <typename AT, int FMT>
static int q8_segments_run(const Q8SegArgs& a, bool pack, unsigned blocks, void* stream) {
  if (pack) CSN_LAUNCH((q8_segments_kernel<AT, FMT, true>), dim3(blocks), dim3(CSN_BLOCK), 0, stream, a);
  else CSN_LAUNCH((q8_segments_kernel<AT, FMT, false>), dim3(blocks), dim3(CSN_BLOCK), 0, stream, a);
  return (int)hipGetLastError();
}
int csn_launch_q8_segments(Q8Seg* seg, int n, bool pack, int a16, int fmt, void* stream) {
  for (int i = 0; i < n;) {
    Q8SegArgs a;
    int64_t blocks = 0;
    for (a.n = 0; i < n && a.n < Q8_MAX_SEGS; ++i) {
      Q8Seg g = seg[i];
      if (g.cols % 32 == 0) { g.cols *= g.rows; g.rows = 1; }
      g.per_row = (g.cols + 31) / 32 * (a16 ? 2 : 4);
      g.items = g.rows * g.per_row;
      if (g.items == 0) continue;
      const int64_t nb = (g.items + Q8_SEG_PIECES - 1) / Q8_SEG_PIECES;
      if (blocks + nb > 0x7fffffff) { if (a.n == 0) return -1; break; }
      g.block0 = (int32_t)blocks;
      blocks += nb;
      a.seg[a.n++] = g;
    }
    if (a.n == 0) break;
    const int e = fmt == Q8_INT8 ? (a16 ? q8_segments_run<csn_bf16, Q8_INT8>(a, pack, (unsigned)blocks, stream) : q8_segments_run<float, Q8_INT8>(a, pack, (unsigned)blocks, stream))
                                 : (a16 ? q8_segments_run<csn_bf16, Q8_E4M3>(a, pack, (unsigned)blocks, stream) : q8_segments_run<float, Q8_E4M3>(a, pack, (unsigned)blocks, stream));
    if (e != 0) return e;
  }
  return 0;
}
#endif  // CSN_EMU_SEQ

// ---- plain copies of small tensors, many in one launch (multiples of 4 bytes) --------------------------------------------------
__global__ __launch_bounds__(CSN_BLOCK) void copy_segments_kernel(CopySegArgs a) {
  int s = 0;
  while (s + 1 < a.n && (int)blockIdx.x >= a.seg[s + 1].block0) ++s;
  const CopySeg& g = a.seg[s];
  const int64_t i0 = (int64_t)((int)blockIdx.x - g.block0) * (4 * CSN_BLOCK) + threadIdx.x;
  for (int r = 0; r < 4; ++r)
    if (i0 + r * CSN_BLOCK < g.words) g.dst[i0 + r * CSN_BLOCK] = g.src[i0 + r * CSN_BLOCK];
}
int csn_launch_copy_segments(CopySeg* seg, int n, void* stream) {
  for (int i = 0; i < n;) {
    CopySegArgs a;
    int64_t blocks = 0;
    for (a.n = 0; i < n && a.n < Q8_MAX_SEGS; ++i) {
      if (seg[i].words == 0) continue;
      const int64_t nb = (seg[i].words + 4 * CSN_BLOCK - 1) / (4 * CSN_BLOCK);
      if (blocks + nb > 0x7fffffff) { if (a.n == 0) return -1; break; }
      seg[i].block0 = (int32_t)blocks;
      blocks += nb;
      a.seg[a.n++] = seg[i];
    }
    if (a.n == 0) break;
    CSN_LAUNCH(copy_segments_kernel, dim3((unsigned)blocks), dim3(CSN_BLOCK), 0, stream, a);
    const int e = (int)hipGetLastError();
    if (e != 0) return e;
  }
  return 0;
}
