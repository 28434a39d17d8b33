// k_q8_wgrad.hip -- weight and bias gradient of a product (1x1 convolution / linear layer) from the 8-bit checkpoint of its input.
//
//     dW[o][i] = sum_t dY[t][o] X[t][i],   db[o] = sum_t dY[t][o]        (X: the values of the checkpoint, q8_core.h)
//
// A matrix product whose reduction runs over the tokens.  A value of the checkpoint is a code of at most 8 significant bits times a
// power of two, that is a bfloat16 number, and the product of two bfloat16 numbers is exact in float: bfloat16 dY goes to
// v_mfma_f32_32x32x16_bf16 as it is.  A float dY is cut by truncation into three bfloat16 numbers of 8 bits each (exact), whose
// products with X go into the same accumulators: three matrix instructions, nothing lost but the accumulation's own rounding.
//
// Block = TM x TN of dW over a slab of the tokens, four waves of (TM / 2) x (TN / 2).  64 tokens are staged at a time into
// two LDS buffers as [row][64 tokens] bfloat16, a row being an output (dY) or an input channel (X): the operand order of the matrix
// instruction, 16 bytes = 8 tokens of a channel.  Planar maps hold 8 consecutive pixels of a channel together already; of token rows
// a thread loads 8 tokens x 4 channels and transposes in registers.  The 16-byte piece c of row r lies at c ^ f(r), f(r) =
// (r ^ r >> 3) & 7: eight consecutive rows (operand reads) and eight rows four apart (the transposed writes) both fall on
// eight different pieces.  The global loads of step s + 1 are in flight while step s is multiplied.
//
// Few tiles and many tokens are the usual case (the channels of a map against its pixels), so the tokens are cut into slabs whose
// partial tiles a second kernel adds in order.
#include "q8_core.h"
#include "slab_sum.h"
#include "train_ops.h"

#ifdef CSN_EMU_SEQ
int csn_launch_q8_wgrad(const Q8WgradArgs&, int, int, int, void*) { return -1; }   // (matrix instructions: lane-exact mode only)
int64_t csn_q8_wgrad_partial_floats(int, int, int64_t, int64_t, int64_t, int64_t) { return 0; }
#else

#define WG_STEP 64      // tokens of a step
#define WG_ROWB 128     // bytes of a staged row

__device__ __forceinline__ unsigned wg_piece(int row, int c) { return (unsigned)(row * WG_ROWB + ((c ^ ((row ^ (row >> 3)) & 7)) << 4)); }
__device__ __forceinline__ csn_u4 wg_u4(unsigned a, unsigned b, unsigned c, unsigned d) {
  csn_u4 r;
  r.x = a; r.y = b; r.z = c; r.w = d;
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

// eight tokens of one row of dY as they were loaded
template <typename AT> struct WgY;
template <> struct WgY<csn_bf16> {
  uint4 u;
  __device__ __forceinline__ void zero() { u = make_uint4(0, 0, 0, 0); }
  __device__ __forceinline__ void load(const csn_bf16* p) { u = *reinterpret_cast<const uint4*>(p); }
  __device__ __forceinline__ void load_some(const csn_bf16* p, int n) {
    unsigned short h[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) h[j] = j < n ? p[j].u : (unsigned short)0;
    u = make_uint4(h[0] | (unsigned)h[1] << 16, h[2] | (unsigned)h[3] << 16, h[4] | (unsigned)h[5] << 16, h[6] | (unsigned)h[7] << 16);
  }
  __device__ __forceinline__ void get(float (&f)[8]) const {
    const unsigned w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) { f[2 * j] = csn_bits_f(w[j] << 16); f[2 * j + 1] = csn_bits_f(w[j] & 0xffff0000u); }
  }
  __device__ __forceinline__ void put(unsigned char* lds, unsigned at, unsigned) const { *reinterpret_cast<csn_u4*>(lds + at) = wg_u4(u.x, u.y, u.z, u.w); }
};
template <> struct WgY<float> {
  float4 a, b;
  __device__ __forceinline__ void zero() { a = b = make_float4(0.f, 0.f, 0.f, 0.f); }
  __device__ __forceinline__ void load(const float* p) { a = *reinterpret_cast<const float4*>(p); b = *reinterpret_cast<const float4*>(p + 4); }
  __device__ __forceinline__ void load_some(const float* p, int n) {
    float f[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) f[j] = j < n ? p[j] : 0.f;
    a = make_float4(f[0], f[1], f[2], f[3]); b = make_float4(f[4], f[5], f[6], f[7]);
  }
  __device__ __forceinline__ void get(float (&f)[8]) const {
    f[0] = a.x; f[1] = a.y; f[2] = a.z; f[3] = a.w; f[4] = b.x; f[5] = b.y; f[6] = b.z; f[7] = b.w;
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
// four channels of one token of dY
template <typename AT> struct WgY4;
template <> struct WgY4<csn_bf16> {
  uint2 u;
  __device__ __forceinline__ void zero() { u = make_uint2(0, 0); }
  __device__ __forceinline__ void load(const csn_bf16* p) { u = *reinterpret_cast<const uint2*>(p); }
  __device__ __forceinline__ void load_some(const csn_bf16* p, int n) {
    unsigned short h[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) h[j] = j < n ? p[j].u : (unsigned short)0;
    u = make_uint2(h[0] | (unsigned)h[1] << 16, h[2] | (unsigned)h[3] << 16);
  }
  __device__ __forceinline__ float get(int j) const {
    const unsigned w = j < 2 ? u.x : u.y;
    return csn_bits_f((j & 1) ? w & 0xffff0000u : w << 16);
  }
};
template <> struct WgY4<float> {
  float4 a;
  __device__ __forceinline__ void zero() { a = make_float4(0.f, 0.f, 0.f, 0.f); }
  __device__ __forceinline__ void load(const float* p) { a = *reinterpret_cast<const float4*>(p); }
  __device__ __forceinline__ void load_some(const float* p, int n) {
    a = make_float4(n > 0 ? p[0] : 0.f, n > 1 ? p[1] : 0.f, n > 2 ? p[2] : 0.f, n > 3 ? p[3] : 0.f);
  }
  __device__ __forceinline__ float get(int j) const { return j == 0 ? a.x : j == 1 ? a.y : j == 2 ? a.z : a.w; }
};

// n = 0 .. 4 codes from an address of any alignment
__device__ __forceinline__ unsigned wg_codes(const uint8_t* p, int n) {
  unsigned w = 0;
#pragma unroll
  for (int j = 0; j < 4; ++j) w |= j < n ? (unsigned)p[j] << (8 * j) : 0u;
  return w;
}

// what a thread holds of the step in flight
template <typename AT, bool ROWS, int TM, int TN> struct WgRegs;
template <typename AT, int TM, int TN> struct WgRegs<AT, false, TM, TN> {
  WgY<AT> y[TM / 32];
  uint2 x[TN / 32];
  unsigned s[TN / 32];
};
template <typename AT, int TM, int TN> struct WgRegs<AT, true, TM, TN> {
  WgY4<AT> y[8];
  unsigned x[8], s[8];
};

template <typename AT, int FMT, bool ROWS, int TM, int TN>
__global__ __launch_bounds__(CSN_BLOCK) void q8_wgrad_kernel(Q8WgradArgs a) {
  CSN_DYN_SMEM(unsigned char, sm);
  constexpr int PARTS = sizeof(AT) == 4 ? 3 : 1;
  constexpr unsigned YB = TM * WG_ROWB, BUF = PARTS * YB + TN * WG_ROWB;
  constexpr int MI = TM / 64, NJ = TN / 64;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  // (slab, tile) items in order over the XCDs (block b runs on XCD b % 8): the tiles of a slab read the same tokens, through one L2
  const int ntile = a.mtiles * a.ntiles, total = ntile * a.slabs, per = (total + 7) >> 3;
  const int item = (int)(blockIdx.x & 7u) * per + (int)(blockIdx.x >> 3);
  if (item >= total || (int)(blockIdx.x >> 3) >= per) return;
  const int slab = item / ntile, tile = item - slab * ntile;
  const int mt = tile / a.ntiles, nt = tile - mt * a.ntiles;
  const int o0 = mt * TM, i0 = nt * TN;
  const int s0 = slab * a.steps_per_slab, s1 = min(s0 + a.steps_per_slab, a.steps);
  const bool bias = a.dbias != nullptr && nt == 0;

  float bsum[4] = {0.f, 0.f, 0.f, 0.f};
  WgRegs<AT, ROWS, TM, TN> rg;

  auto load = [&](int step) {
    if constexpr (!ROWS) {
      const unsigned g = (unsigned)step * 8u + (unsigned)(tid & 7);
      const unsigned o = g / (unsigned)a.chunks, c = g - o * (unsigned)a.chunks;
      const int64_t p = (int64_t)c * 8;
      const int n = (int64_t)o < a.outer ? (int)min((int64_t)8, a.inner - p) : 0;
      const AT* py = reinterpret_cast<const AT*>(a.dy) + (int64_t)o * a.dy_so + p;
#pragma unroll
      for (int j = 0; j < TM / 32; ++j) {
        const int r = o0 + (tid >> 3) + 32 * j;
        rg.y[j].zero();
        if (r < a.cout && n > 0) {
          if (a.vec_y) rg.y[j].load(py + (int64_t)r * a.dy_sc);
          else rg.y[j].load_some(py + (int64_t)r * a.dy_sc, n);
        }
      }
#pragma unroll
      for (int j = 0; j < TN / 32; ++j) {
        const int r = i0 + (tid >> 3) + 32 * j;
        rg.x[j] = make_uint2(0, 0);
        rg.s[j] = 127;
        if (r < a.cin && n > 0) {
          const int64_t row = (int64_t)o * a.cin + r;
          const uint8_t* px = a.codes + row * a.inner + p;
          if (a.vec_x) rg.x[j] = *reinterpret_cast<const uint2*>(px);
          else rg.x[j] = make_uint2(wg_codes(px, n), wg_codes(px + 4, n - 4));
          rg.s[j] = a.exps[row * a.nblk + (p >> 5)];
        }
      }
    } else {
      constexpr int GY = TM / 4, GX = TN / 4;
      {
        const int c = o0 + 4 * (tid & (GY - 1)), k = tid / GY;
        const int n = k < 8 ? (int)min((int64_t)4, a.cout - c) : 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const int64_t t = (int64_t)step * WG_STEP + 8 * k + j;
          rg.y[j].zero();
          if (n > 0 && t < a.outer) {
            const AT* py = reinterpret_cast<const AT*>(a.dy) + t * a.dy_so + c;
            if (a.vec_y && n == 4) rg.y[j].load(py);
            else rg.y[j].load_some(py, n);
          }
        }
      }
      {
        const int c = i0 + 4 * (tid & (GX - 1)), k = tid / GX;
        const int n = k < 8 ? (int)min((int64_t)4, a.cin - c) : 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const int64_t t = (int64_t)step * WG_STEP + 8 * k + j;
          rg.x[j] = 0;
          rg.s[j] = 127;
          if (n > 0 && t < a.outer) {
            const uint8_t* px = a.codes + t * a.cin + c;
            rg.x[j] = a.vec_x && n == 4 ? *reinterpret_cast<const unsigned*>(px) : wg_codes(px, n);
            rg.s[j] = a.exps[t * a.nblk + (c >> 5)];
          }
        }
      }
    }
  };

  auto store = [&](unsigned char* buf) {
    unsigned char* bx = buf + PARTS * YB;
    if constexpr (!ROWS) {
#pragma unroll
      for (int j = 0; j < TM / 32; ++j) {
        rg.y[j].put(buf, wg_piece((tid >> 3) + 32 * j, tid & 7), YB);
        if (bias) {
          float f[8];
          rg.y[j].get(f);
          bsum[j] += ((f[0] + f[1]) + (f[2] + f[3])) + ((f[4] + f[5]) + (f[6] + f[7]));
        }
      }
#pragma unroll
      for (int j = 0; j < TN / 32; ++j) {
        const float sc = q8_scale(rg.s[j]);
        const unsigned w[2] = {rg.x[j].x, rg.x[j].y};
        float f[8];
        q8_decode_vec<FMT, 8>(w, sc, f);
        *reinterpret_cast<csn_u4*>(bx + wg_piece((tid >> 3) + 32 * j, tid & 7)) =
            wg_u4(wg_hi2(f[0], f[1]), wg_hi2(f[2], f[3]), wg_hi2(f[4], f[5]), wg_hi2(f[6], f[7]));
      }
    } else {
      constexpr int GY = TM / 4, GX = TN / 4;
      if (tid / GY < 8) {
        const int c = 4 * (tid & (GY - 1)), k = tid / GY;
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          float f[8];
#pragma unroll
          for (int j = 0; j < 8; ++j) f[j] = rg.y[j].get(q);
          if (bias) bsum[q] += ((f[0] + f[1]) + (f[2] + f[3])) + ((f[4] + f[5]) + (f[6] + f[7]));
#pragma unroll
          for (int part = 0; part < PARTS; ++part) {
            float h[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) h[j] = PARTS == 1 ? f[j] : wg_cut(f[j]);
            *reinterpret_cast<csn_u4*>(buf + part * YB + wg_piece(c + q, k)) =
                wg_u4(wg_hi2(h[0], h[1]), wg_hi2(h[2], h[3]), wg_hi2(h[4], h[5]), wg_hi2(h[6], h[7]));
          }
        }
      }
      if (tid / GX < 8) {
        const int c = 4 * (tid & (GX - 1)), k = tid / GX;
        float f[8][4];
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const unsigned w[1] = {rg.x[j]};
          q8_decode_vec<FMT, 4>(w, q8_scale(rg.s[j]), f[j]);
        }
#pragma unroll
        for (int q = 0; q < 4; ++q)
          *reinterpret_cast<csn_u4*>(bx + wg_piece(c + q, k)) =
              wg_u4(wg_hi2(f[0][q], f[1][q]), wg_hi2(f[2][q], f[3][q]), wg_hi2(f[4][q], f[5][q]), wg_hi2(f[6][q], f[7][q]));
      }
    }
  };

  csn_f16v acc[MI][NJ];
#pragma unroll
  for (int i = 0; i < MI; ++i)
#pragma unroll
    for (int j = 0; j < NJ; ++j)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.f;

  const int wr = (wave >> 1) * (TM / 2), wc = (wave & 1) * (TN / 2);
  int cur = 0;
  if (s0 < s1) {
    load(s0);
    store(sm);
  }
  for (int s = s0; s < s1; ++s) {
    if (s + 1 < s1) load(s + 1);
    __syncthreads();
    const unsigned char* buf = sm + cur * BUF;
#pragma unroll
    for (int kk = 0; kk < WG_STEP / 16; ++kk) {
      const int c = 2 * kk + (lane >> 5);
      csn_u4 b[NJ];
#pragma unroll
      for (int j = 0; j < NJ; ++j) b[j] = *reinterpret_cast<const csn_u4*>(buf + PARTS * YB + wg_piece(wc + 32 * j + (lane & 31), c));
#pragma unroll
      for (int part = 0; part < PARTS; ++part)
#pragma unroll
        for (int i = 0; i < MI; ++i) {
          const csn_u4 y = *reinterpret_cast<const csn_u4*>(buf + part * YB + wg_piece(wr + 32 * i + (lane & 31), c));
#pragma unroll
          for (int j = 0; j < NJ; ++j) acc[i][j] = csn_mfma_32x32x16_bf16(y, b[j], acc[i][j]);
        }
    }
    cur ^= 1;
    if (s + 1 < s1) store(sm + cur * BUF);
  }

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
  if (bias) {   // the block's sums of dY: eight threads hold a row's
    __syncthreads();
    float* sb = reinterpret_cast<float*>(sm);   // [TM][8]
    if constexpr (!ROWS) {
#pragma unroll
      for (int j = 0; j < TM / 32; ++j) sb[((tid >> 3) + 32 * j) * 8 + (tid & 7)] = bsum[j];
    } else {
      constexpr int GY = TM / 4;
      if (tid / GY < 8)
#pragma unroll
        for (int q = 0; q < 4; ++q) sb[(4 * (tid & (GY - 1)) + q) * 8 + tid / GY] = bsum[q];
    }
    __syncthreads();
    if (tid < TM && o0 + tid < a.cout) {
      float v = 0.f;
#pragma unroll
      for (int j = 0; j < 8; ++j) v += sb[tid * 8 + j];
      (a.slabs > 1 ? out + a.cout * a.cin : a.dbias)[o0 + tid] = v;   // (behind the slab's dW)
    }
  }
}

struct WgPlan { int tm, tn, mtiles, ntiles, steps, steps_per_slab, slabs, chunks; };

// Tiles of 128 where the channels fill more than 64.  About 512 blocks (two per CU), but at least four steps of 64 tokens each: a
// slab costs a partial tile written and read again.
static bool wg_plan(int rows, int64_t outer, int64_t inner, int64_t cin, int64_t cout, WgPlan& p) {
  p.tm = cout > 64 ? 128 : 64;
  p.tn = cin > 64 ? 128 : 64;
  const int64_t mt = (cout + p.tm - 1) / p.tm, nt = (cin + p.tn - 1) / p.tn;
  const int64_t chunks = rows ? 1 : (inner + 7) / 8;
  const int64_t all = rows ? (outer + 7) / 8 : outer * chunks, steps = (all + 7) / 8;
  if (mt * nt > (1 << 20) || all > 0x7ffffff0LL || chunks > 0x7ffffff0LL) return false;
  int64_t slabs = (512 + mt * nt - 1) / (mt * nt);
  slabs = std::min(slabs, (steps + 3) / 4);
  if (slabs < 1) slabs = 1;
  p.mtiles = (int)mt; p.ntiles = (int)nt; p.steps = (int)steps; p.chunks = (int)(chunks < 1 ? 1 : chunks);
  p.steps_per_slab = (int)((steps + slabs - 1) / slabs);
  if (p.steps_per_slab < 1) p.steps_per_slab = 1;
  p.slabs = (int)((steps + p.steps_per_slab - 1) / p.steps_per_slab);
  if (p.slabs < 1) p.slabs = 1;
  return true;
}

int64_t csn_q8_wgrad_partial_floats(int rows, int, int64_t outer, int64_t inner, int64_t cin, int64_t cout) {
  WgPlan p;
  if (!wg_plan(rows, outer, inner, cin, cout, p) || p.slabs <= 1) return 0;
  return (int64_t)p.slabs * (cout * cin + cout);
}

template <typename AT, int FMT, bool ROWS, int TM, int TN>
static int q8_wgrad_run(const Q8WgradArgs& a, void* stream) {
  constexpr int smem = 2 * ((sizeof(AT) == 4 ? 3 : 1) * TM + TN) * WG_ROWB;
#ifndef CSN_CPU_EMU
  static CsnPerDeviceOnce once;
  const int st = once.run([] {
    return (int)hipFuncSetAttribute(reinterpret_cast<const void*>(&q8_wgrad_kernel<AT, FMT, ROWS, TM, TN>),
                                    hipFuncAttributeMaxDynamicSharedMemorySize, smem);
  });
  if (st != 0) return st;
#endif
  const int total = a.mtiles * a.ntiles * a.slabs;
  CSN_LAUNCH((q8_wgrad_kernel<AT, FMT, ROWS, TM, TN>), dim3((unsigned)((total + 7) / 8 * 8)), dim3(CSN_BLOCK), smem, stream, a);
  if (a.slabs > 1) {
    const int e = (int)hipGetLastError();
    if (e != 0) return e;
    SlabSumArgs r;
    r.partial = a.partial; r.out0 = a.dweight; r.out1 = a.dbias; r.n0 = a.cout * a.cin; r.n = r.n0 + a.cout; r.slabs = a.slabs;
    return csn_launch_slab_sum(r, stream);
  }
  return (int)hipGetLastError();
}

template <typename AT, int FMT, bool ROWS>
static int q8_wgrad_tile(const Q8WgradArgs& a, const WgPlan& p, void* stream) {
  if (p.tm == 128) return p.tn == 128 ? q8_wgrad_run<AT, FMT, ROWS, 128, 128>(a, stream) : q8_wgrad_run<AT, FMT, ROWS, 128, 64>(a, stream);
  return p.tn == 128 ? q8_wgrad_run<AT, FMT, ROWS, 64, 128>(a, stream) : q8_wgrad_run<AT, FMT, ROWS, 64, 64>(a, stream);
}

int csn_launch_q8_wgrad(const Q8WgradArgs& a0, int rows, int a16, int fmt, void* stream) {
  Q8WgradArgs a = a0;
  WgPlan p;
  if (!wg_plan(rows, a.outer, a.inner, a.cin, a.cout, p)) return -1;
  a.mtiles = p.mtiles; a.ntiles = p.ntiles; a.steps = p.steps; a.steps_per_slab = p.steps_per_slab; a.slabs = p.slabs; a.chunks = p.chunks;
  const uintptr_t es = a16 ? 2 : 4, py = (uintptr_t)a.dy, px = (uintptr_t)a.codes;
  if (rows) {   // 4 channels of a token at once
    a.vec_y = py % (4 * es) == 0 && a.dy_so % 4 == 0;
    a.vec_x = px % 4 == 0 && a.cin % 4 == 0;
  } else {      // 8 pixels of a channel at once, no plane ending inside them
    a.vec_y = a.inner % 8 == 0 && py % 16 == 0 && a.dy_so % 8 == 0 && a.dy_sc % 8 == 0;
    a.vec_x = a.inner % 8 == 0 && px % 8 == 0;
  }
  if (fmt == Q8_INT8) {
    if (rows) return a16 ? q8_wgrad_tile<csn_bf16, Q8_INT8, true>(a, p, stream) : q8_wgrad_tile<float, Q8_INT8, true>(a, p, stream);
    return a16 ? q8_wgrad_tile<csn_bf16, Q8_INT8, false>(a, p, stream) : q8_wgrad_tile<float, Q8_INT8, false>(a, p, stream);
  }
  if (rows) return a16 ? q8_wgrad_tile<csn_bf16, Q8_E4M3, true>(a, p, stream) : q8_wgrad_tile<float, Q8_E4M3, true>(a, p, stream);
  return a16 ? q8_wgrad_tile<csn_bf16, Q8_E4M3, false>(a, p, stream) : q8_wgrad_tile<float, Q8_E4M3, false>(a, p, stream);
}
#endif  // CSN_EMU_SEQ
