// train_ops.h -- argument blocks and launchers of the training operators beside the plan (k_q8.hip, k_norm.hip, k_q8_wgrad.hip).
// Launchers return a hipError_t (0 = fine) or a negative number where no kernel takes the arguments.
#pragma once
#include <stdint.h>
#include <stddef.h>

#include <algorithm>

struct Q8PackArgs {
  const void* x;
  uint8_t* codes;
  uint8_t* exps;
  int64_t outer, rows, cols, so, sr;   // element (o, r, c) at o * so + r * sr + c
  int64_t nblk;                        // blocks of a row
  int64_t nrows, per_row, items;       // (set by the launcher) rows, pieces of a row, pieces
};
struct Q8UnpackArgs {
  const uint8_t* codes;
  const uint8_t* exps;
  void* y;
  int64_t rows, cols, nblk;
  int64_t per_row, items;              // (set by the launcher)
};
int csn_launch_q8_pack(const Q8PackArgs& a, int a16, int fmt, void* stream);
int csn_launch_q8_unpack(const Q8UnpackArgs& a, int a16, int fmt, void* stream);

// one tensor among many (dense rows): x <-> codes, exps
struct Q8Seg {
  void* x;
  uint8_t* codes;
  uint8_t* exps;
  int64_t rows, cols;
  int64_t per_row, items;   // (set by the launcher)
  int32_t block0, pad;
};
#define Q8_MAX_SEGS 48      // of a launch: they travel in its arguments
struct Q8SegArgs { Q8Seg seg[Q8_MAX_SEGS]; int32_t n, pad; };
int csn_launch_q8_segments(Q8Seg* seg, int n, bool pack, int a16, int fmt, void* stream);
struct CopySeg { const uint32_t* src; uint32_t* dst; int64_t words; int32_t block0, pad; };
struct CopySegArgs { CopySeg seg[Q8_MAX_SEGS]; int32_t n, pad; };
int csn_launch_copy_segments(CopySeg* seg, int n, void* stream);

struct NormArgs {
  const void* x;            // null: the checkpoint below is the input (backward)
  const void* dy;
  const uint8_t* codes_in;
  const uint8_t* exps_in;
  void* y;                  // forward: y, backward: dx
  uint8_t* codes;           // forward: checkpoint of x (or null)
  uint8_t* exps;
  const float* weight;
  const float* bias;
  float* mean;
  float* rstd;
  float* dweight;
  float* dbias;
  float* partial;           // backward: [slabs][2][channels]
  int64_t outer, C, inner;
  int64_t x_so, x_sc, dy_so, dy_sc;
  int64_t nblk;             // checkpoint blocks of a plane / row
  float eps;
  // set by the launcher
  int32_t slabs;            // blocks of the register forms
  int32_t tiles, items;     // planar: pixel tiles of an image, (image, tile) items
  int32_t runs;             // planar: items by XCD
};
int csn_launch_norm_fwd(const NormArgs& a, int rows, int a16, int fmt, void* stream);
int csn_launch_norm_bwd(const NormArgs& a, int rows, int a16, int fmt, void* stream);
int64_t csn_norm_partial_floats(int rows, int a16, int64_t outer, int64_t C, int64_t inner);

struct Q8WgradArgs {
  const void* dy;
  const uint8_t* codes;
  const uint8_t* exps;
  float* dweight;
  float* dbias;
  float* partial;           // [slabs][cout * cin + cout]
  int64_t outer, inner, cin, cout;
  int64_t dy_so, dy_sc;
  int64_t nblk;             // checkpoint blocks of a plane / row
  // set by the launcher
  int32_t mtiles, ntiles, slabs, steps_per_slab, chunks;   // chunks: 8-pixel pieces of a plane
};
int csn_launch_q8_wgrad(const Q8WgradArgs& a, int rows, int a16, int fmt, void* stream);
int64_t csn_q8_wgrad_partial_floats(int rows, int a16, int64_t outer, int64_t inner, int64_t cin, int64_t cout);
