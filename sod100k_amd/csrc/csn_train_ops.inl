// csn_train_ops.inl -- C entry points of the training operators beside the plan (include/csnet_hip.h): argument checks, workspaces.
// Included by csn_plan.hip.

#ifdef CSN_CPU_EMU
// The emulator may be built from the plan's units alone: the launchers of k_q8.hip, k_norm.hip and k_q8_wgrad.hip are then null and the entry
// points below refuse every call.  (The product library names them firmly: a missing unit does not load.)
#define WEAK_LAUNCHER(f) extern decltype(f) f __attribute__((weak))
WEAK_LAUNCHER(csn_launch_q8_pack); WEAK_LAUNCHER(csn_launch_q8_unpack); WEAK_LAUNCHER(csn_launch_q8_segments); WEAK_LAUNCHER(csn_launch_copy_segments);
WEAK_LAUNCHER(csn_launch_norm_fwd); WEAK_LAUNCHER(csn_launch_norm_bwd); WEAK_LAUNCHER(csn_norm_partial_floats);
WEAK_LAUNCHER(csn_launch_q8_wgrad); WEAK_LAUNCHER(csn_q8_wgrad_partial_floats);
#undef WEAK_LAUNCHER
#endif

namespace {

#ifdef CSN_CPU_EMU
inline bool train_ops_linked() { return csn_launch_q8_pack && csn_launch_norm_fwd && csn_launch_q8_wgrad; }
#else
inline bool train_ops_linked() { return true; }
#endif
#define REFUSE(why) do { g_hip_err = (why); return CSN_E_INVALID; } while (0)
#define REFUSE_UNLINKED() do { if (!train_ops_linked()) { g_hip_err = "built without the training operators' kernels"; return CSN_E_UNSUPPORTED; } } while (0)

// element counts and byte offsets of all tensors stay far inside 63 bits, block counts inside a grid
const int64_t kMaxElems = (int64_t)1 << 46;
const int64_t kMaxChannels = (int64_t)1 << 24;

inline bool mul_ok(int64_t a, int64_t b) { return a == 0 || b <= kMaxElems / a; }
inline bool aligned(const void* p, int dtype) { return ((uintptr_t)p & (dtype == CSN_BF16 ? 1u : 3u)) == 0; }
inline bool aligned4(const void* p) { return ((uintptr_t)p & 3u) == 0; }
inline int64_t q8_blocks(int64_t cols) { return (cols + CSN_Q8_BLOCK - 1) / CSN_Q8_BLOCK; }
inline bool dtype_ok(int32_t t) { return t == CSN_F32 || t == CSN_BF16; }
inline bool format_ok(int32_t f) { return f == CSN_Q8_INT8 || f == CSN_Q8_E4M3; }
inline bool layout_ok(int32_t l) { return l == CSN_LAYOUT_PLANAR || l == CSN_LAYOUT_ROWS; }
inline bool stride_ok(int64_t s, int64_t n) { return s >= 0 && mul_ok(n, s); }

int norm_check(const csn_norm_desc* d) {
  REFUSE_UNLINKED();
  if (!d) REFUSE("layer norm: null descriptor");
  if (!layout_ok(d->layout) || !dtype_ok(d->dtype)) REFUSE("layer norm: unknown layout or dtype");
  if (d->outer < 0 || d->inner < 0 || d->channels < 1 || d->channels > kMaxChannels)
    REFUSE("layer norm: negative sizes, no channels or more than 2^24");
  if (d->layout == CSN_LAYOUT_ROWS && d->inner != 1) REFUSE("layer norm: rows have inner = 1");
  if (!mul_ok(d->outer, d->inner) || !mul_ok(d->outer * d->inner, d->channels)) REFUSE("layer norm: too many elements");
  if (!(d->eps > 0.f) || !std::isfinite(d->eps)) REFUSE("layer norm: eps must be positive and finite");
  return CSN_OK;
}
int product_check(const csn_product_desc* d) {
  REFUSE_UNLINKED();
  if (!d) REFUSE("product gradient: null descriptor");
  if (!layout_ok(d->layout) || !dtype_ok(d->dtype) || !format_ok(d->format)) REFUSE("product gradient: unknown layout, dtype or format");
  if (d->outer < 0 || d->inner < 0 || d->cin < 1 || d->cout < 1 || d->cin > kMaxChannels || d->cout > kMaxChannels || d->cin * d->cout > ((int64_t)1 << 40))
    REFUSE("product gradient: negative sizes, no channels or too many");
  if (d->layout == CSN_LAYOUT_ROWS && d->inner != 1) REFUSE("product gradient: rows have inner = 1");
  if (!mul_ok(d->outer, d->inner) || !mul_ok(d->outer * d->inner, d->cin) || !mul_ok(d->outer * d->inner, d->cout))
    REFUSE("product gradient: too many elements");
  return CSN_OK;
}
size_t norm_ws(const csn_norm_desc* d) {
  return (size_t)csn_norm_partial_floats(d->layout == CSN_LAYOUT_ROWS, d->dtype == CSN_BF16, d->outer, d->channels, d->inner) * sizeof(float);
}
size_t product_ws(const csn_product_desc* d) {
  return (size_t)csn_q8_wgrad_partial_floats(d->layout == CSN_LAYOUT_ROWS, d->dtype == CSN_BF16, d->outer, d->inner, d->cin, d->cout) *
         sizeof(float);
}

// What csn_backward reads of a train-mode forward, in a fixed order: q(tensor in the workspace, planes, pixels) for activation-typed
// tensors -- the stored activations, the raw convolution outputs, pooled inputs -- and r(pointer, bytes) for the rest: the per-image |GAP|
// tables of the penalty, the bfloat16 copy of the images and the plan's packed tables, whose BatchNorm scale / shift / mean / invstd
// are the batch's.  (The other workspace regions are scratch of one pass.)
template <class Q, class R>
void plan_saved(const csn_plan* P, Q&& q, R&& r) {
  auto act = [&](int64_t off, int C, int lvl) {
    if (off >= 0 && C > 0) q(off, (int64_t)P->S * C, (int64_t)(P->H >> lvl) * (P->W >> lvl));
  };
  for (int i = 1; i < (int)P->acts.size(); ++i) {
    if (P->virt_cons[i] < 0) act(P->acts[i].ws_off, P->acts[i].channels, P->acts[i].lvl);
    act(P->tz_off[i], P->acts[i].channels, P->acts[i].lvl);
  }
  for (const UnitPlan& u : P->units)
    for (int i = 0; i < CSN_MAX_BRANCH; ++i) {
      act(u.pooled_off[i], u.d.cin[i], u.base_lvl + i);
      act(u.mp_off[i], u.d.cin[i], u.base_lvl + i + 1);
      if (u.gap_off[i] >= 0) r(u.gap_off[i], (int64_t)u.d.cout[i] * P->S * (int64_t)sizeof(float));
    }
  if (P->act16) r(P->x16_off, (int64_t)P->S * P->acts[0].channels * P->H * P->W * 2);
  r((int64_t)-1, P->packed_floats * (int64_t)sizeof(float));   // (-1: the packed tables, not a workspace region)
}
int64_t plan_saved_bytes(const csn_plan* P) {
  int64_t n = 0;
  plan_saved(P, [&](int64_t, int64_t rows, int64_t cols) { n += align_up(rows * cols, 256) + align_up(rows * q8_blocks(cols), 256); },
             [&](int64_t, int64_t bytes) { n += align_up(bytes, 256); });
  return n;
}
int plan_saved_move(csn_plan* P, char* ws, char* ck, int format, bool pack, void* stream) try {
  std::vector<Q8Seg> qs;
  std::vector<CopySeg> cs;
  int64_t at = 0;
  plan_saved(P,
             [&](int64_t off, int64_t rows, int64_t cols) {
               Q8Seg g{};
               g.x = ws + off; g.rows = rows; g.cols = cols;
               g.codes = reinterpret_cast<uint8_t*>(ck + at); at += align_up(rows * cols, 256);
               g.exps = reinterpret_cast<uint8_t*>(ck + at); at += align_up(rows * q8_blocks(cols), 256);
               qs.push_back(g);
             },
             [&](int64_t off, int64_t bytes) {
               CopySeg g{};
               uint32_t* t = off >= 0 ? reinterpret_cast<uint32_t*>(ws + off) : reinterpret_cast<uint32_t*>(P->packed);
               uint32_t* c = reinterpret_cast<uint32_t*>(ck + at);
               g.src = pack ? t : c; g.dst = pack ? c : t; g.words = bytes / 4; at += align_up(bytes, 256);
               cs.push_back(g);
             });
  LAUNCH_TRY(csn_launch_q8_segments(qs.data(), (int)qs.size(), pack, P->act16 ? 1 : 0, format, stream));
  LAUNCH_TRY(csn_launch_copy_segments(cs.data(), (int)cs.size(), stream));
  return CSN_OK;
} catch (const std::bad_alloc&) {
  REFUSE("plan checkpoint: out of host memory");
}

}  // namespace

extern "C" {

size_t csn_plan_checkpoint_bytes(const csn_plan* P) { return P && P->train ? (size_t)plan_saved_bytes(P) : 0; }

int csn_plan_checkpoint_save(csn_plan* P, const void* workspace, int32_t format, void* checkpoint, size_t checkpoint_bytes, void* stream) {
  REFUSE_UNLINKED();
  if (!P || !workspace || !checkpoint || ((uintptr_t)checkpoint & 255u) || !format_ok(format)) REFUSE("plan checkpoint: null or misaligned (256 bytes) buffer, unknown format");
  if (!P->train || !P->bn_tables_train) { g_hip_err = "plan checkpoint: no train-mode forward of a training plan to save"; return CSN_E_STATE; }
  if (checkpoint_bytes < (size_t)plan_saved_bytes(P)) REFUSE("plan checkpoint: buffer smaller than csn_plan_checkpoint_bytes");
  return plan_saved_move(P, static_cast<char*>(const_cast<void*>(workspace)), static_cast<char*>(checkpoint), format, true, stream);
}

int csn_plan_checkpoint_restore(csn_plan* P, void* workspace, int32_t format, const void* checkpoint, size_t checkpoint_bytes, void* stream) {
  REFUSE_UNLINKED();
  if (!P || !workspace || !checkpoint || ((uintptr_t)checkpoint & 255u) || !format_ok(format)) REFUSE("plan checkpoint: null or misaligned (256 bytes) buffer, unknown format");
  if (!P->train || !P->trained) { g_hip_err = "plan checkpoint: a training plan that has run a forward is needed"; return CSN_E_STATE; }
  if (checkpoint_bytes < (size_t)plan_saved_bytes(P)) REFUSE("plan checkpoint: buffer smaller than csn_plan_checkpoint_bytes");
  P->bn_tables_train = true;   // (the packed tables are among what comes back, whatever refreshed them since)
  return plan_saved_move(P, static_cast<char*>(workspace), static_cast<char*>(const_cast<void*>(checkpoint)), format, false, stream);
}

int csn_q8_pack(const void* x, int32_t dtype, int64_t outer, int64_t rows, int64_t cols, int64_t outer_stride, int64_t row_stride,
                int32_t format, uint8_t* codes, uint8_t* exponents, void* stream) {
  REFUSE_UNLINKED();
  if (!dtype_ok(dtype) || !format_ok(format)) REFUSE("q8 pack: unknown dtype or format");
  if (outer < 0 || rows < 0 || cols < 0 || !mul_ok(outer, rows) || !mul_ok(outer * rows, cols)) REFUSE("q8 pack: negative or too large sizes");
  if (!stride_ok(outer_stride, outer) || !stride_ok(row_stride, rows)) REFUSE("q8 pack: negative or too large strides");
  if (outer == 0 || rows == 0 || cols == 0) return CSN_OK;
  if (!x || !codes || !exponents || !aligned(x, dtype)) REFUSE("q8 pack: null or misaligned tensor");
  Q8PackArgs a;
  a.x = x; a.codes = codes; a.exps = exponents; a.outer = outer; a.rows = rows; a.cols = cols;
  a.so = outer_stride; a.sr = row_stride; a.nblk = q8_blocks(cols);
  LAUNCH_TRY(csn_launch_q8_pack(a, dtype == CSN_BF16, format, stream));
  return CSN_OK;
}

int csn_q8_unpack(const uint8_t* codes, const uint8_t* exponents, int32_t format, int64_t rows, int64_t cols, void* y, int32_t dtype,
                  void* stream) {
  REFUSE_UNLINKED();
  if (!dtype_ok(dtype) || !format_ok(format)) REFUSE("q8 unpack: unknown dtype or format");
  if (rows < 0 || cols < 0 || !mul_ok(rows, cols)) REFUSE("q8 unpack: negative or too large sizes");
  if (rows == 0 || cols == 0) return CSN_OK;
  if (!y || !codes || !exponents || !aligned(y, dtype)) REFUSE("q8 unpack: null or misaligned tensor");
  Q8UnpackArgs a;
  a.codes = codes; a.exps = exponents; a.y = y; a.rows = rows; a.cols = cols; a.nblk = q8_blocks(cols);
  LAUNCH_TRY(csn_launch_q8_unpack(a, dtype == CSN_BF16, format, stream));
  return CSN_OK;
}

int csn_layer_norm_forward(const csn_norm_desc* d, const void* x, int64_t x_outer_stride, int64_t x_channel_stride,
                           const float* weight, const float* bias, void* y, float* mean, float* rstd, uint8_t* codes,
                           uint8_t* exponents, void* stream) {
  const int st = norm_check(d);
  if (st != CSN_OK) return st;
  const bool rows = d->layout == CSN_LAYOUT_ROWS;
  if (!stride_ok(x_outer_stride, d->outer) || (!rows && !stride_ok(x_channel_stride, d->channels))) REFUSE("layer norm: negative or too large strides");
  if (!codes != !exponents) REFUSE("layer norm: codes without exponents or exponents without codes");
  if (codes && !format_ok(d->format)) REFUSE("layer norm: unknown checkpoint format");
  if (d->outer * d->inner == 0) return CSN_OK;
  if (!x || !y || !aligned(x, d->dtype) || !aligned(y, d->dtype)) REFUSE("layer norm: null or misaligned tensor");
  if (!aligned4(weight) || !aligned4(bias) || !aligned4(mean) || !aligned4(rstd)) REFUSE("layer norm: misaligned parameters");
  NormArgs a{};
  a.x = x; a.y = y; a.codes = codes; a.exps = exponents; a.weight = weight; a.bias = bias; a.mean = mean; a.rstd = rstd;
  a.outer = d->outer; a.C = d->channels; a.inner = d->inner; a.x_so = x_outer_stride; a.x_sc = rows ? 0 : x_channel_stride;
  a.nblk = q8_blocks(rows ? d->channels : d->inner); a.eps = d->eps;
  LAUNCH_TRY(csn_launch_norm_fwd(a, rows, d->dtype == CSN_BF16, codes ? d->format : 0, stream));
  return CSN_OK;
}

size_t csn_layer_norm_workspace_bytes(const csn_norm_desc* d) { return norm_check(d) == CSN_OK ? norm_ws(d) : 0; }

int csn_layer_norm_backward(const csn_norm_desc* d, const void* dy, int64_t dy_outer_stride, int64_t dy_channel_stride,
                            const void* x, int64_t x_outer_stride, int64_t x_channel_stride, const uint8_t* codes,
                            const uint8_t* exponents, const float* mean, const float* rstd, const float* weight, void* dx,
                            float* dweight, float* dbias, void* workspace, size_t workspace_bytes, void* stream) {
  const int st = norm_check(d);
  if (st != CSN_OK) return st;
  const bool rows = d->layout == CSN_LAYOUT_ROWS, empty = d->outer * d->inner == 0;
  if (!stride_ok(dy_outer_stride, d->outer) || (!rows && !stride_ok(dy_channel_stride, d->channels)))
    REFUSE("layer norm: negative or too large strides");
  if (!stride_ok(x_outer_stride, d->outer) || (!rows && !stride_ok(x_channel_stride, d->channels)))
    REFUSE("layer norm: negative or too large strides");
  if (!codes != !exponents || (x && codes)) REFUSE("layer norm: the input is x or a checkpoint (codes and exponents), not both");
  if (codes && !format_ok(d->format)) REFUSE("layer norm: unknown checkpoint format");
  if (!empty) {
    if (!dy || !dx || !mean || !rstd || (!x && !codes)) REFUSE("layer norm: null tensor");
    if (!aligned(dy, d->dtype) || !aligned(dx, d->dtype) || !aligned(x, d->dtype) || !aligned4(mean) || !aligned4(rstd) || !aligned4(weight))
      REFUSE("layer norm: misaligned tensor");
  }
  if (!aligned4(dweight) || !aligned4(dbias)) REFUSE("layer norm: misaligned tensor");
  if ((dweight || dbias) && norm_ws(d) > 0 && (!workspace || !aligned4(workspace) || workspace_bytes < norm_ws(d)))
    REFUSE("layer norm: workspace missing, misaligned or smaller than csn_layer_norm_workspace_bytes");
  NormArgs a{};
  a.x = x; a.dy = dy; a.codes_in = codes; a.exps_in = exponents; a.y = dx; a.weight = weight;
  a.mean = const_cast<float*>(mean); a.rstd = const_cast<float*>(rstd); a.dweight = dweight; a.dbias = dbias;
  a.partial = static_cast<float*>(workspace);
  a.outer = d->outer; a.C = d->channels; a.inner = d->inner;
  a.x_so = x_outer_stride; a.x_sc = rows ? 0 : x_channel_stride; a.dy_so = dy_outer_stride; a.dy_sc = rows ? 0 : dy_channel_stride;
  a.nblk = q8_blocks(rows ? d->channels : d->inner); a.eps = d->eps;
  LAUNCH_TRY(csn_launch_norm_bwd(a, rows, d->dtype == CSN_BF16, codes ? d->format : 0, stream));
  return CSN_OK;
}

size_t csn_product_weight_grad_workspace_bytes(const csn_product_desc* d) { return product_check(d) == CSN_OK ? product_ws(d) : 0; }

int csn_product_weight_grad(const csn_product_desc* d, const void* dy, int64_t dy_outer_stride, int64_t dy_channel_stride,
                            const uint8_t* codes, const uint8_t* exponents, float* dweight, float* dbias, void* workspace,
                            size_t workspace_bytes, void* stream) {
  const int st = product_check(d);
  if (st != CSN_OK) return st;
  const bool rows = d->layout == CSN_LAYOUT_ROWS, empty = d->outer * d->inner == 0;
  if (!stride_ok(dy_outer_stride, d->outer) || (!rows && !stride_ok(dy_channel_stride, d->cout)))
    REFUSE("product gradient: negative or too large strides");
  if (!dweight || !aligned4(dweight) || !aligned4(dbias)) REFUSE("product gradient: null or misaligned gradient");
  if (!empty && (!dy || !codes || !exponents || !aligned(dy, d->dtype))) REFUSE("product gradient: null or misaligned tensor");
  if (product_ws(d) > 0 && (!workspace || !aligned4(workspace) || workspace_bytes < product_ws(d)))
    REFUSE("product gradient: workspace missing, misaligned or smaller than csn_product_weight_grad_workspace_bytes");
  Q8WgradArgs a{};
  a.dy = dy; a.codes = codes; a.exps = exponents; a.dweight = dweight; a.dbias = dbias; a.partial = static_cast<float*>(workspace);
  a.outer = d->outer; a.inner = d->inner; a.cin = d->cin; a.cout = d->cout;
  a.dy_so = dy_outer_stride; a.dy_sc = rows ? 0 : dy_channel_stride; a.nblk = q8_blocks(rows ? d->cin : d->inner);
  LAUNCH_TRY(csn_launch_q8_wgrad(a, rows, d->dtype == CSN_BF16, d->format, stream));
  return CSN_OK;
}

}  // extern "C"
