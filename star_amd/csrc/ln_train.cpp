// ln_train.cpp -- launchers of the LayerNorm training passes (ln_train.h)
#include "ops.h"
#include "ln_train.h"

namespace star {

constexpr int LN_TRAIN_MAX_C = 16384;     // one workgroup per row, eight chunks of eight columns per thread

// How a row is spread: lpr lanes with cpl chunks of eight columns each; lpr 0: a workgroup per row.  Backward: the first of 1, 2, 3, 5 chunks that
// keeps three quarters of the lanes busy -- few chunks per lane hold few registers, and more waves hide the loads (640 columns: 3 instead of
// 5, 251 -> 211 us for 214272 rows).  Forward: the one that leaves the fewest lanes idle (320 columns: 5 instead of 3, 214 -> 201 us for 843264 rows).
struct LnShape { int lpr, cpl; };
static LnShape ln_shape(int C, bool vec, bool backward) {
  const int chunks = (C + 7) / 8;
  if (chunks > 64 * 5) return LnShape{0, chunks <= 256 * 3 ? 3 : 8};
  int least = 1;
  while (least < 8 && least < chunks) least <<= 1;
  auto lanes = [&](int cpl) { int l = least; while (l * cpl < chunks) l <<= 1; return l; };
  LnShape best{lanes(5), 5};
  if (vec)
    for (int cpl : {3, 2, 1}) {
      const int l = lanes(cpl);
      if (l > 64) break;
      if (backward ? 4 * chunks >= 3 * l * cpl : l * cpl <= best.lpr * best.cpl) best = LnShape{l, cpl};
    }
  return best;
}

// workgroups of the backward pass: at most four per compute unit, each writes one partial row of 2 C sums
static int ln_bwd_blocks(Ctx* ctx, int rows, int lpr) {
  const long long rpb = lpr ? 4 * (64 / lpr) : 1;
  const long long steps = (rows + rpb - 1) / rpb;
  const long long most = 4LL * ctx->num_cus;
  return (int)(steps < most ? steps : most);
}

// (the least rows per workgroup over both forms of access, so that the answer does not depend on the pointers)
size_t ln_train_bwd_workspace(Ctx* ctx, int rows, int C) {
  if (rows <= 0 || C <= 0 || C > LN_TRAIN_MAX_C) return 0;
  const int a = ln_bwd_blocks(ctx, rows, ln_shape(C, true, true).lpr), b = ln_bwd_blocks(ctx, rows, ln_shape(C, false, true).lpr);
  return (size_t)(a > b ? a : b) * 2 * C * sizeof(float);
}

static bool al16(const void* p) { return ((uintptr_t)p & 15) == 0; }

template <class T, bool VEC, int CPL, bool WG>
static void ln_fwd_go(Ctx* ctx, const LnTrainParams& p) {
  const long long rpb = WG ? 1 : 4 * (64 / p.lpr);
  STAR_LAUNCH((ln_train_fwd_kernel<T, VEC, CPL, WG>), dim3((unsigned)((p.rows + rpb - 1) / rpb)), dim3(256), (size_t)(WG ? 64 : 0), ctx->stream, p);
}
template <class T, bool VEC, int CPL, bool WG>
static void ln_bwd_go(Ctx* ctx, const LnTrainParams& p, int blocks) {
  const size_t smem = WG ? 64 : (size_t)(4 * 2 * p.lpr * 8 * 4);
  STAR_LAUNCH((ln_train_bwd_kernel<T, VEC, CPL, WG>), dim3((unsigned)blocks), dim3(256), smem, ctx->stream, p);
}
// blocks < 0: the forward pass
template <class T, bool VEC>
static void ln_go(Ctx* ctx, const LnTrainParams& p, int cpl, int blocks) {
  const bool f = blocks < 0;
  if (!p.lpr) {
    if (cpl == 3) f ? ln_fwd_go<T, VEC, 3, true>(ctx, p) : ln_bwd_go<T, VEC, 3, true>(ctx, p, blocks);
    else f ? ln_fwd_go<T, VEC, 8, true>(ctx, p) : ln_bwd_go<T, VEC, 8, true>(ctx, p, blocks);
    return;
  }
  if constexpr (VEC) {
    if (cpl == 1) return f ? ln_fwd_go<T, VEC, 1, false>(ctx, p) : ln_bwd_go<T, VEC, 1, false>(ctx, p, blocks);
    if (cpl == 2) return f ? ln_fwd_go<T, VEC, 2, false>(ctx, p) : ln_bwd_go<T, VEC, 2, false>(ctx, p, blocks);
    if (cpl == 3) return f ? ln_fwd_go<T, VEC, 3, false>(ctx, p) : ln_bwd_go<T, VEC, 3, false>(ctx, p, blocks);
  }
  f ? ln_fwd_go<T, VEC, 5, false>(ctx, p) : ln_bwd_go<T, VEC, 5, false>(ctx, p, blocks);
}

// an output past half of the 256 MB memory-side cache is not there any more when its reader comes: stores that do not allocate on the way
// (843264 x 320 forward 201 -> 195 us); a smaller one stays cached for it
static int ln_streams(int rows, int C) { return (long long)rows * C * 2 > (128LL << 20); }

static int ln_check(Ctx* ctx, const char* who, int rows, int C) {
  if (rows < 0) return ctx->fail(std::string(who) + ": negative row count");
  if (C < 1 || C > LN_TRAIN_MAX_C) return ctx->fail(std::string(who) + ": C must be 1 .. 16384");
  return 0;
}

int op_layer_norm_train(Ctx* ctx, const void* x, long long ldx, void* y, long long ldy, const float* gamma, const float* beta, float* stats,
                        int rows, int C, float eps) {
  if (ln_check(ctx, "layer_norm_train", rows, C)) return 1;
  if (rows == 0) return 0;
  if (!x || !y) return ctx->fail("layer_norm_train: null tensor");
  if (ldx < C || ldy < C) return ctx->fail("layer_norm_train: row strides must be at least C");
  if (y == x && rows > 1 && ldy != ldx) return ctx->fail("layer_norm_train: y over x needs x's row stride");
  ProfScope ps(ctx, PK_LN, 0.0, 4.0 * rows * (double)C);
  const bool v = !((C | ldx | ldy) & 7) && al16(x) && al16(y) && al16(gamma) && al16(beta);
  const LnShape sh = ln_shape(C, v, false);
  const long long rpb = sh.lpr ? 4 * (64 / sh.lpr) : 1;   // (a launch counts its threads in 32 bits)
  if ((rows + rpb - 1) / rpb * 256 > 0xffffffffLL) return ctx->fail("layer_norm_train: too many rows for this width");
  LnTrainParams p{x, nullptr, y, gamma, beta, stats, nullptr, ldx, 0, ldy, rows, C, sh.lpr, ln_streams(rows, C), eps};
  if (ctx->dtype == DT_F16) v ? ln_go<f16, true>(ctx, p, sh.cpl, -1) : ln_go<f16, false>(ctx, p, sh.cpl, -1);
  else v ? ln_go<bf16, true>(ctx, p, sh.cpl, -1) : ln_go<bf16, false>(ctx, p, sh.cpl, -1);
  return 0;
}

int op_layer_norm_bwd(Ctx* ctx, const void* dy, long long lddy, const void* x, long long ldx, const float* stats, const float* gamma, void* dx,
                      long long lddx, float* dgamma, float* dbeta, int rows, int C, void* workspace, size_t workspace_bytes) {
  if (ln_check(ctx, "layer_norm_bwd", rows, C)) return 1;
  const bool sums = dgamma || dbeta;
  int blocks = 0;
  if (rows > 0) {
    if (!dy || !x || !dx || !stats) return ctx->fail("layer_norm_bwd: null tensor");
    if (ldx < C || lddy < C || lddx < C) return ctx->fail("layer_norm_bwd: row strides must be at least C");
    if (rows > 1 && ((dx == x && lddx != ldx) || (dx == dy && lddx != lddy))) return ctx->fail("layer_norm_bwd: dx over x or dy needs its row stride");
    const bool v = !((C | ldx | lddy | lddx) & 7) && al16(x) && al16(dy) && al16(dx) && al16(gamma);
    const LnShape sh = ln_shape(C, v, true);
    blocks = ln_bwd_blocks(ctx, rows, sh.lpr);
    if (sums && (!workspace || workspace_bytes < (size_t)blocks * 2 * C * sizeof(float) || !al16(workspace)))
      return ctx->fail("layer_norm_bwd: workspace missing, too small (star_layer_norm_bwd_workspace) or not 16-byte aligned");
    ProfScope ps(ctx, PK_LN, 0.0, 6.0 * rows * (double)C);
    LnTrainParams p{x, dy, dx, gamma, nullptr, const_cast<float*>(stats), sums ? (float*)workspace : nullptr, ldx, lddy, lddx, rows, C, sh.lpr, ln_streams(rows, C), 0.f};
    if (ctx->dtype == DT_F16) v ? ln_go<f16, true>(ctx, p, sh.cpl, blocks) : ln_go<f16, false>(ctx, p, sh.cpl, blocks);
    else v ? ln_go<bf16, true>(ctx, p, sh.cpl, blocks) : ln_go<bf16, false>(ctx, p, sh.cpl, blocks);
  }
  if (sums) {
    ProfScope ps(ctx, PK_LN, 0.0, 8.0 * blocks * (double)C);
    LnReduceParams r{(const float*)workspace, dgamma, dbeta, C, blocks};
    STAR_LAUNCH(ln_train_reduce_kernel, dim3((unsigned)((2 * C + 15) / 16)), dim3(256), (size_t)(16 * 16 * 4), ctx->stream, r);
  }
  return 0;
}

}  // namespace star
