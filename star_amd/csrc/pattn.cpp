// pattn.cpp -- launchers of the position-dependent attention (pattn.h, pattn_bwd.h)
#include "ops.h"
#include "pattn.h"
#include "pattn_bwd.h"

namespace star {

constexpr int PA_MAX_N = 1 << 28;         // queries and keys of a sequence
constexpr int PA_MAX_LD = 1 << 23;        // elements: a tile's rows stay within 31 bits of bytes
constexpr int PA_MAX_R = 1024;            // reach of the bias: its table and the sums by relative position live in LDS
constexpr int PA_MAX_BUCKETS = 4096;      // a row block's sums by bucket go through the workspace
constexpr int PA_NOLIM = 1 << 30;

static bool al16(const void* p) { return ((uintptr_t)p & 15) == 0; }

// Rows that see at most this many keys: P and dS with what their rounding left (COMP), so that an output is off by its own rounding alone; above,
// by 1.38 - 1.46 times that at every length.  What it costs, f16, 16 heads, all keys visible, us without / with: 16 x 128 tokens forward 15.2 / 15.1,
// backward 34.6 / 33.0; 16 x 226 16.1 / 16.8, 46 / 54; 8 x 512 19.3 / 22.8, 69 / 85; 8 x 768 32.6 / 48, 142 / 179; 4 x 1024 30 / 37, 113 / 140;
// 1 x 4096 94 / 124, 378 / 488: a few us while a call is mostly latency, a quarter to a half of the call from there on
constexpr int PA_COMP_SPAN = 512;

struct PPlan { int gp, rows, units, qb, nw, nq, nblk, nsplit, per, comp; };
// the dK / dV pass: units (sequence, K / V head), key blocks, how many of them hold first tokens, in how many parts each kind, slots per unit
struct PKPlan { int units, nblk, sblk, split_s, split_n, slots; size_t part_slots; };

// Which form, and how many splits of the key tiles.  Up to 32 rows (a token's heads of one group, a few tokens): one wave per workgroup, and
// about ten workgroups per compute unit, at least four tiles each (LDS holds five at a time; with a bias's table four, from a reach of 900 three, which
// the count does not ask for).  More rows: 256-row workgroups where they give every
// compute unit its two, else 128-row ones, split along the keys while fewer than half of the places are taken.
static PPlan pa_plan(Ctx* ctx, const PAttnArgs& a, bool backward) {
  PPlan q{};
  const int G = a.heads / a.kv_heads;
  q.gp = a.table ? 1 : G;
  q.rows = q.gp * a.Nq;
  q.units = a.batch * (a.heads / q.gp);
  const long long cus = ctx->num_cus;
  q.nsplit = 1;
  const long long left = a.left < 0 ? PA_NOLIM : a.left, right = a.right < 0 ? PA_NOLIM : a.right;
  const long long seen = left + right + 1 + a.sinks < a.Nk ? left + right + 1 + a.sinks : a.Nk;
  q.comp = seen <= PA_COMP_SPAN;
  if (!backward && q.rows <= 32) { q.nw = 1; q.nq = 1; }
  else {
    q.nw = 4;
    q.nq = !backward && !q.comp && (long long)q.units * ((q.rows + 255) / 256) >= 2 * cus ? 2 : 1;
  }
  q.qb = 32 * q.nq * q.nw;
  q.nblk = (q.rows + q.qb - 1) / q.qb;
  if (!backward) {
    // the most tiles a block of rows sees: its window, wherever it begins in a tile, and the first tokens
    const long long all = (a.Nk + 63LL) / 64;
    long long tiles = (left + right + 2 + q.qb / q.gp + 63) / 64 + 1 + (a.sinks + 63LL) / 64;
    if (tiles > all) tiles = all;
    const long long base = (long long)q.units * q.nblk, places = (q.nw == 1 ? 5 : 2) * cus;
    // tiles per split: the same for all, so that sequences of different lengths make different counts of equal shares; about two workgroups
    // per place, which evens out what one to the place leaves (one frame of 1350 tokens against a cache: 117 -> 103 us; a token of 32 sequences: 65 -> 61 us in the kernels, 68 with the call)
    long long per = base > 0 ? (tiles * base + places - 1) / places : tiles;
    per = (per + 1) / 2;
    if (per < 4) per = 4;
    if (per < (tiles + 127) / 128) per = (tiles + 127) / 128;
    long long s = tiles > 0 ? (tiles + per - 1) / per : 1;
    if (q.nw != 1 && 2 * base > places) s = 1;
    if (s < 1) s = 1;
    q.nsplit = (int)s;
    q.per = s == 1 ? 0x3fffffff : (int)per;
  }
  return q;
}

// Key blocks of 128.  A block's row tiles are bounded by the window; those of the first tokens are seen by every row.  Parts of at least eight
// tiles, and no more of them than there are places (two workgroups per compute unit): a second round of few would wait for one workgroup.
static PKPlan pa_kplan(Ctx* ctx, const PAttnArgs& a, const PPlan& q) {
  PKPlan k{};
  const bool shared = a.batch > 1 && a.bsk == 0 && a.bsv == 0;
  k.units = (shared ? 1 : a.batch) * a.kv_heads;
  k.nblk = (a.Nk + 127) / 128;
  const long long loops = (long long)(shared ? a.batch : 1) * (a.heads / a.kv_heads / q.gp);
  const long long left = a.left < 0 ? PA_NOLIM : a.left, right = a.right < 0 ? PA_NOLIM : a.right;
  const long long toks = left + right + 128 < a.Nq ? left + right + 128 : a.Nq;
  const long long tn = loops * ((toks * q.gp + 63) / 64), ts = loops * (((long long)a.Nq * q.gp + 63) / 64);
  k.sblk = ts > tn ? (int)(((a.sinks < a.Nk ? a.sinks : a.Nk) + 127) / 128) : 0;
  const long long work = (long long)k.units * ((k.nblk - k.sblk) * tn + k.sblk * ts), places = 2LL * ctx->num_cus;
  long long part = (work + places - 1) / places;
  if (part < 8) part = 8;
  auto parts = [&](long long t) { const long long s = t / part; return (int)(s < 1 ? 1 : s > 64 ? 64 : s); };
  k.split_s = k.sblk ? parts(ts) : 1;
  k.split_n = parts(tn);
  const long long slots = (long long)k.sblk * k.split_s + (long long)(k.nblk - k.sblk) * k.split_n;
  if (slots > 0x7fffffffLL) { k.split_s = k.split_n = 1; k.slots = k.nblk; }
  else k.slots = (int)slots;
  k.part_slots = k.split_n > 1 ? (size_t)k.units * k.slots : k.split_s > 1 ? (size_t)k.units * k.sblk * k.split_s : 0;
  return k;
}

static int pa_check(Ctx* ctx, const PAttnArgs& a, const char* who) {
  const std::string w = std::string(who) + ": ";
  if (a.batch < 0 || a.Nq < 0 || a.Nk < 0 || a.Nq > PA_MAX_N || a.Nk > PA_MAX_N) return ctx->fail(w + "batch and sequence lengths must be 0 .. 2^28");
  if (a.heads < 1 || a.kv_heads < 1 || a.heads % a.kv_heads) return ctx->fail(w + "kv_heads must divide heads");
  if ((long long)a.heads * a.Nq > 0x7fff0000LL || (long long)a.batch * a.heads > 0x7fffffffLL) return ctx->fail(w + "too many rows");
  if (a.sinks < 0) return ctx->fail(w + "sinks must not be negative");
  if (!(a.scale - a.scale == 0.f)) return ctx->fail(w + "scale must be finite");
  const int ld[4] = {a.ldq, a.ldk, a.ldv, a.ldo};
  const int wd[4] = {a.heads * 64, a.kv_heads * 64, a.kv_heads * 64, a.heads * 64};
  for (int i = 0; i < 4; ++i) if ((ld[i] & 7) || ld[i] < wd[i] || ld[i] > PA_MAX_LD) return ctx->fail(w + "row strides must be multiples of 8 elements, at least the row's width and at most 2^23");
  if ((a.bsq | a.bsk | a.bsv | a.bso) & 7) return ctx->fail(w + "batch strides must be multiples of 8 elements");
  if (a.batch > 1 && (a.bsk == 0) != (a.bsv == 0)) return ctx->fail(w + "K and V are shared by the batch together or not at all");
  if ((a.table == nullptr) != (a.buckets == nullptr)) return ctx->fail(w + "the bias needs its table and its buckets");
  if (a.table && (a.num_buckets < 1 || a.num_buckets > PA_MAX_BUCKETS || a.R < 0 || a.R > PA_MAX_R)) return ctx->fail(w + "the bias needs 1 .. 4096 buckets and a range of 0 .. 1024");
  if (a.batch > 0 && a.Nq > 0 && (!a.Q || !al16(a.Q))) return ctx->fail(w + "Q is null or not 16-byte aligned");
  if (a.batch > 0 && a.Nk > 0 && (!a.K || !a.V || !al16(a.K) || !al16(a.V))) return ctx->fail(w + "K or V is null or not 16-byte aligned");
  return 0;
}

static PAttnParams pa_params(const PAttnArgs& a, const PPlan& q) {
  PAttnParams p{};
  p.Q = a.Q; p.K = a.K; p.V = a.V; p.O = a.O; p.lse = a.lse;
  p.dO = a.dO; p.dQ = a.dQ; p.dK = a.dK; p.dV = a.dV;
  p.ldq = a.ldq; p.ldk = a.ldk; p.ldv = a.ldv; p.ldo = a.ldo; p.lddo = a.lddo; p.lddq = a.lddq; p.lddk = a.lddk; p.lddv = a.lddv;
  p.bsq = a.bsq; p.bsk = a.bsk; p.bsv = a.bsv; p.bso = a.bso; p.bsdo = a.bsdo; p.bsdq = a.bsdq; p.bsdk = a.bsdk; p.bsdv = a.bsdv;
  p.Nq = a.Nq; p.Nk = a.Nk; p.heads = a.heads; p.kv_heads = a.kv_heads; p.batch = a.batch;
  p.gp = q.gp; p.rows = q.rows; p.nblk = q.nblk; p.nsplit = q.nsplit; p.per = q.per; p.qb = q.qb;
  p.scale = a.scale; p.c = a.scale * PA_LOG2E;
  p.left = a.left < 0 || a.left > PA_NOLIM ? PA_NOLIM : a.left;
  p.right = a.right < 0 || a.right > PA_NOLIM ? PA_NOLIM : a.right;
  p.sinks = a.sinks < PA_MAX_N ? a.sinks : PA_MAX_N;
  p.q_start = a.q_start; p.kv_len = a.kv_len; p.start0 = a.Nk - a.Nq;
  p.table = a.table; p.buckets = a.buckets; p.num_buckets = a.num_buckets; p.R = a.table ? a.R : 0;
  return p;
}

// items to workgroups: contiguous runs per XCD where there are units enough for each (its L2 keeps the unit's K and V), else one after the other
// (false: more threads than the 32 bits that a launch counts them in)
static bool pa_grid(PAttnParams& p, long long items, int units, int threads, dim3& grid) {
  p.items = items;
  p.swz = units >= 8 ? 1 : 0;
  const long long g = p.swz ? 8 * ((items + 7) / 8) : items;
  if (g * threads > 0xffffffffLL) return false;
  grid = dim3((unsigned)g);
  return true;
}

// the backward pass's workspace: row statistics, sums of dS by bucket, parts of dK and dV
struct PBwdLayout { size_t large, dsum, part, bytes; };
static PBwdLayout pa_bwd_layout(const PAttnArgs& a, const PPlan& q, const PKPlan& k) {
  auto up = [](size_t n) { return (n + 15) & ~(size_t)15; };
  PBwdLayout l;
  l.large = up(4 * (size_t)q.units * q.rows * 4);
  l.dsum = l.large + up((size_t)q.units * q.nblk * 4 * 4);
  l.part = l.dsum + up(a.table ? (size_t)q.units * q.nblk * a.num_buckets * 4 : 0);
  l.bytes = l.part + k.part_slots * 128 * 128 * 4;
  return l;
}

size_t pos_attn_workspace(Ctx* ctx, const PAttnArgs& a, bool backward) {
  if (a.batch <= 0 || a.heads < 1 || a.kv_heads < 1 || a.heads % a.kv_heads || a.Nq <= 0 || a.Nk < 0) return 0;
  const PPlan q = pa_plan(ctx, a, backward);
  if (!backward) return q.nsplit > 1 ? (size_t)q.units * q.nsplit * q.rows * PA_PART * 4 : 0;
  return pa_bwd_layout(a, q, pa_kplan(ctx, a, q)).bytes;
}

template <class T, int BIAS>
static int fwd_t(Ctx* ctx, PAttnParams& p, const PPlan& q, dim3 grid) {
  const size_t smem = 4 * PA_TILE + (BIAS ? (size_t)(2 * p.R + 1 + 2 * PA_PAD) * 4 : 0);
  if (q.nw == 1) STAR_LAUNCH((pattn_fwd_kernel<T, BIAS, 1, 1, 1>), grid, dim3(64), smem, ctx->stream, p);
  else if (q.comp) STAR_LAUNCH((pattn_fwd_kernel<T, BIAS, 1, 4, 1>), grid, dim3(256), smem, ctx->stream, p);
  else if (q.nq == 1) STAR_LAUNCH((pattn_fwd_kernel<T, BIAS, 1, 4, 0>), grid, dim3(256), smem, ctx->stream, p);
  else STAR_LAUNCH((pattn_fwd_kernel<T, BIAS, 2, 4, 0>), grid, dim3(256), smem, ctx->stream, p);
  if (q.nsplit > 1) {
    const long long rows = (long long)q.units * q.rows;
    STAR_LAUNCH((pattn_combine_kernel<T>), dim3((unsigned)((rows + 15) / 16)), dim3(256), (size_t)0, ctx->stream, p);
  }
  return 0;
}

int op_pos_attn_fwd(Ctx* ctx, const PAttnArgs& a) {
  if (pa_check(ctx, a, "pos_attn_fwd")) return 1;
  if (a.batch == 0 || a.Nq == 0) return 0;
  if (a.batch > 1 && a.bso == 0) return ctx->fail("pos_attn_fwd: the sequences' outputs lie on top of each other");
  if (!a.O || !al16(a.O)) return ctx->fail("pos_attn_fwd: O is null or not 16-byte aligned");
  if (a.O == a.Q || (a.Nk > 0 && (a.O == a.K || a.O == a.V))) return ctx->fail("pos_attn_fwd: O must not be Q, K or V");
  const PPlan q = pa_plan(ctx, a, false);
  PAttnParams p = pa_params(a, q);
  const size_t need = pos_attn_workspace(ctx, a, false);
  if (need && (!a.workspace || a.workspace_bytes < need || !al16(a.workspace)))
    return ctx->fail("pos_attn_fwd: workspace missing, too small (star_pos_attn_workspace) or not 16-byte aligned");
  p.part = (float*)a.workspace;
  dim3 grid;
  if (!pa_grid(p, (long long)q.units * q.nblk * q.nsplit, q.units, 64 * q.nw, grid)) return ctx->fail("pos_attn_fwd: too many workgroups");
  ProfScope ps(ctx, PK_ATTN_SELF, 0.0, 0.0, a.batch, a.heads, a.Nq, a.Nk);
  if (ctx->dtype == DT_F16) return a.table ? fwd_t<f16, 1>(ctx, p, q, grid) : fwd_t<f16, 0>(ctx, p, q, grid);
  return a.table ? fwd_t<bf16, 1>(ctx, p, q, grid) : fwd_t<bf16, 0>(ctx, p, q, grid);
}

template <class T, int BIAS, int COMP>
static int bwd_t(Ctx* ctx, PAttnParams p, const PPlan& q, const PKPlan& kp, float* dtable) {
  const int R2 = 2 * p.R + 1;
  dim3 grid;
  if (p.batch > 0 && p.Nq > 0) {
    pa_grid(p, (long long)q.units * q.nblk, q.units, 256, grid);
    const size_t smem = 4 * PA_TILE + (BIAS ? (size_t)(5 * (R2 + 2 * PA_PAD_Q) + 64 * PA_SKEW + 16) * 4 : 0);
    STAR_LAUNCH((pattn_dq_kernel<T, BIAS, COMP>), grid, dim3(256), smem, ctx->stream, p);
  }
  if (p.batch > 0 && p.Nk > 0) {
    PAttnParams k = p;
    k.nblk = kp.slots; k.sblk = kp.sblk; k.split_s = kp.split_s; k.split_n = kp.split_n;
    pa_grid(k, (long long)kp.units * kp.slots, kp.units, 256, grid);
    const size_t smem = 2 * (2 * PA_TILE + PA_ROWB) + (BIAS ? (size_t)(R2 + 2 * PA_PAD_K) * 4 : 0);
    STAR_LAUNCH((pattn_dkdv_kernel<T, BIAS, COMP>), grid, dim3(256), smem, ctx->stream, k);
    if (kp.part_slots) {
      const long long blocks = (long long)kp.units * (kp.split_n > 1 ? kp.nblk : kp.sblk);
      STAR_LAUNCH((pattn_dkdv_join_kernel<T>), dim3((unsigned)blocks, 8), dim3(256), (size_t)0, ctx->stream, k);
    }
  }
  if (BIAS) {
    PDTableParams t{p.dsum, dtable, p.Nq > 0 ? p.batch : 0, p.heads, q.nblk, p.num_buckets};
    STAR_LAUNCH(pattn_dtable_kernel, dim3((unsigned)p.heads), dim3(256), (size_t)(256 * 8), ctx->stream, t);
  }
  return 0;
}

int op_pos_attn_bwd(Ctx* ctx, const PAttnArgs& a, float* dtable) {
  if (pa_check(ctx, a, "pos_attn_bwd")) return 1;
  const int ld[4] = {a.lddo, a.lddq, a.lddk, a.lddv};
  const int wd[4] = {a.heads * 64, a.heads * 64, a.kv_heads * 64, a.kv_heads * 64};
  for (int i = 0; i < 4; ++i) if ((ld[i] & 7) || ld[i] < wd[i] || ld[i] > PA_MAX_LD) return ctx->fail("pos_attn_bwd: row strides must be multiples of 8 elements, at least the row's width and at most 2^23");
  if ((a.bsdo | a.bsdq | a.bsdk | a.bsdv) & 7) return ctx->fail("pos_attn_bwd: batch strides must be multiples of 8 elements");
  const bool any = a.batch > 0 && a.Nq > 0;
  if (any && (!a.dO || !a.dQ || !a.lse || !al16(a.dO) || !al16(a.dQ))) return ctx->fail("pos_attn_bwd: dO, dQ or lse is null or not 16-byte aligned");
  if (a.batch > 0 && a.Nk > 0 && (!a.dK || !a.dV || !al16(a.dK) || !al16(a.dV))) return ctx->fail("pos_attn_bwd: dK or dV is null or not 16-byte aligned");
  const void* in[4] = {any ? a.Q : nullptr, any ? a.dO : nullptr, a.K, a.V};
  const void* gr[3] = {any ? a.dQ : nullptr, a.Nk > 0 ? a.dK : nullptr, a.Nk > 0 ? a.dV : nullptr};
  for (int i = 0; i < 3; ++i) {
    bool twice = false;
    for (int j = 0; j < 4; ++j) twice = twice || (gr[i] && gr[i] == in[j]);
    for (int j = 0; j < i; ++j) twice = twice || (gr[i] && gr[i] == gr[j]);
    if (twice) return ctx->fail("pos_attn_bwd: dQ, dK and dV must not be each other or one of the inputs");
  }
  const bool shared = a.bsk == 0 && a.bsv == 0;
  if (a.batch > 1 && ((a.Nq > 0 && a.bsdq == 0) || (!shared && a.Nk > 0 && (a.bsdk == 0 || a.bsdv == 0))))
    return ctx->fail("pos_attn_bwd: the sequences' gradients lie on top of each other");
  if (a.table && !dtable) return ctx->fail("pos_attn_bwd: no place for the table's gradient");
  const PPlan q = pa_plan(ctx, a, true);
  PAttnParams p = pa_params(a, q);
  const size_t need = pos_attn_workspace(ctx, a, true);
  if (need && (!a.workspace || a.workspace_bytes < need || !al16(a.workspace)))
    return ctx->fail("pos_attn_bwd: workspace missing, too small (star_pos_attn_workspace) or not 16-byte aligned");
  const PKPlan kp = pa_kplan(ctx, a, q);
  dim3 grid;                                             // (before the first launch: nothing is left half done)
  if (!pa_grid(p, (long long)q.units * q.nblk, q.units, 256, grid) || !pa_grid(p, (long long)kp.units * kp.slots, kp.units, 256, grid))
    return ctx->fail("pos_attn_bwd: too many workgroups");
  const PBwdLayout l = pa_bwd_layout(a, q, kp);
  const size_t st = (size_t)q.units * q.rows;
  p.st_ref = (float*)a.workspace; p.st_log = p.st_ref + st; p.st_delta = p.st_log + st; p.st_amax = p.st_delta + st;
  p.st_large = (int*)((char*)a.workspace + l.large); p.nlarge = 4 * q.nblk;
  p.dsum = (float*)((char*)a.workspace + l.dsum);
  p.part = (float*)((char*)a.workspace + l.part);
  ProfScope ps(ctx, PK_ATTN_SELF, 0.0, 0.0, a.batch, a.heads, a.Nq, a.Nk);
  auto go = [&](auto t, auto bias) {
    using T = decltype(t);
    constexpr int B = decltype(bias)::value;
    return q.comp ? bwd_t<T, B, 1>(ctx, p, q, kp, dtable) : bwd_t<T, B, 0>(ctx, p, q, kp, dtable);
  };
  using B0 = std::integral_constant<int, 0>;
  using B1 = std::integral_constant<int, 1>;
  if (ctx->dtype == DT_F16) return a.table ? go(f16{}, B1{}) : go(f16{}, B0{});
  return a.table ? go(bf16{}, B1{}) : go(bf16{}, B0{});
}

// ---- bucket of each relative position, on the host: the borders of the geometric part in whole numbers (a logarithm in floating point is off
// beside one).  With near = exact buckets and steps = the geometric ones, d lies past the k-th border iff
// d^steps near^k >= near^steps distance^k
namespace {
struct Big {                                            // a non-negative integer, 32-bit limbs, least first
  std::vector<uint32_t> v{1u};
  void mul(uint32_t m) {
    uint64_t c = 0;
    for (auto& x : v) { c += (uint64_t)x * m; x = (uint32_t)c; c >>= 32; }
    if (c) v.push_back((uint32_t)c);
  }
  void mul_pow(uint32_t m, int e) { for (int i = 0; i < e; ++i) mul(m); }
  bool operator>=(const Big& o) const {
    if (v.size() != o.v.size()) return v.size() > o.v.size();
    for (size_t i = v.size(); i-- > 0;) if (v[i] != o.v[i]) return v[i] > o.v[i];
    return true;
  }
};
}

// out: 2 * distance + 1 buckets of j - p = -distance .. distance; 0, or 1 for arguments out of range
int rel_buckets(int num_buckets, int distance, bool bidirectional, int* out) {
  const int n = bidirectional ? num_buckets / 2 : num_buckets;
  if (!out || num_buckets < (bidirectional ? 2 : 1) || num_buckets > 256 || (bidirectional && num_buckets % 2) || distance < 1 || distance > PA_MAX_R) return 1;
  const int near = n / 2, steps = n - near;
  if (near > 0 && distance <= near) return 1;           // no room for the geometric part
  int k = 0;
  for (int d = 0; d <= distance; ++d) {
    int bk = d;
    if (d >= near) {
      while (k + 1 < steps) {                           // borders rise with k: d passes them one after the other
        if (near == 0) break;
        Big l, r;
        l.mul_pow((uint32_t)d, steps); l.mul_pow((uint32_t)near, k + 1);
        r.mul_pow((uint32_t)near, steps); r.mul_pow((uint32_t)distance, k + 1);
        if (!(l >= r)) break;
        ++k;
      }
      bk = near + k;
    }
    out[distance - d] = bk;                             // keys before the query
    out[distance + d] = bidirectional ? (d > 0 ? n + bk : bk) : 0;
  }
  return 0;
}

}  // namespace star
