// pattn.h -- attention whose scores depend on positions: a sliding window with first tokens that stay visible, key lengths per sequence,
// query positions in a cache, and a learned relative position bias by buckets; head dim 64, grouped heads.  Forward; the backward pass
// is in pattn_bwd.h.
//
//   p_i = q_start[b] + i;  key j is visible to row i for 0 <= j < kv_len[b], j <= p + right, and (j >= p - left or j < sinks)
//   s_ij = scale q_i k_j + table[buckets[clamp(j - p, -R, R) + R]][h];  O = softmax over the visible keys of s, times V; a row that sees
//   no key: O = 0, lse = -inf.  lse_i = log sum_j exp s_ij.
//
// Layout as in attn5.h: S^T = K Q^T with the operands swapped, so that a lane owns one query row and its probabilities are the B operand
// of O^T = V^T P^T in place; K / V tiles of 64 keys in LDS by DMA, two buffers.  What differs, and why:
//   * Q is not scaled before the product (that would round it to 16 bits once more, beside P): the scale, the bias and the running maximum meet
//     in one fma per score.
//   * A tile is "plain" when every row of the workgroup sees all of its keys and the bias is one constant there (past +-R it is: the far
//     tiles, nearly all of a long sequence).  Plain tiles take the lazy path: P = exp2(fma(s, c, off)) against the running maximum as it
//     stands, the row sum as overflow probe.  Every other tile, every tile until each row of the wave has seen one, and every tile of a wave
//     with a maximum past 2^12 (base 2) takes the exact path: masks and bias per score, the tile's maximum, rescale.  Past that a score's
//     own rounding, which the exact path's maximum has and one fma with it has not, is no longer small: equal scores would weigh differently from
//     tile to tile.  Tiles that no row of the workgroup sees are not visited.
//   * Rows of the heads that share a K / V head are packed token-major into one workgroup's rows (GP of them), so that a group reads its
//     keys once; with a bias a workgroup keeps to one head (one table column in LDS).
//   * K / V rows that no row of the workgroup sees are staged as zeros through the descriptor's range check: what lies behind kv_len or
//     outside the window is not read.
//   * Few rows against long key ranges (a decoding step): the key tiles are dealt to NSPLIT workgroups in equal shares -- sequences of
//     different lengths make different counts of shares -- each writes its (m, l, O) of the rows in fp32, pattn_combine_kernel joins them
//     in a fixed order.
// What bounds it, measured: long inputs no one unit (f16, 17 776 tokens, 16 heads, a window of 5400 either way: 790 - 810 us, 0.85 PFLOP/s of the
// visible pairs; vector unit busy 59 % of the cycles, matrix unit 41 %), and 1120 workgroups on the card's 512 places, the last round a fifth full
// (32 rows per wave instead of 64 would read each fragment twice); a chunk of 1350 tokens against a window of 10 800, 16 heads in groups of 4: 104 us, 8 of
// them the join, 1032 workgroups on 512 places.  A token at a time is bound by HBM: bf16, 32 sequences x 8 K / V heads, 4160 of 32 800 keys: 56 us + 5 us
// of join, 4.8 TB/s of the 272 MB; 16 sequences x 16 heads of up to 8200 keys with a bias: 87 us + 6 us.  Few short rows (8 x 226 tokens, 32 heads, a
// bias: 18 us) are latencies one after the other: lengths, Q, the table's two dependent loads, a barrier, then the first tile, four tiles, store.
// NQ: 32-row blocks per wave (2: 256-row workgroups for long inputs, 1: 128 rows, more workgroups); NW = 1: a wave by itself, 32 rows.
// COMP: P is rounded to the 16-bit type, and so is what the rounding left, and both take part in the second product: O is then off by its own
// rounding alone (1.00 x, without 1.28 - 1.41 x, the gradients 1.40 - 1.46 x).  Four more matrix instructions per 32 x 32 block, taken where they cost
// little: rows that see few keys (PA_COMP_SPAN in pattn.cpp has both sides) and the single-wave form, which waits for its keys.
#pragma once
#include "attn.h"

namespace star {

struct PAttnParams {
  const void* Q; const void* K; const void* V; void* O; float* lse;
  const void* dO; void* dQ; void* dK; void* dV;
  int ldq, ldk, ldv, ldo, lddo, lddq, lddk, lddv;      // row strides (elements)
  long long bsq, bsk, bsv, bso, bsdo, bsdq, bsdk, bsdv; // batch strides (elements)
  int Nq, Nk, heads, kv_heads, batch;
  int gp;                             // heads packed into one unit's rows (1, or heads / kv_heads)
  int rows, qb;                       // gp * Nq; rows per workgroup
  float c, scale;                     // scale * log2(e), scale
  int left, right, sinks;             // left / right past every position: no limit
  const int* q_start; const int* kv_len;
  int start0;                         // position of row 0 where q_start is null
  const float* table; const int* buckets; int num_buckets, R;
  int nblk, nsplit, per;              // row blocks per unit; key splits, key tiles of each
  long long items;                    // units * nblk * nsplit
  int swz;                            // 1: each XCD walks a contiguous run of items
  float* part;                        // nsplit > 1: [unit][split][rows][68]: O[64], m, l
  // backward
  float* st_ref; float* st_log; float* st_delta; float* st_amax;   // [unit][rows]
  int* st_large; int nlarge;          // [unit][nlarge]: 32 rows with a large reference point among them
  float* dsum;                        // [unit][row block][num_buckets] sums of dS
  int sblk, split_s, split_n;         // dK / dV: the first sblk key blocks (those of the first tokens) in split_s parts each, the others in split_n
};

constexpr int PA_KT = 64, PA_TILE = PA_KT * 128;       // keys per tile, bytes of a K or V tile
constexpr int PA_PART = 68;                            // floats per row of a split's partial result (16-byte rows)
constexpr float PA_LOG2E = 1.4426950408889634f, PA_LN2 = 0.6931471805599453f;
constexpr float PA_NINF = -__builtin_inff();
// Of scores in base 2: half a step of fp32 there is a relative 1.7e-4 of exp2, a third of f16's half step; twice as much would no longer be small beside
// it.  Logits of a trained layer are tens, and the rows above it take 1.1 - 1.6 x as long (video window 0.80 -> 1.18 ms, long bias backward 1.0 -> 1.6 ms)
constexpr float PA_LARGE = 4096.0f;

struct PRange { int n, qs; };                          // keys in hand, position of row 0 -- both clamped to what the kernels can index
STAR_DEV PRange pa_range(const PAttnParams& p, int b) {
  int n = p.kv_len ? p.kv_len[b] : p.Nk;
  n = n < 0 ? 0 : n > p.Nk ? p.Nk : n;
  int s = p.q_start ? p.q_start[b] : p.start0;
  const int lim = 1 << 29;
  s = s < -lim ? -lim : s > lim ? lim : s;
  return PRange{wave_uniform(n), wave_uniform(s)};
}
// the window [lo, hi) of the row at position pos, and the count of first tokens beside it
STAR_DEV int pa_hi(const PAttnParams& p, int n, int pos) { const int h = pos + p.right + 1; return h < 0 ? 0 : h > n ? n : h; }
STAR_DEV int pa_lo(const PAttnParams& p, int pos) { const int l = pos - p.left; return l < 0 ? 0 : l; }

// the key tiles that rows at positions [p0, p1] see: [0, na) and [b0, b0 + nb)
struct PTiles { int na, b0, nb, lo, hi, sk; };
STAR_DEV PTiles pa_tiles(const PAttnParams& p, int n, int p0, int p1) {
  PTiles t;
  t.hi = pa_hi(p, n, p1);
  t.lo = pa_lo(p, p0);
  if (t.lo > t.hi) t.lo = t.hi;
  t.sk = p.sinks < t.hi ? p.sinks : t.hi;
  t.na = (t.sk + PA_KT - 1) / PA_KT;
  t.b0 = t.lo / PA_KT;
  const int end = (t.hi + PA_KT - 1) / PA_KT;
  if (t.b0 < t.na) t.b0 = t.na;
  t.nb = t.lo < t.hi && end > t.b0 ? end - t.b0 : 0;
  return t;
}

// which item this workgroup has; units (batch, head group) outermost, then row blocks, then splits
STAR_DEV long long pa_item(const PAttnParams& p) {
  const long long bid = blockIdx.x;
  if (!p.swz) return bid;
  const long long per = (p.items + 7) / 8, slot = bid >> 3;
  return slot >= per ? p.items : (bid & 7) * per + slot;
}

// The bias of one head by relative position, times log2(e), in LDS: tab[i] belongs to j - p = i - R - PAD.  The end values go on for PAD
// entries either way, so that in a tile that reaches into (-R, R) every score's entry is at a fixed distance from its lane's first: no
// clamping per score.  The type's lowest and highest values stay finite: whatever leaves the range in base 2 (beyond +-2.36e38) is held at
// +-3.40e38, the log-sum-exp of a row that sees nothing better is the type's lowest (highest) value
constexpr float PA_MOST = 3.4028235e38f;
constexpr int PA_PAD = 128, PA_PAD_Q = 96, PA_PAD_K = 192;     // a wave's 64 rows against 64 keys; dQ: 32 rows; dK / dV: 64 rows against 128 keys
STAR_DEV float pa_bias_at(const PAttnParams& p, int head, int k) {       // of bucket k
  k = k < 0 ? 0 : k >= p.num_buckets ? p.num_buckets - 1 : k;
  const float v = p.table[(size_t)k * p.heads + head];
  const float w = v * PA_LOG2E;
  return __builtin_fabsf(w) > PA_MOST && __builtin_fabsf(v) <= PA_MOST ? __builtin_copysignf(PA_MOST, v) : w;
}
// log sum exp in base e from the maximum and the sum relative to it
STAR_DEV float pa_lse(float m, float l) {
  return l == 0.f ? PA_NINF : __builtin_fabsf(m) == PA_MOST ? m : (m + __builtin_log2f(l)) * PA_LN2;
}
template <int NT, int PAD>
STAR_DEV void pa_bias_table(const PAttnParams& p, int head, float* tab) {
  constexpr int U = 4;                                 // entries in flight per thread: two dependent loads each
  const int n = 2 * p.R + 1 + 2 * PAD;
  for (int i = threadIdx.x; i < n; i += U * NT) {
    int k[U];
    float w[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      int j = i + u * NT - PAD;
      j = j < 0 ? 0 : j > 2 * p.R ? 2 * p.R : j;
      k[u] = p.buckets[j];
    }
#pragma unroll
    for (int u = 0; u < U; ++u) w[u] = pa_bias_at(p, head, k[u]);
#pragma unroll
    for (int u = 0; u < U; ++u) if (i + u * NT < n) tab[i + u * NT] = w[u];
  }
}

// copies rows of 64 elements (128 bytes) into a swizzled LDS tile, 16 bytes per lane and step; rows that `ok` refuses become zeros.
// base: wave-uniform address of the tile's first row; the byte offset of a row from it stays below 2^31 (the launcher checks strides)
template <int NT, class OFF>
STAR_DEV void pa_stage(const void* base, char* smem, int dst, int tid, int wv, OFF off) {
  const BufDesc d = make_desc(base, GLDS_BUF_RANGE);
#pragma unroll
  for (int j = 0; j < 512 / NT; ++j) {
    const int r = (j * NT + tid) >> 3;
    const int ch = (tid & 7) ^ ((r >> 1) & 7);
    glds16_desc(d, off(r, ch), 0, smem + wave_uniform(dst + (j * NT + wv * 64) * 16));
  }
}

// row of a unit -> token and head within the unit
// (a division's result is in vector registers even where it is the same for all lanes: what steers the DMA goes through wave_uniform)
struct PRow { int i, g; };
STAR_DEV PRow pa_row(const PAttnParams& p, int r) {
  if (p.gp == 1) return PRow{r, 0};
  const int i = r / p.gp;
  return PRow{i, r - i * p.gp};
}

// a wave's rows [r, r + cnt): positions of the first and the last of them, the widest and the narrowest end of their windows.  None: hi = 0
struct PWave { int p0, p1, hi, lo, hi_min, lo_max; };
STAR_DEV PWave pa_wave(const PAttnParams& p, const PRange& rg, int r, int cnt) {
  PWave w;
  const int last = r + cnt - 1 < p.rows - 1 ? r + cnt - 1 : p.rows - 1;
  w.p0 = wave_uniform(rg.qs + pa_row(p, r < p.rows ? r : p.rows - 1).i);
  w.p1 = wave_uniform(rg.qs + pa_row(p, last).i);
  w.hi = r < p.rows ? pa_hi(p, rg.n, w.p1) : 0;
  w.lo = pa_lo(p, w.p0);
  w.hi_min = pa_hi(p, rg.n, w.p0);
  w.lo_max = pa_lo(p, w.p1);
  return w;
}
// some row sees a key of the tile at k0; every row sees all of its keys
STAR_DEV bool pa_sees(const PAttnParams& p, const PWave& w, int k0) { return k0 < w.hi && (k0 + PA_KT > w.lo || k0 < p.sinks); }
STAR_DEV bool pa_sees_whole(const PAttnParams& p, const PWave& w, int k0) {
  return k0 + PA_KT <= w.hi_min && (k0 >= w.lo_max || k0 + PA_KT <= p.sinks);
}

// eight rows of d per lane half: acc[db] holds d = 32 db + (r & 3) + 8 (r >> 2) + 4 h2 of the lane's row; 16-byte stores
template <class T>
STAR_DEV void pa_store_row(const f32x16* acc, float mul, T* row, bool ok) {
  const int h2 = (threadIdx.x & 63) >> 5;
#pragma unroll
  for (int db = 0; db < 2; ++db)
#pragma unroll
    for (int a = 0; a < 2; ++a) {
      u32x2 w[2];
#pragma unroll
      for (int gg = 0; gg < 2; ++gg) {
        vec<T, 4> o4;
#pragma unroll
        for (int e = 0; e < 4; ++e) o4[e] = from_f32<T>(acc[db][(2 * a + gg) * 4 + e] * mul);
        w[gg] = __builtin_bit_cast(u32x2, o4);
      }
      const u32x2 x0 = permlane32_swap(w[0][0], w[1][0]);
      const u32x2 x1 = permlane32_swap(w[0][1], w[1][1]);
      u32x4 out;
      out[0] = x0[0]; out[1] = x1[0]; out[2] = x0[1]; out[3] = x1[1];
      if (ok) *reinterpret_cast<u32x4*>(row + 32 * db + 16 * a + 8 * h2) = out;
    }
}

template <class T, int BIAS, int NQ, int NW, int COMP>
STAR_GLOBAL void STAR_LAUNCH_BOUNDS(NW * 64, NW == 1 ? 1 : 2)
pattn_fwd_kernel(const PAttnParams p) {
  constexpr int NT = NW * 64, QW = 32 * NQ, QB = NW * QW;
  constexpr float LAZY_BIG = 1024.0f;
  char* smem = dyn_smem();                             // two buffers of (K tile | V tile), then the bias table
  float* tab = reinterpret_cast<float*>(smem + 4 * PA_TILE);
  const long long item = pa_item(p);
  if (item >= p.items) return;
  const int tid = threadIdx.x, lane = tid & 63, wv = wave_uniform(tid >> 6);
  const int h2 = lane >> 5, lq = lane & 31;
  const int split = wave_uniform((int)(item % p.nsplit));
  const long long ub = item / p.nsplit;
  const int qb = wave_uniform(p.nblk - 1 - (int)(ub % p.nblk));      // the rows that see most keys first
  const int unit = wave_uniform((int)(ub / p.nblk));
  const int upb = p.heads / p.gp;                      // units per sequence
  const int b = wave_uniform(unit / upb), head0 = wave_uniform((unit - b * upb) * p.gp);
  const int kvh = wave_uniform(head0 / (p.heads / p.kv_heads));
  const PRange rg = pa_range(p, b);
  const int n = rg.n;
  const T* Qg = (const T*)p.Q + (size_t)b * p.bsq + head0 * 64;
  const T* Kg = (const T*)p.K + (size_t)b * p.bsk + kvh * 64;
  const T* Vg = (const T*)p.V + (size_t)b * p.bsv + kvh * 64;

  const int r_base = qb * QB;
  const int r_last = r_base + QB - 1 < p.rows - 1 ? r_base + QB - 1 : p.rows - 1;
  const int p0 = wave_uniform(rg.qs + pa_row(p, r_base).i), p1 = wave_uniform(rg.qs + pa_row(p, r_last).i);
  const PTiles tl = pa_tiles(p, n, p0, p1);
  // the wave's own rows: whether they see a tile, see it whole, and how the bias looks there, is asked for them
  const PWave w = pa_wave(p, rg, r_base + wv * QW, QW);

  vec<T, 8> qf[NQ][4];
  int pos[NQ];                                         // position of the lane's row
#pragma unroll
  for (int qi = 0; qi < NQ; ++qi) {
    int r = r_base + wv * QW + qi * 32 + lq;
    if (r > p.rows - 1) r = p.rows - 1;
    const PRow rw = pa_row(p, r);
    pos[qi] = rg.qs + rw.i;
    const T* q = Qg + (size_t)rw.i * p.ldq + rw.g * 64;
#pragma unroll
    for (int ks = 0; ks < 4; ++ks) qf[qi][ks] = *reinterpret_cast<const vec<T, 8>*>(q + ks * 16 + h2 * 8);
  }
  const int total = tl.na + tl.nb;
  const int it0 = split * p.per < total ? split * p.per : total;
  const int it1 = split == p.nsplit - 1 || it0 + p.per > total ? total : it0 + p.per;
  auto tile_of = [&](int it) STAR_ALWAYS_INLINE { return it < tl.na ? it : it - tl.na + tl.b0; };
  float far_l = 0.f, far_r = 0.f;
  if constexpr (BIAS) {
    far_l = pa_bias_at(p, head0, p.buckets[0]); far_r = pa_bias_at(p, head0, p.buckets[2 * p.R]);
    // where all of the workgroup's tiles are far on the left (most splits of a long cache) only the table's left end is read
    if (it0 < it1 && tile_of(it1 - 1) * PA_KT + PA_KT - 1 - p0 > -p.R) pa_bias_table<NT, PA_PAD>(p, head0, tab);
    else for (int i = tid; i <= PA_PAD; i += NT) tab[i] = far_l;
    block_sync();
  }
  auto stage = [&](int it, int buf) STAR_ALWAYS_INLINE {
    const int t = tile_of(it), k0 = t * PA_KT;
    const int kd = buf * 2 * PA_TILE;
    const T* kb = Kg + (size_t)k0 * p.ldk;
    const T* vb = Vg + (size_t)k0 * p.ldv;
    const bool whole = k0 + PA_KT <= tl.hi && (k0 >= tl.lo || k0 + PA_KT <= tl.sk);
    if (whole) {
      pa_stage<NT>(kb, smem, kd, tid, wv, [&](int r, int ch) { return (uint32_t)(r * p.ldk + ch * 8) * 2u; });
      pa_stage<NT>(vb, smem, kd + PA_TILE, tid, wv, [&](int r, int ch) { return (uint32_t)(r * p.ldv + ch * 8) * 2u; });
    } else {
      auto seen = [&](int r) { const int key = k0 + r; return key < tl.hi && (key >= tl.lo || key < tl.sk); };
      pa_stage<NT>(kb, smem, kd, tid, wv, [&](int r, int ch) { return seen(r) ? (uint32_t)(r * p.ldk + ch * 8) * 2u : GLDS_BUF_OOB; });
      pa_stage<NT>(vb, smem, kd + PA_TILE, tid, wv, [&](int r, int ch) { return seen(r) ? (uint32_t)(r * p.ldv + ch * 8) * 2u : GLDS_BUF_OOB; });
    }
  };

  // loop-invariant fragment addresses (attn5.h): K row kb * 32 + lq, chunk ks * 2 + h2; V^T by transposing reads
  const char* kfo[4];
#pragma unroll
  for (int ks = 0; ks < 4; ++ks) kfo[ks] = opaque(smem + swz_off(lq, ks * 2 + h2));
  const char* vfo[2][2];
  {
    const int i = lane & 15, g = lane >> 4;
#pragma unroll
    for (int half = 0; half < 2; ++half)
#pragma unroll
      for (int db = 0; db < 2; ++db) {
        const int key = 8 * half + 4 * h2 + (i >> 2), d = 32 * db + 16 * (g & 1) + 4 * (i & 3);
        vfo[half][db] = opaque(smem + PA_TILE + swz_off(key, d >> 3) + (d & 7) * 2);
      }
  }

  f32x16 oacc[NQ][2];
#pragma unroll
  for (int a = 0; a < NQ; ++a)
#pragma unroll
    for (int c2 = 0; c2 < 2; ++c2)
#pragma unroll
      for (int r = 0; r < 16; ++r) oacc[a][c2][r] = 0.f;
  float m_run[NQ], l_run[NQ];                          // base 2; m = -inf: the row has seen no key yet
#pragma unroll
  for (int qi = 0; qi < NQ; ++qi) { m_run[qi] = PA_NINF; l_run[qi] = 0.f; }
  bool fresh = true;                                   // wave-uniform: some row may not have seen a key yet, or its maximum is large

  auto tile = [&](int it, int buf) STAR_ALWAYS_INLINE {
    const int k0 = tile_of(it) * PA_KT;
    const int bofs = buf * 2 * PA_TILE;
    if (!pa_sees(p, w, k0)) return;
    const bool masked = !pa_sees_whole(p, w, k0);
    bool near = false;
    float far = 0.f;
    if constexpr (BIAS) {
      const bool fl = k0 + PA_KT - 1 - w.p0 <= -p.R, fr = k0 - w.p1 >= p.R;
      near = !(fl || fr);
      far = fl ? far_l : far_r;
    }
    f32x16 s[NQ][2];
    auto scores = [&]() STAR_ALWAYS_INLINE {
#pragma unroll
      for (int a = 0; a < NQ; ++a)
#pragma unroll
        for (int kb = 0; kb < 2; ++kb)
#pragma unroll
          for (int r = 0; r < 16; ++r) s[a][kb][r] = 0.f;
#pragma unroll
      for (int ks = 0; ks < 4; ++ks)
#pragma unroll
        for (int kb = 0; kb < 2; ++kb) {
          const vec<T, 8> kf = *reinterpret_cast<const vec<T, 8>*>(kfo[ks] + bofs + kb * 4096);
#pragma unroll
          for (int qi = 0; qi < NQ; ++qi) s[qi][kb] = mfma32<T>(kf, qf[qi][ks], s[qi][kb]);
        }
    };
    vec<T, 8> pf[NQ][4], pl[COMP ? NQ : 1][4];
    float lsum[NQ];
    // P = exp2(fma(s, c, off)): the row sum in four chains of fp32 adds on the unrounded values
    auto expo = [&](int qi, float c, float off) STAR_ALWAYS_INLINE {
      float ls0 = 0.f, ls1 = 0.f, ls2 = 0.f, ls3 = 0.f;
#pragma unroll
      for (int kb = 0; kb < 2; ++kb)
#pragma unroll
        for (int u = 0; u < 2; ++u) {
          vec<T, 8> pk, pr;
#pragma unroll
          for (int e = 0; e < 8; e += 4) {
            const float a0 = fast_exp2(__builtin_fmaf(s[qi][kb][8 * u + e], c, off)), a1 = fast_exp2(__builtin_fmaf(s[qi][kb][8 * u + e + 1], c, off));
            const float a2 = fast_exp2(__builtin_fmaf(s[qi][kb][8 * u + e + 2], c, off)), a3 = fast_exp2(__builtin_fmaf(s[qi][kb][8 * u + e + 3], c, off));
            ls0 += a0; ls1 += a1; ls2 += a2; ls3 += a3;
            pk[e] = from_f32<T>(a0); pk[e + 1] = from_f32<T>(a1); pk[e + 2] = from_f32<T>(a2); pk[e + 3] = from_f32<T>(a3);
            if constexpr (COMP) {
              pr[e] = from_f32<T>(a0 - to_f32<T>(pk[e])); pr[e + 1] = from_f32<T>(a1 - to_f32<T>(pk[e + 1]));
              pr[e + 2] = from_f32<T>(a2 - to_f32<T>(pk[e + 2])); pr[e + 3] = from_f32<T>(a3 - to_f32<T>(pk[e + 3]));
            }
          }
          pf[qi][kb * 2 + u] = pk;
          if constexpr (COMP) pl[qi][kb * 2 + u] = pr;
        }
      lsum[qi] = (ls0 + ls1) + (ls2 + ls3);
    };
    bool exact = masked || near || fresh;
    if (!exact) {
      scores();
      bool bad = false;
#pragma unroll
      for (int qi = 0; qi < NQ; ++qi) {
        expo(qi, p.c, far - m_run[qi]);
        bad = bad || !(lsum[qi] <= LAZY_BIG);
      }
      exact = wave_any(bad);                           // some P is large (or overflowed): move the maximum and do the tile again
    }
    if (exact) {
      scores();                                        // (the K tile is still there; scores kept beside P would not fit the registers)
      bool unseen = false;
#pragma unroll
      for (int qi = 0; qi < NQ; ++qi) {
        const int hi = pa_hi(p, n, pos[qi]), lo = pa_lo(p, pos[qi]);
        float mx = PA_NINF;
        // the table's entry of the lane's first key; a tile past +-R reads the end values that go on there
        int at = k0 + 4 * h2 - pos[qi];
        at = at < -p.R - PA_PAD ? -p.R - PA_PAD : at > p.R + PA_PAD - 64 ? p.R + PA_PAD - 64 : at;
        const float* row = tab + at + p.R + PA_PAD;
#pragma unroll
        for (int kb = 0; kb < 2; ++kb)
#pragma unroll
          for (int r = 0; r < 16; ++r) {
            const int j = kb * 32 + (r & 3) + 8 * (r >> 2), key = k0 + 4 * h2 + j;
            float y = __builtin_fmaf(s[qi][kb][r], p.c, BIAS ? row[j] : 0.f);
            if (masked) y = (key < hi) & ((key >= lo) | (key < p.sinks)) ? y : PA_NINF;
            s[qi][kb][r] = y;
            mx = fmaxf(mx, y);
          }
        mx = pair_max(mx);
        const float m_new = fmaxf(m_run[qi], mx);
        const float alpha = m_new == PA_NINF ? 1.f : fast_exp2(m_run[qi] - m_new);
        m_run[qi] = m_new;
        l_run[qi] *= alpha;
#pragma unroll
        for (int db = 0; db < 2; ++db)
#pragma unroll
          for (int r = 0; r < 16; ++r) oacc[qi][db][r] *= alpha;
        unseen = unseen || !(__builtin_fabsf(m_new) <= PA_LARGE);
        expo(qi, 1.f, m_new == PA_NINF ? 0.f : -m_new);
      }
      fresh = wave_any(unseen);
    }
#pragma unroll
    for (int qi = 0; qi < NQ; ++qi) l_run[qi] += lsum[qi];
#pragma unroll
    for (int tt = 0; tt < 4; ++tt)
#pragma unroll
      for (int db = 0; db < 2; ++db) {
        vec<T, 8> vf;
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          const vec<T, 4> r = lds_read_tr<T>(vfo[half][db] + bofs + tt * 2048);
#pragma unroll
          for (int e = 0; e < 4; ++e) vf[half * 4 + e] = r[e];
        }
#pragma unroll
        for (int qi = 0; qi < NQ; ++qi) {
          oacc[qi][db] = mfma32<T>(vf, pf[qi][tt], oacc[qi][db]);
          if constexpr (COMP) oacc[qi][db] = mfma32<T>(vf, pl[qi][tt], oacc[qi][db]);
        }
      }
  };

  if (p.nsplit > 1 && it0 >= it1 && split) return;      // (the first split writes what a row that sees nothing gets)
  glds_wait();                                         // the Q loads are done before the first hand-written LDS-DMA
  if (it0 < it1) stage(it0, 0);
  for (int it = it0; it < it1; ++it) {
    const int buf = wave_uniform((it - it0) & 1);
    glds_wait(); block_sync();
    if (it + 1 < it1) stage(it + 1, buf ^ 1);
    tile(it, buf);
  }

#pragma unroll
  for (int qi = 0; qi < NQ; ++qi) {
    const float l = pair_sum(l_run[qi]);
    const int r = r_base + wv * QW + qi * 32 + lq;
    const bool ok = r < p.rows;
    const PRow rw = pa_row(p, ok ? r : p.rows - 1);
    if (p.nsplit > 1) {
      if (ok) {
        float* o = p.part + (((size_t)unit * p.nsplit + split) * p.rows + r) * PA_PART;
#pragma unroll
        for (int db = 0; db < 2; ++db)
#pragma unroll
          for (int g = 0; g < 4; ++g) {
            f32x4 v;
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = oacc[qi][db][g * 4 + e];
            *reinterpret_cast<f32x4*>(o + 32 * db + 8 * g + 4 * h2) = v;
          }
        if (h2 == 0) { o[64] = m_run[qi]; o[65] = l; }
      }
    } else {
      pa_store_row<T>(oacc[qi], l > 0.f ? 1.0f / l : l == 0.f ? 0.f : l, (T*)p.O + (size_t)b * p.bso + (size_t)rw.i * p.ldo + (head0 + rw.g) * 64, ok);
      if (p.lse && ok && h2 == 0)
        p.lse[((size_t)b * p.heads + head0 + rw.g) * p.Nq + rw.i] = pa_lse(m_run[qi], l);
    }
  }
}

// joins the splits of a row, in their order: sixteen lanes per row, four values of d each
template <class T>
STAR_GLOBAL void STAR_LAUNCH_BOUNDS(256)
pattn_combine_kernel(const PAttnParams p) {
  const int sub = threadIdx.x & 15;
  const int upb = p.heads / p.gp;
  const long long rows = (long long)p.batch * upb * p.rows;
  const long long row = (long long)blockIdx.x * 16 + (threadIdx.x >> 4);
  if (row >= rows) return;
  const int unit = (int)(row / p.rows), r = (int)(row - (long long)unit * p.rows);
  const float* base = p.part + ((size_t)unit * p.nsplit * p.rows + r) * PA_PART;
  const size_t step = (size_t)p.rows * PA_PART;
  const PRow rw = pa_row(p, r);
  const int b = unit / upb;
  // only the splits that had tiles wrote anything
  int n = p.kv_len ? p.kv_len[b] : p.Nk;
  n = n < 0 ? 0 : n > p.Nk ? p.Nk : n;
  int qs = p.q_start ? p.q_start[b] : p.start0;
  qs = qs < -(1 << 29) ? -(1 << 29) : qs > 1 << 29 ? 1 << 29 : qs;
  const int blk = r / p.qb * p.qb, end = blk + p.qb - 1 < p.rows - 1 ? blk + p.qb - 1 : p.rows - 1;
  const PTiles tl = pa_tiles(p, n, qs + pa_row(p, blk).i, qs + pa_row(p, end).i);
  const int need = (tl.na + tl.nb + p.per - 1) / p.per, ns = need < 1 ? 1 : need > p.nsplit ? p.nsplit : need;
  float m = PA_NINF;
#pragma unroll 4
  for (int s = 0; s < ns; ++s) m = fmaxf(m, base[s * step + 64]);
  float l = 0.f;
  f32x4 o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
  for (int s = 0; s < ns; ++s) {
    const float ms = base[s * step + 64];
    const float w = ms == PA_NINF ? 0.f : fast_exp2(ms - m);
    const f32x4 v = *reinterpret_cast<const f32x4*>(base + s * step + 4 * sub);
    l += w * base[s * step + 65];
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] += w * v[e];
  }
  const int head = (unit - b * upb) * p.gp + rw.g;
  const float mul = l > 0.f ? 1.0f / l : l == 0.f ? 0.f : l;
  vec<T, 4> out;
#pragma unroll
  for (int e = 0; e < 4; ++e) out[e] = from_f32<T>(o[e] * mul);
  *reinterpret_cast<vec<T, 4>*>((T*)p.O + (size_t)b * p.bso + (size_t)rw.i * p.ldo + head * 64 + 4 * sub) = out;
  if (p.lse && sub == 0) p.lse[((size_t)b * p.heads + head) * p.Nq + rw.i] = pa_lse(m, l);
}

}  // namespace star
