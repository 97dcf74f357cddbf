// pattn_bwd.h -- backward pass of the position-dependent attention (pattn.h).
//
//   P = exp(s - lse), dV = P^T dO, dP = dO V^T, delta = sum_j P dP, dS = P (dP - delta),
//   dQ = scale dS K, dK = scale dS^T Q, dtable[k][h] = sum over the pairs of bucket k of dS
//
// Two kernels, so that every sum has one owner and a fixed order (no atomics): the same call gives the same bits.
//   pattn_dq_kernel    a wave owns query rows and walks the keys twice.  First walk: delta, and the log-sum-exp once more (the caller's is
//                      rounded to fp32 and in base e), as two numbers: the row's reference point, and log2 of the sum relative to it.  Second walk:
//                      dS, dQ, and the sums of dS by relative position.
//   pattn_dkdv_kernel  a wave owns 32 keys and walks the query rows of every head of the group (and of every sequence, where the batch
//                      shares K and V): dK, dV.
// The reference is the caller's log-sum-exp; for a wave with one past 2^12 (base 2), whose roundings are no small factors of exp2, it is the row's maximum,
// found anew in the first walk, and each score is rounded as in the forward pass before the reference is subtracted.
// delta is not taken as rowsum(dO O): O is rounded to 16 bits and comes from rounded P, and where a softmax is peaked dP - delta is a small
// difference -- the error of dQ and dK would be several times their own rounding.  The first walk costs 8 of 36 matrix instructions
// per 32 x 32 block.  dP is the same sum in the same order in both kernels, so that a row with one visible key has dS = 0 exactly.
// f16 only: P and dS are scaled by powers of two before they are rounded, so that they neither leave f16's range nor fall below its
// normal one: P by 2^10 (P <= 1), dS by the largest |dP| among the row's visible keys (dQ), which the first walk keeps, or among those of the
// rows walked so far (dK): P <= 1 and |dP - delta| <= 2 max |dP| bound it, whatever the sizes of dO and V.
// COMP: as in the forward pass, dS and P with what their rounding left, for short rows.
// Key blocks that many rows see (those of the first tokens: every row), or few blocks on many compute units, are dealt to several
// workgroups along the rows; each writes its part in fp32, pattn_dkdv_join_kernel adds the parts in their order.
// What bounds them: no one unit, and how the workgroups fill the card.  bf16, 2 x 4099 tokens, 16 heads, a bias: 1.0 ms (traced dQ 0.53 - 0.56, dK / dV
// 0.47 - 0.49 ms); 10 d flops a pair make 0.33 PFLOP/s, 0.6 with the products that are taken again (18 d).  Counters, dQ / dK dV: vector unit busy 56 /
// 44 % of a busy compute unit's cycles, matrix unit 33 / 34 %, waves waiting 29 / 40 %; but a compute unit is busy 75 / 66 % of the time only: 1056 workgroups on
// 512 places are two rounds and a few that make a third, and a block of three rows walks all its keys like a full one.  Short sequences (4 x 226 tokens, 16
// heads: 30 + 22 + 5 us) are one chain of product -> exponential -> pack -> product after the other on 128 of 256 compute units, and a launch each.  A window of
// 1024 over 4500 tokens, 16 heads in groups of 4: 173 us (dQ 80, dK / dV 86, join 10 traced), 0.26 PFLOP/s, compute units busy 70 / 74 %.  Tried and no faster:
// 64 rows per wave in dQ (spills), three waves per SIMD with a bias, halves of a tile in step with each other, the transposed fragments read before the
// exponentials.
#pragma once
#include "pattn.h"

namespace star {

// 2^e with |x| 2^e in [2^13, 2^14), so that twice that is below f16's 65504: the exponent as an integer, 0 for zero and non-finite x.  x is a sum
// of 64 products of f16 values, which lies between 2^-48 and 2^38: e within [-40, 60], and so is 2^(e - e') for two of them
constexpr int PA_EXP_MAX = 60;
STAR_DEV int pa_fit_exp(float x) {
  const uint32_t ex = (__builtin_bit_cast(uint32_t, x) >> 23) & 255u;
  if (ex == 0u) return x == 0.f ? 0 : PA_EXP_MAX;
  if (ex == 255u) return 0;
  const int e = 140 - (int)ex;
  return e < -40 ? -40 : e > PA_EXP_MAX ? PA_EXP_MAX : e;
}
STAR_DEV float pa_pow2(int e) { return __builtin_bit_cast(float, (uint32_t)(e + 127) << 23); }

// hi + lo += x, lo gathers what the additions to hi rounded away
STAR_DEV void pa_add2(float& hi, float& lo, float x) {
  const float s = hi + x, t = s - hi;
  lo += (hi - (s - t)) + (x - t);
  hi = s;
}

// the rounded value, and what that left
template <class T, int COMP>
STAR_DEV void pa_round(float v, T& hi, T& lo) {
  hi = from_f32<T>(v);
  if constexpr (COMP) lo = from_f32<T>(v - to_f32<T>(hi));
}

constexpr int PA_ROWB = 64 * 20 + 16;                  // dK / dV: bytes of a tile's row statistics
constexpr int PA_SKEW = 48;                            // floats per row of the skewed buffer: 16 keys + 32 rows - 1 diagonals, and one to spare

// LDS past the tiles with a bias: table | a wave's sums by relative position, four arrays like the table | four skewed buffers
template <class T, int BIAS, int COMP>
STAR_GLOBAL void STAR_LAUNCH_BOUNDS(256, BIAS || COMP ? 2 : 3)
pattn_dq_kernel(const PAttnParams p) {
  constexpr int NT = 256, QW = 32, QB = 4 * QW, PAD = PA_PAD_Q;
  char* smem = dyn_smem();                             // two buffers of (K tile | V tile)
  const long long item = pa_item(p);
  if (item >= p.items) return;
  const int tid = threadIdx.x, lane = tid & 63, wv = wave_uniform(tid >> 6);
  const int h2 = lane >> 5, lq = lane & 31;
  const int qb = wave_uniform(p.nblk - 1 - (int)(item % p.nblk));
  const int unit = wave_uniform((int)(item / p.nblk));
  const int upb = p.heads / p.gp;
  const int b = wave_uniform(unit / upb), head0 = wave_uniform((unit - b * upb) * p.gp);
  const int kvh = wave_uniform(head0 / (p.heads / p.kv_heads));
  const PRange rg = pa_range(p, b);
  const int n = rg.n, RT = 2 * p.R + 1 + 2 * PAD;
  float* tab = reinterpret_cast<float*>(smem + 4 * PA_TILE);
  float* dsum = tab + (1 + wv) * RT;
  float* skew = tab + 5 * RT + wv * (16 * PA_SKEW);
  const T* Qg = (const T*)p.Q + (size_t)b * p.bsq + head0 * 64;
  const T* Gg = (const T*)p.dO + (size_t)b * p.bsdo + head0 * 64;
  const T* Kg = (const T*)p.K + (size_t)b * p.bsk + kvh * 64;
  const T* Vg = (const T*)p.V + (size_t)b * p.bsv + kvh * 64;

  const int r_base = qb * QB;
  const int r_last = r_base + QB - 1 < p.rows - 1 ? r_base + QB - 1 : p.rows - 1;
  const int p0 = wave_uniform(rg.qs + pa_row(p, r_base).i), p1 = wave_uniform(rg.qs + pa_row(p, r_last).i);
  const PTiles tl = pa_tiles(p, n, p0, p1);
  const PWave w = pa_wave(p, rg, r_base + wv * QW, QW);

  vec<T, 8> qf[4], gf[4];
  const int row = r_base + wv * QW + lq;
  const bool row_ok = row < p.rows;
  const PRow rw = pa_row(p, row_ok ? row : p.rows - 1);
  const int pos = rg.qs + (row_ok ? rw.i : row);       // (past the last row: any position, its dS is zero)
  {
    const T* q = Qg + (size_t)rw.i * p.ldq + rw.g * 64;
    const T* g = Gg + (size_t)rw.i * p.lddo + rw.g * 64;
#pragma unroll
    for (int ks = 0; ks < 4; ++ks) {
      qf[ks] = *reinterpret_cast<const vec<T, 8>*>(q + ks * 16 + h2 * 8);
      gf[ks] = *reinterpret_cast<const vec<T, 8>*>(g + ks * 16 + h2 * 8);
    }
  }
  const float lse_in = p.lse[((size_t)b * p.heads + head0 + rw.g) * p.Nq + rw.i];
  const bool dead = !row_ok || lse_in == PA_NINF;      // P = 0
  float ref = dead ? -PA_NINF : lse_in * PA_LOG2E, ll = 0.f;   // P = exp2(y - ref - ll), y the score in base 2
  const bool large = wave_any(!dead && !(__builtin_fabsf(ref) <= PA_LARGE));
  if (lane == 0) p.st_large[((size_t)unit * p.nblk + qb) * 4 + wv] = large;
  if (large) ref = PA_NINF;                            // (the running maximum)
  const int hi = pa_hi(p, n, pos), lo0 = pa_lo(p, pos), lo = lo0;
  const int lo_c = lo0 < hi ? lo0 : hi;
  const bool sole = hi - lo_c + (p.sinks < lo_c ? p.sinks : lo_c) == 1;        // the row sees one key: P = 1
  constexpr bool FIT = __is_same(T, f16);              // dS is rounded as 2^ex dS: 2^ex and 2^-ex, known after the first walk
  float pw = 1.f, ipw = 1.f, amax = 0.f;               // amax: the largest |dP| of the visible keys
  float delta = 0.f, lsum = 0.f, delta_lo = 0.f, lsum_lo = 0.f, far_l = 0.f, far_r = 0.f;
  float sum_l = 0.f, sum_r = 0.f;                      // dS of far tiles: keys at -R or before, at R or past it; what the adds rounded away
  float low_l = 0.f, low_r = 0.f;
  if constexpr (BIAS) {
    pa_bias_table<NT, PAD>(p, head0, tab);
    for (int i = tid; i < 4 * RT + 64 * PA_SKEW; i += NT) tab[RT + i] = 0.f;
    block_sync();
    far_l = tab[0]; far_r = tab[RT - 1];
  }

  const int total = tl.na + tl.nb;
  auto tile_of = [&](int it) STAR_ALWAYS_INLINE { return it < tl.na ? it : it - tl.na + tl.b0; };
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
  const char* kfo[4];                                  // K rows (and V rows, one tile further) as the A operand of S^T and dP^T
#pragma unroll
  for (int ks = 0; ks < 4; ++ks) kfo[ks] = opaque(smem + swz_off(lq, ks * 2 + h2));
  const char* tfo[2][2];                               // K^T by transposing reads: the A operand of dQ^T = K^T dS^T
  {
    const int i = lane & 15, g = lane >> 4;
#pragma unroll
    for (int half = 0; half < 2; ++half)
#pragma unroll
      for (int db = 0; db < 2; ++db) {
        const int key = 8 * half + 4 * h2 + (i >> 2), d = 32 * db + 16 * (g & 1) + 4 * (i & 3);
        tfo[half][db] = opaque(smem + swz_off(key, d >> 3) + (d & 7) * 2);
      }
  }
  f32x16 acc[2];
#pragma unroll
  for (int c2 = 0; c2 < 2; ++c2)
#pragma unroll
    for (int r = 0; r < 16; ++r) acc[c2][r] = 0.f;

  // one tile of 64 keys.  WALK 0: delta and the row sum, 2: the same with the maximum (large rows, KIND 2 or 3), 1: dS and dQ.  KIND 0: every row sees
  // every key, the bias is one constant; 1: masks; 2: masks, the bias from the table, dS into the sums by relative position; 3: large rows, masks,
  // the bias one constant.  With a bias (two waves per SIMD: the table's LDS) KIND 0 takes
  // both halves' products first, the second half's run beside the first half's vector work; without, three waves per SIMD leave no registers for that
  auto body = [&](int k0, int bofs, bool masked, bool fl, float far, vec<T, 8>* ds, vec<T, 8>* dr, auto walk_tag, auto kind_tag) STAR_ALWAYS_INLINE {
    constexpr int WALK = decltype(walk_tag)::value, KIND = decltype(kind_tag)::value;
    constexpr bool AHEAD = KIND == 0 && !COMP && BIAS;
    f32x16 s[2], dp[2];
    auto products = [&](int kb) STAR_ALWAYS_INLINE {
#pragma unroll
      for (int r = 0; r < 16; ++r) { s[kb][r] = 0.f; dp[kb][r] = 0.f; }
#pragma unroll
      for (int ks = 0; ks < 4; ++ks) {
        const vec<T, 8> kf = *reinterpret_cast<const vec<T, 8>*>(kfo[ks] + bofs + kb * 4096);
        const vec<T, 8> vf = *reinterpret_cast<const vec<T, 8>*>(kfo[ks] + bofs + PA_TILE + kb * 4096);
        s[kb] = mfma32<T>(kf, qf[ks], s[kb]);
        dp[kb] = mfma32<T>(vf, gf[ks], dp[kb]);
      }
    };
    if constexpr (AHEAD) { products(0); products(1); }
    const float off = (far - ref) - ll;
    float t0 = 0.f, t1 = 0.f, l0 = 0.f, l1 = 0.f;        // this tile's sums
#pragma unroll
    for (int kb = 0; kb < 2; ++kb) {
      if constexpr (!AHEAD) { STAR_SCHED_FENCE(); products(kb); }
      const int at = k0 + kb * 32 + 4 * h2 - pos + p.R + PAD;                  // the table's entry of the lane's first key
      float base = 0.f;                                  // WALK 2: the maximum, 0 while there is none
      if constexpr (WALK == 2) {
        float mx = PA_NINF;
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const int j = (r & 3) + 8 * (r >> 2), key = k0 + kb * 32 + j + 4 * h2;
          const float y = __builtin_fmaf(s[kb][r], p.c, KIND == 2 ? tab[at + j] : far);
          s[kb][r] = !masked | ((key < hi) & ((key >= lo) | (key < p.sinks))) ? y : PA_NINF;
          mx = fmaxf(mx, s[kb][r]);
        }
        const float m_new = fmaxf(ref, pair_max(mx));
        const float f = m_new == PA_NINF ? 1.f : fast_exp2(ref - m_new);
        ref = m_new;
        base = m_new == PA_NINF ? 0.f : m_new;
        lsum *= f; lsum_lo *= f; delta *= f; delta_lo *= f;
        t0 *= f; t1 *= f; l0 *= f; l1 *= f;
      }
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const int j = (r & 3) + 8 * (r >> 2), key = k0 + kb * 32 + j + 4 * h2;
        float x;
        if constexpr (WALK == 2) x = s[kb][r] - base;
        else if constexpr (KIND >= 2) {
          x = __builtin_fmaf(s[kb][r], p.c, KIND == 2 ? tab[at + j] : far) - ref;
          if constexpr (WALK == 1) x -= ll;
        } else x = __builtin_fmaf(s[kb][r], p.c, off);
        bool see = true;
        if constexpr (WALK == 2) see = s[kb][r] != PA_NINF;
        else if constexpr (KIND != 0) {
          see = !masked | ((key < hi) & ((key >= lo) | (key < p.sinks)));
          if constexpr (WALK == 1) x = sole ? 0.f : x;
        }
        float pr = fast_exp2(x);
        if constexpr (KIND != 0) pr = see ? pr : 0.f;
        if constexpr (WALK != 1) {
          const float d = KIND != 0 ? (see ? dp[kb][r] : 0.f) : dp[kb][r];
          if constexpr (FIT) amax = fmaxf(amax, __builtin_fabsf(d));
          const float wt = KIND != 0 && sole ? 1.f : pr; // (delta is dP itself, whatever the last bit of P)
          if (r & 1) { l1 += pr; t1 = __builtin_fmaf(wt, d, t1); }
          else { l0 += pr; t0 = __builtin_fmaf(wt, d, t0); }
        } else {
          // (subtracted at the end: a row with one visible key has dP - delta = 0 exactly, and sums that start at -delta cost the table's
          // gradient half of its digits past 1e-6)
          float v = pr * (FIT ? __builtin_fmaf(dp[kb][r], pw, -delta) : dp[kb][r] - delta);
          if constexpr (KIND != 0) v = see ? v : 0.f;
          T hi16, lo16{};
          pa_round<T, COMP>(v, hi16, lo16);
          ds[2 * kb + (r >> 3)][r & 7] = hi16;
          if constexpr (COMP) dr[2 * kb + (r >> 3)][r & 7] = lo16;
          if constexpr (BIAS && KIND != 2) { if (r & 1) t1 += v; else t0 += v; }
          if constexpr (KIND == 2) {
            // sums along the diagonals, sixteen keys at a time: each row of values is stored one word further on, so that a relative
            // position becomes a column (the other cells of a row stay zero), and a lane adds up a column.  The rows' positions go
            // up by one lane by lane: with a bias a unit is one head
            skew[((j & 15) + 4 * h2) * (PA_SKEW + 1) - lq + 31] = v * ipw;
            if ((r & 7) == 7) {
              wave_lds_order();
              if (lane < PA_SKEW - 1) {
                float c0 = 0.f, c1 = 0.f;
#pragma unroll
                for (int i = 0; i < 16; i += 2) { c0 += skew[i * PA_SKEW + lane]; c1 += skew[(i + 1) * PA_SKEW + lane]; }
                float* to = dsum + (k0 + kb * 32 + 16 * (r >> 3) - (w.p0 + 31) + p.R + PAD) + lane;
                *to += c0 + c1;
              }
              wave_lds_order();
            }
          }
        }
      }
    }
    if constexpr (WALK != 1) {
      // (with a bias to 2^-48: what delta is off by stays in the sums over millions of pairs that make up the table's gradient)
      if constexpr (BIAS) { pa_add2(lsum, lsum_lo, l0 + l1); pa_add2(delta, delta_lo, t0 + t1); }
      else { lsum += l0 + l1; delta += t0 + t1; }
    }
    else if constexpr (BIAS && KIND != 2) {
      const float t = (t0 + t1) * ipw;
      pa_add2(sum_l, low_l, fl ? t : 0.f);
      pa_add2(sum_r, low_r, fl ? 0.f : t);
    }
  };
  auto tile = [&](int it, int buf, auto walk_tag, auto large_tag) STAR_ALWAYS_INLINE {
    constexpr bool LARGE = decltype(large_tag)::value;
    const int k0 = tile_of(it) * PA_KT, bofs = buf * 2 * PA_TILE;
    if (!pa_sees(p, w, k0)) return;
    const bool masked = !pa_sees_whole(p, w, k0);
    bool near = false, fl = false;
    float far = 0.f;
    if constexpr (BIAS) {
      fl = k0 + PA_KT - 1 - w.p0 <= -p.R;
      near = !(fl || k0 - w.p1 >= p.R);
      far = fl ? far_l : far_r;
    }
    vec<T, 8> ds[4], dr[4];                            // 2^ex dS, sixteen keys each, and what its rounding left
    auto with = [&](auto kind_tag) STAR_ALWAYS_INLINE { body(k0, bofs, masked, fl, far, ds, dr, walk_tag, kind_tag); };
    if (BIAS && near) with(std::integral_constant<int, BIAS ? 2 : 3>{});
    else if constexpr (LARGE) with(std::integral_constant<int, 3>{});
    else if (masked) with(std::integral_constant<int, 1>{});
    else with(std::integral_constant<int, 0>{});
    if constexpr (decltype(walk_tag)::value == 1) {    // (outside the kinds: accumulators that they all write are copied from one to the other)
#pragma unroll
      for (int u = 0; u < 4; ++u)
#pragma unroll
        for (int db = 0; db < 2; ++db) {
          vec<T, 8> kt;
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            const vec<T, 4> r = lds_read_tr<T>(tfo[half][db] + bofs + u * 2048);
#pragma unroll
            for (int e = 0; e < 4; ++e) kt[half * 4 + e] = r[e];
          }
          acc[db] = mfma32<T>(kt, ds[u], acc[db]);
          if constexpr (COMP) acc[db] = mfma32<T>(kt, dr[u], acc[db]);
        }
    }
  };

  glds_wait();
  if (total) stage(0, 0);
  // both walks; a wave with large rows has its own copy of them (with the same barriers), so that the others' code stays as it is without: kinds for
  // them in one copy cost 13 %
  auto walks = [&](auto large_tag) STAR_ALWAYS_INLINE {
    int buf = 0;
    for (int it = 0; it < total; ++it, buf ^= 1) {
      glds_wait(); block_sync();
      stage(it + 1 < total ? it + 1 : 0, buf ^ 1);     // (the second walk's first tile behind the last)
      tile(it, buf, std::integral_constant<int, decltype(large_tag)::value ? 2 : 0>{}, large_tag);
    }
    const float l = pair_sum(lsum + lsum_lo), d = pair_sum(delta + delta_lo);
    delta = sole ? d : l > 0.f ? d / l : l == 0.f ? 0.f : l;
    if (l > 0.f) ll = __builtin_log2f(l);
    if (dead || ref == PA_NINF) ref = -PA_NINF;
    if constexpr (FIT) amax = pair_max(amax);
    if (row_ok && h2 == 0) {
      const size_t at = (size_t)unit * p.rows + row;
      p.st_ref[at] = ref;
      p.st_log[at] = ll;
      p.st_delta[at] = delta;
      if constexpr (FIT) p.st_amax[at] = amax;
    }
    if constexpr (FIT) {
      const int ex = pa_fit_exp(amax);
      pw = pa_pow2(ex); ipw = pa_pow2(-ex);
      delta *= pw;                                     // (a power of two: dP 2^ex - delta 2^ex is as exact as dP - delta)
    }
    for (int it = 0; it < total; ++it, buf ^= 1) {
      glds_wait(); block_sync();
      if (it + 1 < total) stage(it + 1, buf ^ 1);
      tile(it, buf, std::integral_constant<int, 1>{}, large_tag);
    }
  };
  if (__builtin_expect(large, 0)) walks(std::true_type{});
  else walks(std::false_type{});
  pa_store_row<T>(acc, p.scale * ipw, (T*)p.dQ + (size_t)b * p.bsdq + (size_t)rw.i * p.lddq + (head0 + rw.g) * 64, row_ok);
  if constexpr (BIAS) {
    const float tl2 = wave_sum(sum_l + low_l), tr2 = wave_sum(sum_r + low_r);
    block_sync();                                      // every wave is past its last read of a tile: the buffers' first words are free
    float* ends = reinterpret_cast<float*>(smem);
    if (lane == 0) { ends[wv] = tl2; ends[4 + wv] = tr2; }
    block_sync();
    // entry i of the arrays belongs to j - p = i - R - PAD; what lies at +-R and past it joins the far tiles' sums
    auto column = [&](int i) { return (tab[RT + i] + tab[2 * RT + i]) + (tab[3 * RT + i] + tab[4 * RT + i]); };
    const int R2 = 2 * p.R + 1;
    float* rel = ends + 16;                            // [R2] sums by relative position, their buckets [R2], the threads' parts [256]
    int* of = reinterpret_cast<int*>(rel + R2);
    float* part = rel + 2 * R2;
    for (int i = tid; i < R2; i += NT) {
      const int c = p.buckets[i];
      of[i] = c < 0 ? 0 : c >= p.num_buckets ? p.num_buckets - 1 : c;
      if (i > 0 && i < R2 - 1) rel[i] = column(i + PAD);
    }
    float e = 0.f;                                     // first wave: the columns up to -R; last wave: from R on (R = 0: past it)
    if (wv == 0) for (int i = lane; i <= PAD; i += 64) e += column(i);
    if (wv == 3) for (int i = lane; i <= PAD - (p.R == 0); i += 64) e += column(RT - 1 - i);
    e = wave_sum(e);
    if (lane == 0) ends[8 + wv] = e;
    block_sync();
    if (tid == 0) {
      const float left = ends[8] + ((ends[0] + ends[1]) + (ends[2] + ends[3])), right = ends[11] + ((ends[4] + ends[5]) + (ends[6] + ends[7]));
      if (p.R > 0) { rel[0] = left; rel[R2 - 1] = right; }
      else rel[0] = left + right;
    }
    block_sync();
    // by bucket: its entries are shared out among `slices` threads, joined in a fixed order
    float* out = p.dsum + ((size_t)unit * p.nblk + qb) * p.num_buckets;
    int nb = 1;
    while (nb < p.num_buckets && nb < NT) nb <<= 1;
    const int slices = NT / nb, me = tid / nb;
    for (int b0 = 0; b0 < p.num_buckets; b0 += nb) {
      const int k = b0 + tid % nb;
      float v = 0.f;
#pragma unroll 4
      for (int i = me; i < R2; i += slices) { const float x = rel[i]; v += of[i] == k ? x : 0.f; }
      part[tid] = v;
      block_sync();
      if (me == 0 && k < p.num_buckets) {
        for (int j = 1; j < slices; ++j) v += part[j * nb + tid];
        out[k] = v;
      }
      block_sync();
    }
  }
}

// the part of a key block that a slot of a unit stands for
struct PSlot { int kblk, part, parts; };
STAR_DEV PSlot pa_slot(const PAttnParams& p, int slot) {
  const int first = p.sblk * p.split_s;
  if (slot < first) { const int k = wave_uniform(slot / p.split_s); return PSlot{k, slot - k * p.split_s, p.split_s}; }
  const int k = wave_uniform((slot - first) / p.split_n);
  return PSlot{p.sblk + k, slot - first - k * p.split_n, p.split_n};
}

template <class T, int BIAS, int COMP>
STAR_GLOBAL void STAR_LAUNCH_BOUNDS(256, 2)
pattn_dkdv_kernel(const PAttnParams p) {
  constexpr int NT = 256, KB = 128, QT = 64;           // keys per workgroup, query rows per tile
  constexpr int SHIFT = __is_same(T, f16) ? 10 : 0;    // P is rounded as 2^SHIFT P
  constexpr int ROWB = PA_ROWB, BUF = 2 * PA_TILE + ROWB;        // Q tile | dO tile | off[64] | -delta[64] | pos[64] | ref[64] | log[64] | exponent
  char* smem = dyn_smem();                             // two such buffers, then the bias table
  const long long item = pa_item(p);
  if (item >= p.items) return;
  const int tid = threadIdx.x, lane = tid & 63, wv = wave_uniform(tid >> 6);
  const int h2 = lane >> 5, lq = lane & 31;
  const PSlot sl = pa_slot(p, wave_uniform((int)(item % p.nblk)));    // nblk: slots per unit
  const int kblk = sl.kblk;
  const int ku = wave_uniform((int)(item / p.nblk));   // (sequence, K / V head); one sequence where the batch shares K and V
  const int kb0 = wave_uniform(ku / p.kv_heads), kvh = ku - kb0 * p.kv_heads;
  const bool shared = p.batch > 1 && p.bsk == 0 && p.bsv == 0;
  const int j0 = kblk * KB, jw = j0 + wv * 32, key = jw + lq;
  float* tab = reinterpret_cast<float*>(smem + 2 * BUF);

  vec<T, 8> kf[4], vf[4];
  {
    const int nk = shared ? p.Nk : pa_range(p, kb0).n;
    const T* K = (const T*)p.K + (size_t)kb0 * p.bsk + kvh * 64 + (size_t)(key < nk ? key : 0) * p.ldk;
    const T* V = (const T*)p.V + (size_t)kb0 * p.bsv + kvh * 64 + (size_t)(key < nk ? key : 0) * p.ldv;
#pragma unroll
    for (int ks = 0; ks < 4; ++ks) {
#pragma unroll
      for (int e = 0; e < 8; ++e) { kf[ks][e] = from_f32<T>(0.f); vf[ks][e] = from_f32<T>(0.f); }
      if (key < nk) {
        kf[ks] = *reinterpret_cast<const vec<T, 8>*>(K + ks * 16 + h2 * 8);
        vf[ks] = *reinterpret_cast<const vec<T, 8>*>(V + ks * 16 + h2 * 8);
      }
    }
  }
  f32x16 dk[2], dv[2];
#pragma unroll
  for (int c2 = 0; c2 < 2; ++c2)
#pragma unroll
    for (int r = 0; r < 16; ++r) { dk[c2][r] = 0.f; dv[c2][r] = 0.f; }

  const char* afo[4];                                  // Q rows (and dO rows, one tile further) as the A operand of S and dP
#pragma unroll
  for (int ks = 0; ks < 4; ++ks) afo[ks] = opaque(smem + swz_off(lq, ks * 2 + h2));
  const char* tfo[2][2];                               // Q^T (and dO^T) by transposing reads: the A operands of dK^T and dV^T
  {
    const int i = lane & 15, g = lane >> 4;
#pragma unroll
    for (int half = 0; half < 2; ++half)
#pragma unroll
      for (int db = 0; db < 2; ++db) {
        const int q = 8 * half + 4 * h2 + (i >> 2), d = 32 * db + 16 * (g & 1) + 4 * (i & 3);
        tfo[half][db] = opaque(smem + swz_off(q, d >> 3) + (d & 7) * 2);
      }
  }

  const int G = wave_uniform(p.heads / p.kv_heads), subs = wave_uniform(G / p.gp), upb = wave_uniform(p.heads / p.gp);
  const int nb = shared ? p.batch : 1;
  // the tiles [t0, t1) of the rows of sequence b that see some key of the block
  auto tiles_of = [&](const PRange& rg, int& t0, int& t1) STAR_ALWAYS_INLINE {
    const int j1 = j0 + KB - 1 < rg.n - 1 ? j0 + KB - 1 : rg.n - 1;
    int i0 = j0 - p.right - rg.qs, i1 = j0 < p.sinks ? p.Nq : j1 + p.left - rg.qs + 1;
    i0 = i0 < 0 ? 0 : i0; i1 = i1 > p.Nq ? p.Nq : i1;
    t0 = 0; t1 = 0;
    if (j0 < rg.n && i0 < i1) { t0 = (int)((long long)i0 * p.gp / QT); t1 = (int)(((long long)i1 * p.gp + QT - 1) / QT); }
  };
  // this part's share of all tiles, counted over the heads of the group and the sequences one after the other
  long long first = 0, last = 0x7fffffffffffLL;
  if (sl.parts > 1) {
    long long all = 0;
    for (int b = shared ? 0 : kb0; b < (shared ? p.batch : kb0 + 1); ++b) {
      int t0, t1;
      tiles_of(pa_range(p, b), t0, t1);
      all += (long long)(t1 - t0) * subs;
    }
    first = all * sl.part / sl.parts; last = all * (sl.part + 1) / sl.parts;
  }
  long long done = 0;                                  // tiles before the current head's
  int E = PA_EXP_MAX;                                  // f16: dK is summed as 2^E dK
  for (int w = 0; w < nb * subs; ++w) {
    const int b = shared ? wave_uniform(w / subs) : kb0, sub = shared ? w - b * subs : w;
    const int head0 = kvh * G + sub * p.gp, unit = b * upb + kvh * subs + sub;
    const PRange rg = pa_range(p, b);
    const int n = rg.n;
    int t0, t1;
    tiles_of(rg, t0, t1);
    const long long here = done;
    done += t1 - t0;
    if (sl.parts > 1) {
      const long long lo = first - here, hi = last - here;
      const int base = t0, cnt = t1 - t0;
      t0 = wave_uniform(base + (int)(lo < 0 ? 0 : lo > cnt ? cnt : lo)); t1 = wave_uniform(base + (int)(hi < 0 ? 0 : hi > cnt ? cnt : hi));
    }
    if (t0 >= t1) continue;
    const T* Qg = (const T*)p.Q + (size_t)b * p.bsq + head0 * 64;
    const T* Gg = (const T*)p.dO + (size_t)b * p.bsdo + head0 * 64;
    float far_l = 0.f, far_r = 0.f;
    if constexpr (BIAS) {
      block_sync();                                    // the last tile's readers are done with the table
      pa_bias_table<NT, PA_PAD_K>(p, head0, tab);
      block_sync();
      far_l = tab[0]; far_r = tab[2 * p.R + 2 * PA_PAD_K];
    } else block_sync();
    bool large = false;                                  // (no bias) some of the rows are large
    int reach = p.R;                                     // where the bias is one constant

    auto bounds = [&](int t, int& pa, int& pb) STAR_ALWAYS_INLINE {    // positions of a tile's first and last row
      const int rl = t * QT + QT - 1 < p.rows - 1 ? t * QT + QT - 1 : p.rows - 1;
      pa = wave_uniform(rg.qs + pa_row(p, t * QT).i); pb = wave_uniform(rg.qs + pa_row(p, rl).i);
    };
    auto stage = [&](int t, int buf) STAR_ALWAYS_INLINE {
      const int d = buf * BUF;
      const int r0 = t * QT, i_first = wave_uniform(pa_row(p, r0).i);
      const T* qb = Qg + (size_t)i_first * p.ldq;
      const T* gb = Gg + (size_t)i_first * p.lddo;
      auto at = [&](int r, int ch, int ld) {
        const PRow rw = pa_row(p, r0 + r);
        return r0 + r < p.rows ? (uint32_t)((rw.i - i_first) * ld + rw.g * 64 + ch * 8) * 2u : GLDS_BUF_OOB;
      };
      pa_stage<NT>(qb, smem, d, tid, wv, [&](int r, int ch) { return at(r, ch, p.ldq); });
      pa_stage<NT>(gb, smem, d + PA_TILE, tid, wv, [&](int r, int ch) { return at(r, ch, p.lddo); });
    };
    // a row's statistics: loaded by the first wave a tile ahead, written to LDS when the tile's turn comes
    float x_ref = 0.f, x_log = 0.f, x_delta = 0.f, x_amax = 0.f;
    auto load_rows = [&](int t) STAR_ALWAYS_INLINE {
      const int r = t * QT + tid;
      x_ref = -PA_NINF; x_log = 0.f; x_delta = 0.f; x_amax = 0.f;
      if (tid < QT && r < p.rows) {
        const size_t a = (size_t)unit * p.rows + r;
        x_ref = p.st_ref[a]; x_log = p.st_log[a]; x_delta = p.st_delta[a];
        if constexpr (SHIFT) x_amax = p.st_amax[a];
      }
    };
    int e_row = E;                                       // (first wave) the exponent up to the tile being written
    auto write_rows = [&](int t, int buf) STAR_ALWAYS_INLINE {
      if (wv) return;
      float* o = reinterpret_cast<float*>(smem + buf * BUF + 2 * PA_TILE);
      float far = 0.f;
      if constexpr (BIAS) {
        int pa, pb;
        bounds(t, pa, pb);
        if (j0 + KB - 1 - pa <= -p.R) far = far_l;
        else if (j0 - pb >= p.R) far = far_r;
      }
      if constexpr (SHIFT) {
        const float m = wave_max(x_amax);
        if (m > 0.f) { const int e = pa_fit_exp(m); if (e < e_row) e_row = e; }
      }
      o[tid] = (far - x_ref) - x_log + (float)SHIFT;
      o[64 + tid] = -x_delta;
      reinterpret_cast<int*>(o)[128 + tid] = rg.qs + pa_row(p, t * QT + tid).i;
      o[192 + tid] = x_ref;
      o[256 + tid] = (float)SHIFT - x_log;
      if (SHIFT && tid == 0) reinterpret_cast<int*>(o)[320] = e_row;
    };

    auto tile = [&](int t, int buf) STAR_ALWAYS_INLINE {
      int pa, pb;
      bounds(t, pa, pb);
      const int jl = jw + 31;
      const int bofs = buf * BUF;
      const float* o = reinterpret_cast<const float*>(smem + bofs + 2 * PA_TILE);
      float pw = 1.f;
      if constexpr (SHIFT) {
        const int e = wave_uniform(reinterpret_cast<const int*>(o)[320]);
        if (e != E) {                                    // larger gradients than so far: lower the common exponent
          const float f = pa_pow2(e - E);
#pragma unroll
          for (int c2 = 0; c2 < 2; ++c2)
#pragma unroll
            for (int r = 0; r < 16; ++r) dk[c2][r] *= f;
          E = e;
        }
        pw = pa_pow2(E - SHIFT);
      }
      if (jw >= n || jw > pb + p.right || (jl < pa - p.left && jw >= p.sinks)) return;   // no row of the tile sees a key of the wave
      const bool masked = !(jl < n && jl <= pa + p.right && (jw >= pb - p.left || jl < p.sinks));
      const bool near = BIAS ? !(j0 + KB - 1 - pa <= -reach || j0 - pb >= reach) : false;
      const bool table = BIAS && near, plain = !table && !masked && !large;
#pragma unroll
      for (int qs = 0; qs < 2; ++qs) {
        f32x16 s, dp;
#pragma unroll
        for (int r = 0; r < 16; ++r) { s[r] = 0.f; dp[r] = 0.f; }
        if (plain) {                                     // the sums of dP start at -delta (else it is added at the end, as in dQ)
#pragma unroll
          for (int g = 0; g < 4; ++g) {
            const f32x4 dl = *reinterpret_cast<const f32x4*>(o + 64 + qs * 32 + 8 * g + 4 * h2);
#pragma unroll
            for (int e = 0; e < 4; ++e) dp[4 * g + e] = dl[e];
          }
        }
#pragma unroll
        for (int ks = 0; ks < 4; ++ks) {
          const vec<T, 8> a = *reinterpret_cast<const vec<T, 8>*>(afo[ks] + bofs + qs * 4096);
          const vec<T, 8> g = *reinterpret_cast<const vec<T, 8>*>(afo[ks] + bofs + PA_TILE + qs * 4096);
          s = mfma32<T>(a, kf[ks], s);
          dp = mfma32<T>(g, vf[ks], dp);
        }
        vec<T, 8> pf[2], df[2], pl[2], dl8[2];           // P and dS, sixteen rows each, and what their rounding left
        // KIND 0: every row sees every key, the bias is one constant (in off); 1: masks; 2: masks, and the bias from the table (past its ends too: the
        // end values go on there); 3: large rows without a bias, masks.  2 and 3 (EACH) round the score as the forward pass does before the row's
        // reference is subtracted
        auto weights = [&](auto kind_tag) STAR_ALWAYS_INLINE {
          constexpr int KIND = decltype(kind_tag)::value;
#pragma unroll
          for (int g = 0; g < 4; ++g) {                  // rows 8 g + 4 h2 + (0 .. 3) of the 32
            const int row = qs * 32 + 8 * g + 4 * h2;
            constexpr bool EACH = KIND == (BIAS ? 2 : 3);
            f32x4 off{};
            if constexpr (!EACH) off = *reinterpret_cast<const f32x4*>(o + row);
            vec<int, 4> ps{};
            f32x4 dl{};
            if constexpr (KIND != 0) {
              dl = *reinterpret_cast<const f32x4*>(o + 64 + row);
              ps = *reinterpret_cast<const vec<int, 4>*>(reinterpret_cast<const int*>(o) + 128 + row);
            }
            // (with a bias a unit is one head: row by row the positions go up by one)
            const float* tb = nullptr;
            f32x4 ref{}, lg{};
            if constexpr (EACH) {
              ref = *reinterpret_cast<const f32x4*>(o + 192 + row);
              lg = *reinterpret_cast<const f32x4*>(o + 256 + row);
              int at = key - (rg.qs + t * QT + row + 3) + p.R + PA_PAD_K;
              at = at < 0 ? 0 : at > 2 * p.R + 2 * PA_PAD_K - 3 ? 2 * p.R + 2 * PA_PAD_K - 3 : at;
              tb = tab + at;
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const int r = 4 * g + e;
              float x;
              if constexpr (EACH) x = (__builtin_fmaf(s[r], p.c, BIAS ? tb[3 - e] : 0.f) - ref[e]) + lg[e];
              else x = __builtin_fmaf(s[r], p.c, off[e]);
              float pr = fast_exp2(x);
              const float d0 = KIND == 0 ? dp[r] : dp[r] + dl[e];
              float v = pr * (SHIFT ? d0 * pw : d0);
              if constexpr (KIND != 0) {
                const int rel = key - ps[e];
                const bool see = !masked | ((key < n) & (rel <= p.right) & ((rel >= -p.left) | (key < p.sinks)));
                pr = see ? pr : 0.f;
                v = see ? v : 0.f;
              }
              T a, al{}, d, dl_{};
              pa_round<T, COMP>(pr, a, al);
              pa_round<T, COMP>(v, d, dl_);
              pf[g >> 1][(g & 1) * 4 + e] = a; df[g >> 1][(g & 1) * 4 + e] = d;
              if constexpr (COMP) { pl[g >> 1][(g & 1) * 4 + e] = al; dl8[g >> 1][(g & 1) * 4 + e] = dl_; }
            }
          }
        };
        if (table) weights(std::integral_constant<int, BIAS ? 2 : 1>{});
        else if (!BIAS && large) weights(std::integral_constant<int, BIAS ? 1 : 3>{});
        else if (masked) weights(std::integral_constant<int, 1>{});
        else weights(std::integral_constant<int, 0>{});
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
          for (int db = 0; db < 2; ++db) {
            vec<T, 8> qt, gt;
#pragma unroll
            for (int half = 0; half < 2; ++half) {
              const vec<T, 4> a = lds_read_tr<T>(tfo[half][db] + bofs + (qs * 2 + u) * 2048);
              const vec<T, 4> g = lds_read_tr<T>(tfo[half][db] + bofs + PA_TILE + (qs * 2 + u) * 2048);
#pragma unroll
              for (int e = 0; e < 4; ++e) { qt[half * 4 + e] = a[e]; gt[half * 4 + e] = g[e]; }
            }
            dv[db] = mfma32<T>(gt, pf[u], dv[db]);
            dk[db] = mfma32<T>(qt, df[u], dk[db]);
            if constexpr (COMP) {
              dv[db] = mfma32<T>(gt, pl[u], dv[db]);
              dk[db] = mfma32<T>(qt, dl8[u], dk[db]);
            }
          }
      }
    };

    int some = 0;                                        // of the tiles' rows, 32 to a word
    for (int i = 2 * t0 + lane; i < 2 * t1; i += 64) some |= p.st_large[(size_t)unit * p.nlarge + i];
    load_rows(t0);
    glds_wait();                                         // no compiler-visible load in flight beside the hand-written DMA's first use
    // with a large row among them all tiles take the kind that rounds the scores one by one; with a bias as if all were near.  (This costs the others
    // 2 % of this kernel; a kind of its own with a bias, too, or a flag per tile 4 - 5 %)
    if (wave_any(some)) { if (BIAS) reach = 1 << 30; else large = true; }
    stage(t0, 0);
    for (int t = t0; t < t1; ++t) {
      const int buf = (t - t0) & 1;
      write_rows(t, buf);
      glds_wait(); block_sync();
      if (t + 1 < t1) { load_rows(t + 1); stage(t + 1, buf ^ 1); }
      tile(t, buf);
    }
  }

  const float mk = p.scale * (SHIFT ? pa_pow2(-E) : 1.f), mv = pa_pow2(-SHIFT);
  if (sl.parts > 1) {
    // [unit][slot][key][dK 64 | dV 64]; only blocks in parts have slots there
    const int per = p.split_n > 1 ? p.nblk : p.sblk * p.split_s;
    float* o = p.part + (((size_t)ku * per + (int)(item % p.nblk)) * KB + wv * 32 + lq) * 128;
#pragma unroll
    for (int db = 0; db < 2; ++db)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        f32x4 a, c;
#pragma unroll
        for (int e = 0; e < 4; ++e) { a[e] = dk[db][g * 4 + e] * mk; c[e] = dv[db][g * 4 + e] * mv; }
        *reinterpret_cast<f32x4*>(o + 32 * db + 8 * g + 4 * h2) = a;
        *reinterpret_cast<f32x4*>(o + 64 + 32 * db + 8 * g + 4 * h2) = c;
      }
    return;
  }
  const int ob = shared ? 0 : kb0;
  const bool ok = key < p.Nk;
  pa_store_row<T>(dk, mk, (T*)p.dK + (size_t)ob * p.bsdk + (size_t)(ok ? key : 0) * p.lddk + kvh * 64, ok);
  pa_store_row<T>(dv, mv, (T*)p.dV + (size_t)ob * p.bsdv + (size_t)(ok ? key : 0) * p.lddv + kvh * 64, ok);
}

// adds the parts of the key blocks that were split, in their order: eight workgroups per block, a thread per eight values
template <class T>
STAR_GLOBAL void STAR_LAUNCH_BOUNDS(256)
pattn_dkdv_join_kernel(const PAttnParams p) {
  const int first = p.sblk * p.split_s;                // slots of the first blocks
  const int nsplit = p.split_n > 1 ? p.sblk + (p.nblk - first) / p.split_n : p.sblk;      // blocks in parts (all, or those of the first tokens)
  const int ku = blockIdx.x / nsplit, k = blockIdx.x - ku * nsplit;
  const int parts = k < p.sblk ? p.split_s : p.split_n;
  const int slot = k < p.sblk ? k * p.split_s : first + (k - p.sblk) * p.split_n;
  const int per = p.split_n > 1 ? p.nblk : first;
  const int b = ku / p.kv_heads, kvh = ku - b * p.kv_heads;
  const float* src = p.part + ((size_t)ku * per + slot) * 128 * 128;
  for (int i = blockIdx.y * 256 + threadIdx.x; i < 128 * 16; i += 256 * gridDim.y) {
    const int row = i >> 4, c = (i & 15) * 8, key = k * 128 + row;
    if (key >= p.Nk) continue;
    float v[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = 0.f;
    for (int q = 0; q < parts; ++q) {
      const f32x4* a = reinterpret_cast<const f32x4*>(src + ((size_t)q * 128 + row) * 128 + c);
#pragma unroll
      for (int e = 0; e < 4; ++e) { v[e] += a[0][e]; v[4 + e] += a[1][e]; }
    }
    vec<T, 8> o;
#pragma unroll
    for (int e = 0; e < 8; ++e) o[e] = from_f32<T>(v[e]);
    T* dst = c < 64 ? (T*)p.dK + (size_t)b * p.bsdk + (size_t)key * p.lddk + kvh * 64 + c : (T*)p.dV + (size_t)b * p.bsdv + (size_t)key * p.lddv + kvh * 64 + c - 64;
    *reinterpret_cast<vec<T, 8>*>(dst) = o;
  }
}

// dtable[k][h]: the row blocks' sums of a head by bucket, in double and in a fixed order; the blocks are shared out among `slices` threads
struct PDTableParams { const float* dsum; float* dtable; int batch, heads, nblk, num_buckets; };
STAR_GLOBAL void STAR_LAUNCH_BOUNDS(256)
pattn_dtable_kernel(const PDTableParams p) {
  double* part = reinterpret_cast<double*>(dyn_smem());               // [256]
  const int h = blockIdx.x, tid = threadIdx.x;
  const long long n = (long long)p.batch * p.nblk;
  int nb = 1;
  while (nb < p.num_buckets && nb < 256) nb <<= 1;
  const int slices = 256 / nb, me = tid / nb;
  for (int b0 = 0; b0 < p.num_buckets; b0 += nb) {
    const int k = b0 + tid % nb;
    double s = 0.0;
    if (k < p.num_buckets) {
#pragma unroll 4
      for (long long i = me; i < n; i += slices) {
        const long long b = i / p.nblk;
        s += (double)p.dsum[((size_t)(b * p.heads + h) * p.nblk + (i - b * p.nblk)) * p.num_buckets + k];
      }
    }
    part[tid] = s;
    block_sync();
    if (me == 0 && k < p.num_buckets) {
      for (int j = 1; j < slices; ++j) s += part[j * nb + tid];
      p.dtable[(size_t)k * p.heads + h] = (float)s;
    }
    block_sync();
  }
}

}  // namespace star
