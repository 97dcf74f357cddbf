// ln_train.h -- LayerNorm for training: the forward pass that keeps its row statistics, and the backward pass with the reduction of
// the weight's gradient.  x, y, dy, dx: rows in the context's 16-bit type; gamma, beta, their gradients and the statistics: fp32.
//
//   mu = mean(x), r = 1 / sqrt(mean((x - mu)^2) + eps), xh = (x - mu) r, y = xh gamma + beta        stats[row] = (mu, r)
//   a = dy gamma, dx = r (a - mean(a) - xh mean(a xh)),  dgamma = sum_rows dy xh,  dbeta = sum_rows dy
//
// Both passes move every row once (forward 4 bytes per element, backward 6) and are bound by HBM: f16, 843 264 x 320 forward 199 us = 5.4 TB/s,
// 214 272 x 640 backward 197 us = 4.2 TB/s, where a copy of 2 GiB runs at 4.9.  A few hundred rows are the latency of the launches:
// 154 x 1024 forward 4 us, 616 x 1024 backward 8 us + 3 us for the sums.  (The next row's loads ahead of this one's sums lost: 207 -> 262 us.)  A row is held in registers as it
// was read (16-bit, four registers per 16-byte chunk), the two moments are taken from it there: one read, no second pass over memory.
// LPR lanes share a row (the least power of two that holds it in CPL chunks per lane, at least eight where the row has eight chunks,
// so that a group reads whole 128-byte lines); rows past 64 x CPL chunks take a whole workgroup (WG).
// The weight's gradient: a lane owns the same columns in every row that its group visits and adds dy xh and dy up in registers; a
// workgroup walks many rows, joins its groups in LDS and writes one partial row of 2 C sums; a second launch adds the partial rows in a
// fixed order.  No atomics: the same call gives the same bits.
#pragma once
#include "prim.h"

namespace star {

struct LnTrainParams {
  const void* x; const void* dy; void* out;       // out: y (forward) or dx (backward)
  const float* gamma; const float* beta;          // null: 1 and 0
  float* stats;                                   // [rows][2]
  float* partial;                                 // backward: [gridDim.x][2][C] or null
  long long ldx, lddy, ldo;
  int rows, C, lpr;                               // lpr: lanes per row (unused in the WG form)
  int stream;                                     // the output is larger than the caches: store past them
  float eps;
};

// chunk of eight columns; VEC: 16-byte access (C, strides and bases multiples of eight elements), else element by element
template <class T, bool VEC>
STAR_DEV vec<T, 8> ln_load(const T* p, int n) {
  if constexpr (VEC) return *reinterpret_cast<const vec<T, 8>*>(p);
  vec<T, 8> v;
#pragma unroll
  for (int e = 0; e < 8; ++e) v[e] = e < n ? p[e] : from_f32<T>(0.f);
  return v;
}
template <class T, bool VEC, bool STREAM>
STAR_DEV void ln_store(T* p, vec<T, 8> v, int n) {
  if constexpr (VEC) {
    if constexpr (STREAM) store_nt(reinterpret_cast<vec<T, 8>*>(p), v);
    else *reinterpret_cast<vec<T, 8>*>(p) = v;
    return;
  }
#pragma unroll
  for (int e = 0; e < 8; ++e) if (e < n) p[e] = v[e];
}
template <bool VEC>
STAR_DEV void ln_load_f32(const float* p, int n, float fill, float* v) {
  if (!p) {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = fill;
    return;
  }
  if constexpr (VEC) {
    const f32x4 a = *reinterpret_cast<const f32x4*>(p), b = *reinterpret_cast<const f32x4*>(p + 4);
#pragma unroll
    for (int e = 0; e < 4; ++e) { v[e] = a[e]; v[4 + e] = b[e]; }
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = e < n ? p[e] : fill;
  }
}

// sum over the lanes of a row; WG: over the workgroup, through LDS words sm[4 * slot ...] (the caller hands out slots so that one is not
// rewritten before every wave has passed a later barrier)
template <bool WG>
STAR_DEV float ln_row_sum(float v, int lpr, float* sm, int slot) {
  if constexpr (!WG) {
    for (int m = lpr >> 1; m >= 1; m >>= 1) v += shfl_xor(v, m);
    return v;
  }
  v = wave_sum(v);
  if ((threadIdx.x & 63) == 0) sm[4 * slot + (threadIdx.x >> 6)] = v;
  block_sync();
  return (sm[4 * slot] + sm[4 * slot + 1]) + (sm[4 * slot + 2] + sm[4 * slot + 3]);
}

template <class T, bool VEC, int CPL, bool WG>
STAR_GLOBAL void STAR_LAUNCH_BOUNDS(256)
ln_train_fwd_kernel(const LnTrainParams p) {
  float* sm = reinterpret_cast<float*>(dyn_smem());
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int LPR = WG ? 256 : p.lpr;
  const int sub = WG ? (int)threadIdx.x : lane & (LPR - 1);
  const int rpw = WG ? 1 : 64 / LPR;
  const long long row = WG ? (long long)blockIdx.x : ((long long)blockIdx.x * 4 + wave) * rpw + lane / LPR;
  const bool active = row < p.rows;
  const long long rr = active ? row : p.rows - 1;
  const T* x = (const T*)p.x + rr * p.ldx;
  vec<T, 8> v[CPL];
  float sum = 0.f;
#pragma unroll
  for (int i = 0; i < CPL; ++i) {
    const int c = (sub + LPR * i) * 8;
    if (c < p.C) {
      v[i] = ln_load<T, VEC>(x + c, p.C - c);
#pragma unroll
      for (int e = 0; e < 8; ++e) sum += to_f32<T>(v[i][e]);
    }
  }
  const float inv_c = 1.0f / (float)p.C;
  const float mean = ln_row_sum<WG>(sum, LPR, sm, 0) * inv_c;
  float sq = 0.f;
#pragma unroll
  for (int i = 0; i < CPL; ++i) {
    const int c = (sub + LPR * i) * 8;
    if (c < p.C) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float d = to_f32<T>(v[i][e]) - mean;
        if (VEC || c + e < p.C) sq += d * d;
      }
    }
  }
  const float rstd = 1.0f / sqrtf(ln_row_sum<WG>(sq, LPR, sm, 1) * inv_c + p.eps);
  if (!active) return;
  if (sub == 0 && p.stats) { p.stats[2 * row] = mean; p.stats[2 * row + 1] = rstd; }
  T* y = (T*)p.out + row * p.ldo;
  auto write = [&](auto stream_tag) STAR_ALWAYS_INLINE {
#pragma unroll
  for (int i = 0; i < CPL; ++i) {
    const int c = (sub + LPR * i) * 8;
    if (c < p.C) {
      float g[8], b[8];
      ln_load_f32<VEC>(p.gamma ? p.gamma + c : nullptr, p.C - c, 1.f, g);
      ln_load_f32<VEC>(p.beta ? p.beta + c : nullptr, p.C - c, 0.f, b);
      vec<T, 8> o;
#pragma unroll
      for (int e = 0; e < 8; ++e) o[e] = from_f32<T>((to_f32<T>(v[i][e]) - mean) * rstd * g[e] + b[e]);
      ln_store<T, VEC, decltype(stream_tag)::value>(y + c, o, p.C - c);
    }
  }
  };
  if (VEC && p.stream) write(std::integral_constant<bool, VEC>{});
  else write(std::false_type{});
}

template <class T, bool VEC, int CPL, bool WG>
STAR_GLOBAL void STAR_LAUNCH_BOUNDS(256)
ln_train_bwd_kernel(const LnTrainParams p) {
  float* sm = reinterpret_cast<float*>(dyn_smem());
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int LPR = WG ? 256 : p.lpr;
  const int sub = WG ? (int)threadIdx.x : lane & (LPR - 1);
  const int rpw = WG ? 1 : 64 / LPR;
  const int rpb = WG ? 1 : 4 * rpw;                                  // rows per workgroup and step
  const long long steps = ((long long)p.rows + rpb - 1) / rpb;
  const float inv_c = 1.0f / (float)p.C;
  float dg[CPL][8], db[CPL][8];
#pragma unroll
  for (int i = 0; i < CPL; ++i)
#pragma unroll
    for (int e = 0; e < 8; ++e) { dg[i][e] = 0.f; db[i][e] = 0.f; }
  int par = 0;
  for (long long it = blockIdx.x; it < steps; it += gridDim.x, par ^= 1) {
    const long long row = WG ? it : it * rpb + wave * rpw + lane / LPR;
    const bool active = row < p.rows;
    // a row past the end is all zeros: it adds nothing to the sums, and it reads no row that its owner may be writing (dx may be x or dy)
    const T* x = (const T*)p.x + row * p.ldx;
    const T* dy = (const T*)p.dy + row * p.lddy;
    float mean = 0.f, rstd = 0.f;
    if (active) { mean = p.stats[2 * row]; rstd = p.stats[2 * row + 1]; }
    vec<T, 8> vx[CPL], vd[CPL];
#pragma unroll
    for (int i = 0; i < CPL; ++i) {
      const int c = (sub + LPR * i) * 8;
      if (c < p.C) {
        if (active) {
          vx[i] = ln_load<T, VEC>(x + c, p.C - c);
          vd[i] = ln_load<T, VEC>(dy + c, p.C - c);
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e) { vx[i][e] = from_f32<T>(0.f); vd[i][e] = from_f32<T>(0.f); }
        }
      }
    }
    float s1 = 0.f, s2 = 0.f;
#pragma unroll
    for (int i = 0; i < CPL; ++i) {
      const int c = (sub + LPR * i) * 8;
      if (c < p.C) {
        float g[8];
        ln_load_f32<VEC>(p.gamma ? p.gamma + c : nullptr, p.C - c, 1.f, g);
#pragma unroll
        for (int e = 0; e < 8; ++e) {                                 // columns past C hold dy = 0: nothing is added for them
          const float d = to_f32<T>(vd[i][e]), xh = (to_f32<T>(vx[i][e]) - mean) * rstd, a = d * g[e];
          s1 += a;
          s2 += a * xh;
          dg[i][e] += d * xh;
          db[i][e] += d;
        }
      }
    }
    s1 = ln_row_sum<WG>(s1, LPR, sm, par * 2) * inv_c;
    s2 = ln_row_sum<WG>(s2, LPR, sm, par * 2 + 1) * inv_c;
    if (!active) continue;
    T* dx = (T*)p.out + row * p.ldo;
    auto write = [&](auto stream_tag) STAR_ALWAYS_INLINE {
#pragma unroll
    for (int i = 0; i < CPL; ++i) {
      const int c = (sub + LPR * i) * 8;
      if (c < p.C) {
        float g[8];
        ln_load_f32<VEC>(p.gamma ? p.gamma + c : nullptr, p.C - c, 1.f, g);
        vec<T, 8> o;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float xh = (to_f32<T>(vx[i][e]) - mean) * rstd;
          o[e] = from_f32<T>(rstd * (to_f32<T>(vd[i][e]) * g[e] - s1 - xh * s2));
        }
        ln_store<T, VEC, decltype(stream_tag)::value>(dx + c, o, p.C - c);
      }
    }
    };
    if (VEC && p.stream) write(std::integral_constant<bool, VEC>{});
    else write(std::false_type{});
  }
  if (!p.partial) return;
  float* part = p.partial + (size_t)blockIdx.x * 2 * p.C;
  if constexpr (WG) {                                                 // a thread owns its columns alone
#pragma unroll
    for (int i = 0; i < CPL; ++i) {
      const int c = (sub + LPR * i) * 8;
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (c + e < p.C) { part[c + e] = dg[i][e]; part[p.C + c + e] = db[i][e]; }
    }
  } else {
    // the row groups of a wave, then the four waves through LDS [4][2][LPR * 8] per chunk index
    float* buf = sm;
#pragma unroll
    for (int i = 0; i < CPL; ++i) {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        for (int m = LPR; m < 64; m <<= 1) { dg[i][e] += shfl_xor(dg[i][e], m); db[i][e] += shfl_xor(db[i][e], m); }
      block_sync();
      if (lane < LPR) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          buf[(wave * 2 + 0) * LPR * 8 + sub * 8 + e] = dg[i][e];
          buf[(wave * 2 + 1) * LPR * 8 + sub * 8 + e] = db[i][e];
        }
      }
      block_sync();
      for (int k = threadIdx.x; k < 2 * LPR * 8; k += 256) {
        const int which = k / (LPR * 8), c = LPR * i * 8 + k % (LPR * 8);
        float s = 0.f;
#pragma unroll
        for (int w = 0; w < 4; ++w) s += buf[w * 2 * LPR * 8 + k];
        if (c < p.C) part[(size_t)which * p.C + c] = s;
      }
    }
  }
}

// dgamma | dbeta [2 C] from the partial rows: 16 columns per workgroup, sixteen threads per column share the rows, joined in a fixed order
struct LnReduceParams { const float* partial; float* dgamma; float* dbeta; int C, parts; };
STAR_GLOBAL void STAR_LAUNCH_BOUNDS(256)
ln_train_reduce_kernel(const LnReduceParams p) {
  float* sm = reinterpret_cast<float*>(dyn_smem());                   // [16][16]
  const int col = threadIdx.x & 15, slice = threadIdx.x >> 4;
  const int c = blockIdx.x * 16 + col, n = 2 * p.C;
  float s = 0.f;
  if (c < n) {
#pragma unroll 8
    for (int r = slice; r < p.parts; r += 16) s += p.partial[(size_t)r * n + c];
  }
  sm[slice * 16 + col] = s;
  block_sync();
  if (slice || c >= n) return;
  float t = 0.f;
#pragma unroll
  for (int k = 0; k < 16; ++k) t += sm[k * 16 + col];
  if (c < p.C) { if (p.dgamma) p.dgamma[c] = t; }
  else if (p.dbeta) p.dbeta[c - p.C] = t;
}

}  // namespace star
